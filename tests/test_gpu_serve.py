"""DecoderLayer.serve: the layer on sequences whose keys and values lie in the 4-bit cache (cache4.py), against its pieces put together in float64."""
import math

import pytest
import torch

from oracle import cache4 as oracle

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def T():
    import triton_int8_amd as T
    return T


def _layer(T, dev, hidden, heads, int8):
    gen = torch.Generator().manual_seed(hidden + heads)
    layer = T.DecoderLayer(hidden=hidden, heads=heads, mlp=2 * hidden, int8=int8, device=dev)
    with torch.no_grad():
        for p in layer.parameters():
            if p.dim() == 2:
                p.copy_((torch.randn(p.shape, generator=gen) * p.shape[1] ** -0.5).to(torch.bfloat16))
    return layer


class _Reference:
    """The layer on calls of new tokens [batch, tokens, hidden], piece by piece as they are served (the scale of a block of int8 codes depends on the tokens
    that a call puts together): its own norms and linears; keys and values as the cache stores them, attention in float64."""

    def __init__(self, layer, batch):
        self.layer, self.k, self.v = layer, [[] for _ in range(batch)], [[] for _ in range(batch)]

    @torch.no_grad()
    def __call__(self, x, counts=None):
        import triton_int8_amd.decoder as D
        layer, (B, S, H) = self.layer, x.shape
        h = layer.input_norm(x)
        q, k, v = (t.view(B, S, layer.heads, layer.head_dim) for t in D._projections(h, layer.q_proj, layer.k_proj, layer.v_proj))
        a = torch.zeros(B, S, layer.heads, layer.head_dim, dtype=torch.bfloat16)
        for b in range(B):
            n, old = S if counts is None else counts[b], len(self.k[b])
            cos, sin = (t[old:old + n] for t in D.rope_tables(old + n, layer.head_dim, x.device))
            qb, kb = (t[0].cpu() for t in D._rope_pair(q[b:b + 1, :n], k[b:b + 1, :n], cos, sin))
            self.k[b] += list(oracle.decode(*oracle.encode(kb)))
            self.v[b] += list(oracle.decode(*oracle.encode(v[b, :n].cpu())))
            keys, values = torch.stack(self.k[b]), torch.stack(self.v[b])
            s = torch.einsum("ihd,jhd->hij", qb.double(), keys) / math.sqrt(layer.head_dim)
            p = s.masked_fill(torch.ones(n, old + n, dtype=torch.bool).triu(old + 1), float("-inf")).softmax(-1)
            a[b, :n] = torch.einsum("hij,jhd->ihd", p, values).to(torch.bfloat16)
        x = x + layer.o_proj(a.to(x.device).view(B, S, H))
        h = layer.post_norm(x)
        return x + layer.down_proj(D._swiglu(*D._projections(h, layer.gate_proj, layer.up_proj)))


def _rel(a, b):
    return float((a.double() - b.double()).norm() / b.double().norm())


# Differences: attention's roundings (a bf16 ulp of its elements), which the int8 codes of the linears behind it turn into steps of 1/127 of a row's or a
# block's largest element here and there, and keys whose rotation is rounded differently now and then, a whole 4-bit code for those.  Without the cache's
# rounding (4 bits: an eighth of an element's size at most, 6 % rms) the outputs are several times further away, as the last check shows.
CLOSE = 1.5e-2


@pytest.mark.parametrize("hidden,heads,int8", [(512, 4, True), (512, 8, True), (256, 2, False)])
def test_prompts_and_steps(T, dev, hidden, heads, int8):
    layer = _layer(T, dev, hidden, heads, int8)
    gen = torch.Generator(device=dev).manual_seed(1)
    x = torch.randn(2, 130, hidden, generator=gen, device=dev).to(torch.bfloat16)
    rotary = T.decoder.rope_tables(256, layer.head_dim, dev)
    for pieces in ([130], [100, 17] + [1] * 13):        # in one piece; in parts, then token by token
        cache, reference = T.Cache4(2, 200, heads, layer.head_dim, page_size=16, device=dev), _Reference(layer, 2)
        got, want = [], []
        for piece in x.split(pieces, dim=1):
            got.append(layer.serve(piece, cache, rotary))
            want.append(reference(piece))
        assert _rel(torch.cat(got, dim=1), torch.cat(want, dim=1)) <= CLOSE
        assert cache.lengths.tolist() == cache.positions.tolist() == [130, 130]
    with torch.no_grad():
        assert _rel(layer(x), _Reference(layer, 2)(x)) > CLOSE


def test_sequences_of_different_lengths(T, dev):
    """Prompts of different lengths in one call, then steps at each sequence's own position."""
    layer = _layer(T, dev, 512, 4, True)
    gen = torch.Generator(device=dev).manual_seed(2)
    x = torch.randn(3, 60, 512, generator=gen, device=dev).to(torch.bfloat16)
    lengths = [50, 7, 31]
    rotary = T.decoder.rope_tables(64, 128, dev)
    cache = T.Cache4(3, 64, 4, 128, page_size=32, device=dev)
    counts = torch.tensor(lengths, dtype=torch.int32, device=dev)
    reference = _Reference(layer, 3)
    out, want = layer.serve(x[:, :50], cache, rotary, counts=counts), reference(x[:, :50], lengths)
    for b, n in enumerate(lengths):
        assert _rel(out[b, :n], want[b, :n]) <= CLOSE
    for i in range(3):
        token = torch.stack([x[b, n + i:n + i + 1] for b, n in enumerate(lengths)])
        assert _rel(layer.serve(token, cache, rotary), reference(token)) <= CLOSE
    assert cache.lengths.tolist() == [n + 3 for n in lengths]


def test_a_budget_is_kept(T, dev):
    """What gets little attention goes: with a budget that holds everything nothing changes, and with a smaller one the cache stays within it while the
    newest entries and the heaviest of the others stay."""
    layer = _layer(T, dev, 512, 4, True)
    gen = torch.Generator(device=dev).manual_seed(3)
    x = torch.randn(2, 160, 512, generator=gen, device=dev).to(torch.bfloat16)
    rotary = T.decoder.rope_tables(160, 128, dev)
    run = {}
    for budget in (None, 120, 48):
        cache = T.Cache4(2, 180, 4, 128, page_size=16, budget=budget, device=dev)
        parts = [layer.serve(x[:, :100], cache, rotary)]
        for i in range(100, 160):
            if budget is not None and i % 10 == 0:
                before = cache.weights[cache.table.long()].transpose(1, 2).flatten(2).cpu()
                n = int(cache.lengths[0])
                kept = cache.evict(16).cpu()
                for b in range(2):
                    for h in range(4):
                        stay = oracle.kept(before[b, h, :n].tolist(), min(16, n), budget)
                        assert kept[b, h, :len(stay)].tolist() == stay
            if budget == 120 and i >= 120:
                break
            parts.append(layer.serve(x[:, i:i + 1], cache, rotary))
        run[budget] = torch.cat(parts, dim=1)
        if budget == 48:
            assert cache.lengths.tolist() == [58, 58] and cache.positions.tolist() == [160, 160]
    assert torch.equal(run[120][:, :120], run[None][:, :120])
    assert torch.equal(run[48][:, :100], run[None][:, :100]) and torch.isfinite(run[48].float()).all()


def test_a_recorded_step(T, dev):
    """A decode step as a graph: the cache's lengths and positions go on from replay to replay."""
    layer = _layer(T, dev, 512, 4, True)
    gen = torch.Generator(device=dev).manual_seed(4)
    x = torch.randn(2, 40, 512, generator=gen, device=dev).to(torch.bfloat16)
    rotary = T.decoder.rope_tables(64, 128, dev)
    eager, recorded = (T.Cache4(2, 64, 4, 128, page_size=16, device=dev) for _ in range(2))
    step = T.GraphedStep(lambda t: layer.serve(t, recorded, rotary), x[:, :1])
    recorded.reset()
    layer.serve(x[:, :30], recorded, rotary)
    layer.serve(x[:, :30], eager, rotary)
    for i in range(30, 40):
        assert torch.equal(step(x[:, i:i + 1]), layer.serve(x[:, i:i + 1], eager, rotary))
        torch.cuda.synchronize()
    assert recorded.lengths.tolist() == [40, 40]


def test_refusals(T, dev):
    layer = _layer(T, dev, 256, 2, True)
    cache = T.Cache4(1, 8, 2, 128, page_size=16, device=dev)
    x = torch.zeros(1, 5, 256, dtype=torch.bfloat16, device=dev)
    with pytest.raises(ValueError, match="rotary"):
        layer.serve(x, cache, T.decoder.rope_tables(4, 128, dev))
    rotary = T.decoder.rope_tables(64, 128, dev)
    layer.serve(x, cache, rotary)
    with pytest.raises(ValueError, match="room"):
        layer.serve(x, cache, rotary)
