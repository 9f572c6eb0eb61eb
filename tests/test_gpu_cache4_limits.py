"""The 4-bit cache (csrc/cache4.hip, csrc/cache4_attention.hip) at the ends of what its calls take, against its definition in float64."""
import math

import pytest
import torch

from oracle import cache4 as oracle
from test_gpu_cache4 import C, _check_attention, _ints, _pool, _table  # noqa: F401

pytestmark = pytest.mark.gpu


def _gains(pool, page, dim, length, q, scale):
    """What every entry gets of one token's heads q [heads, dim], which share the pool's only kv head and see all of `length` entries (in the pool's order), and
    the largest sum of |q k| scale: float64, on the GPU, a part of the entries at a time."""
    magnitudes = torch.cat((oracle.MAGNITUDES, -oracle.MAGNITUDES)).to(pool.device)
    codes, _, scales, _ = (t[:, 0].flatten(0, 1)[:length] for t in oracle.parts(pool, page, dim))
    q, step = q.double() * scale, 1 << 15

    def keys(at):
        c = codes[at:at + step]
        k = torch.stack((magnitudes[(c & 15).long()], magnitudes[(c >> 4).long()]), -1).flatten(-2)
        return k * torch.exp2(scales[at:at + step].double() - 127).repeat_interleave(32, dim=-1)
    lse, largest = torch.full((len(q),), float("-inf"), dtype=torch.float64, device=pool.device), 0.0
    for at in range(0, length, step):
        k = keys(at)
        lse = torch.logaddexp(lse, (q @ k.T.contiguous()).logsumexp(-1))
        largest = max(largest, float((q.abs() @ k.abs().T.contiguous()).max()))
    return torch.cat([torch.exp(q @ keys(at).T.contiguous() - lse[:, None]).sum(0) for at in range(0, length, step)]), largest


@pytest.mark.parametrize("heads,length", [(4096, (1 << 19) + 70000), (300, 5000)])
def test_weights_of_many_entries_that_many_heads_share(C, dev, heads, length):
    """An entry's distance from the tokens times the heads that share it passes 32 bits in the first of these."""
    page, dim = 256, 64
    gen = torch.Generator(device=dev).manual_seed(heads)
    mine = -(-length // page)
    pool = torch.randint(0, 256, (mine, 1, C.page_bytes(page, dim)), generator=gen, dtype=torch.uint8, device=dev)
    for s in oracle.parts(pool, page, dim)[2:]:
        s.copy_(torch.randint(122, 128, s.shape, generator=gen, dtype=torch.uint8, device=dev))
    table = torch.arange(mine, dtype=torch.int32, device=dev).view(1, -1)
    weights = torch.zeros(mine, 1, page, device=dev)
    q = torch.randn(1, 1, heads, dim, generator=gen, device=dev).bfloat16()
    C.attention(pool, table, _ints([length], dev), q, weights=weights)
    want, logits = _gains(pool, page, dim, length, q[0, 0], 1 / math.sqrt(dim))
    rel = 2.0 ** -18 + 4 * (dim + 8) * 2.0 ** -24 * logits + heads * 2.0 ** -24          # as in test_attention
    got = weights.flatten().double()
    assert not bool(got[length:].any())
    assert bool(((got[:length] - want).abs() <= (rel + 2.0 ** -23) * want).all()), float(((got[:length] - want).abs() / want).max())
    assert abs(float(want.sum()) - heads) < 1e-6 * heads


@pytest.mark.parametrize("tokens,heads,hkv", [(1, 4, 2), (6, 8, 1), (40, 4, 2), (150, 2, 2)])
@pytest.mark.parametrize("dim,page", [(64, 16), (128, 64)])
def test_weights_of_pages_that_sequences_share(C, dev, tokens, heads, hkv, dim, page):
    """Sequences with a common beginning, one of which comes upon a page twice: weights get what all of them give."""
    gen = torch.Generator().manual_seed(tokens + dim)
    lengths, common = [800, 500, 650, 700, 513], 448
    batch, mine = len(lengths), -(-800 // page)
    pool, table = _pool(gen, batch * mine, hkv, page, dim), _table(gen, batch, mine, batch * mine)
    table[:, :common // page] = table[0, :common // page]
    table[3, common // page] = table[3, 0]
    weights = torch.rand(pool.shape[0], hkv, page, generator=gen)
    q = torch.randn(batch, tokens, heads, dim, generator=gen).bfloat16()
    want = oracle.attention(pool, table, lengths, q, [tokens] * batch, 1 / math.sqrt(dim), page)
    expected = weights.double()
    for b, n in enumerate(lengths):
        j = torch.arange(n)
        for h in range(hkv):
            expected[:, h].index_put_((table[b].long()[j // page], j % page), want[2][b][h], accumulate=True)
    # as in test_attention, and a rounding for each addition to a weight
    rel = 2.0 ** -18 + 4 * (dim + 8) * 2.0 ** -24 * float(want[3].max()) + tokens * heads * 2.0 ** -24
    bound = rel * (expected - weights) + (batch + 2) * 2.0 ** -24 * expected
    for _ in range(3):
        got = weights.to(dev)
        out, lse = C.attention(pool.to(dev), table.to(dev), _ints(lengths, dev), q.to(dev), weights=got)
        _check_attention(out, lse, want, dim, max(lengths))
        assert bool(((got.cpu().double() - expected).abs() <= bound).all()), float(((got.cpu().double() - expected).abs() / expected).max())
