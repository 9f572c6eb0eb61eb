"""Cache4 and DecoderLayer.serve on sequences that grow by different numbers of tokens."""
import math

import pytest
import torch

from oracle import cache4 as oracle
from test_gpu_cache4 import C, _check_attention, _ints  # noqa: F401

pytestmark = pytest.mark.gpu


def test_counts_of_more_and_less_than_the_tokens(C, dev):
    """What counts of no sense add is what was written: no entry becomes visible that nobody wrote, and no sequence gets shorter."""
    gen = torch.Generator().manual_seed(1)
    cache = C.Cache4(3, 64, 2, 64, page_size=16, device=dev)
    cache.pool.fill_(255)         # scales that are no numbers
    k, v = (torch.randn(3, 12, 2, 64, generator=gen).bfloat16() for _ in range(2))
    q = torch.randn(3, 5, 2, 64, generator=gen).bfloat16()
    cache.append(k[:, :7].to(dev), v[:, :7].to(dev))
    cache.append(k[:, 7:].to(dev), v[:, 7:].to(dev), counts=_ints([40, -3, 2], dev))
    assert cache.lengths.tolist() == cache.positions.tolist() == [12, 7, 9]
    out, lse = C.attention(cache.pool, cache.table, cache.lengths, q.to(dev), counts=_ints([40, -3, 2], dev))
    want = oracle.attention(cache.pool.cpu(), cache.table.cpu(), [12, 7, 9], q, [5, 0, 2], 1 / math.sqrt(64), 16)
    assert bool(torch.isfinite(out).all())
    _check_attention(out, lse, want, 64, 12)


@pytest.mark.parametrize("int8,scheme", [(True, "block_channel"), (True, "double_channel"), (True, "row_block"), (False, "block_channel")])
def test_blank_rows_change_nothing(dev, int8, scheme):
    """Rows behind a sequence's tokens share blocks of 128 rows, and a scale, with other sequences' tokens: taken for blank, they may hold anything."""
    import triton_int8_amd as T
    gen = torch.Generator().manual_seed(2)
    layer = T.DecoderLayer(hidden=512, heads=4, mlp=1024, int8=int8, scheme=scheme, device=dev)
    with torch.no_grad():
        for p in layer.parameters():
            if p.dim() == 2:
                p.copy_((torch.randn(p.shape, generator=gen) * p.shape[1] ** -0.5).bfloat16())
    rotary = T.decoder.rope_tables(64, 128, dev)
    x = torch.randn(4, 40, 512, generator=gen).bfloat16().to(dev)
    counts = [40, 3, 0, 17]
    padding = torch.arange(40, device=dev)[None] >= torch.tensor(counts, device=dev)[:, None]
    results = []
    for fill in (0.0, 1.0, -3e4, float("inf"), float("nan")):
        cache = T.Cache4(4, 64, 4, 128, page_size=16, budget=64, device=dev)
        cache.pool.zero_()
        prompt = x.masked_fill(padding[..., None], fill)
        before = prompt.clone()
        out = layer.serve(prompt, cache, rotary, counts=_ints(counts, dev), blank=True)
        assert torch.equal(prompt.view(torch.int16), before.view(torch.int16))        # the caller's tensor stays as it is
        assert bool(torch.isfinite(out).all()) and not bool(out[padding].any())
        results.append((out, cache.pool.clone(), cache.weights.clone(), layer.serve(x[:, :1], cache, rotary)))
    for other in results[1:]:
        for a, b in zip(results[0], other):
            assert torch.equal(a, b)


def test_serving_goes_on_while_there_is_room(dev):
    """Drafts of which most are no tokens in the end: neither the cache nor the rotary tables run out before the sequences need them."""
    import triton_int8_amd as T
    layer = T.DecoderLayer(hidden=256, heads=2, mlp=512, int8=False, device=dev)
    rotary = T.decoder.rope_tables(24, 128, dev)
    gen = torch.Generator().manual_seed(3)
    cache = T.Cache4(2, 20, 2, 128, page_size=16, budget=12, device=dev)
    for i in range(9):
        layer.serve(torch.randn(2, 4, 256, generator=gen).bfloat16().to(dev), cache, rotary, counts=_ints([2, i % 2], dev))
    assert cache.lengths.tolist() == [18, 4]
    cache.evict(4)
    layer.serve(torch.randn(2, 6, 256, generator=gen).bfloat16().to(dev), cache, rotary, counts=_ints([6, 0], dev))
    assert cache.lengths.tolist() == [18, 4] and cache.positions.tolist() == [24, 4]
    with pytest.raises(ValueError, match="rotary"):
        layer.serve(torch.randn(2, 1, 256, generator=gen).bfloat16().to(dev), cache, rotary)
    x = torch.randn(2, 3, 256, generator=gen).bfloat16().to(dev)
    with pytest.raises(ValueError, match="room"):
        cache.append(*(t.view(2, 3, 2, 128) for t in (x, x)), counts=_ints([3, 3], dev))


def test_rejected_drafts_and_sequences_that_begin_again(C, dev):
    """Entries that were taken back are not seen, and written over by the next tokens, whose weights begin at zero."""
    gen = torch.Generator().manual_seed(4)
    rand = lambda *shape: torch.randn(*shape, generator=gen).bfloat16().to(dev)  # noqa: E731
    k, v, q = rand(2, 30, 2, 64), rand(2, 30, 2, 64), rand(2, 2, 4, 64)
    drafted, straight = (C.Cache4(2, 40, 2, 64, page_size=16, budget=40, device=dev) for _ in range(2))
    drafted.append(k[:, :20], v[:, :20])
    drafted.append(rand(2, 6, 2, 64), rand(2, 6, 2, 64))
    drafted.attend(rand(2, 6, 4, 64))
    drafted.take_back(_ints([6, 2], dev))
    drafted.take_back(_ints([0, 4], dev))
    drafted.weights.zero_()
    straight.append(k[:, :20], v[:, :20])
    for cache in (drafted, straight):
        cache.append(k[:, 20:22], v[:, 20:22])
    assert torch.equal(drafted.attend(q), straight.attend(q)) and torch.equal(drafted.lengths, straight.lengths)
    for cache in (drafted, straight):
        cache.reset(1)
        cache.append(k[:, 22:], v[:, 22:], counts=_ints([0, 8], dev))
        assert cache.lengths.tolist() == cache.positions.tolist() == [22, 8]
    assert torch.equal(drafted.attend(q), straight.attend(q))
    seen = torch.arange(48, device=dev) < drafted.lengths[:, None]
    for a, b in ((drafted, straight),):
        wa, wb = (c.weights[c.table.long()].transpose(1, 2).flatten(2).transpose(1, 2)[seen] for c in (a, b))
        assert torch.equal(wa, wb)
