"""The 4-bit cache (csrc/cache4.hip, csrc/cache4_attention.hip) at the ends of what its calls take, against its definition in float64."""
import math

import pytest
import torch

from oracle import cache4 as oracle
from test_gpu_cache4 import C, _check_attention, _ints, _masked_reference, _pool, _table  # noqa: F401

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


def _check_evict(C, dev, gen, page, dim, hkv, lengths, keep, recent, weights, table, pool, new_table):
    """Eviction where some pages are not there: their entries are left out.  Everything that is not written stays as it was."""
    pages = pool.shape[0]
    g_pool, g_weights = pool.to(dev), weights.to(dev)
    kept, new_lengths = C.evict(g_pool, table.to(dev), _ints(lengths, dev), g_weights, new_table.to(dev), keep=keep, recent=recent)
    p = (*oracle.parts(pool, page, dim), weights)
    sizes = []
    for b, n in enumerate(lengths):
        j = torch.arange(n)
        at = table[b].long()[j // page]
        there = (at >= 0) & (at < pages)
        old, new = j[there & (j < n - recent)], j[there & (j >= n - recent)]
        sizes.append(min(int(there.sum()), keep))
        for h in range(hkv):
            w = weights[at[old], h, old % page].double().nan_to_num(nan=float("inf"))
            heavy = old[w.sort(descending=True, stable=True).indices[:sizes[-1] - len(new)]].sort().values
            stay = torch.cat((heavy, new))
            assert kept[b, h].tolist() == stay.tolist() + [-1] * (keep - len(stay)), (b, h)
            i = torch.arange(len(stay))
            for t in p:
                t[new_table[b].long()[i // page], h, i % page] = t[at[stay], h, stay % page]
    assert new_lengths.tolist() == sizes
    assert torch.equal(g_pool.cpu(), pool) and torch.equal(g_weights.cpu(), weights)


@pytest.mark.parametrize("page,dim,hkv,lengths,keep,recent", [
    (16, 64, 2, [300, 1, 0, 16, 17, 299, 150], 100, 40), (64, 128, 1, [2049, 700, 1000], 640, 640), (16, 128, 3, [100, 90, 7], 60, 0), (32, 64, 1, [500, 64], 500, 100),
    (256, 128, 1, [3000, 5000], 1500, 1234)])
@pytest.mark.parametrize("holes", ["old", "recent", "everywhere", "all", "all but one"])
def test_evict_leaves_out_what_is_not_there(C, dev, page, dim, hkv, lengths, keep, recent, holes):
    gen = torch.Generator().manual_seed(page + dim)
    batch, mine, new = len(lengths), -(-max(lengths) // page), -(-keep // page)
    pages = batch * (mine + new)
    pool = _pool(gen, pages, hkv, page, dim, values=False)
    order = torch.randperm(pages, generator=gen).int()
    table, new_table = order[:batch * mine].view(batch, mine).clone(), order[batch * mine:].view(batch, new)
    weights = torch.rand(pages, hkv, page, generator=gen)
    for b, n in enumerate(lengths):
        slots = torch.arange(mine)
        first = max(0, n - recent) // page
        gone = {"old": (slots < first) & (slots % 3 == 1), "recent": (slots >= first) & (slots % 2 == 0), "everywhere": torch.rand(mine, generator=gen) < 0.4,
                "all": slots >= 0, "all but one": slots != min(2, (max(n, 1) - 1) // page)}[holes]
        table[b, gone] = torch.tensor([-1, pages, 1 << 30])[b % 3].int()
    _check_evict(C, dev, gen, page, dim, hkv, lengths, keep, recent, weights, table, pool, new_table)


@pytest.mark.parametrize("kind", ["few", "equal", "random"])
@pytest.mark.parametrize("holes", [False, True])
def test_evict_more_entries_than_lds_holds(C, dev, kind, holes):
    """Orders beyond the 32768 that stay in LDS, with weights that are equal on both sides of it."""
    gen = torch.Generator().manual_seed(7)
    page, dim, hkv, lengths, keep, recent = 64, 64, 2, [40000, 32769, 70001], 35000, 500
    batch, mine, new = 3, -(-70001 // page), -(-keep // page)
    pages = batch * (mine + new)
    pool = _pool(gen, pages, hkv, page, dim, values=False)
    order = torch.randperm(pages, generator=gen).int()
    table, new_table = order[:batch * mine].view(batch, mine).clone(), order[batch * mine:].view(batch, new)
    weights = {"few": torch.randint(0, 3, (pages, hkv, page), generator=gen) * 0.5, "equal": torch.full((pages, hkv, page), 0.25),
               "random": torch.rand(pages, hkv, page, generator=gen)}[kind]
    if holes:
        table[:, 5::7] = -1
    _check_evict(C, dev, gen, page, dim, hkv, lengths, keep, recent, weights, table, pool, new_table)


def test_what_is_not_there_is_not_seen_after_an_eviction(C, dev):
    """The places of a new page that nothing was moved to hold whatever was there before: numbers that are none, here."""
    gen = torch.Generator().manual_seed(5)
    page, dim, lengths = 16, 128, [130, 100]
    pool, table = _pool(gen, 40, 1, page, dim), _table(gen, 2, 9, 30)
    for s in oracle.parts(pool[30:], page, dim)[2:]:
        s.fill_(255)
    table[0, 2:4], table[1, 5:] = -1, 1 << 20
    new_table = torch.arange(30, 40, dtype=torch.int32).view(2, 5)
    weights = torch.rand(40, 1, page, generator=gen)
    q = torch.randn(2, 1, 4, dim, generator=gen).bfloat16().to(dev)
    g_pool, g_table, g_new = pool.to(dev), table.to(dev), new_table.to(dev)
    kept, new_lengths = C.evict(g_pool, g_table, _ints(lengths, dev), weights.to(dev), g_new, keep=80, recent=80)
    assert new_lengths.tolist() == [80, 80]
    out, lse = C.attention(g_pool, g_new, new_lengths, q)
    after = g_pool.cpu()
    want = oracle.attention(after, new_table, new_lengths.tolist(), q.cpu(), [1, 1], 1 / math.sqrt(dim), page)
    assert bool(torch.isfinite(out).all())
    _check_attention(out, lse, want, dim, 80)
    for b, n in enumerate(lengths):         # and they are the entries that were there before
        j = kept[b, 0].cpu().long()
        for x, y in zip(oracle.entries(after, new_table[b], page, dim, 0, 80), oracle.entries(pool, table[b].clamp(0, 39), page, dim, 0, n)):
            assert torch.equal(x, y[j]) and bool((table[b].long()[j // page] < 40).all()) and bool((table[b].long()[j // page] >= 0).all())


# steps with a workgroup for each head and shared out, rows that two waves share, prompts of four and eight waves, entries shared among workgroups
ROWS = [(1, 2, 2, 600), (1, 2, 2, 5000), (7, 4, 1, 600), (7, 4, 1, 5000), (50, 1, 1, 600), (50, 1, 1, 9000), (100, 2, 2, 600), (250, 1, 1, 600), (250, 2, 2, 9000)]


@pytest.mark.parametrize("tokens,heads,hkv,room", ROWS)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("values", ["one", "all", "some", "late"])
def test_values_as_large_as_are_stored(C, dev, tokens, heads, hkv, room, dim, values):
    """Up to 1.5 2^127: a single entry's come out as they are, and sums of many, of either sign and beside small ones, as the definition has them; rows that are
    none are zeros."""
    gen = torch.Generator().manual_seed(tokens + dim)
    page, lengths, counts = 32, [1, 600, 333, 597], [1, tokens, max(tokens - 3, 0), tokens // 2]
    mine = -(-600 // page)
    pool, table = _pool(gen, 4 * mine, hkv, page, dim), _table(gen, 4, mine, 4 * mine)
    scales = oracle.parts(pool, page, dim)[3]
    if values == "some":        # here and there a group of 32, of any size
        some = torch.rand(scales.shape, generator=gen) < 0.05
        scales[some] = torch.randint(180, 253, (int(some.sum()),), generator=gen, dtype=torch.uint8)
    elif values == "late":      # the last entries alone, behind many of usual size
        for b, n in enumerate(lengths):
            for j in range(max(0, n - 3), n):
                scales[int(table[b, j // page]), :, j % page] = 252
    else:
        scales.fill_({"one": 127 + 110, "all": 252}[values])
    if values == "one":
        lengths = [1] * 4
        counts = [1, min(tokens, 1), 0, 1]
    if values == "all":         # all positive for some entries' elements: sums of equal signs
        oracle.parts(pool, page, dim)[1][:, :, ::2] &= 0x77
    wide = torch.full((4, -(-room // page)), -1, dtype=torch.int32)
    wide[:, :mine] = table
    q = torch.randn(4, tokens, heads, dim, generator=gen).bfloat16()
    want = oracle.attention(pool, table, lengths, q, counts, 1 / math.sqrt(dim), page)
    weights = torch.zeros(4 * mine, hkv, page, device=dev)
    out, lse = C.attention(pool.to(dev), wide.to(dev), _ints(lengths, dev), q.to(dev), counts=_ints(counts, dev), weights=weights)
    assert bool(torch.isfinite(out).all()), out[~torch.isfinite(out)][:4]
    _check_attention(out, lse, want, dim, max(lengths))
    if values == "one":
        for b in range(4):
            for h in range(hkv):
                v = oracle.entries(pool, table[b], page, dim, h, 1)[1][0]
                for t in range(counts[b]):
                    for head in range(h * (heads // hkv), (h + 1) * (heads // hkv)):
                        assert torch.equal(out[b, t, head].cpu().double(), v)


@pytest.mark.parametrize("tokens,heads,hkv", [(1, 2, 2), (5, 4, 2), (12, 2, 1), (50, 1, 1), (100, 2, 2), (300, 1, 1)])
@pytest.mark.parametrize("dim", [64, 128])
def test_lengths_beyond_the_table(C, dev, tokens, heads, hkv, dim):
    """Entries that the table has no room for are not seen; up to where a query sees the others goes by the length that the sequence says it has."""
    gen = torch.Generator().manual_seed(tokens + dim)
    page, room = 16, 208
    lengths, counts = [room + 1, room + 3, room + tokens + 40, room, 2 ** 31 - 1], [tokens, max(tokens - 1, 1), tokens, tokens, tokens]
    pool, table = _pool(gen, 5 * room // page, hkv, page, dim), _table(gen, 5, room // page, 5 * room // page)
    q = torch.randn(5, tokens, heads, dim, generator=gen).bfloat16()
    said = [min(n, room + 1000) for n in lengths]
    wide = torch.full((5, -(-(room + 1000) // page)), -1, dtype=torch.int32)
    wide[:, :room // page] = table
    want = _masked_reference(pool, wide, said, q, counts, 1 / math.sqrt(dim), page)
    for narrow in (table, wide[:, :40]):        # (pages that are none: what there is room for then)
        weights = torch.zeros(pool.shape[0], hkv, page, device=dev)
        out, lse = C.attention(pool.to(dev), narrow.to(dev), _ints(lengths, dev), q.to(dev), counts=_ints(counts, dev), weights=weights)
        _check_attention(out, lse, want, dim, room)
        expected = torch.zeros(pool.shape[0], hkv, page, dtype=torch.float64)
        j = torch.arange(room)
        for b in range(5):
            for h in range(hkv):
                expected[table[b].long()[j // page], h, j % page] += want[2][b][h][:room]
        rel = 2.0 ** -18 + 4 * (dim + 8) * 2.0 ** -24 * float(want[3].max()) + tokens * heads * 2.0 ** -24      # as in test_attention
        assert bool(((weights.cpu().double() - expected).abs() <= (rel + 2.0 ** -22) * expected).all())
