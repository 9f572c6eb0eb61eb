"""The 4-bit cache (csrc/cache4.hip, csrc/cache4_attention.hip) against its definition in float64 (oracle/cache4.py)."""
import math

import pytest
import torch

from oracle import cache4 as oracle

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def C():
    import triton_int8_amd as T
    return T.cache4


def _pool(gen, pages, heads, page, dim, values=True):
    """A pool on the CPU: random bytes (scales of 255 among them, which are no numbers), or random codes with scales around one."""
    pool = torch.randint(0, 256, (pages, heads, page * (dim + dim // 16)), generator=gen, dtype=torch.uint8)
    if values:
        for s in oracle.parts(pool, page, dim)[2:]:
            s.copy_(torch.randint(122, 128, s.shape, generator=gen, dtype=torch.uint8))
    return pool


def _table(gen, batch, mine, pages, lengths=None, page=None):
    """Pages of the sequences in any order; those behind a sequence's end are none of the pool's."""
    table = torch.randperm(pages, generator=gen)[:batch * mine].view(batch, mine).int()
    if lengths is not None:
        for b, n in enumerate(lengths):
            table[b, -(-n // page):] = torch.tensor([-1, 1 << 30, pages])[b % 3]
    return table


def _ints(values, dev):
    return torch.tensor(values, dtype=torch.int32, device=dev)


def _odd(t, dev, layout):
    """The same values on the GPU in another layout: dense, a slice of a wider tensor, or heads outside tokens."""
    if layout == "sliced":
        wide = torch.zeros((*t.shape[:2], t.shape[2] + 3, t.shape[3]), dtype=t.dtype, device=dev)
        wide[:, :, 1:-2] = t.to(dev)
        return wide[:, :, 1:-2]
    if layout == "heads":
        return t.to(dev).transpose(1, 2).contiguous().transpose(1, 2)
    if layout == "unaligned":       # neither the strides nor the address fit 16 bytes
        flat = torch.zeros(t.numel() // t.shape[3] * (t.shape[3] + 1) + 1, dtype=t.dtype, device=dev)
        view = flat[1:].view(*t.shape[:3], t.shape[3] + 1)[..., :t.shape[3]]
        view.copy_(t)
        return view
    return t.to(dev)


# a token; the edges of a wave's 16 tokens and of pages; several tiles; odd numbers of heads
@pytest.mark.parametrize("batch,tokens,heads,page", [(1, 1, 1, 16), (7, 1, 8, 64), (2, 15, 3, 16), (3, 17, 2, 32), (2, 130, 5, 128), (1, 600, 1, 256)])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("layout", ["dense", "sliced", "heads", "unaligned"])
def test_append_and_read(C, dev, batch, tokens, heads, page, dim, layout):
    gen = torch.Generator().manual_seed(tokens + dim)
    lengths = [5 + 9 * b for b in range(batch)]
    counts = [tokens if b % 3 != 1 else tokens // 2 for b in range(batch)]
    mine = -(-(max(lengths) + tokens) // page)
    pool, table = _pool(gen, batch * mine + 2, heads, page, dim, values=False), _table(gen, batch, mine, batch * mine + 2)
    weights = torch.rand(pool.shape[0], heads, page, generator=gen)
    k, v = (torch.randn(batch, tokens, heads, dim, generator=gen) * torch.exp(3 * torch.randn(batch, tokens, heads, dim, generator=gen)) for _ in range(2))
    k, v = k.bfloat16(), v.bfloat16()
    g_pool, g_table, g_weights = pool.to(dev), table.to(dev), weights.to(dev)
    ragged = _ints(counts, dev) if batch > 1 else None
    C.append(g_pool, g_table, _ints(lengths, dev), _odd(k, dev, layout), _odd(v, dev, layout), counts=ragged, weights=g_weights)
    got_k, got_v = C.read(g_pool, g_table, _ints(lengths, dev), tokens, dim, counts=ragged)
    want_k, want_v = torch.zeros(k.shape, dtype=torch.float64), torch.zeros(k.shape, dtype=torch.float64)
    for b in range(batch):
        for t in range(counts[b] if batch > 1 else tokens):
            j = lengths[b] + t
            at, row = int(table[b, j // page]), j % page
            for h in range(heads):
                oracle.put(pool, page, dim, at, row, h, k[b, t, h], v[b, t, h])
                weights[at, h, row] = 0.0
                want_k[b, t, h], want_v[b, t, h] = (oracle.decode(*oracle.encode(x[b, t, h])) for x in (k, v))
    assert torch.equal(g_pool.cpu(), pool)          # nothing but the new entries' bytes is touched
    assert torch.equal(g_weights.cpu(), weights)
    assert torch.equal(got_k.cpu().double(), want_k) and torch.equal(got_v.cpu().double(), want_v)


def test_every_bf16_is_stored_as_defined(C, dev):
    """All 65536 of them, beside others of their size and beside anything: NaN counts as zero, infinities as the largest value."""
    gen = torch.Generator().manual_seed(1)
    every = torch.arange(65536).to(torch.int32).to(torch.int16).view(torch.bfloat16)
    x = torch.cat((every, every[torch.randperm(65536, generator=gen)], every.repeat_interleave(32)[:65536 * 4])).view(1, -1, 1, 128)
    n, page = x.shape[1], 256
    mine = -(-n // page)
    pool = torch.zeros((mine, 1, C.page_bytes(page, 128)), dtype=torch.uint8, device=dev)
    table = torch.arange(mine, dtype=torch.int32, device=dev).view(1, -1)
    C.append(pool, table, _ints([0], dev), x.to(dev), x.flip(1).to(dev))
    codes, scales = oracle.encode(x[0, :, 0])
    p = [t.flatten(0, 2)[:n].cpu() for t in oracle.parts(pool, page, 128)]
    packed = codes[:, 0::2] | (codes[:, 1::2] << 4)
    assert torch.equal(p[0], packed) and torch.equal(p[2], scales)
    assert torch.equal(p[1], packed.flip(0)) and torch.equal(p[3], scales.flip(0))
    k, v = C.read(pool, table, _ints([0], dev), n, 128)
    want = oracle.decode(codes, scales)
    assert torch.isfinite(k).all() and torch.equal(k[0, :, 0].double().cpu(), want) and torch.equal(v[0, :, 0].double().cpu(), want.flip(0))


def test_append_leaves_out_what_has_no_room(C, dev):
    """Entries behind the table's pages, in front of the first and in pages that the pool does not have are not written, and read as zeros."""
    gen = torch.Generator().manual_seed(2)
    pool = _pool(gen, 4, 2, 16, 64, values=False)
    table = torch.tensor([[1, 4], [2, -1], [3, 0]], dtype=torch.int32)
    k, v = (torch.randn(3, 40, 2, 64, generator=gen).bfloat16() for _ in range(2))
    g_pool, starts = pool.to(dev), _ints([0, 10, -20], dev)
    C.append(g_pool, table.to(dev), starts, k.to(dev), v.to(dev))
    got = C.read(g_pool, table.to(dev), starts, 40, 64)
    want = torch.zeros(2, 3, 40, 2, 64, dtype=torch.float64)
    for b, start in enumerate([0, 10, -20]):
        for t in range(40):
            j = start + t
            if 0 <= j < 32 and 0 <= int(table[b, j // 16]) < 4:
                for h in range(2):
                    oracle.put(pool, 16, 64, int(table[b, j // 16]), j % 16, h, k[b, t, h], v[b, t, h])
                    want[0, b, t, h], want[1, b, t, h] = (oracle.decode(*oracle.encode(x[b, t, h])) for x in (k, v))
    assert torch.equal(g_pool.cpu(), pool)
    assert torch.equal(got[0].cpu().double(), want[0]) and torch.equal(got[1].cpu().double(), want[1])


def _check_attention(got_out, got_lse, want, dim, entries):
    """Errors by what the kernels round: a score is a sum of `dim` exact products in fp32, (dim + 8) 2^-24 of the sum of their magnitudes at most;
    an exponential and a sum over the entries 2^-20 (2^-24 per addition in any tree over at most 2^17 entries would be 2^-7; sums that meet in
    chunks stay below (64 + entries / 64) 2^-24); probabilities are rounded to bf16 (2^-8 of sum p |v|: 2^-9 each, twice for their product's order), the
    result to bf16 (2^-9); what is below 2^-126 may be zero."""
    out, lse, _, logits, spread = want
    chain = (64 + entries / 64) * 2.0 ** -24
    score = (dim + 8) * 2.0 ** -24 * logits
    seen = torch.isfinite(lse)
    assert torch.equal(torch.isfinite(got_lse.cpu()), seen) and bool((got_lse.cpu()[~seen] == float("-inf")).all())
    bound = score + 2.0 ** -20 + chain + 2.0 ** -22 * (lse.abs() + logits)
    assert bool(((got_lse.cpu().double() - lse).abs()[seen] <= bound[seen]).all()), float(((got_lse.cpu().double() - lse).abs()[seen] / bound[seen]).max())
    rel = 2 * (score + 2.0 ** -22 * logits) + 2.0 ** -19 + 2 * chain
    bound = 2.0 ** -8 * out.abs() + (2.0 ** -8 + rel.unsqueeze(-1)) * spread + 2.0 ** -126
    assert bool(((got_out.cpu().double() - out).abs() <= bound).all()), float(((got_out.cpu().double() - out).abs() - bound).max())


SIZES = [
    # tokens, heads, kv heads, page, lengths, counts
    (1, 1, 1, 16, [1], None),
    (1, 4, 4, 16, [0, 1, 15, 16, 17, 31, 32, 33], None),            # nothing in a cache; the edges of pages and tiles
    (1, 8, 2, 64, [127, 128, 129, 700], None),
    (1, 14, 2, 32, [1000, 3], None),                                 # seven heads share one
    (1, 32, 1, 128, [300, 0, 257], None),
    (1, 64, 2, 256, [5000, 1, 64], None),                            # thirty-two heads share one
    (3, 4, 2, 16, [2, 40, 3, 100], [3, 3, 1, 0]),                    # more new tokens than entries: rows that see nothing; no new token
    (5, 16, 4, 32, [63, 64, 65, 515], [5, 4, 1, 5]),
    (7, 10, 5, 16, [200, 33], None),
    (16, 16, 1, 64, [333, 16], None),
    (31, 2, 2, 16, [31, 100, 29, 64], [31, 17, 31, 1]),
    (40, 12, 3, 64, [200, 40, 41], [40, 40, 23]),
    (129, 2, 1, 32, [129, 400, 1], [129, 100, 1]),
    (200, 3, 3, 128, [200, 1100], None),
    (300, 8, 2, 16, [517], None),
]


@pytest.mark.parametrize("size", SIZES, ids=str)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("layout", ["dense", "sliced", "heads"])
def test_attention(C, dev, size, dim, layout):
    tokens, heads, hkv, page, lengths, counts = size
    gen = torch.Generator().manual_seed(tokens * heads + dim)
    batch = len(lengths)
    mine = -(-max(lengths) // page) + 1
    pages = batch * mine + 3
    pool, table = _pool(gen, pages, hkv, page, dim, values=False), _table(gen, batch, mine, pages, lengths, page)
    p = oracle.parts(pool, page, dim)
    for b, n in enumerate(lengths):         # entries have scales around one, everything else is whatever it is
        for j in range(n):
            for s in p[2:]:
                s[int(table[b, j // page]), :, j % page] = torch.randint(122, 128, s.shape[1:2] + s.shape[3:], generator=gen, dtype=torch.uint8)
    weights = torch.rand(pages, hkv, page, generator=gen)
    q = torch.randn(batch, tokens, heads, dim, generator=gen).bfloat16()
    want = oracle.attention(pool, table, lengths, q, counts or [tokens] * batch, 1 / math.sqrt(dim), page)
    args = pool.to(dev), table.to(dev), _ints(lengths, dev), _odd(q, dev, layout)
    ragged = None if counts is None else _ints(counts, dev)
    out, lse = C.attention(*args, counts=ragged)
    _check_attention(out, lse, want, dim, max(lengths))
    g_weights = weights.to(dev)
    out2, lse2 = C.attention(*args, counts=ragged, weights=g_weights)
    assert torch.equal(out2, out) and torch.equal(lse2, lse)        # sums in a fixed order
    gains, logits = want[2], want[3]
    rel = 2.0 ** -18 + 4 * (dim + 8) * 2.0 ** -24 * float(logits.max()) + tokens * heads * 2.0 ** -24
    expected, bound = weights.double(), torch.zeros_like(weights, dtype=torch.float64)
    for b, n in enumerate(lengths):
        j = torch.arange(n)
        for h in range(hkv):
            at = table[b].long()[j // page]
            expected[at, h, j % page] += gains[b][h]
            bound[at, h, j % page] = rel * gains[b][h] + 2.0 ** -23 * expected[at, h, j % page]
    assert bool(((g_weights.cpu().double() - expected).abs() <= bound).all())
    again = weights.to(dev)
    C.attention(*args, counts=ragged, weights=again)
    assert torch.equal(again, g_weights)


@pytest.mark.parametrize("tokens", [1, 100])
def test_attention_scale_and_large_scores(C, dev, tokens):
    """A scale of the caller's, and scores far apart (a key that takes everything in each tile)."""
    gen = torch.Generator().manual_seed(tokens)
    page, dim, n = 32, 64, 600
    pool = _pool(gen, 20, 2, page, dim)
    for s in oracle.parts(pool, page, dim)[2:3]:
        s.add_(torch.randint(0, 6, s.shape, generator=gen, dtype=torch.uint8))
    table = _table(gen, 1, 19, 20)
    q = (4 * torch.randn(1, tokens, 4, dim, generator=gen)).bfloat16()
    for scale in (1.0, 0.01, 0.0, -0.5):
        want = oracle.attention(pool, table, [n], q, [tokens], scale, page)
        out, lse = C.attention(pool.to(dev), table.to(dev), _ints([n], dev), q.to(dev), scale=scale)
        magnitude = oracle.attention(pool, table, [n], q, [tokens], abs(scale), page)[3]
        _check_attention(out, lse, (*want[:3], magnitude, want[4]), dim, n)


def test_attention_values_that_are_no_numbers_stay_in_their_rows(C, dev):
    """A query with NaN gives NaN in its own row and head only; what lies behind a sequence's end is never seen."""
    gen = torch.Generator().manual_seed(4)
    pool, table = _pool(gen, 12, 2, 32, 128).to(dev), _table(gen, 2, 6, 12).to(dev)
    for tokens in (2, 70):
        q = torch.randn(2, tokens, 4, 128, generator=gen).bfloat16().to(dev)
        lengths = _ints([150, 171], dev)
        want = C.attention(pool, table, lengths, q)
        q[1, 1, 2, 7] = float("nan")
        out, lse = C.attention(pool, table, lengths, q)
        assert torch.isnan(out[1, 1, 2]).all() and torch.isnan(lse[1, 1, 2])
        out[1, 1, 2], lse[1, 1, 2] = want[0][1, 1, 2], want[1][1, 1, 2]
        assert torch.equal(out, want[0]) and torch.equal(lse, want[1])


def test_attention_many_sequences(C, dev):
    """More sequences than lanes of a wave, with none, one and many entries, and two far longer than the rest."""
    gen = torch.Generator().manual_seed(6)
    batch, page, dim, hkv, heads = 150, 16, 64, 2, 4
    lengths = [int(x) for x in torch.randint(0, 60, (batch,), generator=gen)]
    lengths[77], lengths[149] = 2500, 1100
    mine = -(-2500 // page)
    used = torch.randperm(sum(-(-n // page) for n in lengths), generator=gen).int()
    table, at = torch.full((batch, mine), -7, dtype=torch.int32), 0
    for b, n in enumerate(lengths):
        table[b, :-(-n // page)] = used[at:at + -(-n // page)]
        at += -(-n // page)
    pool = _pool(gen, at, hkv, page, dim)
    q = torch.randn(batch, 1, heads, dim, generator=gen).bfloat16()
    want = oracle.attention(pool, table, lengths, q, [1] * batch, 1 / 8, page)
    out, lse = C.attention(pool.to(dev), table.to(dev), _ints(lengths, dev), q.to(dev))
    _check_attention(out, lse, want, dim, 2500)


def test_offsets_beyond_32_bits(C, dev):
    """A pool of more than 4 GiB, of which the last pages are used; a table whose rows lie apart."""
    page, dim, hkv = 256, 128, 32
    pages = (5 << 30) // (hkv * C.page_bytes(page, dim))
    pool = torch.zeros((pages, hkv, C.page_bytes(page, dim)), dtype=torch.uint8, device=dev)
    weights = torch.zeros((pages, hkv, page), dtype=torch.float32, device=dev)
    table = torch.arange(pages - 1, pages - 9, -1, dtype=torch.int32, device=dev).view(2, 4)[:, :2]
    gen = torch.Generator().manual_seed(8)
    k, v = (torch.randn(2, 300, hkv, dim, generator=gen).bfloat16() for _ in range(2))
    starts = _ints([0, 200], dev)
    C.append(pool, table, starts, k.to(dev), v.to(dev), weights=weights)
    got = C.read(pool, table, starts, 300, dim)
    for x, y in zip(got, (k, v)):
        assert torch.equal(x.cpu().double(), oracle.decode(*oracle.encode(y)))
    small, small_table = pool[pages - 8:].cpu(), table.cpu() - (pages - 8)
    for tokens in (1, 80):
        q = torch.randn(2, tokens, hkv, dim, generator=gen).bfloat16()
        want = oracle.attention(small, small_table, [300, 500], q, [tokens] * 2, 1 / math.sqrt(dim), page)
        out, lse = C.attention(pool, table, _ints([300, 500], dev), q.to(dev), weights=weights)
        _check_attention(out, lse, want, dim, 500)
    new_table = torch.tensor([[0], [1]], dtype=torch.int32, device=dev)
    kept, lengths = C.evict(pool, table, _ints([300, 500], dev), weights, new_table, keep=200, recent=50)
    moved = C.read(pool, new_table, _ints([0, 0], dev), 200, dim)
    before = C.read(pool, table, _ints([0, 0], dev), 500, dim)
    for x, y in zip(moved, before):
        index = kept.long().transpose(1, 2)[..., None].expand(-1, -1, -1, dim)
        assert torch.equal(x, y.gather(1, index))


@pytest.mark.parametrize("kind", ["random", "equal", "few", "odd"])
@pytest.mark.parametrize("page,dim,hkv,lengths,keep,recent", [
    (16, 64, 1, [1, 0, 5, 6, 7], 6, 2), (16, 128, 3, [40, 16, 100], 16, 0), (64, 128, 2, [2049, 1024, 1025, 3000], 1024, 1000), (32, 64, 4, [300], 77, 77),
    (128, 128, 1, [9000, 130], 4097, 1), (64, 64, 2, [70], 500, 3)])
def test_evict(C, dev, kind, page, dim, hkv, lengths, keep, recent):
    gen = torch.Generator().manual_seed(keep + dim)
    batch = len(lengths)
    mine, new = -(-max(lengths) // page), -(-keep // page)
    pages = batch * (mine + new)
    pool = _pool(gen, pages, hkv, page, dim, values=False)
    order = torch.randperm(pages, generator=gen).int()
    table, new_table = order[:batch * mine].view(batch, mine), order[batch * mine:].view(batch, new)
    weights = torch.rand(pages, hkv, page, generator=gen).exp()
    if kind == "equal":
        weights.fill_(0.25)
    elif kind == "few":
        weights = torch.randint(0, 3, weights.shape, generator=gen) * 0.5
    elif kind == "odd":         # zeros of both signs, negative numbers, infinities and no numbers
        values = torch.tensor([0.0, -0.0, -1.0, 1e-45, -1e-45, float("inf"), float("-inf"), float("nan"), -float("nan"), 3.0, 3e38])
        weights = values[torch.randint(0, len(values), weights.shape, generator=gen)]
    g_pool, g_weights = pool.to(dev), weights.to(dev)
    kept, new_lengths = C.evict(g_pool, table.to(dev), _ints(lengths, dev), g_weights, new_table.to(dev), keep=keep, recent=recent)
    assert new_lengths.tolist() == [min(n, keep) for n in lengths]
    p = (*oracle.parts(pool, page, dim), weights)
    for b, n in enumerate(lengths):
        j = torch.arange(n)
        for h in range(hkv):
            stay = oracle.kept(weights[table[b].long()[j // page], h, j % page].tolist(), recent, keep)
            assert kept[b, h].tolist() == stay + [-1] * (keep - len(stay)), (b, h)
            i, stay = torch.arange(len(stay)), torch.tensor(stay, dtype=torch.int64)
            for t in p:
                t[new_table[b].long()[i // page], h, i % page] = t[table[b].long()[stay // page], h, stay % page]
    assert torch.equal(g_pool.cpu(), pool)
    assert torch.equal(g_weights.cpu().view(torch.int32), weights.view(torch.int32))


def test_on_another_stream_and_in_a_graph(C, dev):
    """Steps of a decode loop recorded once: the lengths change on the GPU between replays; every replay has the eager results."""
    gen = torch.Generator(device=dev).manual_seed(9)
    rand = lambda *shape: torch.randn(*shape, generator=gen, device=dev).bfloat16()
    make = lambda: C.Cache4(3, 500, 2, 128, page_size=32, budget=200, device=dev)
    eager, recorded = make(), make()
    side = torch.cuda.Stream()
    k, v, q = rand(3, 300, 2, 128), rand(3, 300, 2, 128), rand(3, 300, 4, 128)
    counts = _ints([300, 250, 1], dev)
    want = [eager.append(k, v, counts=counts), eager.attend(q, counts=counts)][1]
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        recorded.append(k, v, counts=counts)
        assert torch.equal(recorded.attend(q, counts=counts), want)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(eager.evict(100), recorded.evict(100))
    for a, b in ((eager.lengths, recorded.lengths), (eager.table, recorded.table), (eager.positions, recorded.positions)):
        assert torch.equal(a, b)
    assert eager.lengths.tolist() == [200, 200, 1] and eager.positions.tolist() == [300, 250, 1]
    k, v, q = rand(3, 1, 2, 128), rand(3, 1, 2, 128), rand(3, 1, 4, 128)
    state = [t.clone() for t in (recorded.pool, recorded.weights, recorded.lengths, recorded.positions)]
    recorded.append(k, v), recorded.attend(q)
    torch.cuda.synchronize()
    for t, s in zip((recorded.pool, recorded.weights, recorded.lengths, recorded.positions), state):
        t.copy_(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        recorded.append(k, v)
        out = recorded.attend(q)
    for _ in range(4):
        for t, shape in ((k, k.shape), (v, v.shape), (q, q.shape)):
            t.copy_(rand(*shape))
        graph.replay()
        eager.append(k, v)
        assert torch.equal(eager.attend(q), out)
        torch.cuda.synchronize()
    assert torch.equal(eager.weights, recorded.weights) and torch.equal(eager.lengths, recorded.lengths)


def test_refusals(C, dev):
    """What the kernels cannot take is refused before anything is launched."""
    pool = torch.zeros((8, 2, C.page_bytes(16, 64)), dtype=torch.uint8, device=dev)
    table, one = torch.zeros((1, 4), dtype=torch.int32, device=dev), _ints([1], dev)
    weights = torch.zeros((8, 2, 16), dtype=torch.float32, device=dev)
    kv, q = torch.zeros((1, 3, 2, 64), dtype=torch.bfloat16, device=dev), torch.zeros((1, 3, 6, 64), dtype=torch.bfloat16, device=dev)
    before = pool.clone()
    for what in (lambda: C.append(pool, table, one, kv.float(), kv), lambda: C.append(pool, table, one, kv.cpu(), kv), lambda: C.append(pool, table, one, kv, kv[:, :2]),
                 lambda: C.append(pool, table, one, q, q), lambda: C.append(pool, table, one.long(), kv, kv), lambda: C.append(pool, table, _ints([1, 2], dev), kv, kv),
                 lambda: C.append(pool, table.long(), one, kv, kv), lambda: C.append(pool, table[:, ::2], one, kv, kv), lambda: C.append(pool, table, one, kv[:, :0], kv[:, :0]),
                 lambda: C.append(pool, table, one, kv, kv, weights=weights[:7]), lambda: C.append(pool[..., :-1].contiguous(), table, one, kv, kv),
                 lambda: C.append(pool, table, one, kv[..., :32].contiguous(), kv[..., :32].contiguous()), lambda: C.append(pool[:, :, ::2], table, one, kv, kv),
                 lambda: C.append(pool, table, one.cpu(), kv, kv), lambda: C.append(pool, table, one, kv, kv, counts=_ints([1, 1], dev)),
                 lambda: C.append(pool, table, one, kv.clone().requires_grad_(True), kv),
                 lambda: C.read(pool, table, one, 0, 64), lambda: C.read(pool, table, one, 3, 96), lambda: C.read(pool.cpu(), table, one, 3, 64),
                 lambda: C.attention(pool, table, one, q[:, :, :5]), lambda: C.attention(pool, table, one, q.half()), lambda: C.attention(pool, table, one, q[0]),
                 lambda: C.attention(pool, table, one, q.clone().requires_grad_(True)), lambda: C.attention(pool, table, one, q, weights=weights.double()),
                 lambda: C.attention(pool, table[0], one, q),
                 lambda: C.evict(pool, table, one, weights, table, keep=0, recent=0), lambda: C.evict(pool, table, one, weights, table, keep=65, recent=0),
                 lambda: C.evict(pool, table, one, weights, table, keep=8, recent=9), lambda: C.evict(pool, table, one, weights.half(), table, keep=8, recent=1),
                 lambda: C.evict(pool, table, one, weights, table.long(), keep=8, recent=1), lambda: C.evict(pool, table, one, None, table, keep=8, recent=1),
                 lambda: C.Cache4(0, 10, 2, 64), lambda: C.Cache4(1, 10, 2, 80), lambda: C.Cache4(1, 10, 2, 64, page_size=48), lambda: C.Cache4(1, 10, 2, 64, budget=11)):
        with pytest.raises(ValueError):
            what()
    cache = C.Cache4(1, 10, 2, 64, device=dev)
    for _ in range(3):
        cache.append(kv, kv)
    with pytest.raises(ValueError, match="room"):
        cache.append(kv, kv)
    with pytest.raises(ValueError, match="budget"):
        cache.evict(1)
    with torch.no_grad():
        C.append(pool, table, one, kv.clone().requires_grad_(True), kv)
    assert not torch.equal(pool, before)


def _masked_reference(pool, table, lengths, q, counts, scale, page):
    """As oracle.attention, for tables with pages that the pool does not have: their entries are not seen."""
    B, S, H, D = q.shape
    hkv, pages = pool.shape[1], pool.shape[0]
    out, lse = torch.zeros(B, S, H, D, dtype=torch.float64), torch.full((B, S, H), float("-inf"), dtype=torch.float64)
    logits, spread = torch.zeros(B, S, H, dtype=torch.float64), torch.zeros(B, S, H, D, dtype=torch.float64)
    gains = [[torch.zeros(n, dtype=torch.float64) for _ in range(hkv)] for n in lengths]
    for b, n in enumerate(lengths):
        j = torch.arange(n)
        there = (table[b].long()[j // page] >= 0) & (table[b].long()[j // page] < pages)
        for h in range(hkv):
            k, v = oracle.entries(pool, table[b].clamp(0, pages - 1), page, D, h, n)
            for t in range(counts[b]):
                sees = there & (j <= n - counts[b] + t)
                if not sees.any():
                    continue
                x = slice(h * (H // hkv), (h + 1) * (H // hkv))
                rows = q[b, t, x].double()
                s = (rows @ k[sees].T) * scale
                p = s.softmax(-1)
                out[b, t, x], lse[b, t, x] = p @ v[sees], s.logsumexp(-1)
                logits[b, t, x] = (rows.abs() @ k[sees].abs().T * scale).amax(-1)
                spread[b, t, x] = p @ v[sees].abs()
                gains[b][h][sees] += p.sum(0)
    return out, lse, gains, logits, spread


# 4, 32, 36, 64, 65, 200 and 400 rows that share a kv head; several pages that are not there, a whole sequence of them, and one that is there alone
@pytest.mark.parametrize("tokens,heads", [(1, 4), (8, 4), (9, 4), (16, 4), (65, 1), (50, 4), (100, 4)])
@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("dim", [64, 128])
def test_pages_that_are_not_there(C, dev, tokens, heads, page, dim):
    gen = torch.Generator().manual_seed(tokens + page)
    lengths = [700, 333, 128, 640]
    mine = -(-700 // page)
    pool, table = _pool(gen, 4 * mine, 1, page, dim), _table(gen, 4, mine, 4 * mine)
    table[0, 1::3] = torch.tensor([-1, 4 * mine, 1 << 30]).repeat(mine)[:len(table[0, 1::3])]
    table[2] = -5
    table[3, :5], table[3, 6:] = 1 << 29, -1
    weights = torch.rand(4 * mine, 1, page, generator=gen)
    q = torch.randn(4, tokens, heads, dim, generator=gen).bfloat16()
    want = _masked_reference(pool, table, lengths, q, [tokens] * 4, 1 / math.sqrt(dim), page)
    g_weights = weights.to(dev)
    out, lse = C.attention(pool.to(dev), table.to(dev), _ints(lengths, dev), q.to(dev), weights=g_weights)
    _check_attention(out, lse, want, dim, 700)
    rel = 2.0 ** -18 + 4 * (dim + 8) * 2.0 ** -24 * float(want[3].max()) + tokens * heads * 2.0 ** -24      # as in test_attention
    for b, n in enumerate(lengths):
        for j in range(n):
            at = int(table[b, j // page])
            if 0 <= at < 4 * mine:
                weights[at, 0, j % page] += want[2][b][0][j]
    assert bool(((g_weights.cpu().double() - weights.double()).abs() <= rel * weights.double() + 2.0 ** -22 * weights.double()).all())


@pytest.mark.parametrize("tokens,heads,hkv", [(9, 4, 1), (13, 8, 2), (64, 3, 3), (33, 1, 1), (2, 40, 2), (128, 2, 1), (257, 1, 1)])
@pytest.mark.parametrize("dim", [64, 128])
def test_rows_of_every_form(C, dev, tokens, heads, hkv, dim):
    """33 to 64 rows (two waves share them), 128, 256 and 257; entries shared among many workgroups, and few of them."""
    gen = torch.Generator().manual_seed(tokens + dim)
    for page, lengths, counts in ((64, [3000, tokens, 1111], None), (16, [tokens + 1, 700], [tokens, tokens - 1])):
        batch, mine = len(lengths), -(-max(lengths) // page)
        pool, table = _pool(gen, batch * mine, hkv, page, dim), _table(gen, batch, mine, batch * mine)
        q = torch.randn(batch, tokens, heads, dim, generator=gen).bfloat16()
        want = oracle.attention(pool, table, lengths, q, counts or [tokens] * batch, 1 / math.sqrt(dim), page)
        out, lse = C.attention(pool.to(dev), table.to(dev), _ints(lengths, dev), q.to(dev), counts=None if counts is None else _ints(counts, dev))
        _check_attention(out, lse, want, dim, max(lengths))


@pytest.mark.parametrize("dim", [64, 128])
def test_evict_sequences_of_every_length(C, dev, dim):
    """Sequences that end anywhere within the entries that a wave moves, shorter and longer than the budget: only what is kept is written, and only to its place."""
    gen = torch.Generator().manual_seed(dim)
    page, keep, lengths = 16, 70, list(range(0, 101))
    mine, new = -(-100 // page), -(-keep // page)
    pages = len(lengths) * (mine + new)
    pool = _pool(gen, pages, 1, page, dim, values=False)
    order = torch.randperm(pages, generator=gen).int()
    table, new_table = order[:len(lengths) * mine].view(-1, mine), order[len(lengths) * mine:].view(-1, new)
    weights = torch.rand(pages, 1, page, generator=gen)
    g_pool, g_weights = pool.to(dev), weights.to(dev)
    kept, _ = C.evict(g_pool, table.to(dev), _ints(lengths, dev), g_weights, new_table.to(dev), keep=keep, recent=30)
    p = (*oracle.parts(pool, page, dim), weights)
    for b, n in enumerate(lengths):
        j = torch.arange(n)
        stay = oracle.kept(weights[table[b].long()[j // page], 0, j % page].tolist(), 30, keep)
        assert kept[b, 0].tolist() == stay + [-1] * (keep - len(stay)), n
        i, stay = torch.arange(len(stay)), torch.tensor(stay, dtype=torch.int64)
        for t in p:
            t[new_table[b].long()[i // page], 0, i % page] = t[table[b].long()[stay // page], 0, stay % page]
    assert torch.equal(g_pool.cpu(), pool) and torch.equal(g_weights.cpu(), weights)


@pytest.mark.parametrize("tokens,heads,hkv,page,lengths,counts", [s for s in SIZES if s[0] * s[1] // s[2] <= 32 and max(s[4]) <= 1000], ids=str)
@pytest.mark.parametrize("dim", [64, 128])
def test_steps_whatever_room_the_table_has(C, dev, tokens, heads, hkv, page, lengths, counts, dim):
    """The same entries in tables of short and long rows, which decide how they are shared out; some pages are not there, some values are no numbers."""
    gen = torch.Generator().manual_seed(tokens + heads + dim)
    batch, mine = len(lengths), -(-max(lengths) // page)
    pool, table = _pool(gen, batch * mine, hkv, page, dim), _table(gen, batch, mine, batch * mine)
    for b in range(1, batch, 2):
        table[b, (mine - 1) // 2] = batch * mine + b
    q = torch.randn(batch, tokens, heads, dim, generator=gen).bfloat16()
    want = _masked_reference(pool, table, lengths, q, counts or [tokens] * batch, 1 / math.sqrt(dim), page)
    q = q.to(dev)
    ragged = None if counts is None else _ints(counts, dev)
    for room in (mine * page, 512, 528, 1024, 1280, 2048, 2304, 5120):
        if room >= mine * page and room % page == 0:
            wide = torch.full((batch, room // page), -1, dtype=torch.int32)
            wide[:, :mine] = table
            weights = torch.zeros(pool.shape[0], hkv, page, device=dev)
            out, lse = C.attention(pool.to(dev), wide.to(dev), _ints(lengths, dev), q, counts=ragged, weights=weights)
            _check_attention(out, lse, want, dim, max(lengths))
            odd = q.clone()
            odd[0, 0, -1, 3] = float("inf")
            out2, lse2 = C.attention(pool.to(dev), wide.to(dev), _ints(lengths, dev), odd, counts=ragged)
            out2[0, 0, -1], lse2[0, 0, -1] = out[0, 0, -1], lse[0, 0, -1]
            assert torch.equal(out2, out) and torch.equal(lse2, lse)


@pytest.mark.parametrize("heads,room", [(100, 512), (100, 528), (200, 512), (200, 528), (86, 2048), (85, 2048), (86, 2064), (128, 1040), (171, 256), (171, 528)])
@pytest.mark.parametrize("dim,tokens", [(64, 1), (64, 20), (128, 1), (128, 20)])
def test_steps_of_many_heads(C, dev, heads, room, dim, tokens):
    """Around one, two and more heads per CU, of sequences with none, few and all the entries that there is room for."""
    gen = torch.Generator().manual_seed(heads + room + dim)
    page, lengths = 16, [room, 0, room // 3]
    mine = room // page
    pool, table = _pool(gen, 2 * mine + 5, heads, page, dim), _table(gen, 3, 2 * mine // 3, 2 * mine + 5)
    table = torch.cat((table, torch.full((3, mine - table.shape[1]), -1, dtype=torch.int32)), 1)
    table[0] = torch.randperm(2 * mine + 5, generator=gen)[:mine].int()
    q = torch.randn(3, tokens, heads, dim, generator=gen).bfloat16()
    out, lse = C.attention(pool.to(dev), table.to(dev), _ints(lengths, dev), q.to(dev))
    some = [0, heads // 2, heads - 1]
    want = oracle.attention(pool[:, some].contiguous(), table, lengths, q[:, :, some], [tokens] * 3, 1 / math.sqrt(dim), page)
    _check_attention(out[:, :, some], lse[:, :, some], want, dim, room)
    assert bool((lse[1] == float("-inf")).all()) and not bool(out[1].any())
    assert bool(torch.isfinite(lse[0, -1]).all()) and bool(torch.isfinite(out).all())


@pytest.mark.parametrize("batch,tokens,heads,hkv,page", [(7, 150, 7, 1, 64), (5, 90, 32, 8, 16), (40, 44, 8, 8, 32), (3, 300, 2, 1, 16), (4, 70, 40, 40, 16)])
@pytest.mark.parametrize("dim", [64, 128])
def test_prompts_of_no_and_few_entries_in_tables_of_any_width(C, dev, batch, tokens, heads, hkv, page, dim):
    """Prompts whose blocks are shared out or left whole by what the table has room for and by what there is: none, a few entries, several tiles."""
    gen = torch.Generator().manual_seed(batch + tokens + dim)
    counts = [(0, tokens, tokens // 3, 1)[b % 4] for b in range(batch)]
    lengths = [n + (0, 0, 200, 500)[(b // 2) % 4] for b, n in enumerate(counts)]
    lengths[-1] = 0
    mine = -(-max(lengths) // page)
    pool, table = _pool(gen, batch * mine, hkv, page, dim), _table(gen, batch, mine, batch * mine)
    some = [0, hkv - 1] if hkv > 1 else [0]
    q = torch.randn(batch, tokens, heads, dim, generator=gen).bfloat16()
    rows = [h * (heads // hkv) + g for h in some for g in range(heads // hkv)]
    want = oracle.attention(pool[:, some].contiguous(), table, lengths, q[:, :, rows], counts, 1 / math.sqrt(dim), page)
    for room in (mine, mine + 1, -(-2000 // page), -(-8192 // page), -(-60000 // page)):
        wide = torch.full((batch, max(room, mine)), -1, dtype=torch.int32)
        wide[:, :mine] = table
        out = torch.full_like(q, float("nan"), device=dev)        # (memory that the outputs may come from)
        del out
        out, lse = C.attention(pool.to(dev), wide.to(dev), _ints(lengths, dev), q.to(dev), counts=_ints(counts, dev))
        _check_attention(out[:, :, rows], lse[:, :, rows], want, dim, max(lengths))
        assert bool(torch.isfinite(out).all())
