"""What serving from a 4-bit key/value cache is judged by: the cases, their plain form, and the calls of ``triton_int8_amd.cache4``.

The cache is a pool of pages, uint8 [pages, kv heads, bytes of a page], a page table int32 [batch, pages of a sequence] and the number of
entries of every sequence.  A page of a head holds P entries (head dim D): codes of the keys [P][D / 2], codes of the values [P][D / 2],
scales of the keys [P][D / 32], scales of the values [P][D / 32].  A code is a 4-bit float (sign, magnitude 0 .5 1 1.5 2 3 4 6; the even
element in the low half of a byte), a scale the exponent byte e of 2^(e - 127) for 32 elements.

Operators:
  append   keys and values of new tokens into their places, and those places read back
  attend   queries of the new tokens over all entries up to their own; with ``weights`` the probabilities that every entry got are added up
  evict    the newest entries and the heaviest of the others, in order, into other pages
"""
import math
import random

import torch

own = False
DEVICE = "cuda:0"
GROUP = 32
MAGNITUDES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
_tables = {}


def _case(op, batch, new, length, heads, kv_heads, dim, page, *, ragged=False, fused=False, weights=False, keep=0, recent=0):
    return {"op": op, "batch": batch, "new": new, "length": length, "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page,
            "ragged": ragged, "fused": fused, "weights": weights, "keep": keep, "recent": recent}


def listed():
    return [
        # one token of each stream of a decode batch goes into the cache: launches and latency
        {"name": "append_step", **_case("append", 32, 1, 4096, 32, 8, 128, 64, weights=True)},
        # prompts of different lengths that share a call, cut out of one projection of q, k and v, on pages of 16
        {"name": "append_ragged", **_case("append", 5, 333, 700, 16, 4, 64, 16, ragged=True, fused=True)},
        # the prompts of the benchmark's decoder layer: 4 x 4096 tokens, 32 heads of 128
        {"name": "append_prompt", **_case("append", 4, 4096, 4096, 32, 32, 128, 64)},
        # a single decode stream in a short conversation: latency is all there is
        {"name": "step_1", **_case("attend", 1, 1, 1021, 32, 8, 128, 16)},
        # a decode batch of the decoder layer (as many kv heads as heads), streams of different lengths, one of them new
        {"name": "step_batch", **_case("attend", 16, 1, 4096, 32, 32, 128, 64, ragged=True)},
        # long documents, one far longer than most: a pure stream through the cache
        {"name": "step_long", **_case("attend", 8, 1, 131072, 32, 8, 128, 64, ragged=True)},
        # a decode batch that keeps a budget: every entry's attention weight is added up
        {"name": "step_weights", **_case("attend", 32, 1, 2048, 32, 8, 128, 64, weights=True)},
        # drafted tokens of several streams are looked at together, heads of 64
        {"name": "drafts_weights", **_case("attend", 8, 5, 8191, 16, 4, 64, 32, ragged=True, weights=True, fused=True)},
        # the last part of two long prompts that go through in parts of 2048 tokens
        {"name": "prompt", **_case("attend", 2, 2048, 8192, 32, 8, 128, 64)},
        # prompts of different lengths behind what their caches hold already, weights added up
        {"name": "prompt_weights", **_case("attend", 3, 1000, 1777, 32, 32, 128, 16, ragged=True, weights=True, fused=True)},
        # a decode batch that went over its budget by some tokens
        {"name": "evict_step", **_case("evict", 8, 0, 2112, 8, 8, 128, 64, weights=True, keep=2048, recent=1024)},
        # long prompts cut down to a budget
        {"name": "evict_prompt", **_case("evict", 16, 0, 16384, 8, 8, 128, 64, ragged=True, weights=True, keep=2048, recent=500)},
    ]


def _log(rng, low, high):
    return min(high, max(low, int(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def _cost(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / 50)


def draw(rng):
    most = {op: max(_cost(c) for c in listed() if c["op"] == op) for op in ("append", "attend", "evict")}
    while True:
        op = rng.choice(("append", "attend", "attend", "attend", "attend", "evict"))
        kv_heads, dim, page, ragged = rng.choice((1, 2, 4, 5, 8, 32)), rng.choice((64, 128, 128)), rng.choice((16, 32, 64, 128)), rng.random() < 0.5
        heads = kv_heads * rng.choice((1, 2, 4, 7, 8, 16))
        weights, fused = rng.random() < 0.4, rng.random() < 0.3
        if op == "append":
            new = _log(rng, 1, 4096)
            c = _case(op, _log(rng, 1, 64), new, new + _log(rng, 1, 4096), heads, kv_heads, dim, page, ragged=ragged, fused=fused, weights=weights)
        elif op == "attend":
            new = rng.choice((1, 1, _log(rng, 2, 16), _log(rng, 16, 4096)))
            c = _case(op, _log(rng, 1, 64), new, max(new, _log(rng, 1, 131072)), heads, kv_heads, dim, page, ragged=ragged, fused=fused, weights=weights)
        else:
            length = _log(rng, 32, 32768)
            keep = max(1, int(length * rng.uniform(0.05, 0.99)))
            c = _case(op, _log(rng, 1, 32), 0, length, kv_heads, kv_heads, dim, page, ragged=ragged, weights=True, keep=keep, recent=int(keep * rng.uniform(0, 0.9)))
        # (the plain form holds every score and every value in 32 bits)
        fits = c["batch"] * max(c["heads"] * max(1, c["new"]), 2 * c["kv_heads"] * dim) * c["length"] <= 2 ** 31
        if heads <= 128 and fits and _cost(c) <= most[op]:
            return c


def _sizes(case):
    """(entries of every sequence, new tokens of every sequence): from the case alone, so that its work is the same for all seeds.
    Sequences behind each other: one of full length, and where they are ragged one that has just begun and one without a new token."""
    batch, new, length = case["batch"], case["new"], case["length"]
    lengths, counts = [length] * batch, [new] * batch
    if case["ragged"]:
        r = random.Random("%d %d %d" % (batch, new, length))
        for b in range(1, batch):
            counts[b] = r.randint((new + 1) // 2, new)
            lengths[b] = max(counts[b], int(length * r.uniform(0.02, 1.0) ** 2))
        if batch > 2:
            lengths[1] = counts[1]
        if batch > 3 and new > 1:
            counts[2] = 0
    return lengths, counts


def _pages(case):
    """pages of a sequence, and of the budget that it is cut down to"""
    return -(-case["length"] // case["page"]), -(-case["keep"] // case["page"])


def work(case):
    lengths, counts = _sizes(case)
    dim, hkv = case["dim"], case["kv_heads"]
    entry = dim + dim // 16        # bytes of a token's key and value of a head
    if case["op"] == "append":
        n = sum(counts) * hkv
        return {"bytes": n * (4 * dim + entry + 4 * case["weights"]) + case["batch"] * case["new"] * hkv * 4 * dim, "flops": 0}
    if case["op"] == "evict":
        kept = sum(min(n, case["keep"]) for n in lengths) * hkv
        return {"bytes": 4 * hkv * sum(lengths) + kept * (2 * (entry + 4) + 4), "flops": 0}
    pairs = sum(n * length - n * (n - 1) // 2 for n, length in zip(counts, lengths))
    rows = case["batch"] * case["new"] * case["heads"]
    return {"bytes": sum(lengths) * hkv * (entry + 8 * case["weights"]) + rows * (4 * dim + 4), "flops": 4 * dim * case["heads"] * pairs}


def _table(name, values, device):
    key = name, device
    if key not in _tables:
        _tables[key] = torch.tensor(values, dtype=torch.float32, device=device)
    return _tables[key]


def _encode(x):
    """float32 [..., D] -> codes uint8 [..., D / 2], scales uint8 [..., D / 32]."""
    g = x.unflatten(-1, (-1, GROUP))
    amax = g.abs().amax(-1)
    # the smallest power of two by which the largest of a group is no more than 6 (1.5 2^2): up by one where the fraction is over 1.5
    scale = (((amax.view(torch.int32) + 0x3fffff) >> 23) - 2).clamp(1, 252)
    y = (g * ((254 - scale) << 23).view(torch.float32).unsqueeze(-1)).flatten(-2)
    a = y.abs()
    code = ((a > 0.25).byte() + (a >= 0.75).byte() + (a > 1.25).byte() + (a >= 1.75).byte() + (a > 2.5).byte() + (a >= 3.5).byte() + (a > 5.0).byte()
            + (y < 0).byte() * 8)
    return code[..., 0::2] | (code[..., 1::2] << 4), scale.byte()


def _decode(codes, scales):
    """codes uint8 [..., D / 2], scales uint8 [..., D / 32] -> float32 [..., D]."""
    value = list(MAGNITUDES) + [-m for m in MAGNITUDES]
    pairs = _table("pairs", [[value[b & 15], value[b >> 4]] for b in range(256)], codes.device)
    x = pairs[codes.int()].flatten(-2)
    return (x.unflatten(-1, (-1, GROUP)) * (scales.int() << 23).view(torch.float32).unsqueeze(-1)).flatten(-2)


def _parts(pool, page, dim):
    """Views of a pool [..., bytes]: codes of keys, codes of values [..., P, D / 2], scales of keys, scales of values [..., P, D / 32]."""
    c, s = page * dim // 2, page * dim // GROUP
    k, v, ks, vs = pool.split((c, c, s, s), dim=-1)
    return tuple(t.unflatten(-1, (page, -1)) for t in (k, v, ks, vs))


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    batch, new, hkv, heads, dim, page = (case[n] for n in ("batch", "new", "kv_heads", "heads", "dim", "page"))
    lengths, counts = _sizes(case)
    mine, spare = _pages(case)
    pages = batch * (mine + spare)
    pool = torch.empty((pages, hkv, page * (dim + dim // 16)), dtype=torch.uint8, device=DEVICE)
    # keys have a few channels that are far larger than the others, as keys of trained models have
    channels = torch.ones((hkv, 1, dim), device=DEVICE)
    channels[:, :, torch.randperm(dim, generator=gen, device=DEVICE)[:dim // 32]] = 8.0
    parts, step = _parts(pool, page, dim), max(1, (1 << 26) // (hkv * page * dim))
    for p in range(0, pages, step):
        n = min(step, pages - p)
        k, v = (torch.randn((n, hkv, page, dim), generator=gen, device=DEVICE).bfloat16().float() for _ in range(2))
        for t, at in ((k * channels, 0), (v, 1)):
            codes, scales = _encode(t)
            parts[at][p:p + n], parts[at + 2][p:p + n] = codes, scales
    s = dict(case)
    s["pool"] = pool
    # the pages of the sequences in any order; those of their budgets in any order behind them
    s["table"] = torch.randperm(batch * mine, generator=gen, device=DEVICE).int().view(batch, mine)
    s["lengths"] = torch.tensor(lengths, dtype=torch.int32, device=DEVICE)
    s["counts"] = torch.tensor(counts, dtype=torch.int32, device=DEVICE) if case["ragged"] and new else None
    s["accumulated"] = None
    if case["weights"]:
        # what entries get over a while: few are heavy, most light
        s["accumulated"] = torch.randn((pages, hkv, page), generator=gen, device=DEVICE).mul_(2.0).exp_()
    if new:
        widths = (heads, hkv, hkv)
        shape = lambda h: (batch, new, h, dim)  # noqa: E731
        if case["fused"]:
            qkv = torch.randn(shape(sum(widths)), generator=gen, device=DEVICE).bfloat16().split(widths, dim=2)
        else:
            qkv = tuple(torch.randn(shape(h), generator=gen, device=DEVICE).bfloat16() for h in widths)
        s["q"], s["k"], s["v"] = qkv
        s["starts"] = s["lengths"] - torch.tensor(counts, dtype=torch.int32, device=DEVICE)
    if spare:
        s["new_table"] = torch.randperm(batch * spare, generator=gen, device=DEVICE).int().view(batch, spare) + batch * mine
    return s


def run(s):
    if own:
        from triton_int8_amd import cache4
        if s["op"] == "append":
            cache4.append(s["pool"], s["table"], s["starts"], s["k"], s["v"], counts=s["counts"], weights=s["accumulated"])
            k, v = cache4.read(s["pool"], s["table"], s["starts"], s["new"], s["dim"], counts=s["counts"])
            return [k, v] if s["accumulated"] is None else [k, v, s["accumulated"]]
        if s["op"] == "attend":
            out, lse = cache4.attention(s["pool"], s["table"], s["lengths"], s["q"], counts=s["counts"], weights=s["accumulated"])
            return [out, lse] if s["accumulated"] is None else [out, lse, s["accumulated"]]
        kept, lengths = cache4.evict(s["pool"], s["table"], s["lengths"], s["accumulated"], s["new_table"], keep=s["keep"], recent=s["recent"])
    else:
        if s["op"] == "append":
            return _plain_append(s)
        if s["op"] == "attend":
            return _plain_attend(s)
        kept, lengths = _plain_evict(s)
    # the entries are moved as they are, so their bytes are what comes back: those of the pages that they went to
    first = s["table"].numel()
    return [kept, lengths, s["pool"][first:], s["accumulated"][first:]]


def _places(s, index):
    """Pages and rows of the entries index [batch, n] (those of no sequence among them, at the last page)."""
    at = (index // s["page"]).clamp(0, s["table"].shape[1] - 1).long()
    return s["table"].long().gather(1, at), (index % s["page"]).long()


def _new_rows(s):
    """bool [batch, new]: which rows of q, k and v are tokens"""
    i = torch.arange(s["new"], device=DEVICE)
    return (i < s["counts"][:, None]) if s["counts"] is not None else (i >= 0).expand(s["batch"], -1)


def _plain_append(s):
    i, rows = torch.arange(s["new"], device=DEVICE), _new_rows(s)
    pages, at = (t[rows] for t in _places(s, s["starts"][:, None] + i))
    parts, read = _parts(s["pool"], s["page"], s["dim"]), []
    for x, codes_at, scales_at in ((s["k"], parts[0], parts[2]), (s["v"], parts[1], parts[3])):
        codes, scales = _encode(x[rows].float())
        codes_at[pages, :, at], scales_at[pages, :, at] = codes, scales
        out = torch.zeros(x.shape, dtype=torch.bfloat16, device=DEVICE)
        out[rows] = _decode(codes_at[pages, :, at], scales_at[pages, :, at]).bfloat16()
        read.append(out)
    if s["accumulated"] is None:
        return read
    s["accumulated"][pages, :, at] = 0.0
    return [*read, s["accumulated"]]


def _plain_attend(s):
    batch, new, heads, hkv, dim, page = (s[n] for n in ("batch", "new", "heads", "kv_heads", "dim", "page"))
    mine = s["table"].shape[1]
    held = mine * page
    # [batch, kv heads, entries, ...] of everything that the tables name
    k, v, ks, vs = (t.transpose(1, 2).flatten(2, 3) for t in _parts(s["pool"][s["table"].long()], page, dim))
    j = torch.arange(held, device=DEVICE)
    there = (j < s["lengths"][:, None])[:, None, :, None]
    k, v = (torch.where(there, _decode(c, e), 0.0) for c, e in ((k, ks), (v, vs)))
    # the queries of the heads that share a kv head, one token after the other
    q = s["q"].float().view(batch, new, hkv, heads // hkv, dim).permute(0, 2, 1, 3, 4).reshape(batch, hkv, -1, dim)
    scores = torch.matmul(q, k.transpose(2, 3)) / math.sqrt(dim)
    counts = s["counts"][:, None] if s["counts"] is not None else new
    i, rows = torch.arange(new, device=DEVICE), _new_rows(s)
    sees = (j <= (s["lengths"][:, None] - counts + i)[:, :, None]) & rows[:, :, None]
    scores.masked_fill_(~sees.repeat_interleave(heads // hkv, dim=1)[:, None], float("-inf"))
    largest = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(largest == float("-inf"), 0.0, largest))
    total = p.sum(-1, keepdim=True)
    p /= torch.where(total == 0, 1.0, total)
    out = torch.matmul(p, v)
    lse = torch.where(total == 0, float("-inf"), largest + total.log())
    tokens = lambda t: t.reshape(batch, hkv, new, heads // hkv, -1).permute(0, 2, 1, 3, 4).reshape(batch, new, heads, -1)  # noqa: E731
    out, lse = tokens(out).bfloat16(), tokens(lse)[..., 0].contiguous()
    if s["accumulated"] is None:
        return [out, lse]
    got = p.sum(2).view(batch, hkv, mine, page).transpose(1, 2)
    s["accumulated"].index_add_(0, s["table"].flatten(), got.reshape(batch * mine, hkv, page))
    return [out, lse, s["accumulated"]]


def _plain_evict(s):
    batch, hkv, page, keep = (s[n] for n in ("batch", "kv_heads", "page", "keep"))
    n = s["lengths"][:, None, None]
    held = s["table"].shape[1] * page
    w = s["accumulated"][s["table"].long()].transpose(1, 2).reshape(batch, hkv, held)
    j = torch.arange(held, device=DEVICE)
    w = torch.where(j >= n, float("-inf"), torch.where(j >= n - s["recent"], float("inf"), w))
    # the heaviest first, those in front first among equals; then in their old order, and nothing behind the last
    kept = w.sort(dim=-1, descending=True, stable=True).indices[..., :keep]
    kept = torch.where(torch.arange(kept.shape[-1], device=DEVICE) < n, kept, held).sort(dim=-1).values
    lengths = s["lengths"].clamp(max=keep)
    there = kept < held
    b, h, to = there.nonzero(as_tuple=True)
    pages, at = (t.view(kept.shape)[there] for t in _places(s, kept.flatten(1)))
    new_pages, new_at = s["new_table"].long()[b, to // page], to % page
    for part in (*_parts(s["pool"], page, s["dim"]), s["accumulated"]):
        part[new_pages, h, new_at] = part[pages, h, at]
    return torch.where(there, kept, -1).int(), lengths


def exact(case, seed):
    s = prepare(case, seed)
    lengths, counts = _sizes(case)
    batch, new, heads, hkv, dim, page = (case[n] for n in ("batch", "new", "heads", "kv_heads", "dim", "page"))
    group = heads // hkv
    places = [s["table"][b].long().repeat_interleave(page)[:n] for b, n in enumerate(lengths)]
    weights = None if s["accumulated"] is None else s["accumulated"].double()
    if case["op"] == "append":
        grid = torch.tensor(MAGNITUDES, dtype=torch.float64, device=DEVICE)
        read = []
        for x in (s["k"], s["v"]):
            out = torch.zeros(x.shape, dtype=torch.float64, device=DEVICE)
            for b, n in enumerate(counts):
                g = x[b, :n].double().unflatten(-1, (-1, GROUP))
                scale = torch.exp2(torch.ceil(torch.log2(g.abs().amax(-1, keepdim=True).clamp_min(1e-30) / 6)))
                away = (g.abs().unsqueeze(-1) / scale.unsqueeze(-1) - grid).abs()
                near = away == away.amin(-1, keepdim=True)
                even = near & (torch.arange(8, device=DEVICE) % 2 == 0)     # of two that are as near the even one
                code = torch.where(even.any(-1, keepdim=True), even, near).byte().argmax(-1)
                out[b, :n] = (grid[code] * scale * g.sign()).flatten(-2)
            read.append(out)
        if weights is None:
            return read
        for b, n in enumerate(counts):
            i = torch.arange(lengths[b] - n, lengths[b], device=DEVICE)
            weights[places[b][i], :, i % page] = 0.0
        return [*read, weights]
    value = torch.tensor(list(MAGNITUDES) + [-m for m in MAGNITUDES], dtype=torch.float64, device=DEVICE)
    if case["op"] == "attend":
        out = torch.zeros((batch, new, heads, dim), dtype=torch.float64, device=DEVICE)
        lse = torch.full((batch, new, heads), float("-inf"), dtype=torch.float64, device=DEVICE)
        parts = _parts(s["pool"], page, dim)
        for b, n in enumerate(counts):
            j = torch.arange(lengths[b], device=DEVICE)
            for h in range(hkv):
                k, v = (torch.stack((value[(c & 15).long()], value[(c >> 4).long()]), -1).flatten(-2)
                        * torch.exp2(e.double() - 127).repeat_interleave(GROUP, dim=-1)
                        for c, e in ((parts[a][places[b], h, j % page], parts[a + 2][places[b], h, j % page]) for a in (0, 1)))
                for r in range(0, n, 512):
                    i = torch.arange(r, min(n, r + 512), device=DEVICE)
                    q = s["q"][b, i, h * group:(h + 1) * group].double()
                    scores = (q.flatten(0, 1) @ k.T).view(len(i), group, -1) * dim ** -0.5
                    scores = scores.masked_fill((j > (lengths[b] - n + i)[:, None])[:, None], float("-inf"))
                    lse[b, i, h * group:(h + 1) * group] = scores.logsumexp(-1)
                    p = scores.softmax(-1)
                    out[b, i, h * group:(h + 1) * group] = (p.flatten(0, 1) @ v).view(len(i), group, dim)
                    if weights is not None:
                        weights[places[b], h, j % page] += p.sum((0, 1))
        return [out, lse] if weights is None else [out, lse, weights]
    for b, n in enumerate(lengths):
        j = torch.arange(n, device=DEVICE)
        for h in range(hkv):
            w = s["accumulated"][places[b], h, j % page]
            old = max(0, n - case["recent"])
            heavy = w[:old].sort(descending=True, stable=True).indices[:max(0, min(n, case["keep"]) - (n - old))]
            kept = torch.cat((heavy.sort().values, j[old:]))
            to = torch.arange(len(kept), device=DEVICE)
            weights[s["new_table"][b].long()[to // page], h, to % page] = w[kept].double()
    return [None, None, None, weights[s["table"].numel():]]
