"""The 4-bit key / value cache in plain torch on the CPU: what its codes and scales are, and attention and eviction in float64.

No counterpart in the reference.  Layout and rules: ``include/ti8.h``, ti8_cache4."""
import torch

MAGNITUDES = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)
LARGEST = 1.5 * 2.0 ** 127


def encode(x):
    """bf16 [..., D] -> (codes 0 .. 15 uint8 [..., D], scales uint8 [..., D / 32])."""
    g = torch.nan_to_num(x.double(), nan=0.0, posinf=LARGEST, neginf=-LARGEST).clamp(-LARGEST, LARGEST).unflatten(-1, (-1, 32))
    negative = torch.signbit(g)
    g = g.abs()
    mantissa, exponent = torch.frexp(g.amax(-1, keepdim=True))          # amax = mantissa 2^exponent, 0.5 <= mantissa < 1
    e = torch.where(mantissa == 0, -126, exponent - 3 + (mantissa > 0.75)).clamp(-126, 125)      # 6 = 0.75 2^3
    y = g / torch.exp2(e.double())
    away = (y.unsqueeze(-1) - MAGNITUDES).abs()
    nearest = away == away.amin(-1, keepdim=True)
    even = nearest & (torch.arange(8) % 2 == 0)
    code = torch.where(even.any(-1, keepdim=True), even, nearest).byte().argmax(-1)
    return (code + 8 * negative).flatten(-2).byte(), (e.squeeze(-1) + 127).byte()


def decode(codes, scales):
    """The values in float64."""
    v = MAGNITUDES[(codes & 7).long()] * torch.where(codes >= 8, -1.0, 1.0)
    return (v.unflatten(-1, (-1, 32)) * torch.exp2(scales.double() - 127).unsqueeze(-1)).flatten(-2)


def parts(pool, page, dim):
    """Views of a pool [pages, heads, bytes]: packed codes of keys and of values [.., page, dim / 2], scales of keys and of values [.., page, dim / 32]."""
    sizes = (page * dim // 2, page * dim // 2, page * dim // 32, page * dim // 32)
    return tuple(t.unflatten(-1, (page, -1)) for t in pool.split(sizes, dim=-1))


def put(pool, page, dim, at, row, head, k, v):
    """Key and value bf16 [D] as entry `row` of page `at`."""
    p = parts(pool, page, dim)
    for x, codes_at, scales_at in ((k, p[0], p[2]), (v, p[1], p[3])):
        codes, scales = encode(x)
        codes_at[at, head, row] = codes[0::2] | (codes[1::2] << 4)
        scales_at[at, head, row] = scales


def entries(pool, table_row, page, dim, head, length):
    """(keys, values) float64 [length, D] of a sequence's entries."""
    j = torch.arange(length)
    at = table_row.long()[j // page]
    p, out = parts(pool, page, dim), []
    for codes_at, scales_at in ((p[0], p[2]), (p[1], p[3])):
        packed = codes_at[at, head, j % page]
        out.append(decode(torch.stack((packed & 15, packed >> 4), -1).flatten(-2), scales_at[at, head, j % page]))
    return out


def attention(pool, table, lengths, q, counts, scale, page):
    """(out, lse, weights' gain per entry [batch][kv head][entry], bounds): float64.  `bounds` = per (batch, token, head) the largest sum of
    |q k| scale over the visible keys, and sum p |v| of every output: what roundings scale with."""
    B, S, H, D = q.shape
    hkv = pool.shape[1]
    out, lse = torch.zeros(B, S, H, D, dtype=torch.float64), torch.full((B, S, H), float("-inf"), dtype=torch.float64)
    logits, spread = torch.zeros(B, S, H, dtype=torch.float64), torch.zeros(B, S, H, D, dtype=torch.float64)
    gains = [[torch.zeros(n, dtype=torch.float64) for _ in range(hkv)] for n in lengths]
    for b in range(B):
        n = lengths[b]
        for h in range(hkv):
            k, v = entries(pool, table[b], page, D, h, n)
            for t in range(counts[b]):
                sees = n - counts[b] + t + 1
                if sees <= 0:
                    continue
                x = slice(h * (H // hkv), (h + 1) * (H // hkv))
                rows = q[b, t, x].double()
                s = rows @ k[:sees].T * scale
                p = s.softmax(-1)
                out[b, t, x], lse[b, t, x] = p @ v[:sees], s.logsumexp(-1)
                logits[b, t, x] = (rows.abs() @ k[:sees].abs().T * scale).amax(-1)
                spread[b, t, x] = p @ v[:sees].abs()
                gains[b][h][:sees] += p.sum(0)
    return out, lse, gains, logits, spread


def kept(weights, recent, keep):
    """Which entries of a sequence's head stay, in order (weights [length])."""
    n = len(weights)
    if n <= keep:
        return list(range(n))
    old = n - recent
    key = lambda j: (0, 0.0) if weights[j] != weights[j] else (1, -float(weights[j]) + 0.0)     # NaN in front of every number
    heavy = sorted(range(old), key=lambda j: (key(j), j))[:keep - recent]
    return sorted(heavy) + list(range(old, n))
