"""What the 4-bit linear layer and the norm in front of it are judged by: the cases, their plain form, and the calls of ``triton_int8_amd``.

The 4-bit format: a code is a float of 4 bits (sign, magnitude 0 .5 1 1.5 2 3 4 6; the even element in the low half of a byte); 32 neighbours of a
row share a scale byte e, which stands for 2^(e - 127): the smallest power of two (e at least 1) by which the largest of them is at most 6.  A row's
codes take whole tiles of 256 elements, zeros behind its end: uint8 [rows, tiles * 128]; the scales are uint8 [tiles, rows, 8].

Operators:
  quant   rows, columns (as rows of the transposed tensor) or both into 4 bits, and the values that they stand for
  gemm    A B^T of two tensors in 4 bits
  step    a linear layer's forward and backward, every product in 4 bits: Y = X W^T, dX = dY W, dW = dY^T X
  norm    residual added, root-mean-square norm, result in 4 bits, or in 8 with a scale per row or per 128 columns; and the values that it stands for
"""
import math

import torch

own = False
DEVICE = "cuda:0"
GROUP, TILE = 32, 256
EPS = 1e-5
MAGNITUDES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _quant(rows, cols, way):
    return {"op": "quant", "rows": rows, "cols": cols, "way": way}


def _gemm(m, n, k, *, batch=1, shared=True, wide=False):
    return {"op": "gemm", "batch": batch, "m": m, "n": n, "k": k, "shared": shared, "wide": wide}


def _step(tokens, k, n):
    return {"op": "step", "tokens": tokens, "k": k, "n": n}


def _norm(rows, dim, to, *, group=0, residual=True):
    return {"op": "norm", "rows": rows, "dim": dim, "to": to, "group": group, "residual": residual}


def listed():
    return [
        # gradients of ragged prompts through a narrow layer, both ways as a backward needs them
        {"name": "quant_ragged", **_quant(1001, 1016, "both")},
        # an MLP weight of the benchmark's decoder layer, both ways as a training step needs it
        {"name": "quant_weight", **_quant(14336, 4096, "both")},
        # a single decode stream through a projection: latency and the weight's bytes
        {"name": "gemm_token", **_gemm(1, 4096, 4096)},
        # a decode batch through an MLP projection: a stream of the weight
        {"name": "gemm_decode", **_gemm(32, 14336, 4096)},
        # products of a batch, odd sizes, results in 32 bits
        {"name": "gemm_batch", **_gemm(333, 1001, 1000, batch=5, shared=False, wide=True)},
        # a short prompt through an attention projection: too few rows to fill the card with large tiles
        {"name": "gemm_short", **_gemm(700, 4096, 4096)},
        # prompts of the benchmark's token count through an MLP projection: matrix instructions all the way
        {"name": "gemm_prompt", **_gemm(8192, 14336, 4096)},
        # a small layer on a ragged batch, forward and backward
        {"name": "step_ragged", **_step(1000, 1024, 2560)},
        # the benchmark's layer, forward and backward
        {"name": "step", **_step(8192, 4096, 4096)},
        # one new token of a decoder layer on its way into 4-bit projections: latency is all there is
        {"name": "norm_token", **_norm(1, 4096, "mx4")},
        # a prompt on its way into int8 projections whose scales go by 128 columns
        {"name": "norm_int8", **_norm(2047, 4096, "int8", group=128)},
        # the prompts of the benchmark's decoder layer: 4 x 4096 tokens
        {"name": "norm_prompt", **_norm(16384, 4096, "mx4")},
    ]


def _log(rng, low, high):
    return min(high, max(low, int(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def _cost(case):
    w = work(case)
    return w["bytes"] + w["flops"] / 500


def draw(rng):
    most = {}
    for c in listed():
        most[c["op"]] = max(most.get(c["op"], 0), _cost(c))
    while True:
        op = rng.choice(("quant", "gemm", "gemm", "gemm", "step", "norm", "norm"))
        if op == "quant":
            c = _quant(_log(rng, 1, 16384), _log(rng, 1, 16384), rng.choice(("row", "col_t", "both")))
        elif op == "gemm":
            batch, m = rng.choice((1, 1, _log(rng, 2, 16))), rng.choice((_log(rng, 1, 64), _log(rng, 64, 8192)))
            c = _gemm(m, _log(rng, 1, 16384), _log(rng, 1, 16384), batch=batch, shared=batch == 1 or rng.random() < 0.5, wide=rng.random() < 0.3)
        elif op == "step":
            c = _step(_log(rng, 1, 8192), 8 * _log(rng, 2, 1024), 8 * _log(rng, 2, 1024))
        else:
            to = rng.choice(("mx4", "mx4", "int8"))
            dim = 128 * _log(rng, 1, 64) if to == "int8" else 8 * _log(rng, 1, 1024)
            c = _norm(_log(rng, 1, 16384), dim, to, group=rng.choice((0, 128)) if to == "int8" else 0, residual=rng.random() < 0.7)
        if _cost(c) <= most[op]:
            return c


def _held(elements):
    """bytes of so many elements in 4 bits with their scales"""
    return elements * 17 / 32


def work(case):
    if case["op"] == "quant":
        n = case["rows"] * case["cols"]
        ways = 2 if case["way"] == "both" else 1
        return {"bytes": 2 * n + ways * (_held(n) + 2 * n), "flops": 0}
    if case["op"] == "gemm":
        b, m, n, k = (case[x] for x in ("batch", "m", "n", "k"))
        return {"bytes": _held(b * m * k + (1 if case["shared"] else b) * n * k) + (4 if case["wide"] else 2) * b * m * n, "flops": 2 * b * m * n * k}
    if case["op"] == "step":
        t, k, n = (case[x] for x in ("tokens", "k", "n"))
        return {"bytes": 2 * (2 * t * k + 2 * t * n + 2 * n * k), "flops": 6 * t * k * n}
    n = case["rows"] * case["dim"]
    held = _held(n) if case["to"] == "mx4" else n + 4 * case["rows"] * max(1, case["dim"] // case["group"] if case["group"] else 1)
    return {"bytes": (2 + 4 * case["residual"]) * n + held + 2 * n + 4 * case["rows"] + 2 * case["dim"], "flops": 0}


def _encode(x):
    """float32 [rows, cols] -> codes uint8 [rows, tiles * 128], scales uint8 [tiles, rows, 8]."""
    x = torch.nn.functional.pad(x, (0, -x.shape[1] % TILE))
    g = x.unflatten(-1, (-1, GROUP))
    amax = g.abs().amax(-1)
    # the smallest power of two by which the largest of a group is no more than 6 (1.5 2^2): up by one where the fraction is over 1.5
    scale = (((amax.view(torch.int32) + 0x3fffff) >> 23) - 2).clamp(1, 254)
    y = (g * ((254 - scale) << 23).view(torch.float32).unsqueeze(-1)).flatten(-2)
    a = y.abs()
    code = ((a > 0.25).byte() + (a >= 0.75).byte() + (a > 1.25).byte() + (a >= 1.75).byte() + (a > 2.5).byte() + (a >= 3.5).byte() + (a > 5.0).byte()
            + (y < 0).byte() * 8)
    return code[:, 0::2] | (code[:, 1::2] << 4), scale.byte().unflatten(-1, (-1, 8)).transpose(0, 1).contiguous()


def _decode(codes, scales):
    """codes [.., rows, tiles * 128], scales [tiles, all rows, 8] -> float32 [.., rows, tiles * 256]."""
    value = torch.tensor(list(MAGNITUDES) + [-m for m in MAGNITUDES], device=codes.device)
    x = torch.stack((value[(codes & 15).int()], value[(codes >> 4).int()]), -1).flatten(-2)
    e = scales.transpose(0, 1).reshape(*codes.shape[:-1], -1)
    return (x.unflatten(-1, (-1, GROUP)) * (e.int() << 23).view(torch.float32).unsqueeze(-1)).flatten(-2)


def _quantised(x):
    """The values, float32, that the rows of x have in 4 bits."""
    return _decode(*_encode(x.float()))[:, :x.shape[1]]


def _activations(gen, rows, cols):
    """Normal, with one channel of a hundred twenty times as large."""
    x = torch.randn((rows, cols), generator=gen, device=DEVICE)
    x[:, torch.randperm(cols, generator=gen, device=DEVICE)[:max(1, cols // 100)]] *= 20
    return x.bfloat16()


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    normal = lambda *shape: torch.randn(shape, generator=gen, device=DEVICE)  # noqa: E731
    s = dict(case)
    if case["op"] == "quant":
        s["x"] = _activations(gen, case["rows"], case["cols"])
    elif case["op"] == "gemm":
        b, m, n, k = (case[x] for x in ("batch", "m", "n", "k"))
        s["a"], s["sa"] = _encode(_activations(gen, b * m, k).float())
        s["b"], s["sb"] = _encode((normal(n if case["shared"] else b * n, k) * 0.02).bfloat16().float())
        if b > 1:
            s["a"] = s["a"].view(b, m, -1)
        if not case["shared"]:
            s["b"] = s["b"].view(b, n, -1)
    elif case["op"] == "step":
        s["x"], s["w"], s["dy"] = _activations(gen, case["tokens"], case["k"]), (normal(case["n"], case["k"]) * 0.02).bfloat16(), (normal(case["tokens"], case["n"]) * 1e-3).bfloat16()
    else:
        s["x"] = _activations(gen, case["rows"], case["dim"])
        s["residual"] = _activations(gen, case["rows"], case["dim"]) if s["residual"] else None
        s["weight"] = (1.0 + 0.1 * normal(case["dim"])).bfloat16()
    return s


def run(s):
    if not own:
        return {"quant": _plain_quant, "gemm": _plain_gemm, "step": _plain_step, "norm": _plain_norm}[s["op"]](s)
    from triton_int8_amd import mx4, ops
    if s["op"] == "quant":
        rows, cols = s["x"].shape
        if s["way"] == "row":
            return [mx4.dequant(*mx4.quant_row(s["x"]), cols)]
        if s["way"] == "col_t":
            return [mx4.dequant(*mx4.quant_col_t(s["x"]), rows)]
        q, e, qt, et = mx4.quant_row_col_t(s["x"])
        return [mx4.dequant(q, e, cols), mx4.dequant(qt, et, rows)]
    if s["op"] == "gemm":
        return mx4.gemm_nt(s["a"], s["sa"], s["b"], s["sb"], out_dtype=torch.float32 if s["wide"] else torch.bfloat16)
    if s["op"] == "step":
        return list(mx4.linear_fwd_bwd(s["x"], s["w"], s["dy"]))
    q, e, rstd, *h = ops.rmsnorm_quant(s["x"], s["weight"], EPS, residual=s["residual"], to=s["to"], group=s["group"])
    return [mx4.dequant(q, e, s["dim"]) if s["to"] == "mx4" else ops.dequant_row(q, e), rstd, *h]


def _plain_quant(s):
    ways = {"row": (s["x"],), "col_t": (s["x"].t(),), "both": (s["x"], s["x"].t())}[s["way"]]
    return [_quantised(x).bfloat16() for x in ways]


def _plain_gemm(s):
    out = torch.matmul(_decode(s["a"], s["sa"]), _decode(s["b"], s["sb"]).transpose(-1, -2))
    return out if s["wide"] else out.bfloat16()


def _plain_step(s):
    x, w, dy = s["x"], s["w"], s["dy"]
    return [torch.matmul(_quantised(a), _quantised(b).t()).bfloat16() for a, b in ((x, w), (dy, w.t()), (dy.t(), x.t()))]


def _plain_norm(s):
    x = s["x"] if s["residual"] is None else (s["x"].float() + s["residual"].float()).bfloat16()
    # in 64 bits, so that no code next to a border goes by the order of a sum
    rstd = (1.0 / (x.double().square().mean(-1) + EPS).sqrt()).float()
    y = ((x.float() * rstd[:, None]).bfloat16().float() * s["weight"].float()).bfloat16().float()
    if s["to"] == "mx4":
        values = _quantised(y)
    else:
        g = y.unflatten(-1, (-1, s["group"] or s["dim"]))
        amax = g.abs().amax(-1, keepdim=True).clamp_min(1e-4)
        scale = torch.full_like(amax, 127.0) / amax
        values = ((g * scale + 0.5).floor().clamp(-128, 127) * (torch.ones_like(scale) / scale)).flatten(-2)
    return [values.bfloat16(), rstd, *([] if s["residual"] is None else [x])]


def _exactly(x):
    """The nearest values that the rows of x (64 bits) have in 4 bits, of two that are as near the one with the even code."""
    grid = torch.tensor(MAGNITUDES, dtype=torch.float64, device=DEVICE)
    even = torch.arange(8, device=DEVICE) % 2 == 0
    cols, parts = x.shape[1], []
    for rows in x.split(max(1, (1 << 24) // max(1, x.shape[1]))):
        g = torch.nn.functional.pad(rows, (0, -cols % GROUP)).unflatten(-1, (-1, GROUP))
        scale = torch.exp2(torch.ceil(torch.log2(g.abs().amax(-1, keepdim=True) / 6).clamp_min(-126)))
        away = ((g / scale).abs().unsqueeze(-1) - grid).abs()
        near = away == away.amin(-1, keepdim=True)
        code = torch.where((near & even).any(-1, keepdim=True), near & even, near).byte().argmax(-1)
        parts.append((grid[code] * scale * g.sign()).flatten(-2)[:, :cols])
    return torch.cat(parts)


def _held_values(codes, scales, k):
    """What codes and scales stand for, in 64 bits: [rows, k]."""
    value = torch.tensor(list(MAGNITUDES) + [-m for m in MAGNITUDES], dtype=torch.float64, device=DEVICE)
    rows = codes.reshape(-1, codes.shape[-1])
    x = torch.empty((rows.shape[0], 2 * rows.shape[1]), dtype=torch.float64, device=DEVICE)
    x[:, 0::2], x[:, 1::2] = value[(rows & 15).long()], value[(rows >> 4).long()]
    for g in range(x.shape[1] // GROUP):
        x[:, g * GROUP:(g + 1) * GROUP] *= torch.exp2(scales[g // 8, :, g % 8].double() - 127)[:, None]
    return x[:, :k]


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "quant":
        ways = {"row": [s["x"]], "col_t": [s["x"].t()], "both": [s["x"], s["x"].t()]}[case["way"]]
        return [_exactly(x.double()) for x in ways]
    if case["op"] == "gemm":
        b, m, n, k = (case[x] for x in ("batch", "m", "n", "k"))
        left, right = _held_values(s["a"], s["sa"], k), _held_values(s["b"], s["sb"], k)
        if case["shared"]:
            out = left @ right.t()
            return out.view(b, m, n) if b > 1 else out
        return torch.stack([left[i * m:(i + 1) * m] @ right[i * n:(i + 1) * n].t() for i in range(b)])
    if case["op"] == "step":
        x, w, dy = (s[t].double() for t in ("x", "w", "dy"))
        return [_exactly(x) @ _exactly(w).t(), _exactly(dy) @ _exactly(w.t()).t(), _exactly(dy.t()) @ _exactly(x.t()).t()]
    rounded = lambda t: t.bfloat16().double()  # noqa: E731
    x = s["x"].double() if s["residual"] is None else rounded(s["x"].double() + s["residual"].double())
    rstd = (x.pow(2).sum(-1) / case["dim"] + EPS).rsqrt()
    y = rounded(rounded(x * rstd[:, None]) * s["weight"].double())
    if case["to"] == "mx4":
        values = _exactly(y)
    else:
        values = torch.empty_like(y)
        width = case["group"] or case["dim"]
        for c in range(0, case["dim"], width):
            g = y[:, c:c + width]
            step = g.abs().amax(-1, keepdim=True).clamp_min(1e-4) / 127
            values[:, c:c + width] = torch.floor(g / step + 0.5).clamp(max=127) * step
    return [values, rstd, *([] if s["residual"] is None else [x])]
