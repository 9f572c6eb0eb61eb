"""The norm whose result is quantised on the way out, against the oracle's norm and quantisers.

The mean is taken in 64 bits on both sides and rounded to 32 bits once, after which every operation is a rounding of its own: everything is compared bit for bit."""
import pytest
import torch

from conftest import bits_equal, make_gen, randn_bf16, rel_err
from oracle import mx4 as oracle

pytestmark = pytest.mark.gpu
EPS = 1e-5


@pytest.fixture(scope="module")
def T():
    import triton_int8_amd
    return triton_int8_amd


def inputs(rows, dim, residual=True, seed=0):
    gen = make_gen(rows * 31 + dim + seed)
    x = torch.randn(rows, dim, generator=gen) * torch.exp2(torch.randint(-20, 20, (rows, 1), generator=gen).float())
    x[:, dim // 3] *= 20
    if rows > 3:
        x[2] = 0
    x = x.bfloat16()
    return x, 1.0 + randn_bf16(gen, dim, std=0.2), (x.float() * torch.randn(rows, dim, generator=gen)).bfloat16() if residual else None


def check(T, dev, x, w, r, to="mx4", eps=EPS, **kw):
    y, rstd, h = oracle.norm(x, w, eps, r)
    put = lambda t: None if t is None else t.to(dev)  # noqa: E731
    got = T.ops.rmsnorm_quant(put(x), put(w), eps, residual=put(r), to=to, **kw)
    assert len(got) == (3 if r is None else 4)
    q, s, at = got[:3]
    assert at.shape == x.shape[:-1] and bits_equal(at, rstd.float())
    if r is not None:
        assert bits_equal(got[3], h)
    if to == "mx4":
        codes, scales = oracle.quant_row(y.flatten(0, -2))
        assert q.shape[:-1] == x.shape[:-1] and torch.equal(q.cpu().flatten(0, -2), codes) and torch.equal(s.cpu(), scales)
    else:
        codes, scales = T.ops.quant_row(y.to(dev), **kw)
        assert q.dtype == torch.int8 and s.shape == scales.shape and torch.equal(q, codes) and torch.equal(s, scales)
        values = T.ops.dequant_row(q, s)
        wide = q.float() * (s.unsqueeze(-1) if s.dim() < q.dim() else s.repeat_interleave(128, -1))
        assert bits_equal(values, wide.bfloat16())


@pytest.mark.parametrize("dim", [8, 32, 56, 256, 264, 512, 520, 1000, 1024, 1032, 2048, 2560, 4096, 4104, 8192, 8200, 14336, 16384])
@pytest.mark.parametrize("rows,residual", [(1, True), (5, False), (6, True)])
def test_mx4(T, dev, rows, dim, residual):
    check(T, dev, *inputs(rows, dim, residual))


@pytest.mark.parametrize("dim", [128, 256, 640, 1024, 1152, 2048, 4096, 5120, 8192, 12288, 16384])
@pytest.mark.parametrize("group", [0, 128])
@pytest.mark.parametrize("residual", [True, False])
def test_int8(T, dev, dim, group, residual):
    check(T, dev, *inputs(7, dim, residual), to="int8", group=group)


@pytest.mark.parametrize("group", [0, 128])
def test_int8_other_scales(T, dev, group):
    for mode in (T._lib.INV_AMAX_DIV_127, T._lib.INV_MULTIPLIER, T._lib.INV_AMAX_MUL_RCP127):
        check_mode = dict(to="int8", group=group, inv_mode=mode)
        x, w, r = inputs(5, 384)
        y, _, _ = oracle.norm(x, w, EPS, r)
        q, s, *_ = T.ops.rmsnorm_quant(x.to(dev), w.to(dev), EPS, residual=r.to(dev), **check_mode)
        codes, scales = T.ops.quant_row(y.to(dev), group=group, inv_mode=mode)
        assert torch.equal(q, codes) and torch.equal(s, scales)


@pytest.mark.parametrize("rows", [2, 3, 4, 9, 63, 300, 2100])
def test_many_rows(T, dev, rows):
    for dim in (264, 2304):
        check(T, dev, *inputs(rows, dim))
    check(T, dev, *inputs(rows, 384), to="int8", group=128)


@pytest.mark.parametrize("rows", [1, 7, 300, 400, 401, 402, 403, 404, 405, 900])       # (around 4 MB in all, up to which they share a block)
def test_results_lie_apart(T, dev, rows):
    x, w, r = (t.to(dev) for t in inputs(rows, 4096))
    for results in (T.ops.rmsnorm_quant(x, w, EPS, residual=r), T.ops.rmsnorm_quant(x, w, EPS, residual=r, to="int8", group=128), T.ops.rmsnorm_quant(x, w, EPS),
                    T.mx4.quant_row_col_t(x[:, :1000])):
        spans = sorted((t.data_ptr(), t.data_ptr() + t.numel() * t.element_size()) for t in results)
        assert all(a[1] <= b[0] for a, b in zip(spans, spans[1:])) and all(a % 16 == 0 for a, _ in spans)
        for t in results:
            assert t.is_contiguous() and t.untyped_storage().nbytes() >= (t.storage_offset() + t.numel()) * t.element_size()
        kept = [t.clone() for t in results]
        for i, t in enumerate(results):
            t.zero_()
            assert all(torch.equal(a, b) for a, b in zip(results[i + 1:], kept[i + 1:]))


@pytest.mark.parametrize("eps", [0.0, 1e-12, 1.0])
def test_eps(T, dev, eps):
    x, w, r = inputs(3, 512)
    check(T, dev, x, w, r, eps=eps)
    check(T, dev, (x.float() * 1e-6).bfloat16(), w, None, eps=eps)


def test_views(T, dev):
    x, w, r = inputs(12, 512)
    wide = torch.randn(3, 4, 700, generator=make_gen(1)).bfloat16().to(dev)
    inside = wide[:, :, 8:520]
    got = T.ops.rmsnorm_quant(inside, w.to(dev), EPS, residual=r.to(dev).view(3, 4, 512))
    want = T.ops.rmsnorm_quant(inside.contiguous(), w.to(dev), EPS, residual=r.to(dev).view(3, 4, 512))
    odd = T.ops.rmsnorm_quant(wide[:, :, 3:515], torch.cat((w, w)).to(dev)[1::2], EPS, residual=r.to(dev).view(3, 4, 512))
    odd_want = T.ops.rmsnorm_quant(wide[:, :, 3:515].contiguous(), torch.cat((w, w)).to(dev)[1::2].contiguous(), EPS, residual=r.to(dev).view(3, 4, 512))
    for a, b in ((got, want), (odd, odd_want)):
        assert a[0].shape == (3, 4, 256) and a[2].shape == (3, 4) and a[3].shape == (3, 4, 512)
        assert all(torch.equal(u, v) for u, v in zip(a, b))
    one = T.ops.rmsnorm_quant(x[0].to(dev), w.to(dev), EPS)
    assert one[0].shape == (256,) and one[2].shape == () and torch.equal(one[0], T.ops.rmsnorm_quant(x[:1].to(dev), w.to(dev), EPS)[0][0])


def test_nan_and_infinity_spoil_their_row(T, dev):
    x, w, _ = inputs(4, 512, False)
    x[1, 7], x[3, 500] = float("nan"), float("inf")
    q, s, rstd = T.ops.rmsnorm_quant(x.to(dev), w.to(dev), EPS)
    clean = torch.tensor([0, 2])
    want = T.ops.rmsnorm_quant(x[clean].to(dev), w.to(dev), EPS)
    assert torch.equal(q[clean], want[0]) and torch.equal(s[:, clean], want[1])
    assert bool((s[:, 1] == 255).all()) and rstd[1].isnan() and rstd[3] == 0
    assert s[1, 3].tolist().count(255) == 1         # infinity times zero; the others are zeros


@pytest.mark.parametrize("rows,dim", [(3, 256), (40, 1024)])
def test_gradient_goes_back_through_the_norm_alone(T, dev, rows, dim):
    """The gradient of y, handed to rmsnorm_backward with the h and rstd of the call: against the formula in 64 bits and against differences."""
    x, w, r = inputs(rows, dim, seed=3)
    x, r = (x.float() / x.float().norm(dim=1, keepdim=True).clamp_min(1e-3) * dim ** 0.5).bfloat16(), (0.1 * torch.randn(rows, dim, generator=make_gen(4))).bfloat16()
    dy = randn_bf16(make_gen(5), rows, dim)
    q, s, rstd, h = T.ops.rmsnorm_quant(x.to(dev), w.to(dev), EPS, residual=r.to(dev))
    dh, dw = T.ops.rmsnorm_backward(dy.to(dev), h, w.to(dev), rstd)
    hd, wd, d = h.cpu().double(), w.double(), dy.double()
    norm = lambda t, u: t * torch.rsqrt(t.square().mean(-1, keepdim=True) + EPS) * u  # noqa: E731
    rr = torch.rsqrt(hd.square().mean(-1, keepdim=True) + EPS)
    want = rr * (d * wd) - hd * rr ** 3 * (d * wd * hd).mean(-1, keepdim=True)
    # three roundings to bf16 on the way to dh (dy w, the two terms' sum): half a step each of terms that no component's sum exceeds; dw: product and sum
    assert rel_err(dh, want) <= 3 * 2.0 ** -8
    assert rel_err(dw, (d * hd * rr).sum(0)) <= 4 * 2.0 ** -8
    step = torch.randn(rows, dim, generator=make_gen(6), dtype=torch.float64)
    e = 1e-5
    slope = ((norm(hd + e * step, wd) - norm(hd - e * step, wd)) * d).sum() / (2 * e)
    assert abs(float((want * step).sum() - slope)) <= 1e-6 * float((want.abs() * step.abs()).sum())


def test_norm_then_products(T, dev):
    """Residual, norm and both kinds of linear behind it, as a layer makes them."""
    x, w, r = inputs(50, 512)
    weight = randn_bf16(make_gen(9), 384, 512, std=0.02).to(dev)
    y, _, _ = oracle.norm(x, w, EPS, r)
    q, s, _, h = T.ops.rmsnorm_quant(x.to(dev), w.to(dev), EPS, residual=r.to(dev))
    with torch.no_grad():
        layer = T.Mx4Linear(512, 384, device=dev)
        layer.weight.copy_(weight)
        assert bits_equal(T.mx4.gemm_nt(q, s, *layer.quantised()), layer(y.to(dev)))
    q, s, _, _ = T.ops.rmsnorm_quant(x.to(dev), w.to(dev), EPS, residual=r.to(dev), to="int8")
    wq, ws = T.linear.quantize_weight(weight, "double_channel")
    pad = torch.nn.functional.pad
    got = T.ops.gemm_i8_nt(pad(q, (0, 0, 0, 14))[None], wq, pad(s, (0, 14))[None], T._lib.SCALE_ROW, ws, T._lib.SCALE_ROW, acc_i32_full=True)[0, :50]
    want = (q.double() * s.double()[:, None]) @ (wq.double() * ws.double()[:, None]).t()
    assert rel_err(got, want) <= 2.0 ** -8
