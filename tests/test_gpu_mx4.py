"""Tensors in 4 bits, their product and the layer made of them, against the oracle in 64 bits.

Codes and scales are compared bit for bit.  A product of two codes is exact in fp32 with its scales, so a sum of K of them is off by at most one rounding
per addition, 2^-23 of the sum of magnitudes each (truncations counted in), and by half a step of its own type, 2^-8 of its value in bf16 and 2^-24 in fp32."""
import pytest
import torch

from conftest import bits_equal, make_gen, randn_bf16
from oracle import mx4 as oracle

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def M():
    import triton_int8_amd
    return triton_int8_amd.mx4


def tensor(gen, rows, cols, spread=True):
    """Rows with magnitudes over many powers of two, an outlier channel, ties and zeros."""
    x = torch.randn(rows, cols, generator=gen)
    if spread:
        x *= torch.exp2(torch.randint(-12, 12, (rows, 1), generator=gen).float())
        x[:, cols // 2] *= 20
        x[rows // 2] = 0
        x[:, ::7] = torch.randint(-12, 13, x[:, ::7].shape, generator=gen) / 2
    return x.to(torch.bfloat16)


def same(got, want, what=""):
    for g, w, name in zip(got, want, ("codes", "scales")):
        assert g.shape == w.shape and g.dtype == w.dtype, (what, name, g.shape, w.shape)
        assert torch.equal(g.cpu(), w), (what, name, int((g.cpu() != w).sum()))


SIZES = [(1, 1), (1, 32), (1, 4096), (2, 31), (3, 33), (5, 256), (7, 257), (32, 64), (33, 255), (63, 100), (64, 512), (65, 777), (255, 24), (256, 256), (257, 40), (300, 1000),
         (1001, 1016), (1, 70000), (70000, 1)]


@pytest.mark.parametrize("rows,cols", SIZES)
def test_quantisers(M, dev, rows, cols):
    x = tensor(make_gen(rows * 1000 + cols), rows, cols)
    by_rows, by_columns = oracle.quant_row(x), oracle.quant_row(x.t())
    d = x.to(dev)
    same(M.quant_row(d), by_rows, "row")
    same(M.quant_col_t(d), by_columns, "col_t")
    q, s, qt, st = M.quant_row_col_t(d)
    same((q, s), by_rows, "both, rows")
    same((qt, st), by_columns, "both, columns")
    for (codes, scales), n in ((by_rows, cols), (by_columns, rows)):
        assert bits_equal(M.dequant(codes.to(dev), scales.to(dev), n), oracle.values(codes, scales, n).bfloat16())


def test_quantisers_on_large_tiles(M, dev):
    """Tensors with enough tiles for the quantiser's large ones, ragged at both ends."""
    rows, cols = 256 * 24 + 41, 256 * 22 + 9
    x = tensor(make_gen(5), rows, cols)
    q, s, qt, st = M.quant_row_col_t(x.to(dev))
    same((q, s), oracle.quant_row(x), "rows")
    same((qt, st), oracle.quant_row(x.t()), "columns")
    same(M.quant_col_t(x.to(dev)), oracle.quant_row(x.t()), "columns alone")


@pytest.mark.parametrize("what", ["transposed", "columns", "odd start", "rows apart", "expanded", "three dims", "one row"])
def test_quantisers_read_views(M, dev, what):
    base = tensor(make_gen(3), 130, 301).to(dev)
    x = {"transposed": lambda: base.t(), "columns": lambda: base[:, 3:290], "odd start": lambda: base.flatten()[1:1 + 120 * 300].view(120, 300), "rows apart": lambda: base[::3],
         "expanded": lambda: base[:1].expand(70, -1), "three dims": lambda: base.view(10, 13, 301), "one row": lambda: base[5:6, 7:]}[what]()
    flat = x.reshape(-1, x.shape[-1]).cpu().contiguous()
    q, s = M.quant_row(x)
    assert q.shape[:-1] == x.shape[:-1]
    same((q.view(flat.shape[0], -1), s), oracle.quant_row(flat), what)
    if x.dim() == 2:
        same(M.quant_col_t(x), oracle.quant_row(flat.t()), what)
        same(M.quant_row_col_t(x)[2:], oracle.quant_row(flat.t()), what)


def test_numbers_at_the_ends_of_the_range(M, dev):
    """The largest and smallest numbers, every border between two codes, infinities and NaN: which spoil their own group only."""
    x = torch.zeros(9, 96)
    x[0, :4] = torch.tensor([3.3895313892515355e38, -3.3895313892515355e38, 1e38, 2.0 ** 127])
    x[1, :6] = torch.tensor([2.0 ** -126, 2.0 ** -127, -(2.0 ** -128), 2.0 ** -125, 1.5 * 2.0 ** -126, 2.0 ** -133])
    x[2, :7] = torch.tensor([6.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5]) * 2.0 ** 90
    x[3, :7] = torch.tensor([6.0, 5.0, -5.0, -0.25, 0.24902344, 4.96875, 5.03125]) * 2.0 ** -90
    x[4, :2] = torch.tensor([6.0, 6.03125])
    x[5, 40] = float("inf")
    x[6, 0] = float("nan")
    x[7, 95] = -float("inf")
    x[8, :3] = torch.tensor([-0.0, 1.0, -1e-30])
    x[5:8, 1] = 3.0
    x = x.to(torch.bfloat16)
    codes, scales = oracle.quant_row(x)
    assert scales[0, 0, 0] == 252 and scales[0, 1, 0] == 1 and scales[0, 5].tolist()[:3] == [126, 255, 1] and scales[0, 6, 0] == 255 and scales[0, 7, 2] == 255
    q, s, qt, st = M.quant_row_col_t(x.to(dev))
    same((q, s), (codes, scales))
    same(M.quant_row(x.to(dev)), (codes, scales))
    same((qt, st), oracle.quant_row(x.t()))
    assert bits_equal(M.dequant(q, s, 96).nan_to_num(7.0), oracle.values(codes, scales, 96).nan_to_num(7.0).bfloat16())
    # a product hands NaN on, and only to the rows that have it
    w = torch.ones(5, 96, dtype=torch.bfloat16, device=dev)
    y = M.gemm_nt(q[2:], s[:, 2:], *M.quant_row(w)).cpu()
    assert y.isnan().all(1).tolist() == [False, False, False, True, True, True, False] and not y[[0, 1, 2, 6]].isnan().any()


def products(M, dev, a, b, out_dtype, **shape):
    """gemm_nt of values in 4 bits against the oracle."""
    qa, qb = oracle.quant_row(a.flatten(0, -2)), oracle.quant_row(b.flatten(0, -2))
    K = a.shape[-1]
    va, vb = (oracle.values(*q, K).view(t.shape) for q, t in ((qa, a), (qb, b)))
    want, mag = oracle.gemm_nt(va, vb)
    put = lambda q, t: (q[0].view(*t.shape[:-1], -1).to(dev), q[1].to(dev))  # noqa: E731
    got = M.gemm_nt(*put(qa, a), *put(qb, b), out_dtype=out_dtype)
    assert got.dtype == out_dtype and got.shape == want.shape
    close(got, want, mag, K)
    return got


def close(got, want, mag, K, what=""):
    half = 2.0 ** -8 if got.dtype == torch.bfloat16 else 2.0 ** -24
    bound = (half * want.abs() + (K + 1) * 2.0 ** -23 * mag) * (1 + 2.0 ** -8)
    away = (got.double().cpu() - want).abs()
    assert bool((away <= bound).all()), (what, float((away / bound.clamp_min(1e-300)).max()), int((away > bound).sum()))


PRODUCTS = [(1, 1, 1), (1, 7, 40), (2, 16, 256), (3, 33, 300), (8, 100, 2048), (15, 31, 512), (16, 48, 640), (17, 65, 1000), (31, 96, 777), (32, 64, 4096), (33, 40, 512),
            (48, 130, 1300), (64, 64, 257), (65, 200, 1024), (100, 129, 100), (127, 128, 256), (128, 128, 2560), (129, 255, 512), (200, 333, 900), (256, 512, 768), (257, 1001, 1000),
            (513, 260, 300), (5, 3, 16384), (130, 20, 8000), (1000, 70, 32)]


@pytest.mark.parametrize("m,n,k", PRODUCTS)
@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
def test_products(M, dev, m, n, k, out_dtype):
    gen = make_gen(m * 7 + n * 3 + k)
    products(M, dev, tensor(gen, m, k), tensor(gen, n, k, spread=False), out_dtype)


@pytest.mark.parametrize("batch,m,n,k", [(2, 3, 5, 300), (5, 40, 33, 256), (3, 150, 70, 520), (9, 1, 17, 1000), (3, 40, 30, 9000)])
@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
def test_batches(M, dev, batch, m, n, k, out_dtype):
    gen = make_gen(batch)
    a = tensor(gen, batch * m, k).view(batch, m, k)
    products(M, dev, a, tensor(gen, batch * n, k, spread=False).view(batch, n, k), out_dtype)
    products(M, dev, a, tensor(gen, n, k, spread=False), out_dtype)


def test_large_product(M, dev):
    """Enough tiles for the largest ones, ragged at both ends; values at sampled places."""
    m, n, k = 2048 + 77, 4096 + 33, 1024 + 40
    gen = torch.Generator(device=dev).manual_seed(1)
    a, b = (torch.randn(r, k, generator=gen, device=dev).bfloat16() for r in (m, n))
    qa, qb = M.quant_row(a), M.quant_row(b)
    rows, cols = torch.randint(0, m, (64,), generator=make_gen(2)), torch.randint(0, n, (200,), generator=make_gen(3))
    rows[:4], cols[:4] = torch.tensor([0, m - 1, 255, 256]), torch.tensor([0, n - 1, 255, 256])
    va, vb = oracle.rounded(a[rows.to(dev)].cpu()), oracle.rounded(b[cols.to(dev)].cpu())
    want, mag = oracle.gemm_nt(va, vb)
    for out_dtype in (torch.bfloat16, torch.float32):
        got = M.gemm_nt(*qa, *qb, out_dtype=out_dtype)
        close(got[rows.to(dev)][:, cols.to(dev)], want, mag, k)
        assert torch.equal(got, M.gemm_nt(*qa, *qb, out_dtype=out_dtype))


@pytest.mark.parametrize("m", [1, 4, 20, 40, 130, 300])
def test_products_of_slices(M, dev, m):
    """Rows of larger tensors, in place; what lies around the result is left as it was."""
    gen = make_gen(m)
    a, b = tensor(gen, m + 9, 700), tensor(gen, 90, 700, spread=False)
    (qa, sa), (qb, sb) = M.quant_row(a.to(dev)), M.quant_row(b.to(dev))
    got = M.gemm_nt(qa[5:5 + m], sa[:, 5:5 + m], qb[3:76], sb[:, 3:76])
    want, mag = oracle.gemm_nt(oracle.rounded(a[5:5 + m]), oracle.rounded(b[3:76]))
    close(got, want, mag, 700)


def test_scales_far_apart(M, dev):
    """Scales whose powers of two are each out of a single number's range together with the other's, but not their product."""
    gen = make_gen(8)
    a, b = torch.randn(40, 512, generator=gen), torch.randn(70, 512, generator=gen)
    for up in (-100.0, 100.0):
        products(M, dev, (a * 2.0 ** up).bfloat16(), (b * 2.0 ** -up).bfloat16(), torch.float32)


@pytest.mark.parametrize("tokens,k,n", [(1, 8, 24), (5, 100, 36), (64, 256, 128), (100, 96, 200), (129, 512, 320), (300, 40, 1000)])
def test_layer_forward_and_backward(M, dev, tokens, k, n):
    gen = make_gen(tokens + k)
    x, w, dy = tensor(gen, tokens, k), randn_bf16(gen, n, k, std=0.02), randn_bf16(gen, tokens, n, std=1e-3)
    want = [oracle.gemm_nt(oracle.rounded(a), oracle.rounded(b)) for a, b in ((x, w), (dy, w.t()), (dy.t(), x.t()))]
    got = M.linear_fwd_bwd(x.to(dev), w.to(dev), dy.to(dev))
    for g, (v, mag), depth, name in zip(got, want, (k, n, tokens), ("Y", "dX", "dW")):
        close(g, v, mag, depth, name)
    layer = M.Mx4Linear(k, n, device=dev)
    with torch.no_grad():
        layer.weight.copy_(w)
    xd = x.to(dev).requires_grad_()
    y = layer(xd)
    y.backward(dy.to(dev))
    for g, (v, mag), depth, name in zip((y, xd.grad, layer.weight.grad), want, (k, n, tokens), ("Y", "dX", "dW")):
        close(g.detach(), v, mag, depth, name)
    with torch.no_grad():
        assert bits_equal(layer(xd), y.detach())
        assert bits_equal(layer.pack()(xd), y.detach()) and layer.weight is None and [n for n, _ in layer.named_buffers()] == ["codes", "scales"]


TOGETHER = [[(3, 64, 512), (3, 200, 512), (3, 16, 512)], [(30, 5000, 300), (30, 4000, 300)], [(100, 333, 1000), (257, 100, 40), (40, 1000, 5000)], [(1, 7, 256), (300, 300, 300), (20, 20, 20)],
            [(5, 5, 16384), (8, 8, 10)], [(1000, 513, 700)], [(2050, 1030, 520), (1030, 520, 2050), (2050, 520, 1030)]]


@pytest.mark.parametrize("sizes", TOGETHER, ids=str)
def test_products_together(M, dev, sizes):
    gen = make_gen(len(sizes))
    inputs = [(tensor(gen, m, k), tensor(gen, n, k, spread=False)) for m, n, k in sizes]
    got = M.gemm_nt_multi([(*M.quant_row(a.to(dev)), *M.quant_row(b.to(dev))) for a, b in inputs])
    assert len(got) == len(sizes)
    for c, (a, b), (m, n, k) in zip(got, inputs, sizes):
        assert c.dtype == torch.bfloat16 and c.shape == (m, n)
        close(c, *oracle.gemm_nt(oracle.rounded(a), oracle.rounded(b)), k, (m, n, k))


@pytest.mark.parametrize("sizes", [[(3, 64, 512), (3, 200, 512)], [(100, 333, 1000), (257, 100, 40), (40, 1000, 5000)], [(5, 40, 16384), (300, 100, 600)]], ids=str)
def test_products_together_into_wider_rows(M, dev, sizes):
    """From C: results in either type, rows apart; what lies between them is left as it was."""
    gen = make_gen(3)
    lib, problems, kept, outs = M._lib, (M._lib.Mx4GemmProblem * len(sizes))(), [], []
    for i, (m, n, k) in enumerate(sizes):
        a, b = tensor(gen, m, k), tensor(gen, n, k, spread=False)
        da, db = M._operand(*M.quant_row(a.to(dev)), "a"), M._operand(*M.quant_row(b.to(dev)), "b")
        c = torch.full((m, n + 5), 7.0, dtype=torch.bfloat16 if i % 2 else torch.float32, device=dev)
        problems[i] = lib.Mx4GemmProblem(da[2], db[2], c.data_ptr(), n + 5, m, n, k, 1 - i % 2)
        kept.append((da, db))
        outs.append((c, a, b, n, k))
    need = lib.lib().ti8_mx4_gemm_nt_multi_workspace(problems, len(sizes))
    workspace = torch.empty(max(need, 16), dtype=torch.uint8, device=dev)
    lib.call("ti8_mx4_gemm_nt_multi", problems, len(sizes), workspace.data_ptr(), need, torch.cuda.current_stream().cuda_stream)
    for c, a, b, n, k in outs:
        assert bool((c[:, n:] == 7.0).all())
        close(c[:, :n], *oracle.gemm_nt(oracle.rounded(a), oracle.rounded(b)), k, n)
