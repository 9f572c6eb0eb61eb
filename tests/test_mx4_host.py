"""Tensors in 4 bits and the quantised norm without a GPU: what the entry points and the Python functions refuse, and the shapes that the wrappers make."""
import ctypes

import pytest
import torch

FAKE = 0x10000      # a 16-byte aligned "device pointer"; validation never dereferences it


@pytest.fixture(scope="module")
def lib():
    import triton_int8_amd
    return triton_int8_amd._lib


def mx(lib, rows=64, cols=512, **other):
    tiles = -(-cols // 256)
    return lib.Mx4(**{**dict(codes=FAKE, scales=FAKE, ld=tiles * 128, scale_ld=rows * 8), **other})


def refused(lib, name, code, msg, *args):
    assert getattr(lib.lib(), name)(*args) == code
    text = lib.lib().ti8_last_error().decode()
    assert msg in text and (name in text or text.startswith("unknown")), text       # (what all quantisers have in common)


def operand(lib, **other):
    fields = dict(x=FAKE, ldx=512, rows=64, cols=512)
    return lib.Mx4Operand(**{**fields, **other})


TENSORS = [(dict(codes=None), 1, "required"), (dict(scales=None), 1, "required"), (dict(ld=128), 2, "ld"), (dict(scale_ld=504), 2, "scale_ld"), (dict(codes=FAKE + 8), 3, "aligned"),
           (dict(scales=FAKE + 4), 3, "8-byte"), (dict(ld=264), 3, "ld"), (dict(scale_ld=516), 3, "scale_ld")]


@pytest.mark.parametrize("other,code,msg", TENSORS, ids=str)
def test_tensors_that_are_refused(lib, other, code, msg):
    bad, good = mx(lib, **other), mx(lib)
    if other != dict(codes=None):
        refused(lib, "ti8_mx4_quant", code, msg, operand(lib, by_rows=bad), 1, None)
        refused(lib, "ti8_mx4_quant", code, msg, operand(lib, ldx=64, rows=512, cols=64, by_columns=bad), 1, None)
    refused(lib, "ti8_mx4_dequant", code, msg, bad, 64, 512, FAKE, 512, None)
    for a, b in ((bad, good), (good, bad)):
        refused(lib, "ti8_mx4_gemm_nt", code, msg, a, 0, b, 0, FAKE, 64, 0, 1, 64, 64, 512, 0, None, 0, None)
    if other != dict(codes=None):
        refused(lib, "ti8_rmsnorm_quant", code, msg, norm(lib, dim=512, ldx=512, ldr=512, ldh=512, mx4=bad), None)


@pytest.mark.parametrize("args,code,msg", [
    ((None, 512, 64, 512, 1, 1), 1, "required"), ((FAKE, 512, 64, 512, 0, 0), 1, "required"), ((FAKE, 512, 0, 512, 1, 1), 2, "rows"), ((FAKE, 512, 64, 0, 1, 1), 2, "cols"),
    ((FAKE, 511, 64, 512, 1, 1), 2, "ldx"), ((FAKE, 512, (1 << 28) + 1, 512, 1, 1), 2, "2^28"), ((FAKE + 1, 512, 64, 512, 1, 0), 3, "aligned")])
def test_quant(lib, args, code, msg):
    x, ldx, rows, cols, by_rows, by_columns = args
    o = operand(lib, x=x, ldx=ldx, rows=rows, cols=cols, by_rows=mx(lib) if by_rows else lib.Mx4(), by_columns=mx(lib, 512, 64) if by_columns else lib.Mx4())
    refused(lib, "ti8_mx4_quant", code, msg, o, 1, None)


def test_quant_of_several(lib):
    both = operand(lib, by_rows=mx(lib), by_columns=mx(lib, 512, 64))
    for count in (0, 4, -1):
        refused(lib, "ti8_mx4_quant", 2, "operands", (lib.Mx4Operand * 4)(*[both] * 4), count, None)
    refused(lib, "ti8_mx4_quant", 1, "by rows and by columns", (lib.Mx4Operand * 2)(both, operand(lib, by_rows=mx(lib))), 2, None)
    refused(lib, "ti8_mx4_quant", 2, "ldx", (lib.Mx4Operand * 2)(both, operand(lib, ldx=5, by_rows=mx(lib), by_columns=mx(lib, 512, 64))), 2, None)


@pytest.mark.parametrize("change,code,msg", [
    (dict(X=None), 1, "required"), (dict(dW=None), 1, "required"), (dict(workspace=None), 1, "required"), (dict(T=0), 2, "T"), (dict(K=(1 << 22) + 1), 2, "2^22"), (dict(N=-3), 2, "N"),
    (dict(bytes=4096), 1, "workspace of"), (dict(workspace=FAKE + 16), 3, "256-byte"), (dict(dX=FAKE + 1), 3, "2-byte"), (dict(W=FAKE + 1), 3, "ti8_mx4_quant"),
    (dict(lddy=99), 2, "ti8_mx4_quant")], ids=str)
def test_step(lib, change, code, msg):
    v = {**dict(X=FAKE, W=FAKE, dY=FAKE, Y=FAKE, dX=FAKE, dW=FAKE, T=50, K=200, N=100, lddy=100, workspace=FAKE, bytes=1 << 30), **change}
    got = lib.lib().ti8_mx4_linear_fwd_bwd(v["X"], 200, v["W"], 200, v["dY"], v["lddy"], v["Y"], v["dX"], v["dW"], v["T"], v["K"], v["N"], v["workspace"], v["bytes"], None)
    assert got == code and msg in lib.lib().ti8_last_error().decode()


def problem(lib, **other):
    fields = dict(a=mx(lib), b=mx(lib), c=FAKE, ldc=64, M=64, N=64, K=512, wide=0)
    return lib.Mx4GemmProblem(**{**fields, **other})


@pytest.mark.parametrize("other,code,msg", [
    (dict(c=None), 1, "required"), (dict(M=0), 2, "M"), (dict(K=(1 << 22) + 1), 2, "2^22"), (dict(ldc=63), 2, "ldc"), (dict(c=FAKE + 1), 3, "aligned"), (dict(N=65, ldc=65), 2, "scale_ld"),
    (dict(K=513), 2, "ld")], ids=str)
def test_several_products(lib, other, code, msg):
    for at in range(3):
        problems = (lib.Mx4GemmProblem * 3)(*(problem(lib, **(other if i == at else {})) for i in range(3)))
        refused(lib, "ti8_mx4_gemm_nt_multi", code, msg, problems, 3, None, 0, None)
    for count in (0, 4, -1):
        refused(lib, "ti8_mx4_gemm_nt_multi", 2, "products", (lib.Mx4GemmProblem * 4)(*[problem(lib)] * 4), count, None, 0, None)
        assert lib.lib().ti8_mx4_gemm_nt_multi_workspace((lib.Mx4GemmProblem * 4)(*[problem(lib)] * 4), count) == -1
    refused(lib, "ti8_mx4_gemm_nt_multi", 1, "required", None, 1, None, 0, None)
    long = lib.Mx4GemmProblem(mx(lib, 100, 16384), mx(lib, 100, 16384), FAKE, 100, 100, 100, 16384, 0)
    need = lib.lib().ti8_mx4_gemm_nt_multi_workspace(long, 1)
    assert need == lib.lib().ti8_mx4_gemm_nt_workspace(1, 100, 100, 16384) > 0
    refused(lib, "ti8_mx4_gemm_nt_multi", 1, "workspace of", long, 1, FAKE, need - 1, None)
    refused(lib, "ti8_mx4_gemm_nt_multi", 3, "16-byte", long, 1, FAKE + 8, need, None)


def test_workspaces(lib):
    """Long contractions over few tiles are shared out; sizes that are not taken have no workspace."""
    l = lib.lib()
    assert l.ti8_mx4_gemm_nt_workspace(1, 8192, 8192, 4096) == 0 and l.ti8_mx4_gemm_nt_workspace(1, 1, 1, 1) == 0
    assert l.ti8_mx4_gemm_nt_workspace(1, 100, 100, 16384) in (2 * 40000, 4 * 40000, 8 * 40000)
    assert l.ti8_mx4_gemm_nt_workspace(0, 1, 1, 1) == l.ti8_mx4_gemm_nt_workspace(1, 1, 1, 1 << 23) == -1
    assert l.ti8_mx4_linear_fwd_bwd_workspace(0, 1, 1) == l.ti8_mx4_linear_fwd_bwd_workspace(1, 1 << 23, 1) == -1
    T, K, N = 300, 520, 1000
    held = sum(r * -(-c // 256) * 136 for r, c in ((T, K), (K, T), (N, K), (K, N), (T, N), (N, T)))
    assert held <= l.ti8_mx4_linear_fwd_bwd_workspace(T, K, N) <= held + 13 * 256 + l.ti8_mx4_gemm_nt_workspace(1, N, K, T) + l.ti8_mx4_gemm_nt_workspace(1, T, N, K) + l.ti8_mx4_gemm_nt_workspace(1, T, K, N)


@pytest.mark.parametrize("change,code,msg", [
    (dict(c=None), 1, "required"), (dict(M=0), 2, "M"), (dict(N=0), 2, "N"), (dict(K=0), 2, "K"), (dict(K=(1 << 22) + 1), 2, "2^22"), (dict(batch=0), 2, "batch"),
    (dict(batch=65536), 2, "batch"), (dict(ldc=63), 2, "ldc"), (dict(rows_a=63, batch=2), 2, "rows_a"), (dict(rows_b=1, batch=2), 2, "rows_b"),
    (dict(rows_a=64, batch=2), 2, "scale_ld"), (dict(c=FAKE + 1), 3, "aligned"), (dict(c=FAKE + 2, wide=1), 3, "aligned")], ids=str)
def test_gemm(lib, change, code, msg):
    v = {**dict(rows_a=0, rows_b=0, c=FAKE, ldc=64, bsc=0, batch=1, M=64, N=64, K=512, wide=0), **change}
    refused(lib, "ti8_mx4_gemm_nt", code, msg, mx(lib), v["rows_a"], mx(lib), v["rows_b"], v["c"], v["ldc"], v["bsc"], v["batch"], v["M"], v["N"], v["K"], v["wide"], None, 0, None)


def norm(lib, **other):
    fields = dict(x=FAKE, ldx=256, residual=FAKE, ldr=256, w=FAKE, h=FAKE, ldh=256, rstd=FAKE, rows=64, dim=256, eps=1e-5, mx4=mx(lib, 64, 256))
    return lib.RmsnormQuantArgs(**{**fields, **other})


INT8 = dict(q=FAKE, ldq=256, s=FAKE)


@pytest.mark.parametrize("other,code,msg", [
    (dict(x=None), 1, "required"), (dict(w=None), 1, "required"), (dict(rstd=None), 1, "required"), (dict(h=None), 1, "go together"), (dict(residual=None), 1, "go together"),
    (dict(q=FAKE), 1, "one of"), (dict(mx4=None), 1, "one of"), (dict(rows=0), 2, "rows"), (dict(dim=12), 2, "dim"), (dict(dim=16392), 2, "dim"), (dict(ldx=248), 2, "leading"),
    (dict(ldr=248), 2, "leading"), (dict(ldh=248), 2, "leading"), (dict(x=FAKE + 8), 3, "aligned"), (dict(w=FAKE + 2), 3, "aligned"), (dict(residual=FAKE + 2), 3, "aligned"),
    (dict(h=FAKE + 2), 3, "aligned"), (dict(ldx=260), 3, "aligned"), (dict(rstd=FAKE + 2), 3, "aligned"),
    (dict(mx4=None, **{**INT8, "s": None}), 1, "needs s"), (dict(mx4=None, group=64, **INT8), 4, "group"), (dict(mx4=None, qflags=8, **INT8), 4, "flags"),
    (dict(mx4=None, qflags=64, **INT8), 4, "flags"), (dict(mx4=None, inv_mode=4, **INT8), 4, "inv_mode"), (dict(mx4=None, dim=200, **INT8), 2, "dim%128"),
    (dict(mx4=None, **{**INT8, "ldq": 248}), 2, "ldq"), (dict(mx4=None, **{**INT8, "q": FAKE + 4}), 3, "aligned"), (dict(mx4=None, **{**INT8, "ldq": 260}), 3, "aligned")], ids=str)
def test_rmsnorm_quant(lib, other, code, msg):
    if other.get("mx4", 0) is None:
        other = {**other, "mx4": lib.Mx4()}
    refused(lib, "ti8_rmsnorm_quant", code, msg, norm(lib, **other), None)


@pytest.mark.parametrize("args,code,msg", [
    ((None, 256, FAKE, 4, 256, 0, FAKE, 256), 1, "required"), ((FAKE, 256, None, 4, 256, 0, FAKE, 256), 1, "required"), ((FAKE, 256, FAKE, 0, 256, 0, FAKE, 256), 2, "rows"),
    ((FAKE, 256, FAKE, 4, 252, 0, FAKE, 256), 2, "cols%8"), ((FAKE, 256, FAKE, 4, 200, 128, FAKE, 256), 2, "cols%128"), ((FAKE, 255, FAKE, 4, 256, 0, FAKE, 256), 2, "leading"),
    ((FAKE, 256, FAKE, 4, 256, 64, FAKE, 256), 4, "group"), ((FAKE + 4, 256, FAKE, 4, 256, 0, FAKE, 256), 3, "aligned"), ((FAKE, 256, FAKE, 4, 256, 0, FAKE + 8, 256), 3, "aligned")])
def test_dequant_row(lib, args, code, msg):
    refused(lib, "ti8_dequant_row", code, msg, *args, None)


def test_missing_arguments_are_refused(lib):
    refused(lib, "ti8_rmsnorm_quant", 1, "required", None, None)
    refused(lib, "ti8_mx4_dequant", 1, "required", None, 64, 512, FAKE, 512, None)
    refused(lib, "ti8_mx4_gemm_nt", 1, "required", None, 0, mx(lib), 0, FAKE, 64, 0, 1, 64, 64, 512, 0, None, 0, None)
    refused(lib, "ti8_mx4_dequant", 2, "ldy", mx(lib), 64, 512, FAKE, 511, None)
    refused(lib, "ti8_mx4_dequant", 3, "aligned", mx(lib), 64, 512, FAKE + 1, 512, None)


@pytest.fixture
def recorded(monkeypatch):
    """The library's calls, recorded instead of made, on host tensors."""
    import triton_int8_amd as T
    calls = []
    monkeypatch.setattr(T.ops, "_on_gpu", lambda t: True)
    monkeypatch.setattr(torch.Tensor, "get_device", lambda t: 0)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 0, raising=False)
    monkeypatch.setattr(T.mx4, "_stream", lambda: 0)
    monkeypatch.setattr(T.ops, "_stream", lambda: 0)
    monkeypatch.setattr(T._lib, "native", lambda: None)
    monkeypatch.setattr(T._lib, "call", lambda name, *a: calls.append((name, a)))
    return T, calls


def bf(*shape):
    return torch.zeros(*shape, dtype=torch.bfloat16)


def test_python_refusals(recorded):
    T, calls = recorded
    M = T.mx4
    for bad in (torch.zeros(4, 4), bf(0, 4), bf(()), None, "x"):
        with pytest.raises(ValueError, match="x must be"):
            M.quant_row(bad)
    for f in (M.quant_col_t, M.quant_row_col_t):
        with pytest.raises(ValueError, match="2 dimensions"):
            f(bf(2, 3, 4))
    q, s = M.quant_row(bf(5, 300))
    assert q.shape == (5, 256) and s.shape == (2, 5, 8)
    for codes, scales, msg in ((q.int(), s, "codes of A"), (q[:, :100], s, "codes of A"), (q, s[:1], "scales of A"), (q, s.int(), "scales of A"), (q[:4], s, "scales of A"), (q[0], s, "codes of A")):
        with pytest.raises(ValueError, match=msg):
            M.gemm_nt(codes, scales, q, s)
    q1, s1 = M.quant_row(bf(5, 256))
    with pytest.raises(ValueError, match="tiles along"):
        M.gemm_nt(q, s, q1, s1)
    q3, s3 = M.quant_row(bf(2, 5, 300))
    with pytest.raises(ValueError, match="batches"):
        M.gemm_nt(q, s, q3, s3)
    with pytest.raises(ValueError, match="out_dtype"):
        M.gemm_nt(q, s, q, s, out_dtype=torch.float16)
    for cols in (256, 513, 0, -1, 2.0):
        with pytest.raises(ValueError, match="columns"):
            M.dequant(q, s, cols)
    with pytest.raises(ValueError, match="do not fit"):
        M.linear_fwd_bwd(bf(5, 300), bf(7, 301), bf(5, 7))
    with pytest.raises(ValueError, match="do not fit"):
        M.linear_fwd_bwd(bf(5, 300), bf(7, 300), bf(6, 7))
    with pytest.raises(ValueError, match="positive"):
        M.Mx4Linear(0, 4)
    for problems, msg in (([], "between 1 and 3"), ([(q, s, q, s)] * 4, "between 1 and 3"), ([(q, s, q, s), (q, s, q1, s1)], "as many tiles"), ([(q, s, q), (s, q, s, q, s)], "a product is"), ([(q3, s3, q, s)], "matrices")):
        with pytest.raises(ValueError, match=msg):
            M.gemm_nt_multi(problems)


def test_python_refusals_of_the_norm(recorded):
    T, calls = recorded
    f = T.ops.rmsnorm_quant
    x, w = bf(3, 256), bf(256)
    for args, kw, msg in (((x, w, 1e-5), dict(to="fp8"), "`to`"), ((x, w, 1e-5), dict(group=128), "group"), ((x, w, 1e-5), dict(to="int8", group=64), "group"),
                          ((x.float(), w, 1e-5), {}, "x must be bfloat16"), ((x, w.float(), 1e-5), {}, "weight must be"), ((bf(3, 100), bf(100), 1e-5), {}, "multiple of 8"),
                          ((bf(3, 200), bf(200), 1e-5), dict(to="int8"), "multiple of 128"), ((bf(1, 16392), bf(16392), 1e-5), {}, "up to 16384"), ((bf(0, 256), w, 1e-5), {}, "non-empty"),
                          ((x, bf(128), 1e-5), {}, "do not fit"), ((x, w, 1e-5), dict(residual=bf(4, 256)), "do not fit")):
        with pytest.raises(ValueError, match=msg):
            f(*args, **kw)
    for i in range(3):
        t = [x.clone(), w.clone(), x.clone()]
        t[i].requires_grad_()
        with pytest.raises(ValueError, match="gradient"):
            f(t[0], t[1], 1e-5, residual=t[2])
        with torch.no_grad():
            f(t[0], t[1], 1e-5, residual=t[2])
    q = torch.zeros(3, 256, dtype=torch.int8)
    for args, msg in (((q.float(), torch.zeros(3)), "int8"), ((q, bf(3)), "float32"), ((q, torch.zeros(4)), "do not fit"), ((q, torch.zeros(3, 3)), "do not fit"), ((q[:, :100], torch.zeros(3)), "multiple of 8")):
        with pytest.raises(ValueError, match=msg):
            T.ops.dequant_row(*args)


def test_other_devices_are_refused(recorded, monkeypatch):
    T, calls = recorded
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 1, raising=False)
    for call in (lambda: T.mx4.quant_row(bf(3, 256)), lambda: T.mx4.gemm_nt(*(torch.zeros(3, 128, dtype=torch.uint8), torch.zeros(1, 3, 8, dtype=torch.uint8)) * 2),
                 lambda: T.ops.rmsnorm_quant(bf(3, 256), bf(256), 1e-5), lambda: T.ops.dequant_row(torch.zeros(3, 8, dtype=torch.int8), torch.zeros(3)),
                 lambda: T.mx4.dequant(torch.zeros(3, 128, dtype=torch.uint8), torch.zeros(1, 3, 8, dtype=torch.uint8), 200)):
        with pytest.raises(ValueError, match="current GPU"):
            call()
    assert not calls


def test_one_weight_for_all_batches_is_one_product(recorded):
    T, calls = recorded
    a, b = T.mx4.quant_row(bf(3, 5, 300)), T.mx4.quant_row(bf(7, 300))
    calls.clear()
    assert T.mx4.gemm_nt(*a, *b).shape == (3, 5, 7)
    (name, args), = calls
    assert name == "ti8_mx4_gemm_nt" and args[1] == args[3] == 0 and args[7:11] == (1, 15, 7, 512)
    c = T.mx4.quant_row(bf(3, 7, 300))
    calls.clear()
    assert T.mx4.gemm_nt(*a, *c, out_dtype=torch.float32).dtype == torch.float32
    assert calls[0][1][1] == 5 and calls[0][1][3] == 7 and calls[0][1][7:12] == (3, 5, 7, 512, 1)


def test_layers(recorded):
    T, calls = recorded
    layer = T.Mx4Linear(40, 24, bias=True)
    with pytest.raises(ValueError, match="40 input features"):
        layer(bf(3, 41))
    with torch.no_grad():
        assert layer(bf(2, 3, 40)).shape == (2, 3, 24) and layer(bf(0, 40)).shape == (0, 24)
    x = bf(2, 3, 40).requires_grad_()
    y = layer(x)
    y.sum().backward()
    assert x.grad.shape == x.shape and layer.weight.grad.shape == (24, 40) and layer.bias.grad.shape == (24,)
    with pytest.raises(RuntimeError, match="once"):
        z = layer(x)
        g, = torch.autograd.grad(z.float().square().sum(), x, create_graph=True)
        g.sum().backward()
    empty = bf(0, 40).requires_grad_()
    layer.weight.grad = None
    layer(empty).sum().backward()
    assert empty.grad.shape == (0, 40) and layer.weight.grad.abs().sum() == 0
    layer.pack()
    assert layer.packed and layer.pack() is layer and "packed=True" in repr(layer)
    with pytest.raises(ValueError, match="forward only"):
        layer(x)
    with torch.no_grad():
        assert layer(x).shape == (2, 3, 24)
    assert set(layer.state_dict()) == {"bias", "codes", "scales"}


def test_gradients_that_are_not_wanted_are_not_computed(recorded):
    T, calls = recorded
    names = lambda: [n for n, _ in calls]  # noqa: E731
    w, x = torch.nn.Parameter(bf(24, 40)), bf(3, 40)
    y, = T.mx4.Mx4LinearFunction.apply(x, w)
    calls.clear()
    y.sum().backward()
    assert names() == ["ti8_mx4_quant", "ti8_mx4_gemm_nt_multi"] and calls[0][1][0].by_rows.codes is None
    w.requires_grad_(False)
    y, = T.mx4.Mx4LinearFunction.apply(x.requires_grad_(), w)
    calls.clear()
    y.sum().backward()
    assert names() == ["ti8_mx4_quant", "ti8_mx4_gemm_nt_multi"] and calls[0][1][0].by_columns.codes is None
    # one of several outputs that nobody uses
    a, b = torch.nn.Parameter(bf(24, 40)), torch.nn.Parameter(bf(8, 40))
    y, z = T.mx4.Mx4LinearFunction.apply(x, a, b)
    calls.clear()
    z.sum().backward()
    assert a.grad is None and b.grad.shape == (8, 40) and names() == ["ti8_mx4_quant", "ti8_mx4_gemm_nt_multi"]


def test_tracing_is_refused(recorded):
    """A trace would hold nothing of what a call launches."""
    T, calls = recorded
    x, w, layer = torch.ones(4, 256, dtype=torch.bfloat16), torch.ones(256, dtype=torch.bfloat16), T.Mx4Linear(256, 8).requires_grad_(False)
    q, s = torch.zeros(4, 128, dtype=torch.uint8), torch.zeros(1, 4, 8, dtype=torch.uint8)
    for call in (layer, T.mx4.quant_row, T.mx4.quant_row_col_t, lambda t: T.mx4.linear_fwd_bwd(t, t, t[:, :4]), lambda t: T.ops.rmsnorm_quant(t, w, 1e-5)[0],
                 lambda t: T.mx4.gemm_nt(q, s, q, s) + t[:, :4], lambda t: T.mx4.dequant(q, s, 256) + t, lambda t: T.mx4.gemm_nt_multi([(q, s, q, s)])[0] + t[:, :4],
                 lambda t: T.ops.dequant_row(t.to(torch.int8), torch.ones(4))):
        with pytest.raises(ValueError, match="traced"):
            torch.jit.trace(call, (x,), check_trace=False)
    assert not calls


def test_tangents_are_refused(recorded):
    T, calls = recorded
    from torch.autograd import forward_ad
    x, w = torch.ones(4, 256, dtype=torch.bfloat16), torch.ones(256, dtype=torch.bfloat16)
    layer = T.Mx4Linear(256, 8, bias=True).requires_grad_(False)
    with forward_ad.dual_level():
        d = forward_ad.make_dual(x, x)
        for call in (lambda: layer(d), lambda: T.mx4.linears(d, (layer, layer)), lambda: T.ops.rmsnorm_quant(d, w, 1e-5), lambda: T.ops.rmsnorm_quant(x, w, 1e-5, residual=d)):
            with pytest.raises(ValueError, match="tangent"):
                call()
        assert not calls
        layer(x)        # (no tangent of its own)
    assert [c[0] for c in calls] == ["ti8_mx4_quant", "ti8_mx4_quant", "ti8_mx4_gemm_nt_multi"]
