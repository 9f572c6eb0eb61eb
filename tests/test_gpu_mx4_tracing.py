"""What records operators is refused by calls on tensors in 4 bits where they are made from C++, too; what only watches changes nothing."""
import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx

from conftest import bits_equal, make_gen, randn_bf16

pytestmark = pytest.mark.gpu


@pytest.fixture(params=[True, False], ids=["from C++", "from Python"])
def T(request, monkeypatch):
    import triton_int8_amd
    if not request.param:
        monkeypatch.setattr(triton_int8_amd._lib, "native", lambda: None)
    else:
        assert triton_int8_amd._lib.native() is not None
    return triton_int8_amd


def entry_points(T, dev):
    """Functions of x bf16 [4, 256]."""
    w = torch.ones(256, dtype=torch.bfloat16, device=dev)
    q, s = T.mx4.quant_row(torch.ones(4, 256, dtype=torch.bfloat16, device=dev))
    q8 = torch.ones(4, 256, dtype=torch.int8, device=dev), torch.ones(4, device=dev)
    layer = T.Mx4Linear(256, 8, bias=True, device=dev).requires_grad_(False)
    return [layer, lambda t: T.mx4.linears(t, (layer, layer)), T.mx4.quant_row, T.mx4.quant_col_t, T.mx4.quant_row_col_t, lambda t: T.mx4.linear_fwd_bwd(t, t, t[:, :4]),
            lambda t: T.mx4.gemm_nt(q, s, q, s) + t[:, :4], lambda t: T.mx4.gemm_nt_multi([(q, s, q, s)])[0] + t[:, :4], lambda t: T.mx4.dequant(q, s, 256) + t,
            lambda t: T.ops.rmsnorm_quant(t, w, 1e-5), lambda t: T.ops.rmsnorm_quant(t, w, 1e-5, residual=t, to="int8"), lambda t: T.ops.dequant_row(*q8) + t]


@pytest.mark.parametrize("how", [{}, dict(pre_dispatch=True), dict(tracing_mode="fake"), dict(tracing_mode="symbolic")], ids=str)
def test_make_fx_is_refused(T, dev, how):
    x = torch.ones(4, 256, dtype=torch.bfloat16, device=dev)
    for i, f in enumerate(entry_points(T, dev)):
        with pytest.raises(ValueError, match="traced"):
            make_fx(f, **how)(x)
            print("entry point", i)


def test_functionalize_is_refused(T, dev):
    x = torch.ones(4, 256, dtype=torch.bfloat16, device=dev)
    for i, f in enumerate(entry_points(T, dev)):
        with pytest.raises(ValueError, match="traced"):
            torch.func.functionalize(f)(x)
            print("entry point", i)


def test_modes_that_watch_change_nothing(T, dev):
    from torch.utils.flop_counter import FlopCounterMode
    x = randn_bf16(make_gen(1), 4, 256).to(dev)
    for f in entry_points(T, dev):
        want = f(x)
        with FlopCounterMode(display=False):
            got = f(x)
        for a, b in zip(*((t,) if isinstance(t, torch.Tensor) else t for t in (got, want))):
            assert bits_equal(a, b)
