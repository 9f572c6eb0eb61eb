"""Inputs with a forward-mode tangent are refused by calls in 4 bits where they are made from C++, too."""
import pytest
import torch
from torch.autograd import forward_ad

pytestmark = pytest.mark.gpu


@pytest.fixture(params=[True, False], ids=["from C++", "from Python"])
def T(request, monkeypatch):
    import triton_int8_amd
    if not request.param:
        monkeypatch.setattr(triton_int8_amd._lib, "native", lambda: None)
    return triton_int8_amd


def calls_with(T, x, w, dy):
    q, s = torch.ones(4, 256, dtype=torch.int8, device=x.device), x[:, 0].float()
    return {"x": [lambda: T.mx4.quant_row(x), lambda: T.mx4.quant_row(x.view(2, 2, 256)), lambda: T.mx4.quant_col_t(x), lambda: T.mx4.quant_row_col_t(x), lambda: T.mx4.quant_row(x.t()),
                  lambda: T.mx4.linear_fwd_bwd(x, w, dy), lambda: T.ops.rmsnorm_quant(x, w[0], 1e-5), lambda: T.ops.dequant_row(q, s)],
            "w": [lambda: T.mx4.linear_fwd_bwd(x, w, dy), lambda: T.ops.rmsnorm_quant(x, w[0], 1e-5, residual=x, to="int8")], "dy": [lambda: T.mx4.linear_fwd_bwd(x, w, dy)]}


@pytest.mark.parametrize("which", ["x", "w", "dy"])
def test_tangents_are_refused(T, dev, which):
    plain = {k: torch.ones(s, dtype=torch.bfloat16, device=dev) for k, s in dict(x=(4, 256), w=(8, 256), dy=(4, 8)).items()}
    with forward_ad.dual_level():
        for call in calls_with(T, **{**plain, which: forward_ad.make_dual(plain[which], plain[which].clone())})[which]:
            with pytest.raises(ValueError, match="tangent"):
                call()
        for call in calls_with(T, **plain)[which]:       # (none of them has one here)
            call()
    torch.cuda.synchronize()


@pytest.mark.parametrize("bias", [False, True])
def test_a_backward_refuses_gradients_with_a_tangent(T, dev, bias):
    layer, x = T.Mx4Linear(256, 8, bias=bias, device=dev), torch.ones(4, 256, dtype=torch.bfloat16, device=dev, requires_grad=True)
    with forward_ad.dual_level():
        y = layer(x)
        with pytest.raises(ValueError, match="tangent"):
            torch.autograd.grad(y, x, forward_ad.make_dual(torch.ones_like(y), torch.ones_like(y)), retain_graph=True)
        torch.autograd.grad(y, x, torch.ones_like(y))
