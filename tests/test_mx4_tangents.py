"""Inputs with a forward-mode tangent: no call in 4 bits carries one on, so all refuse them, also where a backward meets one."""
import pytest
import torch
from torch.autograd import forward_ad

from test_mx4_host import bf, recorded  # noqa: F401 (a fixture)


def calls_with(T, x, w, dy):
    """name -> calls on tensors of which some may have a tangent: x [4, 256], w [8, 256], dy [4, 8]."""
    q, s = torch.zeros(4, 256, dtype=torch.int8), x[:, 0].float()
    return {"quant_row": lambda: T.mx4.quant_row(x), "quant_row of a weight": lambda: T.mx4.quant_row(w), "quant_col_t": lambda: T.mx4.quant_col_t(x), "quant_row_col_t": lambda: T.mx4.quant_row_col_t(x),
            "quant_row, transposed": lambda: T.mx4.quant_row(x.t()), "quant_row, three dims": lambda: T.mx4.quant_row(x.view(2, 2, 256)), "step": lambda: T.mx4.linear_fwd_bwd(x, w, dy),
            "norm": lambda: T.ops.rmsnorm_quant(x, w[0], 1e-5, residual=x), "dequant_row": lambda: T.ops.dequant_row(q, s)}


MEETS = {"quant_row": "x", "quant_row of a weight": "w", "quant_col_t": "x", "quant_row_col_t": "x", "quant_row, transposed": "x", "quant_row, three dims": "x", "step": "x w dy", "norm": "x w", "dequant_row": "x"}


@pytest.mark.parametrize("name,which", [(n, w) for n, ws in MEETS.items() for w in ws.split()])
def test_tangents_are_refused(recorded, name, which):  # noqa: F811
    T, calls = recorded
    plain = dict(x=bf(4, 256), w=bf(8, 256), dy=bf(4, 8))
    with forward_ad.dual_level():
        with pytest.raises(ValueError, match="tangent"):
            calls_with(T, **{**plain, which: forward_ad.make_dual(plain[which], plain[which].clone())})[name]()
        assert not calls
        calls_with(T, **plain)[name]()      # (none of them has one here)
        assert calls


@pytest.mark.parametrize("bias,wanted", [(False, "x"), (False, "weight"), (True, "x"), (True, "bias"), (True, "weight")])
def test_a_backward_refuses_gradients_with_a_tangent(recorded, bias, wanted):  # noqa: F811
    """Forward over reverse: a gradient of the output that has a tangent has gradients with one, which the backward's products do not give."""
    T, calls = recorded
    layer, x = T.Mx4Linear(256, 8, bias=bias), bf(4, 256).requires_grad_()
    with forward_ad.dual_level():
        y = layer(x)
        calls.clear()
        d = forward_ad.make_dual(torch.ones_like(y), torch.ones_like(y))
        with pytest.raises(ValueError, match="tangent"):
            torch.autograd.grad(y, x if wanted == "x" else getattr(layer, wanted), d, retain_graph=True)
        assert not calls
        torch.autograd.grad(y, x if wanted == "x" else getattr(layer, wanted), torch.ones_like(y))
        assert calls


def test_a_tangent_of_the_bias(recorded):  # noqa: F811
    T, calls = recorded
    layer = T.Mx4Linear(256, 8, bias=True).requires_grad_(False)
    with forward_ad.dual_level():
        b = forward_ad.make_dual(layer.bias.detach(), torch.ones(8, dtype=torch.bfloat16))
        del layer.bias
        layer.bias = b
        with pytest.raises(ValueError, match="tangent"):
            layer(bf(4, 256))
    assert not calls
