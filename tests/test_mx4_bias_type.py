"""A bias of another type than the layer's: outputs have the sum's type, and the bias's gradient is a sum of numbers of that type."""
import pytest
import torch

from conftest import make_gen
from test_mx4_host import bf, recorded  # noqa: F401 (a fixture)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64])
def test_a_wide_bias(recorded, dtype):  # noqa: F811
    T, calls = recorded
    layer = T.Mx4Linear(40, 24)
    layer.bias = torch.nn.Parameter(torch.zeros(24, dtype=dtype))
    y, dy = layer(bf(5, 40)), torch.randn(5, 24, generator=make_gen(1)).to(dtype)
    assert y.dtype == dtype
    calls.clear()
    y.backward(dy)
    assert layer.bias.grad.dtype == dtype and [n for n, _ in calls] == ["ti8_mx4_quant", "ti8_mx4_gemm_nt_multi"]
    # (five numbers: four additions, each off by half a step of the sum of magnitudes at most; in float64 on both sides)
    additions = 4 if dtype == torch.float32 else 8
    assert bool(((layer.bias.grad.double() - dy.double().sum(0)).abs() <= additions * torch.finfo(dtype).eps / 2 * dy.double().abs().sum(0)).all())


def test_a_bias_of_the_layers_type(recorded):  # noqa: F811
    T, calls = recorded
    layer = T.Mx4Linear(40, 24, bias=True)
    y = layer(bf(5, 40))
    calls.clear()
    y.backward(torch.ones_like(y))
    assert [n for n, _ in calls] == ["ti8_column_sum", "ti8_mx4_quant", "ti8_mx4_gemm_nt_multi"]


@pytest.mark.gpu
@pytest.mark.parametrize("n", [24, 96])
def test_gradients_of_a_wide_bias(dev, n):
    import triton_int8_amd as T
    gen = make_gen(2)
    layer, x, dy = T.Mx4Linear(256, n, device=dev), torch.randn(33, 256, generator=gen).bfloat16().to(dev), torch.randn(33, n, generator=gen).to(dev)
    plain = layer(x)
    layer.bias = torch.nn.Parameter(torch.randn(n, generator=gen).to(dev))
    y = layer(x)
    assert torch.equal(y.detach(), plain.detach() + layer.bias.detach())
    y.backward(dy)
    away = (layer.bias.grad.double() - dy.double().sum(0)).abs()
    assert bool((away <= 32 * 2.0 ** -24 * dy.double().abs().sum(0)).all())      # (32 additions, half a step each)
