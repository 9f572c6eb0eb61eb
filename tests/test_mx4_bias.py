"""A layer in 4 bits of which the bias alone is trained: its gradient is added up as beside a weight's (launches that a graph may hold), also where the layer is packed."""
import pytest
import torch

from conftest import bits_equal, make_gen, randn_bf16
from test_mx4_host import bf, recorded  # noqa: F401 (a fixture)


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("shape", [(5, 40), (2, 3, 40), (40,)], ids=str)
def test_the_bias_alone(recorded, packed, shape):  # noqa: F811
    T, calls = recorded
    layer = T.Mx4Linear(40, 24, bias=True)
    layer.weight.requires_grad_(False)
    if packed:
        layer.pack()
    y = layer(bf(*shape))
    calls.clear()
    y.backward(torch.ones_like(y))
    assert layer.bias.grad.shape == (24,) and [n for n, _ in calls] == ["ti8_column_sum"]
    with torch.no_grad():
        assert not layer(bf(*shape)).requires_grad


@pytest.mark.parametrize("packed", [False, True])
def test_the_bias_alone_without_tokens(recorded, packed):  # noqa: F811
    T, calls = recorded
    layer = T.Mx4Linear(40, 24, bias=True)
    layer.weight.requires_grad_(False)
    if packed:
        layer.pack()
    calls.clear()
    layer(bf(0, 40)).sum().backward()
    assert layer.bias.grad.tolist() == [0.0] * 24 and not calls


def test_frozen_layers_have_no_graph(recorded):  # noqa: F811
    T, calls = recorded
    for bias in (False, True):
        layer = T.Mx4Linear(40, 24, bias=bias).requires_grad_(False)
        assert not layer(bf(5, 40)).requires_grad and not layer.pack()(bf(5, 40)).requires_grad


@pytest.mark.gpu
@pytest.mark.parametrize("packed", [False, True])
def test_captured_with_its_backward(dev, packed):
    """The bias's gradient alone, recorded and replayed with eager work between the replays; many rows, whose sum takes several workgroups."""
    import triton_int8_amd as T
    gen = make_gen(3)
    layer = T.Mx4Linear(64, 96, bias=True, device=dev)
    layer.weight.requires_grad_(False)
    if packed:
        layer.pack()
    sets = [(randn_bf16(gen, 20000, 64).to(dev), randn_bf16(gen, 20000, 96).to(dev)) for _ in range(3)]

    def step(x, dy):
        bias = layer.bias.detach().requires_grad_()
        y = torch.func.functional_call(layer, {"bias": bias}, x)
        return y.detach(), torch.autograd.grad(y, bias, dy)[0]
    want = [[t.clone() for t in step(*s)] for s in sets]
    for s, (y, db) in zip(sets, want):
        exact = s[1].double().sum(0)
        # (19999 additions in fp32 and a rounding to bf16)
        assert bool(((db.double() - exact).abs() <= 2.0 ** -8 * exact.abs() + 20000 * 2.0 ** -24 * (1 + 2.0 ** -8) * s[1].double().abs().sum(0)).all())
    graphed = T.GraphedStep(step, *sets[0])
    for turn in range(6):
        got = graphed(*sets[turn % 3])
        torch.cuda.synchronize()
        assert all(bits_equal(a, b) for a, b in zip(got, want[turn % 3])), turn
        step(*sets[(turn + 1) % 3])
