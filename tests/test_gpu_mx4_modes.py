"""Layers in 4 bits under what torch wraps around a layer: compilation, inference mode, checkpoints, saved tensors that wait elsewhere, copies, rows that are no numbers."""
import copy

import pytest
import torch

from conftest import bits_equal, make_gen, randn_bf16

pytestmark = pytest.mark.gpu


@pytest.fixture(params=[True, False], ids=["from C++", "from Python"])
def T(request, monkeypatch):
    import triton_int8_amd
    if not request.param:
        monkeypatch.setattr(triton_int8_amd._lib, "native", lambda: None)
    return triton_int8_amd


def step(layer, x, dy):
    """(y, dx, dW, db) of a call with its backward."""
    layer.zero_grad(set_to_none=True)
    h = x.detach().requires_grad_()
    y = layer(h)
    y.backward(dy)
    return [y.detach(), h.grad, *(p.grad for p in layer.parameters())]


@pytest.fixture
def made(T, dev):
    gen = make_gen(1)
    m = T.Mx4Linear(300, 96, bias=True, device=dev)
    with torch.no_grad():
        m.weight.copy_(randn_bf16(gen, 96, 300, std=0.06))
        m.bias.copy_(randn_bf16(gen, 96))
    x, dy = randn_bf16(gen, 70, 300).to(dev), randn_bf16(gen, 70, 96).to(dev)
    return m, x, dy, [t.clone() for t in step(m, x, dy)]


@pytest.mark.parametrize("backend", ["eager", "aot_eager"])
def test_compiled(made, backend):
    m, x, dy, want = made
    compiled = torch.compile(m, backend=backend)
    for _ in range(2):
        m.zero_grad(set_to_none=True)
        h = x.clone().requires_grad_()
        y = compiled(h)
        y.backward(dy)
        assert all(bits_equal(a, b) for a, b in zip([y.detach(), h.grad, m.weight.grad, m.bias.grad], want))
        with torch.no_grad():
            assert bits_equal(compiled(x), want[0])
    torch._dynamo.reset()


def test_compiled_functions(T, dev):
    x = randn_bf16(make_gen(2), 33, 520).to(dev)
    w = torch.ones(520, dtype=torch.bfloat16, device=dev)
    for f in (lambda t: T.mx4.quant_row(t), lambda t: T.mx4.quant_row(t.t()), lambda t: T.ops.rmsnorm_quant(t, w, 1e-5, residual=t), lambda t: T.mx4.gemm_nt(*T.mx4.quant_row(t), *T.mx4.quant_row(t))):
        want, got = f(x), torch.compile(f, backend="eager")(x)
        for a, b in zip(*((t,) if isinstance(t, torch.Tensor) else t for t in (got, want))):
            assert bits_equal(a, b)
        torch._dynamo.reset()


def test_inference_mode(made):
    m, x, dy, want = made
    with torch.inference_mode():
        assert bits_equal(m(x), want[0])
        other = copy.deepcopy(m).pack()
        assert bits_equal(other(x), want[0])
    with torch.no_grad():
        assert bits_equal(other(x), want[0])
    assert all(bits_equal(a, b) for a, b in zip(step(m, x, dy), want))


@pytest.mark.parametrize("reentrant", [False, True])
def test_checkpointed(made, reentrant):
    from torch.utils.checkpoint import checkpoint
    m, x, dy, want = made
    got = step_of(lambda h: checkpoint(m, h, use_reentrant=reentrant), m, x, dy)
    assert all(bits_equal(a, b) for a, b in zip(got, want))


def step_of(call, m, x, dy):
    m.zero_grad(set_to_none=True)
    h = x.clone().requires_grad_()
    y = call(h)
    y.backward(dy)
    return [y.detach(), h.grad, m.weight.grad, m.bias.grad]


def test_saved_tensors_that_wait_elsewhere(made):
    m, x, dy, want = made
    with torch.autograd.graph.save_on_cpu():
        got = step_of(m, m, x, dy)
    assert all(bits_equal(a, b) for a, b in zip(got, want))


def test_copies(made):
    m, x, dy, want = made
    other = copy.deepcopy(m)
    assert all(bits_equal(a, b) for a, b in zip(step(other, x, dy), want))
    packed = copy.deepcopy(other.pack())
    with torch.no_grad():
        assert bits_equal(packed(x), want[0])


def test_batched_gradients_are_refused(made):
    m, x, dy, want = made
    y = m(x.clone().requires_grad_())
    with pytest.raises((RuntimeError, ValueError)):
        torch.autograd.grad(y, m.weight, torch.stack((dy, dy)), is_grads_batched=True)
    torch.cuda.synchronize()


def test_the_weight_may_change_before_the_backward(made):
    """(The backward reads what the forward quantised.)"""
    m, x, dy, want = made
    m.zero_grad(set_to_none=True)
    h = x.clone().requires_grad_()
    y = m(h)
    with torch.no_grad():
        m.weight.zero_()
    y.backward(dy)
    assert all(bits_equal(a, b) for a, b in zip([y.detach(), h.grad, m.weight.grad, m.bias.grad], want))


@pytest.mark.parametrize("dim", [512, 4096])
@pytest.mark.parametrize("to,group", [("mx4", 0), ("int8", 0), ("int8", 128)])
def test_rows_that_are_no_numbers(T, dev, dim, to, group):
    """They spoil their own row only, and there give what the quantiser gives for the norm's result."""
    gen = make_gen(dim)
    x, w = randn_bf16(gen, 9, dim), randn_bf16(gen, dim)
    x[1, 5], x[3, dim - 1], x[5, 0], x[7] = float("nan"), float("inf"), -float("inf"), 0.0
    x[8, 7], x[8, 9] = 3e38, -3e38
    x, w = x.to(dev), w.to(dev)
    q, s, rstd = T.ops.rmsnorm_quant(x, w, 1e-5, to=to, group=group)
    y = ((x.float() * rstd[:, None]).bfloat16().float() * w.float()).bfloat16()
    want = T.mx4.quant_row(y) if to == "mx4" else T.ops.quant_row(y, group=group)
    fine = [0, 2, 4, 6, 7, 8]
    assert torch.equal(q[fine], want[0][fine]) and torch.equal(s[:, fine] if to == "mx4" else s[fine], want[1][:, fine] if to == "mx4" else want[1][fine])
    if to == "mx4":
        assert torch.equal(q, want[0]) and torch.equal(s, want[1])
    exact = 1.0 / torch.sqrt(x[fine].double().square().mean(-1) + 1e-5)
    assert bool(((rstd[fine].double() - exact).abs() <= 2.0 ** -24 * (1 + 2.0 ** -20) * exact).all())
    assert rstd[1].isnan() and rstd[3] == 0 and rstd[5] == 0
