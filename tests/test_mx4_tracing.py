"""Calls on tensors in 4 bits, and the quantised norm, under what records operators: a record would hold the outputs' memory and nothing that fills it."""
import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx

from test_mx4_host import bf, recorded  # noqa: F401 (a fixture)


def entry_points(T):
    """name -> a function of x bf16 [4, 256]."""
    w, q, s = bf(256), torch.zeros(4, 128, dtype=torch.uint8), torch.zeros(1, 4, 8, dtype=torch.uint8)
    layer, trained = T.Mx4Linear(256, 8, bias=True).requires_grad_(False), T.Mx4Linear(256, 8)
    return {
        "layer": layer, "layer in training": trained, "several layers": lambda t: T.mx4.linears(t, (layer, layer)), "quant_row": T.mx4.quant_row, "quant_col_t": T.mx4.quant_col_t,
        "quant_row_col_t": T.mx4.quant_row_col_t, "step": lambda t: T.mx4.linear_fwd_bwd(t, t, t[:, :4]), "product": lambda t: T.mx4.gemm_nt(q, s, q, s) + t[:, :4],
        "products": lambda t: T.mx4.gemm_nt_multi([(q, s, q, s)])[0] + t[:, :4], "dequant": lambda t: T.mx4.dequant(q, s, 256) + t, "norm": lambda t: T.ops.rmsnorm_quant(t, w, 1e-5),
        "norm to int8": lambda t: T.ops.rmsnorm_quant(t, w, 1e-5, residual=t, to="int8"), "dequant_row": lambda t: T.ops.dequant_row(torch.zeros(4, 256, dtype=torch.int8), torch.ones(4)) + t}


NAMES = ["layer", "layer in training", "several layers", "quant_row", "quant_col_t", "quant_row_col_t", "step", "product", "products", "dequant", "norm", "norm to int8", "dequant_row"]


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("how", [{}, dict(pre_dispatch=True), dict(tracing_mode="fake"), dict(tracing_mode="symbolic")], ids=str)
def test_make_fx_is_refused(recorded, name, how):  # noqa: F811
    T, calls = recorded
    with pytest.raises(ValueError, match="traced"):
        make_fx(entry_points(T)[name], **how)(bf(4, 256))
    assert not calls


@pytest.mark.parametrize("name", [n for n in NAMES if n != "layer in training"])      # (there torch refuses functions with a backward of their own)
def test_functionalize_is_refused(recorded, name):  # noqa: F811
    T, calls = recorded
    with pytest.raises(ValueError, match="traced"):
        torch.func.functionalize(entry_points(T)[name])(bf(4, 256))
    assert not calls


@pytest.mark.parametrize("name", NAMES)
def test_tensors_without_memory_are_refused(recorded, name):  # noqa: F811
    from torch._subclasses.fake_tensor import FakeTensorMode
    T, calls = recorded
    f = entry_points(T)[name]
    with FakeTensorMode(allow_non_fake_inputs=True), pytest.raises(ValueError, match="traced"):
        f(bf(4, 256))
    assert not calls


@pytest.mark.parametrize("name", ["layer", "quant_row", "step", "norm"])
@pytest.mark.parametrize("transform", [torch.func.vmap, lambda f: torch.func.grad(lambda t: f(t)[0].float().sum()), lambda f: lambda t: torch.func.jvp(f, (t,), (t,))], ids=["vmap", "grad", "jvp"])
def test_transformed_inputs_are_refused(recorded, name, transform):  # noqa: F811
    T, calls = recorded
    with pytest.raises((ValueError, RuntimeError)):
        transform(entry_points(T)[name])(bf(1, 4, 256) if transform is torch.func.vmap else bf(4, 256))
    assert not calls


@pytest.mark.parametrize("name", NAMES)
def test_modes_that_watch_are_no_tracers(recorded, name):  # noqa: F811
    from torch.utils.flop_counter import FlopCounterMode
    T, calls = recorded
    f = entry_points(T)[name]
    with FlopCounterMode(display=False):
        f(bf(4, 256))
    assert calls


def test_constants_of_a_mapped_function(recorded):  # noqa: F811
    T, calls = recorded
    q, s = torch.zeros(4, 128, dtype=torch.uint8), torch.zeros(1, 4, 8, dtype=torch.uint8)
    assert torch.func.vmap(lambda t: t + T.mx4.dequant(q, s, 256))(bf(3, 4, 256)).shape == (3, 4, 256)
    assert [n for n, _ in calls] == ["ti8_mx4_dequant"]


@pytest.mark.parametrize("backend", ["eager", "aot_eager"])
def test_a_compiled_layer_makes_its_calls(recorded, backend):  # noqa: F811
    """(torch.compile leaves them out of its graphs.)"""
    T, calls = recorded
    layer = T.Mx4Linear(256, 8)
    compiled = torch.compile(layer, backend=backend)
    for _ in range(2):
        calls.clear()
        compiled(bf(4, 256).requires_grad_()).sum().backward()
        assert [n for n, _ in calls] == ["ti8_mx4_quant", "ti8_mx4_quant", "ti8_mx4_gemm_nt_multi"] + ["ti8_mx4_quant", "ti8_mx4_gemm_nt_multi"]
    torch._dynamo.reset()
