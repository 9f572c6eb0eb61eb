"""Calls on a 4-bit cache under what records operators: a record would hold nothing of what they write."""
import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx


@pytest.fixture
def called(monkeypatch):
    """A pool, its table and lengths on the host, and the library's calls, recorded instead of made."""
    import triton_int8_amd as T
    calls = []
    monkeypatch.setattr(T.ops, "_on_gpu", lambda t: True)
    monkeypatch.setattr(torch.Tensor, "get_device", lambda t: 0)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 0, raising=False)
    monkeypatch.setattr(T.cache4, "_stream", lambda: 0)
    monkeypatch.setattr(T._lib, "native", lambda: None)
    monkeypatch.setattr(T._lib, "call", lambda name, *a: calls.append(name))
    where = torch.zeros(4, 2, T.cache4.page_bytes(16, 64), dtype=torch.uint8), torch.zeros(1, 4, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    weights, spare = torch.zeros(4, 2, 16), torch.zeros(1, 4, dtype=torch.int32)
    C = T.cache4
    return calls, {"append": lambda t: C.append(*where, t, t), "attention": lambda t: C.attention(*where, t)[0], "read": lambda t: C.read(*where, 3, 64)[0] + t,
                   "evict": lambda t: C.evict(*where, weights, spare, keep=32, recent=1)[0]}


@pytest.mark.parametrize("name", ["append", "attention", "read", "evict"])
@pytest.mark.parametrize("how", [make_fx, lambda f: make_fx(f, pre_dispatch=True), lambda f: make_fx(f, tracing_mode="fake"), torch.func.functionalize, lambda f: lambda x: torch.jit.trace(f, (x,))],
                         ids=["make_fx", "pre_dispatch", "fake", "functionalize", "jit"])
def test_tracers_are_refused(called, name, how):
    calls, entry_points = called
    with pytest.raises(ValueError, match="traced"):
        how(entry_points[name])(torch.ones(1, 3, 2, 64, dtype=torch.bfloat16))
    assert not calls


@pytest.mark.parametrize("name", ["append", "read"])
def test_modes_that_watch_are_no_tracers(called, name, monkeypatch):
    from torch.utils.flop_counter import FlopCounterMode
    calls, entry_points = called
    with FlopCounterMode(display=False):
        entry_points[name](torch.ones(1, 3, 2, 64, dtype=torch.bfloat16))
    assert calls == ["ti8_cache4_" + name]
