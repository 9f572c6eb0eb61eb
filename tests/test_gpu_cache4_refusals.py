"""What the 4-bit cache's calls refuse beyond shapes and types."""
import pytest
import torch
from torch.autograd import forward_ad

from test_gpu_cache4 import C, _ints  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.fixture
def cache(C, dev):
    cache = C.Cache4(1, 64, 2, 64, page_size=16, budget=32, device=dev)
    cache.pool.zero_()
    return cache


def _calls(C, cache, x, weights):
    """Every call that takes values, with x in place of one of them or with these weights."""
    plain, q = x.detach().clone(), torch.cat((x, x), dim=2)
    where = cache.pool, cache.table
    return [lambda: C.append(*where, cache.lengths, x, plain), lambda: C.append(*where, cache.lengths, plain, x), lambda: C.attention(*where, cache.lengths, q)], [
        lambda: C.append(*where, cache.lengths, plain, plain, weights=weights), lambda: C.attention(*where, cache.lengths, plain, weights=weights),
        lambda: C.evict(*where, cache.lengths, weights, cache.spare, keep=32, recent=1)]


@pytest.mark.parametrize("native", [True, False])
def test_tangents(C, dev, cache, native, monkeypatch):
    """A tangent would be dropped without a word; tensors that have none are taken also while tangents are carried on."""
    import triton_int8_amd as T
    if not native:
        monkeypatch.setattr(T._lib, "native", lambda: None)
    x = torch.ones(1, 3, 2, 64, dtype=torch.bfloat16, device=dev)
    before = cache.pool.clone()
    with forward_ad.dual_level():
        for grad in (True, False):
            with torch.set_grad_enabled(grad):
                for call in _calls(C, cache, forward_ad.make_dual(x, torch.ones_like(x)), None)[0] + \
                        _calls(C, cache, x, forward_ad.make_dual(cache.weights, torch.ones_like(cache.weights)))[1]:
                    with pytest.raises(ValueError, match="tangent"):
                        call()
        assert torch.equal(cache.pool, before)
        cache.append(x, x)
    assert cache.lengths.tolist() == [3] and not torch.equal(cache.pool, before)
    out = cache.attend(torch.cat((x, x), dim=2))
    with forward_ad.dual_level():
        assert torch.equal(cache.attend(torch.cat((x, x), dim=2)), out)


@pytest.mark.parametrize("native", [True, False])
def test_weights_that_require_a_gradient(C, dev, cache, native, monkeypatch):
    import triton_int8_amd as T
    if not native:
        monkeypatch.setattr(T._lib, "native", lambda: None)
    x = torch.ones(1, 3, 2, 64, dtype=torch.bfloat16, device=dev)
    weights = cache.weights.clone().requires_grad_(True)
    for call in _calls(C, cache, x, weights)[1]:
        with pytest.raises(ValueError, match="gradient"):
            call()
    with torch.no_grad():
        for call in _calls(C, cache, x, weights)[1]:
            call()


@pytest.mark.parametrize("native", [True, False])
def test_tracing(C, dev, cache, native, monkeypatch):
    """A trace would hold nothing of what a call launches."""
    import triton_int8_amd as T
    if not native:
        monkeypatch.setattr(T._lib, "native", lambda: None)
    x = torch.ones(1, 3, 2, 64, dtype=torch.bfloat16, device=dev)
    cache.append(x, x)
    where = cache.pool, cache.table, cache.lengths
    before = cache.pool.clone()
    for call in (lambda t: C.append(*where, t, t), lambda t: C.attention(*where, t)[0], lambda t: C.read(*where, 3, 64)[0],
                 lambda t: C.evict(*where, cache.weights, cache.spare, keep=32, recent=1)[0]):
        with pytest.raises(ValueError, match="traced"):
            torch.jit.trace(call, (x,), check_trace=False)
    assert torch.equal(cache.pool, before)


@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("scale", [float("nan"), float("inf"), 1e39, -(2 ** 200)])
def test_scales(C, dev, cache, native, scale, monkeypatch):
    import triton_int8_amd as T
    if not native:
        monkeypatch.setattr(T._lib, "native", lambda: None)
    x = torch.ones(1, 3, 2, 64, dtype=torch.bfloat16, device=dev)
    cache.append(x, x)
    with pytest.raises(ValueError, match="scale"):
        C.attention(cache.pool, cache.table, cache.lengths, x, scale=scale)
    assert torch.equal(cache.attend(x, scale=1), cache.attend(x, scale=1.0))
