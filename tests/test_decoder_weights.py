"""DecoderLayer.copy_weights_from: what is copied is told by names, and all of it or nothing is."""
import pytest
import torch

from conftest import make_gen
from triton_int8_amd import DecoderLayer


def filled(seed, *sizes, scheme="mx4", packed=False, **kw):
    """A layer of random weights (hidden == mlp: matrices of all linears have one shape); packed as DecoderLayer.pack leaves it, with random codes."""
    layer, gen = DecoderLayer(*(sizes or (64, 2, 64)), scheme=scheme, **kw), make_gen(seed)
    with torch.no_grad():
        for p in layer.parameters():
            p.copy_(torch.randn(p.shape, generator=gen))
        for m in layer._linears() if packed else ():
            m.codes, m.scales = (torch.randint(0, 250, s, dtype=torch.uint8, generator=gen) for s in ((m.out_features, 128), (1, m.out_features, 8)))
            m.weight = None
    return layer


def state(layer):
    return {k: v.clone() for k, v in layer.state_dict().items()}


@pytest.mark.parametrize("a,b", [(dict(packed=True), {}), ({}, dict(packed=True)), (dict(packed=True), dict(int8=False)), (dict(int8=False), dict(packed=True))], ids=str)
def test_packed_and_unpacked_layers_do_not_mix(a, b):
    to, other = filled(1, **a), filled(2, **b)
    before = state(to)
    with pytest.raises(ValueError, match="pack"):
        to.copy_weights_from(other)
    assert all(torch.equal(v, before[k]) for k, v in to.state_dict().items())


def test_packed_layers_copy_their_codes():
    to, other = filled(1, packed=True), filled(2, packed=True)
    at = {k: v.data_ptr() for k, v in to.state_dict().items()}
    to.copy_weights_from(other)
    want = state(other)
    assert len(want) == 16 and to.state_dict().keys() == want.keys()
    assert all(torch.equal(v, want[k]) and v.data_ptr() == at[k] for k, v in to.state_dict().items())     # (in place: a recorded graph reads them)


@pytest.mark.parametrize("sizes", [(64, 2, 128), (128, 2, 64), (1, 1, 64)], ids=str)
def test_layers_of_other_sizes_are_refused(sizes):
    """(Also those that would fit into the others by broadcasting.)"""
    to, other = filled(1), filled(2, *sizes)
    before = state(to)
    with pytest.raises(ValueError, match="shape"):
        to.copy_weights_from(other)
    assert all(torch.equal(v, before[k]) for k, v in to.state_dict().items())


@pytest.mark.parametrize("a,b", [(dict(), dict(int8=False)), (dict(int8=False), dict()), (dict(scheme="block_channel"), dict()), (dict(scheme="double_channel"), dict(int8=False))], ids=str)
def test_layers_of_any_scheme_share_values(a, b):
    to, other = filled(1, 128, 2, 128, **a), filled(2, 128, 2, 128, **b)
    to.copy_weights_from(other)
    assert all(torch.equal(p, q) for p, q in zip(to.parameters(), other.parameters()))


def test_a_layer_inside_another_module():
    to, other = filled(1), filled(2)
    to.copy_weights_from(torch.nn.Sequential(other))
    assert all(torch.equal(p, q) for p, q in zip(to.parameters(), other.parameters()))
