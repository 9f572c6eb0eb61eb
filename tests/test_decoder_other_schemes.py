"""Layers of other schemes look at one of their linears, not at all seven, before they serve as they always did."""
import pytest
import torch

from triton_int8_amd import DecoderLayer


@pytest.mark.parametrize("how", [dict(), dict(scheme="double_channel"), dict(int8=False)], ids=str)
def test_one_look(monkeypatch, how):
    layer = DecoderLayer(256, 2, 256, **how)
    monkeypatch.setattr(DecoderLayer, "_linears", lambda self: pytest.fail("looked at all"))
    assert not layer._norm_quantises(torch.zeros(1, 1, 256, dtype=torch.bfloat16))
