"""nn.RotaryEmbedding: where its frequencies live and which scalings it takes."""
import pytest
import torch

from immunostruct_amd import functional as HF
from immunostruct_amd.nn import RotaryEmbedding

YARN = dict(kind="yarn", factor=4.0, original_length=4096)


@pytest.mark.parametrize("scaling", [None, dict(kind="linear", factor=4.0), dict(kind="ntk", factor=4.0), YARN], ids=lambda s: "none" if s is None else s["kind"])
def test_frequencies_are_on_the_host_under_a_device_context(scaling):
    """a model built under torch.device(...) or a default device (here: meta, which needs no GPU)"""
    want = RotaryEmbedding(16, scaling=scaling)
    with torch.device("meta"):
        one = RotaryEmbedding(16, scaling=scaling)
    torch.set_default_device("meta")
    try:
        two = RotaryEmbedding(16, scaling=scaling)
    finally:
        torch.set_default_device(None)
    for rope in (one, two):
        assert rope.freq.device.type == "cpu" and torch.equal(rope.freq, want.freq) and rope.amplitude == want.amplitude


@pytest.mark.gpu
def test_turns_under_a_device_context(cuda_device):
    with torch.device("cuda"):
        rope = RotaryEmbedding(16)
        q = torch.randn(2, 5, 3, 16)
        got = rope(q)[0]
    assert torch.equal(got, HF.rotary(q, None, RotaryEmbedding(16).freq)[0])


@pytest.mark.parametrize("scaling", ["linear", "yarn", ("kind", "linear"), 4.0, dict(kind="yarn", factor=4.0), dict(YARN, original_length=None),
                                     dict(YARN, original_length=float("nan")), dict(YARN, original_length=float("inf")), dict(YARN, beta_fast=None),
                                     dict(YARN, beta_fast=float("inf")), dict(kind="linear", factor=None), dict(kind="linear", factor="x"),
                                     dict(YARN, amplitude=float("nan")), dict(YARN, amplitude="x")])
def test_scalings_that_are_none(scaling):
    with pytest.raises(ValueError, match="RotaryEmbedding: unknown scaling"):
        RotaryEmbedding(16, scaling=scaling)


def test_frequencies_have_no_gradient():
    with pytest.raises(ValueError, match="no gradient"):
        HF.rotary(torch.zeros(1, 2, 1, 8), None, torch.ones(4, dtype=torch.float64, requires_grad=True))
