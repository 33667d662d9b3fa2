"""Devices that the wrappers of 4-bit weights and edits look after (no GPU needed: nothing here reaches a launch)."""
import types

import pytest

import gpt2_b200 as G


@pytest.fixture(scope="module")
def torch():
    import torch
    return torch


def test_tensors_of_the_host_do_not_reach_the_library(lib, torch):
    half = dict(dtype=torch.float16)
    x = torch.zeros(3, 100)
    for e in (G.LogitsEdit(lib, torch, 3, 100), G.LogitsEdit(lib, torch, 3, 100, repetition=torch.ones(3))):
        with pytest.raises(ValueError):
            e.apply(x, x)
    w = G.W4Weight(lib, torch, torch.zeros(6, 64, dtype=torch.uint8), torch.zeros(2, 6, **half))
    for call in (lambda: w.quantize(torch.zeros(6, 128, **half)), lambda: w.dequantize(torch.zeros(6, 128, **half)), lambda: w.linear(torch.zeros(2, 6, **half), torch.zeros(2, 128, **half)),
                 lambda: G.W4Weight.pack(lib, torch, torch.zeros(6, 128, **half))):
        with pytest.raises(ValueError):
            call()


class Fake:
    """A tensor of two rows on a device that need not exist."""

    def __init__(self, torch, index):
        self.dtype, self.shape, self.device = torch.float32, torch.Size((2, 8)), torch.device("cuda", index)

    def stride(self):
        return (8, 1)

    def data_ptr(self):
        return 4096


def test_an_edit_without_tensors_checks_the_current_device(lib, torch, monkeypatch):
    """Its launches go to the current device, so the logits have to be there."""
    made = []
    fake = types.SimpleNamespace(cuda=types.SimpleNamespace(current_device=lambda: 0))
    e = G.LogitsEdit(lib, fake, 2, 8)
    monkeypatch.setattr(e, "_edit", lambda *a: made.append(a) or 0)
    with pytest.raises(ValueError):
        e.apply(Fake(torch, 1), Fake(torch, 1))
    with pytest.raises(ValueError):
        e.apply(Fake(torch, 0), Fake(torch, 1))
    assert not made
    e.apply(Fake(torch, 0), Fake(torch, 0))
    assert len(made) == 1
