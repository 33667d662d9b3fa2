"""A decode batch and its 4-bit weights are on one device (no GPU needed: nothing here reaches the library)."""
import types

import pytest

import gpt2_b200 as G


@pytest.mark.parametrize("which", ["layer", "head"])
def test_weights_of_another_device(which):
    import torch
    here, there = (types.SimpleNamespace(codes=types.SimpleNamespace(device=torch.device("cuda", i))) for i in (0, 1))
    layers = [{"qkv": here, "fc": here}, {"qkv": here, "fc": there if which == "layer" else here}]
    w4 = types.SimpleNamespace(layers=layers, head=there if which == "head" else None)
    caches = types.SimpleNamespace(device=torch.device("cuda", 0))
    with pytest.raises(ValueError, match="device"):
        G.DecodeBatch(None, None, caches, w4)
