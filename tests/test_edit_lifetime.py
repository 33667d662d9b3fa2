"""What a generation keeps of its arguments (no GPU needed)."""
import gc
import types
import weakref

import pytest

import gpt2_b200 as G


@pytest.fixture(scope="module")
def torch():
    import torch
    return torch


def test_a_batch_keeps_the_edit_of_its_generation(lib, torch):
    """generate() returns before its steps ran: the edit's tensors have to outlive a caller who drops them."""
    i32 = dict(dtype=torch.int32)
    bt = G.DecodeBatch.__new__(G.DecodeBatch)
    bt.B, bt.caches, bt.h = 2, torch.zeros(1), None
    bt.lib = types.SimpleNamespace(check=lambda rc, what: None, gpt2_b200_batch_generate_edited=lambda *a: 0)
    mask = torch.zeros(1, (G.VOCAB + 31) // 32, **i32)
    alive = weakref.ref(mask)
    bt.generate(torch.zeros(2, 3, **i32), torch.ones(2, **i32), 4, torch.zeros(2, 5, **i32), edit=G.LogitsEdit(lib, torch, 2, G.VOCAB, mask=mask))
    del mask
    gc.collect()
    assert alive() is not None
