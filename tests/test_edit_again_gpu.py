"""Generations with edited logits called again: the graph that is there is taken where nothing changed."""
import ctypes

import numpy as np
import pytest

import gpt2_b200 as G

pytestmark = pytest.mark.gpu
V = G.VOCAB


@pytest.fixture(scope="module")
def weights(cuda):
    return G.ModelWeights(cuda, "cuda", seed=21, hf_init=False)


def batch(torch, lib, weights, B, max_t=32):
    return G.DecodeBatch(lib, weights, torch.zeros(B, 12, 2, 12, max_t, 64, dtype=torch.float16, device="cuda"))


def ints(torch, *values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def test_an_equal_edit_does_not_wait_for_the_device(cuda, lib, weights):
    """A descriptor with the same fields takes the graph that is there, whatever lies in its padding and its unused fields; a new graph
    would wait for everything that the device still has to do."""
    torch = cuda
    B, steps = 2, 4
    prompt, plen = ints(torch, [5], [6]), ints(torch, 1, 1)
    out = torch.empty(B, steps + 1, dtype=torch.int32, device="cuda")
    bt = batch(torch, lib, weights, B)
    edit = G.LogitsEdit(lib, torch, B, V, repetition=torch.full((B,), 1.2, device="cuda"))
    for _ in range(2):
        bt.generate(prompt, plen, steps, out, edit=edit)
    torch.cuda.synchronize()
    want = out.clone()
    side, done = torch.cuda.Stream(), torch.cuda.Event()
    raw = (ctypes.c_uint8 * ctypes.sizeof(edit.c)).from_buffer(edit.c)
    fields = np.zeros(len(raw), bool)
    for name, kind in G.GPT2LogitsEdit._fields_:
        at = getattr(G.GPT2LogitsEdit, name).offset
        fields[at:at + ctypes.sizeof(kind)] = True
    for i in np.nonzero(~fields)[0]:
        raw[int(i)] = 0xA5
    assert not fields.all()
    with torch.cuda.stream(side):
        torch.cuda._sleep(1_000_000_000)  # half a second
        done.record()
    bt.generate(prompt, plen, steps, out, edit=edit)
    assert not done.query()
    torch.cuda.synchronize()
    assert torch.equal(out, want)
    bt.close()
    assert lib.status() == 0
