"""Edited logits bit by bit: the same fp32 operations in the documented order, each rounded to nearest, then one rounding to the type."""
import numpy as np
import pytest

from test_logits_edit_gpu import handle, make

pytestmark = pytest.mark.gpu


def edited32(p):
    x = p["logits"].astype(np.float32)
    rows, vocab = x.shape
    one = np.float32(1)
    for r in range(rows):
        if "history" in p:
            n, start = int(p["length"][r]), int(p["prompt"][r])
            tokens = p["history"][r, :n]
            count = np.bincount(tokens[start:], minlength=vocab)
            seen = np.unique(tokens)
            v = x[r, seen]
            with np.errstate(over="ignore"):
                v = np.where(v > 0, v / p["repetition"][r], v * p["repetition"][r])
                c = count[seen].astype(np.float32)
                v = np.where(c > 0, (v - p["frequency"][r] * c) - p["presence"][r], v)
            x[r, seen] = v
        if "bias" in p:
            sums = {}
            for t, b in zip(p["bias_token"][r, :p["n_bias"][r]], p["bias"][r]):
                if 0 <= t < vocab:
                    sums[t] = np.float32(sums[t] + b) if t in sums else b
            for t, b in sums.items():
                x[r, t] = x[r, t] + b * one
        if "mask" in p and p["mask_row"][r] >= 0:
            t = np.arange(vocab)
            x[r, (p["mask"][p["mask_row"][r]][t // 32] >> (t % 32).astype(np.uint32)) & 1 == 0] = -np.inf
    assert x.dtype == np.float32
    with np.errstate(over="ignore"):
        return x.astype(p["logits"].dtype)


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("rows,vocab,history,biases,masks", [(1, 50257, 300, 0, None), (4, 999, 500, 40, 2), (64, 50257, 1023, 16, 8), (3, 50, 6000, 1024, 1), (2, 131072, 8192, 300, 2),
                                                             (5, 70001, 100, 7, None)])
def test_every_bit(lib, cuda, rows, vocab, history, biases, masks, dtype):
    torch = cuda
    p = make(torch, rows, vocab, history, biases, 7 * rows + vocab, dtype, masks)
    h, logits = handle(lib, torch, p)
    out = torch.empty_like(logits)
    bits = np.uint16 if dtype == np.float16 else np.uint32
    want = edited32(p).view(bits)
    h.apply(out, logits)
    assert np.array_equal(out.cpu().numpy().view(bits), want)
    nxt = torch.empty(rows, dtype=torch.int32, device="cuda")
    h.apply(logits, logits, nxt)
    assert np.array_equal(logits.cpu().numpy().view(bits), want)
    lib.status()
