"""Penalties, biases, masks and the greedy choice against the definition in 64 bits.

Tolerances: an edit is up to 6 operations in fp32, each off by half a step, 2^-24 of what it sees (the logit, the penalties' product and their
sums with it): 8 * 2^-24 of the largest magnitude on the way covers them; the result is rounded once to its type. What no edit
touches is compared bit by bit. The choice is compared with the argmax of what was written.
"""
import math

import numpy as np
import pytest

import gpt2_b200 as G

pytestmark = pytest.mark.gpu


def make(torch, rows, vocab, history, biases, seed, dtype=np.float16, masks=None):
    """The pieces of an edit in numpy."""
    rng = np.random.default_rng(seed)
    p = {"logits": (4 * rng.standard_normal((rows, vocab))).astype(dtype)}
    if history:
        p["history"] = (vocab * rng.random((rows, history)) ** 3).astype(np.int32)
        p["length"] = rng.integers(0, history + 1, rows).astype(np.int32)
        p["prompt"] = (p["length"] * rng.random(rows)).astype(np.int32)
        for name in ("repetition", "frequency", "presence"):
            p[name] = (rng.random(rows) + (0.5 if name == "repetition" else -0.5)).astype(np.float32)
    if biases:
        p["bias_token"] = rng.integers(-2, vocab + 2, (rows, biases)).astype(np.int32)  # some outside, some twice
        p["bias"] = rng.standard_normal((rows, biases)).astype(np.float32)
        p["n_bias"] = rng.integers(0, biases + 1, rows).astype(np.int32)
    if masks:
        p["mask"] = rng.integers(0, 2**32, (masks, (vocab + 31) // 32 + 1), dtype=np.uint32)
        p["mask_row"] = rng.integers(-1, masks, rows).astype(np.int32)
    return p


def edited(p):
    """The edited logits in 64 bits, the largest magnitude on the way, and which were touched."""
    x = p["logits"].astype(np.float64)
    rows, vocab = x.shape
    size, touched = np.abs(x), np.zeros(x.shape, bool)
    for r in range(rows):
        if "history" in p:
            n = int(p["length"][r]) if "length" in p else p["history"].shape[1]
            start = int(p["prompt"][r]) if "prompt" in p else 0
            tokens = p["history"][r, :n]
            ok = (tokens >= 0) & (tokens < vocab)
            count = np.bincount(tokens[start:][ok[start:]], minlength=vocab)
            for t in np.unique(tokens[ok]):
                rep = float(p["repetition"][r]) if "repetition" in p else 1.0
                x[r, t] = x[r, t] / rep if x[r, t] > 0 else x[r, t] * rep
                size[r, t] = max(size[r, t], abs(x[r, t]))
                if count[t]:
                    down = (float(p["frequency"][r]) if "frequency" in p else 0.0) * count[t]
                    size[r, t] += abs(down)
                    x[r, t] -= down
                    x[r, t] -= float(p["presence"][r]) if "presence" in p else 0.0
                    size[r, t] += 1
                touched[r, t] = True
        if "bias" in p:
            for i in range(int(p["n_bias"][r]) if "n_bias" in p else p["bias"].shape[1]):
                t = int(p["bias_token"][r, i])
                if 0 <= t < vocab:
                    x[r, t] += float(p["bias"][r, i])
                    size[r, t] += abs(float(p["bias"][r, i]))
                    touched[r, t] = True
        if "mask" in p:
            m = int(p["mask_row"][r]) if "mask_row" in p else r if p["mask"].shape[0] > 1 else 0
            if m >= 0:
                t = np.arange(vocab)
                out = (p["mask"][m][t // 32] >> (t % 32).astype(np.uint32)) & 1 == 0
                x[r, out] = -np.inf
                touched[r, out] = True
    return x, size, touched


def check(p, got, untouched_from=None):
    want, size, touched = edited(p)
    assert np.array_equal(got[~touched].view(np.uint16 if got.dtype == np.float16 else np.uint32),
                          p["logits"][~touched].view(np.uint16 if got.dtype == np.float16 else np.uint32))
    assert np.array_equal(np.isneginf(got), np.isneginf(want))
    live = touched & ~np.isneginf(want)
    half = float(np.finfo(got.dtype).eps) / 2
    err = np.abs(got[live].astype(np.float64) - want[live])
    assert (err <= half * np.abs(want[live]) + 8 * 2.0**-24 * size[live] + 2.0**-25).all()


def first_max(got):
    return np.array([-1 if np.isneginf(r).all() else int(np.argmax(r)) for r in got.astype(np.float32)])


def handle(lib, torch, p, device="cuda"):
    t = {k: torch.from_numpy(v.view(np.int32) if v.dtype == np.uint32 else v).to(device) for k, v in p.items()}
    logits = t.pop("logits")
    return G.LogitsEdit(lib, torch, *logits.shape, **t), logits


CASES = [(1, 1, 1, 0, None), (1, 9, 3, 2, 1), (2, 33, 40, 5, 2), (3, 100, 0, 7, None), (5, 1000, 100, 0, 3), (1, 50257, 300, 0, None), (1, 50257, 1000, 1024, 1),
         (64, 50257, 1023, 16, 8), (7, 20001, 5000, 300, 4), (2, 262145, 700, 33, 2), (300, 511, 64, 3, 300), (700, 4097, 20, 1, 5), (600, 40001, 3, 2, None),
         (2, 262145, 9000, 33, 2), (3, 50, 6000, 1024, 1), (2, 1000, 20000, 3, 2), (150, 70001, 4097, 1, None)]


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("rows,vocab,history,biases,masks", CASES)
def test_edits_and_the_choice(lib, cuda, rows, vocab, history, biases, masks, dtype):
    torch = cuda
    p = make(torch, rows, vocab, history, biases, rows + vocab, dtype, masks)
    h, logits = handle(lib, torch, p)
    out = torch.empty_like(logits)
    nxt = torch.full((rows,), -7, dtype=torch.int32, device="cuda")
    h.apply(out, logits, nxt)
    got = out.cpu().numpy()
    check(p, got)
    want = first_max(got)
    assert np.array_equal(nxt.cpu().numpy(), want)
    assert lib.status() == (G.ST_EDIT_NO_TOKEN if (want < 0).any() else 0)
    out2 = torch.empty_like(logits)
    h.apply(out2, logits)
    assert np.array_equal(out2.cpu().numpy(), got)
    # in place, with and without the choice
    for n in (None, nxt.zero_()):
        here = logits.clone()
        h.apply(here, here, n)
        assert np.array_equal(here.cpu().numpy(), got)
    assert np.array_equal(nxt.cpu().numpy(), want)
    lib.status()


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("a,b,ld,ldo", [(0, 0, 1001, 1001), (1, 1, 1003, 1003), (1, 2, 1008, 1009), (3, 0, 1005, 1002), (7, 5, 1016, 1016), (2, 2, 1021, 1027)])
def test_rows_that_start_anywhere(lib, cuda, a, b, ld, ldo, dtype):
    """Rows of odd strides and offsets; what lies between them stays as it was."""
    torch = cuda
    rows, vocab = 9, 1001
    p = make(torch, rows, vocab, 200, 9, a + 10 * b, dtype, 2)
    h, logits = handle(lib, torch, p)
    src = torch.full((rows * ld + 16,), 3.0, dtype=logits.dtype, device="cuda")
    dst = torch.full((rows * ldo + 16,), 3.0, dtype=logits.dtype, device="cuda")
    x, y = src[a:a + rows * ld].view(rows, ld)[:, :vocab], dst[b:b + rows * ldo].view(rows, ldo)[:, :vocab]
    x.copy_(logits)
    nxt = torch.empty(rows, dtype=torch.int32, device="cuda")
    h.apply(y, x, nxt)
    check(p, y.cpu().numpy())
    assert np.array_equal(nxt.cpu().numpy(), first_max(y.cpu().numpy()))
    y.fill_(3.0)
    assert bool((dst == 3).all())
    h.apply(x, x)
    check(p, x.cpu().numpy())
    x.fill_(3.0)
    assert bool((src == 3).all())
    lib.status()


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
def test_values_that_are_not_finite_and_rows_with_nothing_left(lib, cuda, dtype):
    torch = cuda
    rows, vocab = 6, 300
    x = np.zeros((rows, vocab), dtype)
    x[0, 5], x[0, 6], x[0, 7] = np.nan, 2, 2          # NaN is never chosen, the first of equals is
    x[1] = -np.inf                                      # nothing there
    x[2, 100] = np.inf                                  # chosen
    x[3] = np.finfo(dtype).min                          # the type's lowest value is a value
    x[4, :] = np.nan                                    # nothing there
    x[5, 3:5] = (-0.0, 0.0)
    x[5, :3], x[5, 5:] = -1, -1                         # zeros of either sign are equal
    p = {"logits": x}
    h, logits = handle(lib, torch, p)
    out, nxt = torch.empty_like(logits), torch.empty(rows, dtype=torch.int32, device="cuda")
    h.apply(out, logits, nxt)
    bits = np.uint16 if dtype == np.float16 else np.uint32
    assert np.array_equal(out.cpu().numpy().view(bits), x.view(bits))
    assert nxt.tolist() == [6, -1, 100, 0, -1, 3]
    assert lib.status() == G.ST_EDIT_NO_TOKEN
    # a mask that leaves nothing, one that leaves a NaN, one token forced by an infinite bias, one -inf that no bias lifts
    mask = np.zeros((rows, 10), np.uint32)
    mask[0, 0] = 1 << 5
    mask[2:] = 0xFFFFFFFF
    p = {"logits": x, "mask": mask, "bias_token": np.full((rows, 1), 42, np.int32), "bias": np.full((rows, 1), np.inf, np.float32)}
    p["bias"][5] = -np.inf
    h, logits = handle(lib, torch, p)
    h.apply(out, logits, nxt)
    got = out.cpu().numpy()
    assert np.isnan(got[0, 5]) and np.isneginf(np.delete(got[0], 5)).all() and np.isneginf(got[1]).all()
    assert nxt.tolist() == [-1, -1, 42, 42, -1, 3] and np.isneginf(got[5, 42])
    assert lib.status() == G.ST_EDIT_NO_TOKEN


def test_counts_lengths_and_prompts(lib, cuda):
    """A repetition counts in the prompt too, frequency and presence behind it alone; tokens outside the vocabulary are passed over."""
    torch = cuda
    vocab = 64
    hist = np.array([[3, 3, 9, 3, -1, 9, 64, 10], [3, 3, 9, 3, -1, 9, 64, 10], [5] * 8, [5] * 8], np.int32)
    p = {"logits": np.ones((4, vocab), np.float32), "history": hist, "length": np.array([8, 5, 0, 8], np.int32), "prompt": np.array([3, 0, 0, 8], np.int32),
         "repetition": np.full(4, 2, np.float32), "frequency": np.full(4, 0.25, np.float32), "presence": np.full(4, 1, np.float32)}
    h, logits = handle(lib, torch, p)
    out = torch.empty_like(logits)
    h.apply(out, logits)
    want = np.ones((4, vocab))
    want[0, [3, 9, 10]] = 0.5 - 0.25 - 1
    want[1, 3], want[1, 9] = 0.5 - 0.75 - 1, 0.5 - 0.25 - 1
    want[3, 5] = 0.5
    assert np.array_equal(out.cpu().numpy().astype(np.float64), want)
    assert lib.status() == 0


def test_bounds_on_the_device(lib, cuda):
    """Lengths, prompts, counts and mask rows outside their bounds are clamped and reported; nothing outside is read."""
    torch = cuda
    p = make(torch, 4, 500, 20, 6, 1, np.float32, 2)
    p["prompt"][:] = 0
    good = dict(p, length=np.array([20, 0, 20, 20], np.int32), n_bias=np.array([6, 0, 6, 6], np.int32), mask_row=np.array([0, -1, -1, -1], np.int32))
    bad = dict(good, length=np.array([21, -5, 2**31 - 1, 20], np.int32), n_bias=np.array([7, -1, 2**30, 6], np.int32), mask_row=np.array([0, -1, -2, 2], np.int32))
    (h, x), (k, _) = handle(lib, torch, good), handle(lib, torch, bad)
    a, b = torch.empty_like(x), torch.empty_like(x)
    h.apply(a, x)
    assert lib.status() == 0
    check(good, a.cpu().numpy())
    k.apply(b, x)
    assert lib.status() == G.ST_EDIT_BAD_INPUT
    assert torch.equal(a, b)
    k, _ = handle(lib, torch, dict(good, prompt=np.array([21, 3, -1, 0], np.int32)))
    k.apply(b, x)
    assert lib.status() == G.ST_EDIT_BAD_INPUT


def test_one_list_and_one_mask_for_all_rows(lib, cuda):
    torch = cuda
    rows, vocab = 5, 777
    p = make(torch, rows, vocab, 0, 11, 2, np.float16, 1)
    del p["mask_row"], p["n_bias"]
    p["bias_token"][:], p["bias"][:] = p["bias_token"][:1], p["bias"][:1]
    t = {k: torch.from_numpy(v.view(np.int32) if v.dtype == np.uint32 else v).cuda() for k, v in p.items()}
    h = G.LogitsEdit(lib, torch, rows, vocab, bias_token=t["bias_token"][:1].expand(rows, -1), bias=t["bias"][:1].expand(rows, -1), mask=t["mask"])
    out = torch.empty_like(t["logits"])
    h.apply(out, t["logits"])
    check(p, out.cpu().numpy())
    assert lib.status() == 0


def test_captured_and_replayed_while_its_inputs_change(lib, cuda):
    torch = cuda
    rows, vocab = 8, 50257
    p = make(torch, rows, vocab, 64, 4, 5, np.float16, 8)
    q = make(torch, rows, vocab, 64, 4, 6, np.float16, 8)
    h, x = handle(lib, torch, p)
    names = ("repetition", "frequency", "presence", "history", "length", "prompt", "bias_token", "bias", "n_bias", "mask", "mask_row")
    out, nxt = torch.empty_like(x), torch.empty(rows, dtype=torch.int32, device="cuda")
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    h.apply(out, x, nxt, stream=st.cuda_stream)
    st.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=st):
        h.apply(out, x, nxt, stream=st.cuda_stream)
    for case in (q, p):
        x.copy_(torch.from_numpy(case["logits"]))
        for name, t in zip(names, h.tensors):
            v = case[name]
            t.copy_(torch.from_numpy(v.view(np.int32) if v.dtype == np.uint32 else v))
        g.replay()
        torch.cuda.synchronize()
        check(case, out.cpu().numpy())
        assert np.array_equal(nxt.cpu().numpy(), first_max(out.cpu().numpy()))
    lib.status()


def test_edited_logits_go_on_to_the_beams(lib, cuda):
    """The beams' selection of edited logits: banned tokens are never chosen, a forced one is."""
    torch = cuda
    B, W, vocab = 3, 4, 5000
    p = make(torch, B * W, vocab, 30, 0, 9, np.float32, 1)
    p["mask_row"][:] = 0
    h, x = handle(lib, torch, p)
    h.apply(x, x)
    token, parent = (torch.empty(B * W, dtype=torch.int32, device="cuda") for _ in range(2))
    score = torch.randn(B * W, device="cuda")
    new = torch.empty_like(score)
    lib.beam_select(token, parent, new, None, x, score, None, B, W, -1, lib.beam_work(torch, B, W, "cuda"))
    total = score.double()[:, None] + torch.log_softmax(x.double(), -1)
    want = torch.sort(total.view(B, -1), descending=True).values[:, :W].flatten()
    assert torch.allclose(new.double(), want, rtol=0, atol=2.0**-17)  # as the selection's own tests have it: sums of about 10, 1e-5
    t = token.cpu().numpy()
    assert ((p["mask"][0][t // 32] >> (t % 32).astype(np.uint32)) & 1 == 1).all()
    assert lib.status() == 0 and math.isfinite(float(new[0]))
