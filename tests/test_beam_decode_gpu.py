"""Beam search end to end: gpt2_b200_beam_generate against a beam search driven from the host over the
fp16 batched decoder.

With the attention's output projection set to zero the cache has no influence on the logits, and both decoders run the
same kernels on the same rows: the host's selection in fp64 must then choose the same tokens wherever its totals are
further apart than fp32 rounding (2^-20 of their size), and scores agree to that. With the projection in place the 8-bit cache
shows: every hypothesis is decoded again, token by token, over the fp16 cache, and its score must agree within the
repository's parity bar for logits (REL_TOL of the largest logit, per step)."""
import ctypes

import numpy as np
import pytest

import gpt2_b200 as G
from conftest import REL_TOL

pytestmark = pytest.mark.gpu
V = G.VOCAB


def run(torch, lib, w, prompt, plen, W, n_steps, eos=-1, kind="int8", page=16, block=16, pages=None):
    B = prompt.shape[0]
    most = -(-(n_steps + 1) // page)
    cache = G.KV8Cache.create(lib, torch, B * W, most, pages or B * W * most, page=page, block=block, kind=kind)
    beam = G.BeamDecoder(lib, w, cache, B, W)
    out = torch.full((B * W, n_steps + 3), -9, dtype=torch.int32, device="cuda")
    score = torch.empty(B * W, dtype=torch.float32, device="cuda")
    d_prompt, d_plen = torch.from_numpy(prompt).cuda(), torch.from_numpy(plen).cuda()
    beam.generate(d_prompt, d_plen, n_steps, out, score, eos)
    torch.cuda.synchronize()
    first = out.cpu().numpy().copy(), score.cpu().numpy().copy()
    beam.generate(d_prompt, d_plen, n_steps, out, score, eos)  # again: the same bits
    torch.cuda.synchronize()
    assert np.array_equal(first[0], out.cpu().numpy()) and np.array_equal(first[1], score.cpu().numpy())
    assert (first[0][:, n_steps + 1:] == -9).all()
    # every page's reference count is the number of table entries that name it
    table, ref = cache.table.cpu(), cache.ref.cpu()
    assert torch.equal(torch.bincount(table[table >= 0].long(), minlength=ref.numel()).to(torch.int32), ref)
    assert bool((cache.length == n_steps).any())
    beam.close()
    return first[0][:, : n_steps + 1], first[1].astype(np.float64)


class Replay:
    """Rows of the fp16 batched decoder, stepped together: logits after each token."""

    def __init__(self, torch, lib, w, rows, max_t):
        self.torch = torch
        self.caches = torch.zeros(rows, 12, 2, 12, max_t, 64, dtype=torch.float16, device="cuda")
        self.batch = G.DecodeBatch(lib, w, self.caches)
        self.logits = torch.empty(rows, V, dtype=torch.float16, device="cuda")

    def step(self, tokens, t):
        torch = self.torch
        wide = torch.empty(self.logits.shape[0], 50264, dtype=torch.float16, device="cuda")
        self.batch.step(torch.tensor(tokens, dtype=torch.int32, device="cuda"), torch.full((len(tokens),), t, dtype=torch.int32, device="cuda"), wide)
        torch.cuda.synchronize()
        return wide[:, :V].double()


@pytest.fixture(scope="module")
def plain_weights(cuda):
    """GPT-2 weights whose attention writes nothing to the residual stream."""
    w = G.ModelWeights(cuda, "cuda", seed=11, hf_init=False, std=0.05)
    for L in range(G.N_LAYER):
        w.t[f"h{L}.attn_proj_w"].zero_()
    return w


@pytest.mark.parametrize("B,W,eos", [(2, 4, -1), (1, 1, -1), (3, 5, -1), (2, 3, 777)])
def test_beam_search_matches_a_host_search(cuda, lib, plain_weights, B, W, eos):
    torch = cuda
    rng = np.random.default_rng(B * 10 + W)
    n_steps = 24
    plen = np.array([1, 7, 19][:B], dtype=np.int32)
    prompt = rng.integers(0, V, (B, 20)).astype(np.int32)
    if eos >= 0:  # a token that the model likes: what a greedy continuation takes first
        probe, _ = run(torch, lib, plain_weights, prompt, plen, 1, n_steps)
        eos = int(probe[0, plen[0] + 2])
    tokens, score = run(torch, lib, plain_weights, prompt, plen, W, n_steps, eos)
    dec = Replay(torch, lib, plain_weights, B * W, n_steps)  # logits depend on the row's token and position alone
    hyps = [[([int(prompt[b, 0])], 0.0, False)] for b in range(B)]
    near = False
    for t in range(n_steps):
        last = [h[w][0][-1] if w < len(h) else 0 for h in hyps for w in range(W)]
        logp = torch.log_softmax(dec.step(last, t), -1).cpu().numpy()
        for b in range(B):
            if t + 1 < plen[b]:
                hyps[b] = [([int(x) for x in prompt[b, : t + 2]], 0.0, False)]
                continue
            total = np.full((len(hyps[b]), V), -np.inf)
            for w, (_, s, d) in enumerate(hyps[b]):
                total[w] = -np.inf if d else s + logp[b * W + w]
                if d:
                    total[w, eos] = s
            order = np.argsort(-total.reshape(-1), kind="stable")[: W + 1]
            vals = total.reshape(-1)[order]
            # within a beam the order is that of the fp16 logits, equal ones by token: only beams can be too near
            near |= bool(((vals[:-1] - vals[1:] < 2.0 ** -20 * (np.abs(vals[:-1]) + 40)) & (order[:-1] // V != order[1:] // V)).any())
            hyps[b] = [(hyps[b][c // V][0] + [int(c % V)], float(total.reshape(-1)[c]), hyps[b][c // V][2] or int(c % V) == eos) for c in order[:W]]
    assert not near, "the inputs have a near tie: choose another seed"
    for b in range(B):
        for w in range(W):
            assert tokens[b * W + w].tolist() == hyps[b][w][0], (b, w)
            assert abs(score[b * W + w] - hyps[b][w][1]) <= n_steps * 2.0 ** -19 * (abs(hyps[b][w][1]) + 40)
    if eos >= 0:
        assert any(h[2] for hs in hyps for h in hs), "no beam met eos: the case does not test it"
    assert lib.status() == 0


@pytest.mark.parametrize("kind,page,block", [("int8", 16, 16), ("e4m3", 32, 16)])
def test_scores_agree_with_the_fp16_cache(cuda, lib, kind, page, block):
    torch = cuda
    w = G.ModelWeights(torch, "cuda", seed=5)
    rng = np.random.default_rng(8)
    B, W, n_steps = 3, 4, 60
    plen = np.array([40, 33, 5], dtype=np.int32)
    prompt = rng.integers(0, V, (B, 40)).astype(np.int32)
    tokens, score = run(torch, lib, w, prompt, plen, W, n_steps, kind=kind, page=page, block=block)
    for b in range(B):
        assert (np.diff(score[b * W:(b + 1) * W]) <= 0).all()  # best first
        assert (tokens[b * W:(b + 1) * W, : plen[b]] == prompt[b, : plen[b]]).all()
        assert len({tuple(t) for t in tokens[b * W:(b + 1) * W]}) == W  # different hypotheses
    dec = Replay(torch, lib, w, B * W, n_steps)
    again, allowed = np.zeros(B * W), np.zeros(B * W)
    for t in range(n_steps):
        x = dec.step(tokens[:, t].tolist(), t)
        logp = torch.log_softmax(x, -1).cpu().numpy()
        big = float(x.abs().max())
        for r in range(B * W):
            if t + 1 >= plen[r // W]:
                again[r] += logp[r, tokens[r, t + 1]]
                allowed[r] += 2 * REL_TOL * big
    assert (np.abs(again - score) <= allowed).all(), (again - score, allowed)
    assert lib.status() == 0


def test_refusals_and_a_pool_that_runs_out(cuda, lib):
    torch = cuda
    w = G.ModelWeights(torch, "cuda", seed=5)
    cache = G.KV8Cache.create(lib, torch, 4, 2, 8)
    h = ctypes.c_void_p()
    create = lib.gpt2_b200_beam_create
    for B, W in ((1, 3), (0, 4), (4, 0), (2, 3)):
        assert create(ctypes.byref(h), ctypes.byref(w.struct), cache.ref_c, B, W) == G.EINVAL and not h.value
    assert create(None, ctypes.byref(w.struct), cache.ref_c, 1, 4) == G.EINVAL
    assert create(ctypes.byref(h), None, cache.ref_c, 1, 4) == G.EINVAL
    assert create(ctypes.byref(h), ctypes.byref(w.struct), None, 1, 4) == G.EINVAL
    other = G.KV8Cache.create(lib, torch, 4, 2, 8, heads=6)
    assert create(ctypes.byref(h), ctypes.byref(w.struct), other.ref_c, 1, 4) == G.EINVAL
    beam = G.BeamDecoder(lib, w, cache, 1, 4)
    prompt = torch.zeros(1, 4, dtype=torch.int32, device="cuda")
    plen = torch.ones(1, dtype=torch.int32, device="cuda")
    out = torch.zeros(4, 40, dtype=torch.int32, device="cuda")
    for bad in (dict(n_steps=0), dict(n_steps=33), dict(n_steps=20, out=torch.zeros(4, 20, dtype=torch.int32, device="cuda")), dict(n_steps=4, eos=V), dict(n_steps=4, eos=-2)):
        with pytest.raises(RuntimeError):
            beam.generate(**{"prompt": prompt, "prompt_len": plen, "out": out, **bad})
    few = G.KV8Cache.create(lib, torch, 4, 2, 5)  # 5 pages for 4 beams of two pages
    short = G.BeamDecoder(lib, w, few, 1, 4)
    short.generate(prompt, plen, 30, out)
    torch.cuda.synchronize()
    assert lib.status() & G.ST_KV8_NO_PAGE
    beam.generate(prompt, plen, 30, out)  # and the device is fine
    torch.cuda.synchronize()
    assert lib.status() == 0
    beam.close()
    beam.close()
