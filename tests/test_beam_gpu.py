"""Beam selection on the GPU against fp64 log-softmax and a sort, planted ties, masks, finished and dead beams.

A total is score + (x - lse) with three fp32 roundings and an lse whose sum of up to V exponentials is off by a
few ulp: at most 2^-21 (|score| + |x| + |lse|) + 2^-20. Where two fp64 totals are further apart than twice that, the order
must be the fp64 order; nearer ones may stand either way round (planted exact ties may not)."""
import numpy as np
import pytest

import gpt2_b200 as G

pytestmark = pytest.mark.gpu


def select(torch, lib, logits, score, done, B, W, eos, inplace=False, work=None):
    token, parent = (torch.full((B * W,), -7, dtype=torch.int32, device="cuda") for _ in range(2))
    new_score = score if inplace else torch.empty_like(score)
    new_done = done if inplace and done is not None else torch.empty_like(token)
    work = work if work is not None else lib.beam_work(torch, B, W, "cuda")
    lib.beam_select(token, parent, new_score, new_done, logits, score, done, B, W, eos, work)
    torch.cuda.synchronize()
    return token.cpu().numpy(), parent.cpu().numpy(), new_score.cpu().numpy().astype(np.float64), new_done.cpu().numpy()


def check(logits, score, done, B, W, eos, got):
    """Every output against the fp64 totals of the same inputs (host arrays)."""
    token, parent, new_score, new_done = got
    V = logits.shape[1]
    for b in range(B):
        x = logits[b * W:(b + 1) * W].astype(np.float64)
        x = np.where(x < np.inf, x, -np.inf)  # NaN and +inf count as masked
        s = score[b * W:(b + 1) * W].astype(np.float64)
        with np.errstate(invalid="ignore", divide="ignore"):
            top = x.max(1, keepdims=True)
            lse = top + np.log(np.exp(x - np.where(np.isfinite(top), top, 0)).sum(1, keepdims=True))
            total = s[:, None] + (x - lse)
        total[np.isnan(total)] = -np.inf
        tol = 2.0 ** -21 * (np.abs(np.where(np.isfinite(s), s, 0))[:, None] + np.abs(np.where(np.isfinite(x), x, 0)) + np.abs(np.where(np.isfinite(lse), lse, 0))) + 2.0 ** -20
        for w in range(W):
            if done is not None and done[b * W + w]:
                total[w] = -np.inf
                total[w, max(eos, 0)] = s[w]
                tol[w] = 0
        order = np.argsort(-total.reshape(-1), kind="stable")[:W]
        flat, ftol = total.reshape(-1), tol.reshape(-1)
        picked = set()
        for j in range(W):
            i = b * W + j
            best = order[j] if j < len(order) else -1
            if best < 0 or flat[best] == -np.inf:  # no candidate left
                assert (token[i], parent[i], new_score[i], new_done[i]) == (max(eos, 0), i, -np.inf, 1), (b, j)
                continue
            w, v = parent[i] - b * W, token[i]
            assert 0 <= w < W and 0 <= v < V, (b, j)
            c = w * V + v
            assert c not in picked
            picked.add(c)
            if c != best:
                assert abs(flat[c] - flat[best]) <= 2 * max(ftol[c], ftol[best]) and flat[c] != flat[best], (b, j, flat[c], flat[best])
            assert abs(new_score[i] - flat[c]) <= ftol[c], (b, j)
            was = bool(done[b * W + w]) if done is not None else False
            assert new_done[i] == int(was or v == eos)


@pytest.mark.parametrize("dtype", ["float16", "float32"])
@pytest.mark.parametrize("B,W,V", [(1, 1, 1), (1, 4, 50257), (3, 5, 50257), (2, 32, 1000), (7, 3, 37), (1, 8, 131), (70, 4, 4099), (2, 2, 200000), (1, 16, 65536)])
def test_selection_matches_fp64(cuda, lib, B, W, V, dtype):
    torch = cuda
    rng = np.random.default_rng(B * 1000 + W + V)
    x = (3.0 * rng.standard_normal((B * W, V))).astype(dtype)
    x[:, rng.integers(0, V, V // 20)] = -np.inf
    if V > 1:
        x[:, 0] = 1.0
    score = (-20 * rng.random(B * W)).astype(np.float32)
    done = (rng.random(B * W) < 0.2).astype(np.int32)
    eos = V - 1
    wide = torch.full((B * W, V + 5), float("nan"), dtype=getattr(torch, dtype), device="cuda")  # a stride that is odd at times
    wide[:, :V] = torch.from_numpy(x)
    d_score, d_done = torch.from_numpy(score).cuda(), torch.from_numpy(done).cuda()
    work = lib.beam_work(torch, B, W, "cuda")
    got = select(torch, lib, wide[:, :V], d_score, d_done, B, W, eos, work=work)
    check(x, score, done, B, W, eos, got)
    same = select(torch, lib, wide[:, :V].contiguous(), d_score, d_done, B, W, eos, inplace=True, work=work)
    for a, b in zip(got, same):
        assert np.array_equal(a, b)
    free = select(torch, lib, wide[:, :V], torch.from_numpy(score).cuda(), None, B, W, -1, work=work)
    check(x, score, None, B, W, -1, free)
    assert lib.status() == 0


def test_equal_totals_go_to_the_lower_beam_then_the_lower_token(cuda, lib):
    torch = cuda
    W, V = 4, 50257
    x = np.full((W, V), -2.0, np.float16)
    x[:, [40000, 17, 30001, 50256]] = 5.0  # the same row in every beam: every total exists four times
    score = np.full(W, -3.0, np.float32)
    token, parent, _, _ = select(torch, lib, torch.from_numpy(x).cuda(), torch.from_numpy(score).cuda(), None, 1, W, -1)
    assert token.tolist() == [17, 30001, 40000, 50256] and parent.tolist() == [0, 0, 0, 0]
    score = np.array([-4.0, -3.0, -np.inf, -3.0], np.float32)
    x[1, 17] = -2.0  # beam 1 now spreads over three tokens, its totals lie above those of beam 3
    token, parent, s, _ = select(torch, lib, torch.from_numpy(x).cuda(), torch.from_numpy(score).cuda(), None, 1, W, -1)
    assert token.tolist() == [30001, 40000, 50256, 17] and parent.tolist() == [1, 1, 1, 3]
    flat = np.zeros((W, V), np.float32)  # every candidate equal
    token, parent, _, _ = select(torch, lib, torch.from_numpy(flat).cuda(), torch.zeros(W, device="cuda"), None, 1, W, -1)
    assert token.tolist() == [0, 1, 2, 3] and parent.tolist() == [0] * 4


def test_masked_rows_dead_beams_and_finished_beams(cuda, lib):
    torch = cuda
    W, V, eos = 3, 101, 7
    x = np.full((3 * W, V), -np.inf, np.float32)
    x[0, 5] = 1.0                      # item 0: one candidate in all (beam 1 masked whole, beam 2 dead)
    x[2] = 0.5
    x[3:6] = np.random.default_rng(0).standard_normal((3, V))  # item 1: all finished
    x[6:9] = x[3:6]                    # item 2: the first step, one beam alive
    score = np.array([-1, -2, -np.inf, -9, -8, -7, 0, -np.inf, -np.inf], np.float32)
    done = np.array([0, 0, 0, 1, 1, 1, 0, 0, 0], np.int32)
    got = select(torch, lib, torch.from_numpy(x).cuda(), torch.from_numpy(score).cuda(), torch.from_numpy(done).cuda(), 3, W, eos)
    check(x, score, done, 3, W, eos, got)
    token, parent, s, d = got
    assert (token[0], parent[0]) == (5, 0) and s[0] == -1.0 and s[1] == s[2] == -np.inf
    assert token[3:6].tolist() == [eos] * 3 and parent[3:6].tolist() == [5, 4, 3] and s[3:6].tolist() == [-7, -8, -9]
    assert parent[6:9].tolist() == [6, 6, 6]
    assert lib.status() == 0


@pytest.mark.parametrize("dtype", ["float16", "float32"])
def test_non_finite_logits_are_never_chosen(cuda, lib, dtype):
    torch = cuda
    B, W, V = 2, 2, 9001
    rng = np.random.default_rng(3)
    x = rng.standard_normal((B * W, V)).astype(dtype)
    x[0, [3, 800, 9000]] = np.nan, np.inf, np.nan
    x[3] = np.nan
    score = np.zeros(B * W, np.float32)
    got = select(torch, lib, torch.from_numpy(x).cuda(), torch.from_numpy(score).cuda(), None, B, W, -1)
    assert lib.status() == G.ST_BEAM_LOGIT
    check(x, score, None, B, W, -1, got)
    big = (x * 0 + 65000 * np.sign(rng.standard_normal(x.shape))).astype(dtype)  # the type's ends: no overflow
    big[np.isnan(big)] = -65000
    got = select(torch, lib, torch.from_numpy(big).cuda(), torch.from_numpy(score).cuda(), None, B, W, -1)
    check(big, score, None, B, W, -1, got)
    assert lib.status() == 0
