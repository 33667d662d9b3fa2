"""Prefill, decode and the cache writers on the GPU against the double-precision oracle alone, for machines on which the
reference's own code has not been built. Tolerances: conftest.ABS_TOL and REL_TOL; the writers move bits."""
import ctypes

import numpy as np
import pytest

import gpt2_b200 as G
import oracle as O
from conftest import assert_close

pytestmark = pytest.mark.gpu
L_ = 12


def host(t):
    return t.float().cpu().numpy()


def u16(t):
    return t.cpu().numpy().view(np.uint16)


@pytest.mark.parametrize("T", [1, 2, 31, 32, 33, 127, 128, 129, 161, 255, 256, 257, 512, 1000, 1024])
def test_prefill(cuda, lib, oracle, T):
    x = O.seeded_qkv(2000 + T, T)
    qkv = cuda.from_numpy(x.astype(np.float16)).cuda()
    att = cuda.full((T, O.E), 12344.0, dtype=cuda.float16, device="cuda")
    lib.prefill(att, qkv, T)
    assert_close(host(att), oracle.prefill(x), f"T={T}")
    lib.gpt2_attention_b200(att.data_ptr(), qkv.data_ptr(), T, O.E, O.H, O.D)
    assert lib.gpt2_b200_last_error() == 0
    assert_close(host(att), oracle.prefill(x), f"T={T}, void entry point")
    assert lib.status() == 0


@pytest.fixture(scope="module")
def cache(cuda):
    rng = np.random.default_rng(123)
    arena = rng.standard_normal((L_, 2, O.H, 1024, O.D), dtype=np.float32).astype(np.float16)
    q = rng.standard_normal((L_, O.QKV), dtype=np.float32).astype(np.float16)
    d_arena = cuda.from_numpy(arena).cuda()
    return arena.astype(np.float32), q.astype(np.float32), d_arena, cuda.from_numpy(q).cuda(), G.cache_view(d_arena.data_ptr(), L_, 1024)


@pytest.mark.parametrize("length", [1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 500, 1023, 1024])
def test_decode_one_layer(cuda, lib, oracle, cache, length):
    arena, q, _, d_q, kv = cache
    for L in (0, 7, 11):
        att = cuda.empty((O.E,), dtype=cuda.float16, device="cuda")
        lib.gpt2_attn_decode_b200(att.data_ptr(), d_q[L].data_ptr(), ctypes.byref(kv), L, length)
        assert lib.gpt2_b200_last_error() == 0
        assert_close(host(att), oracle.decode(q[L, :O.E], arena[L, 0], arena[L, 1], length), f"len={length} L={L}")
    assert lib.status() == 0


def test_scatter_append_and_prefill_that_fills_the_cache(cuda, lib, oracle):
    torch = cuda
    T, maxt = 300, 320
    x = O.seeded_qkv(5, T).astype(np.float16)
    d_qkv = torch.from_numpy(x).cuda()
    mine = torch.zeros((L_, 2, O.H, maxt, O.D), dtype=torch.float16, device="cuda")
    kv = G.cache_view(mine.data_ptr(), L_, maxt)
    att = torch.empty((T, O.E), dtype=torch.float16, device="cuda")
    lib.gpt2_kv_scatter_prefill_b200(ctypes.byref(kv), 4, d_qkv.data_ptr(), T)
    assert lib.gpt2_b200_last_error() == 0
    assert lib.gpt2_attention_kv_b200_stream(att.data_ptr(), d_qkv.data_ptr(), ctypes.byref(kv), 11, T, O.E, O.H, O.D, None) == 0
    for L in (4, 11):
        lib.gpt2_kv_append_one_b200(ctypes.byref(kv), L, d_qkv[40].data_ptr(), T + 3)
        assert lib.gpt2_b200_last_error() == 0
    k, v = (np.zeros((O.H, maxt, O.D), np.uint16) for _ in range(2))
    oracle.kv_scatter(k, v, x.view(np.uint16))
    oracle.kv_scatter(k, v, x[40:41].view(np.uint16), pos0=T + 3)
    got = u16(mine)
    for L in range(L_):
        assert np.array_equal(got[L, 0], k if L in (4, 11) else 0 * k) and np.array_equal(got[L, 1], v if L in (4, 11) else 0 * v), L
    assert_close(host(att), oracle.prefill(x.astype(np.float32)), "prefill that fills the cache")


@pytest.mark.parametrize("use_dev", [False, True])
def test_decode_attn_step(cuda, lib, oracle, use_dev):
    """Append, then attend, for all 12 layers."""
    torch = cuda
    maxt, pos = 256, 200
    rng = np.random.default_rng(8)
    base = rng.standard_normal((L_, 2, O.H, maxt, O.D), dtype=np.float32).astype(np.float16)
    qkv = rng.standard_normal((L_, O.QKV), dtype=np.float32).astype(np.float16)
    mine, d_qkv = torch.from_numpy(base).cuda(), torch.from_numpy(qkv).cuda()
    kv = G.cache_view(mine.data_ptr(), L_, maxt)
    att = torch.empty((L_, O.E), dtype=torch.float16, device="cuda")
    d_pos = torch.tensor([pos], dtype=torch.int32, device="cuda")
    lib.check(lib.gpt2_b200_reserve(L_, O.H, maxt), "reserve")
    lib.check(lib.gpt2_b200_decode_attn_step(att.data_ptr(), O.E, d_qkv.data_ptr(), O.QKV, ctypes.byref(kv), d_pos.data_ptr() if use_dev else None, pos, None), "step")
    got, after = host(att), u16(mine)
    for L in range(L_):
        k, v = base[L, 0].view(np.uint16).copy(), base[L, 1].view(np.uint16).copy()
        oracle.kv_scatter(k, v, qkv[L: L + 1].view(np.uint16), pos0=pos)
        assert np.array_equal(after[L, 0], k) and np.array_equal(after[L, 1], v), f"cache of layer {L}"
        want = oracle.decode(qkv[L, :O.E].astype(np.float32), k.view(np.float16).astype(np.float32), v.view(np.float16).astype(np.float32), pos + 1)
        assert_close(got[L], want, f"layer {L}")
    assert lib.status() == 0


def plain_forward(torch, w, ids):
    """GPT-2's logits after every token of ids [B][T], in fp32 from the same weights."""
    t = {k: v.float() for k, v in w.t.items()}

    def norm(x, g, b):
        return (x - x.mean(-1, keepdim=True)) / torch.sqrt(x.var(-1, unbiased=False, keepdim=True) + 1e-5) * t[g] + t[b]

    B, T = ids.shape
    x = t["wte"][ids] + t["wpe"][:T]
    ahead = torch.ones(T, T, dtype=torch.bool, device=x.device).triu(1)
    for L in range(L_):
        p = f"h{L}."
        q, k, v = (norm(x, p + "ln1_g", p + "ln1_b") @ t[p + "qkv_w"].T + t[p + "qkv_b"]).view(B, T, 3, O.H, O.D).permute(2, 0, 3, 1, 4)
        a = torch.softmax((q @ k.transpose(-1, -2) / O.D ** 0.5).masked_fill(ahead, -np.inf), -1) @ v
        x = x + a.transpose(1, 2).reshape(B, T, -1) @ t[p + "attn_proj_w"].T + t[p + "attn_proj_b"]
        h = norm(x, p + "ln2_g", p + "ln2_b") @ t[p + "fc_w"].T + t[p + "fc_b"]
        h = 0.5 * h * (1 + torch.tanh(0.7978845608028654 * (h + 0.044715 * h ** 3)))
        x = x + h @ t[p + "proj_w"].T + t[p + "proj_b"]
    return norm(x, "lnf_g", "lnf_b") @ t["wte"].T


@pytest.mark.parametrize("B", [1, 5, 40])
def test_batched_decode_step(cuda, lib, B):
    """Teacher-forced steps against a plain fp32 forward, within the bound for fp16 steps against an fp32 forward (tests/test_model_gpu.py: 5e-2)."""
    torch = cuda
    T = 9
    w = G.ModelWeights(torch, "cuda", seed=7, hf_init=False)
    ids = torch.from_numpy(np.random.default_rng(B).integers(0, G.VOCAB, (B, T))).cuda()
    want = plain_forward(torch, w, ids)
    caches = torch.zeros(B, L_, 2, O.H, 16, O.D, dtype=torch.float16, device="cuda")
    batch = G.DecodeBatch(lib, w, caches)
    logits = torch.empty(B, 50264, dtype=torch.float16, device="cuda")
    for t in range(T):
        batch.step(ids[:, t].int(), torch.full((B,), t, dtype=torch.int32, device="cuda"), logits)
        torch.cuda.synchronize()
        assert float((logits[:, :G.VOCAB].float() - want[:, t]).abs().max()) <= 5e-2, f"position {t}"
    assert lib.status() == 0
