"""The decode step over 4-bit weights and generation with edited logits.

A step is compared with the fp16 step over the values that the codes stand for: the sums are the same, the fp16 step rounds once more before
GELU and the residual, half a step 2^-11 of numbers of order 1, which 24 times through layers and LayerNorms stays below the parity bar that
the fp16 step itself is held to against the reference (2e-3, 1e-2 of the largest). Tokens of a generation are those of the same calls made one
by one, exactly.
"""
import numpy as np
import pytest

import gpt2_b200 as G
from conftest import assert_close

pytestmark = pytest.mark.gpu
V, E = G.VOCAB, G.N_EMBD


@pytest.fixture(scope="module", params=[False, True], ids=["symmetric", "least"])
def models(request, cuda, lib):
    """fp16 weights, them in 4 bits, and an fp16 copy that holds what the codes stand for."""
    torch = cuda
    w = G.ModelWeights(torch, "cuda", seed=11, hf_init=False)
    q = G.W4ModelWeights(lib, torch, w, group=128 if request.param else 64, least=request.param)
    plain = G.ModelWeights(torch, "cuda", seed=11, hf_init=False)
    for L, layer in enumerate(q.layers):
        for n, t in q.NAMES:
            layer[n].dequantize(plain.t[f"h{L}.{t}"])
    head = plain.t["wte"].clone()
    q.head.dequantize(head)
    return w, q, plain, head


def caches(torch, B, max_t=32):
    return torch.zeros(B, 12, 2, 12, max_t, 64, dtype=torch.float16, device="cuda")


@pytest.mark.parametrize("B", [1, 5, 8, 9, 17, 64, 130])
def test_steps_match_the_fp16_step_over_the_same_values(cuda, lib, models, B):
    torch = cuda
    w, q, plain, head = models
    rng = np.random.default_rng(B)
    one, two = caches(torch, B), caches(torch, B)
    a, b = G.DecodeBatch(lib, w, one, q), G.DecodeBatch(lib, plain, two)
    la, lb = (torch.empty(B, V + 7, dtype=torch.float16, device="cuda") for _ in range(2))
    na = torch.empty(B, dtype=torch.int32, device="cuda")
    for pos in range(3):
        tok = torch.from_numpy(rng.integers(0, V, B).astype(np.int32)).cuda()
        at = torch.full((B,), pos, dtype=torch.int32, device="cuda")
        a.step(tok, at, la, na)
        b.step(tok, at, lb)
        torch.cuda.synchronize()
        got = la[:, :V].cpu().numpy()
        # (the other step's head has the embedding's own values: logits are compared below, without a 4-bit head)
        assert np.array_equal(na.cpu().numpy(), np.argmax(got.astype(np.float32), 1))
    k, v = one.cpu().numpy(), two.cpu().numpy()
    assert_close(k[:, :, :, :, :3], v[:, :, :, :, :3], f"K/V of {B} sequences", 8e-3, 1e-2)
    assert (k[:, :, :, :, 3:] == 0).all()
    a.close(), b.close()
    assert lib.status() == 0


@pytest.mark.parametrize("B", [1, 6, 16, 70])
def test_logits_with_an_fp16_head(cuda, lib, models, B):
    """Without a 4-bit head the logits are the fp16 step's over the same values, within the parity bar."""
    torch = cuda
    w, q, plain, _ = models
    bare = G.W4ModelWeights.__new__(G.W4ModelWeights)  # the same layers, no head
    bare.layers, bare.head, bare.struct = q.layers, None, G.GPT2W4Weights()
    for L in range(12):
        for n, _ in q.NAMES:
            getattr(bare.struct, n)[L] = q.layers[L][n].c
    a, b = G.DecodeBatch(lib, w, caches(torch, B), bare), G.DecodeBatch(lib, plain, caches(torch, B))
    la, lb = (torch.empty(B, V, dtype=torch.float16, device="cuda") for _ in range(2))
    rng = np.random.default_rng(B)
    for pos in range(4):
        tok = torch.from_numpy(rng.integers(0, V, B).astype(np.int32)).cuda()
        at = torch.full((B,), pos, dtype=torch.int32, device="cuda")
        a.step(tok, at, la)
        b.step(tok, at, lb)
        torch.cuda.synchronize()
        assert_close(la.cpu().numpy(), lb.cpu().numpy(), f"logits of {B} sequences at {pos}", 8e-3, 1e-2)
    a.close(), b.close()
    assert lib.status() == 0


def test_the_4_bit_head_is_its_product(cuda, lib, models):
    """The head's logits are the product of the last LayerNorm's rows, which a head of one-hot rows reads out."""
    torch = cuda
    w, q, _, head = models
    B = 12
    bt = G.DecodeBatch(lib, w, caches(torch, B), q)
    tok = torch.arange(B, dtype=torch.int32, device="cuda") * 97
    at = torch.zeros(B, dtype=torch.int32, device="cuda")
    logits = torch.empty(B, V, dtype=torch.float16, device="cuda")
    bt.step(tok, at, logits)
    eye = torch.zeros(V, E, dtype=torch.float16, device="cuda")
    eye[:E] = torch.eye(E, dtype=torch.float16, device="cuda")
    reader = G.W4ModelWeights.__new__(G.W4ModelWeights)
    reader.layers, reader.head, reader.struct = q.layers, G.W4Weight.pack(lib, torch, eye, 32, True), G.GPT2W4Weights()
    for L in range(12):
        for n, _ in q.NAMES:
            getattr(reader.struct, n)[L] = q.layers[L][n].c
    reader.struct.head = reader.head.c
    back = torch.empty_like(eye)
    reader.head.dequantize(back)
    rd = G.DecodeBatch(lib, w, caches(torch, B), reader)
    rows = torch.empty(B, V, dtype=torch.float16, device="cuda")
    rd.step(tok, at, rows)
    torch.cuda.synchronize()
    # scale rd(1/15) stands for 15 rd(1/15) in the place of a one: rows = that times the LayerNorm's row, rounded
    one = float(back[0, 0])
    x = rows[:, :E].double() / one
    want, size = x @ head.double().T, x.abs() @ head.double().abs().T
    # x is off by half a step of the read-out's rounding, 2^-11 and 2^-25, times the weights; the logits by half a step
    tol = 2.0**-11 * (1 + 2.0**-8) * size + 2.0**-24 * head.double().abs().sum(1) + 2.0**-11 * want.abs() + 2.0**-25
    assert bool(((logits.double() - want).abs() <= tol).all())
    bt.close(), rd.close()
    assert lib.status() == 0


def edit_of(torch, lib, B, seed, **more):
    rng = np.random.default_rng(seed)
    t = {n: torch.from_numpy((rng.random(B) * 0.8 + (0.6 if n == "repetition" else 0.0)).astype(np.float32)).cuda() for n in ("repetition", "frequency", "presence")}
    t["bias_token"] = torch.from_numpy(rng.integers(0, V, (B, 5)).astype(np.int32)).cuda()
    t["bias"] = torch.from_numpy((2 * rng.standard_normal((B, 5))).astype(np.float32)).cuda()
    t["mask"] = torch.from_numpy(rng.integers(-2**31, 2**31, (3, (V + 31) // 32)).astype(np.int32)).cuda()
    t["mask_row"] = torch.from_numpy((np.arange(B) % 4 - 1).astype(np.int32)).cuda()
    return {**t, **more}


@pytest.mark.parametrize("four_bits", [False, True])
@pytest.mark.parametrize("B", [1, 7, 20])
def test_generation_with_edited_logits_is_the_calls_one_by_one(cuda, lib, models, B, four_bits):
    torch = cuda
    w, q, _, _ = models
    steps, plens = 14, [1 + i % 6 for i in range(B)]
    rng = np.random.default_rng(B)
    prompt = torch.from_numpy(rng.integers(0, V, (B, 6)).astype(np.int32)).cuda()
    plen = torch.tensor(plens, dtype=torch.int32, device="cuda")
    t = edit_of(torch, lib, B, B)
    out = torch.full((B, steps + 3), -9, dtype=torch.int32, device="cuda")
    bt = G.DecodeBatch(lib, w, caches(torch, B), q if four_bits else None)
    bt.generate(prompt, plen, steps, out, edit=G.LogitsEdit(lib, torch, B, V, **t))
    torch.cuda.synchronize()
    got = out.clone()
    again = G.DecodeBatch(lib, w, caches(torch, B), q if four_bits else None)
    held = torch.zeros(B, steps + 1, dtype=torch.int32, device="cuda")
    held[:, 0] = prompt[:, 0]
    length = torch.empty(B, dtype=torch.int32, device="cuda")
    start = torch.empty(B, dtype=torch.int32, device="cuda")
    edit = G.LogitsEdit(lib, torch, B, V, history=held, length=length, prompt=start, **t)
    logits, nxt = torch.empty(B, V, dtype=torch.float16, device="cuda"), torch.empty(B, dtype=torch.int32, device="cuda")
    for pos in range(steps):
        length.fill_(pos + 1)
        start.copy_(plen.clamp(max=pos + 1))
        again.step(held[:, pos].contiguous(), torch.full((B,), pos, dtype=torch.int32, device="cuda"), logits)
        edit.apply(logits, logits, nxt)
        for b in range(B):
            held[b, pos + 1] = prompt[b, pos + 1] if pos + 1 < plens[b] else nxt[b]
    assert torch.equal(got[:, :steps + 1], held)
    assert bool((got[:, steps + 1:] == -9).all())
    bt.close(), again.close()
    assert lib.status() == 0


def test_generations_of_one_batch_follow_their_buffers(cuda, lib, models):
    """Greedy into one buffer, edited into another, greedy into that one: each writes where it was told to."""
    torch = cuda
    w, q, _, _ = models
    B, steps = 3, 9
    prompt = torch.randint(0, V, (B, 4), dtype=torch.int32, device="cuda")
    plen = torch.tensor([4, 2, 1], dtype=torch.int32, device="cuda")
    bt = G.DecodeBatch(lib, w, caches(torch, B), q)
    a, b, c = (torch.full((B, steps + 1), -9, dtype=torch.int32, device="cuda") for _ in range(3))
    bt.generate(prompt, plen, steps, a)
    t = edit_of(torch, lib, B, 5)
    edit = G.LogitsEdit(lib, torch, B, V, **t)
    bt.generate(prompt, plen, steps, b, edit=edit)
    torch.cuda.synchronize()
    first, edited = a.clone(), b.clone()
    a.fill_(-9)
    bt.generate(prompt, plen, steps, b)  # greedy into the edited one's buffer
    torch.cuda.synchronize()
    assert torch.equal(b, first) and bool((a == -9).all())
    bt.generate(prompt, plen, steps, c, edit=edit)
    torch.cuda.synchronize()
    assert torch.equal(c, edited) and not torch.equal(edited, first)
    # the edit's tensors may change between generations, its pointers too
    t["mask"].fill_(-1)
    none = G.LogitsEdit(lib, torch, B, V, mask=t["mask"], mask_row=t["mask_row"])
    bt.generate(prompt, plen, steps, c, edit=none)
    torch.cuda.synchronize()
    assert torch.equal(c, first)
    bt.close()
    assert lib.status() == 0


def test_a_sequence_with_nothing_to_choose(cuda, lib, models):
    torch = cuda
    w, q, _, _ = models
    prompt, plen = torch.tensor([[5, 6], [7, 8]], dtype=torch.int32, device="cuda"), torch.tensor([2, 2], dtype=torch.int32, device="cuda")
    mask = torch.zeros(2, (V + 31) // 32, dtype=torch.int32, device="cuda")
    mask[1, 3] = 1 << 4  # token 100 alone
    bt = G.DecodeBatch(lib, w, caches(torch, 2), q)
    out = torch.empty(2, 6, dtype=torch.int32, device="cuda")
    bt.generate(prompt, plen, 5, out, edit=G.LogitsEdit(lib, torch, 2, V, mask=mask))
    torch.cuda.synchronize()
    assert out.tolist() == [[5, 6, -1, -1, -1, -1], [7, 8, 100, 100, 100, 100]]
    assert lib.status() == G.ST_EDIT_NO_TOKEN | G.ST_MODEL_BAD_TOKEN
    bt.close()


def test_greedy_generation_over_4_bits_is_its_steps(cuda, lib, models):
    torch = cuda
    w, q, _, _ = models
    B, steps = 10, 12
    prompt = torch.randint(0, V, (B, 3), dtype=torch.int32, device="cuda")
    plen = torch.tensor([1 + b % 3 for b in range(B)], dtype=torch.int32, device="cuda")
    a, b = G.DecodeBatch(lib, w, caches(torch, B), q), G.DecodeBatch(lib, w, caches(torch, B), q)
    out = torch.empty(B, steps + 1, dtype=torch.int32, device="cuda")
    a.generate(prompt, plen, steps, out)
    tok, nxt = prompt[:, 0].contiguous(), torch.empty(B, dtype=torch.int32, device="cuda")
    want = [tok.clone()]
    for pos in range(steps):
        b.step(tok, torch.full((B,), pos, dtype=torch.int32, device="cuda"), None, nxt)
        tok = torch.where(plen > pos + 1, prompt[:, min(pos + 1, 2)], nxt).contiguous()
        want.append(tok.clone())
    torch.cuda.synchronize()
    assert torch.equal(out, torch.stack(want, 1))
    a.close(), b.close()
    assert lib.status() == 0
