"""4-bit weights and edits at the ends of what their documentation allows: first calls of a process inside a capture, sizes whose offsets pass
32 bits, the longest k of one row, the largest vocabulary, tables that all rows share, calls at once."""
import os
import subprocess
import sys

import numpy as np
import pytest

import gpt2_b200 as G
from test_logits_edit_gpu import check, first_max, handle, make
from test_w4_gpu import close

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

FIRST = """
import sys
sys.path.insert(0, "bare-metal-gpt2_b200")
import torch, gpt2_b200 as G
lib, what = G.load(), sys.argv[1]
half = dict(device="cuda", dtype=torch.float16)
w, x, out = torch.randn(512, 2048, **half), torch.randn(64, 2048, **half), torch.zeros(64, 512, **half)
q = G.W4Weight.create(lib, torch, 512, 2048, 64, True)
back, logits, nxt = torch.zeros_like(w), torch.randn(3, 9000, **half), torch.zeros(3, dtype=torch.int32, device="cuda")
edit = G.LogitsEdit(lib, torch, 3, 9000, bias_token=torch.full((3, 1), 77, dtype=torch.int32, device="cuda"), bias=torch.full((3, 1), 50.0, device="cuda"))
st = torch.cuda.Stream()
calls = {"pack": lambda: q.quantize(w, st.cuda_stream), "back": lambda: q.dequantize(back, st.cuda_stream), "rows": lambda: q.linear(out[:3], x[:3], stream=st.cuda_stream),
         "many": lambda: q.linear(out, x, stream=st.cuda_stream), "edit": lambda: edit.apply(logits, logits, nxt, stream=st.cuda_stream)}
order = [what] + [c for c in calls if c != what]
torch.cuda.synchronize()
g = {}
for c in order:
    g[c] = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g[c], stream=st):
        calls[c]()
for c in ("pack", "back", "rows"):
    g[c].replay()
torch.cuda.synchronize()
few = out[:3].clone()
g["many"].replay(), g["edit"].replay()
torch.cuda.synchronize()
want = x.double() @ back.double().t()
assert float((few.double() - want[:3]).abs().max()) < 0.25 and float((out.double() - want).abs().max()) < 0.25
assert float((back - w).abs().max()) < 0.5 and nxt.tolist() == [77] * 3 and lib.status() == 0
print("fine")
"""


@pytest.mark.parametrize("what", ["pack", "back", "rows", "many", "edit"])
def test_the_first_call_of_a_process_is_captured(cuda, what):
    # outputs of up to about 200: an fp16 step is 0.125, and rounding is off by half of it
    r = subprocess.run([sys.executable, "-c", FIRST, what], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip() == "fine", r.stdout + r.stderr


def test_weights_beyond_32_bits(lib, cuda):
    """4.6e9 weights: elements, bytes of W and of its codes pass 2^31 and 2^32."""
    torch = cuda
    N, K, group, last = 140001, 32768, 32, 65
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    w = torch.empty(N, K, dtype=torch.float16, device="cuda").normal_(generator=g)
    q = G.W4Weight.pack(lib, torch, w, group, True)
    end = G.W4Weight.pack(lib, torch, w[-last:], group, True)
    assert torch.equal(q.codes[-last:], end.codes) and torch.equal(q.scale[:, -last:], end.scale) and torch.equal(q.least[:, -last:], end.least)
    q.dequantize(w)
    values = torch.empty(last, K, dtype=torch.float16, device="cuda")
    end.dequantize(values)
    assert torch.equal(w[-last:], values)
    for B in (1, 20):  # both kernels
        x = torch.randn(B, K, generator=g, device="cuda", dtype=torch.float16)
        out = torch.full((B, N), float("nan"), dtype=torch.float16, device="cuda")
        q.linear(out, x)
        for part in (slice(0, 300), slice(65000, 65300), slice(N - last, N)):
            v, x64 = w[part].cpu().numpy().astype(np.float64), x.cpu().numpy().astype(np.float64)
            close(out[:, part].cpu().numpy(), x64 @ v.T, np.abs(x64) @ np.abs(v).T, K)
        assert not bool(out.isnan().any())
    assert lib.status() == 0


@pytest.mark.parametrize("B,K", [(1, 32800), (1, 131072), (16, 65536), (200, 40960)])
def test_a_long_k(lib, cuda, B, K):
    torch = cuda
    N, group = 300, 32
    g = torch.Generator(device="cuda")
    g.manual_seed(K)
    q = G.W4Weight.pack(lib, torch, torch.randn(N, K, generator=g, device="cuda", dtype=torch.float16), group)
    v = torch.empty(N, K, dtype=torch.float16, device="cuda")
    q.dequantize(v)
    x = torch.randn(B, K, generator=g, device="cuda", dtype=torch.float16)
    out = torch.empty(B, N, dtype=torch.float16, device="cuda")
    q.linear(out, x)
    want, size = x.double() @ v.double().t(), x.double().abs() @ v.double().abs().t()
    close(out.cpu().numpy(), want.cpu().numpy(), size.cpu().numpy(), K)
    assert lib.status() == 0


def test_logits_beyond_32_bits(lib, cuda):
    """4.6 GB of fp32 logits: the last rows as an edit of those alone gives them."""
    torch = cuda
    rows, vocab, last = 1100, 2**20 + 3, 3
    g = torch.Generator(device="cuda")
    g.manual_seed(2)
    x = torch.empty(rows, vocab, device="cuda").normal_(generator=g)
    hist = torch.randint(0, vocab, (rows, 50), generator=g, device="cuda", dtype=torch.int32)
    mask = torch.randint(-2**31, 2**31, (rows, (vocab + 31) // 32), generator=g, device="cuda").to(torch.int32)
    rep = torch.rand(rows, generator=g, device="cuda") + 0.5
    want, out, nxt = x[-last:].clone(), torch.empty_like(x), torch.empty(rows, dtype=torch.int32, device="cuda")
    G.LogitsEdit(lib, torch, last, vocab, history=hist[-last:], mask=mask[-last:], repetition=rep[-last:]).apply(want, want)
    G.LogitsEdit(lib, torch, rows, vocab, history=hist, mask=mask, repetition=rep).apply(out, x, nxt)
    assert torch.equal(out[-last:], want)
    assert torch.equal(nxt[-last:].long(), want.argmax(1)) and torch.equal(nxt[:4].long(), out[:4].argmax(1))
    assert lib.status() == 0


@pytest.mark.parametrize("offset", [0, 3])
def test_the_largest_vocabulary(lib, cuda, offset):
    torch = cuda
    vocab = 2**30
    x = torch.full((vocab + 8,), -1.0, dtype=torch.float16, device="cuda")
    row = x[offset:offset + vocab].view(1, vocab)
    tokens = [0, 5, 2**29 + 1, vocab - 2, vocab - 1]
    edit = G.LogitsEdit(lib, torch, 1, vocab, repetition=torch.full((1,), 2.0, device="cuda"), history=torch.tensor([tokens], dtype=torch.int32, device="cuda"),
                        bias_token=torch.tensor([[vocab - 2, 7]], dtype=torch.int32, device="cuda"), bias=torch.tensor([[4.0, 2.0]], device="cuda"))
    nxt = torch.empty(1, dtype=torch.int32, device="cuda")
    edit.apply(row, row, nxt)
    want = {0: -2.0, 5: -2.0, 2**29 + 1: -2.0, vocab - 2: 2.0, vocab - 1: -2.0, 7: 1.0}
    assert {t: float(row[0, t]) for t in want} == want
    for t in want:
        row[0, t] = -1.0
    assert bool((x == -1).all()) and nxt.item() == vocab - 2
    assert lib.status() == 0


def test_one_history_for_all_rows(lib, cuda):
    """A history of stride 0, lengths and prompts of each row's own."""
    torch = cuda
    p = make(torch, 6, 5000, 700, 0, 3, np.float16)
    p["history"][:] = p["history"][0]
    t = {k: torch.from_numpy(v).cuda() for k, v in p.items()}
    logits = t.pop("logits")
    t["history"] = t["history"][:1].expand(6, -1)
    assert t["history"].stride(0) == 0
    nxt = torch.empty(6, dtype=torch.int32, device="cuda")
    G.LogitsEdit(lib, torch, 6, 5000, **t).apply(logits, logits, nxt)
    got = logits.cpu().numpy()
    check(p, got)
    assert np.array_equal(nxt.cpu().numpy(), first_max(got)) and lib.status() == 0


def test_edits_at_once(lib, cuda):
    """Two captured graphs of one handle, and calls of another, on streams of their own: they share nothing but what they read."""
    torch = cuda
    jobs = []
    p = make(torch, 16, 50257, 400, 20, 1, np.float16, 4)
    h, x = handle(lib, torch, p)
    q = make(torch, 200, 3001, 100, 3, 2, np.float32, 4)
    k, y = handle(lib, torch, q)
    for e, src, n in ((h, x, 16), (h, x, 16), (k, y, 200)):
        st, out, nxt = torch.cuda.Stream(), torch.empty_like(src), torch.empty(n, dtype=torch.int32, device="cuda")
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            e.apply(out, src, nxt, stream=st.cuda_stream)
        jobs.append((g, st, out, nxt))
    torch.cuda.synchronize()
    for _ in range(20):
        for g, st, _, _ in jobs:
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    for (_, _, out, nxt), case in zip(jobs, (p, p, q)):
        got = out.cpu().numpy()
        check(case, got)
        assert np.array_equal(nxt.cpu().numpy(), first_max(got))
    lib.status()


def test_edited_generation_of_256_sequences(lib, cuda):
    """The widest batch, over 4-bit weights: every sequence is forced along tokens of its own."""
    torch = cuda
    B, steps = 256, 5
    w = G.ModelWeights(torch, "cuda", seed=9)
    bt = G.DecodeBatch(lib, w, torch.zeros(B, 12, 2, 12, 8, 64, dtype=torch.float16, device="cuda"), G.W4ModelWeights(lib, torch, w))
    forced = torch.arange(B, device="cuda", dtype=torch.int32)[:, None] * 190 + 11
    prompt, plen = torch.randint(0, G.VOCAB, (B, 3), dtype=torch.int32, device="cuda"), (torch.arange(B, device="cuda", dtype=torch.int32) % 3 + 1)
    out = torch.full((B, steps + 2), -9, dtype=torch.int32, device="cuda")
    bt.generate(prompt, plen, steps, out, edit=G.LogitsEdit(lib, torch, B, G.VOCAB, bias_token=forced, bias=torch.full((B, 1), 30000.0, device="cuda")))
    torch.cuda.synchronize()
    at = torch.arange(steps + 1, device="cuda")[None]
    want = torch.where(at < plen[:, None], prompt[:, [0, 1, 2, 2, 2, 2]], forced)
    assert torch.equal(out[:, :steps + 1], want) and bool((out[:, steps + 1] == -9).all())
    bt.close()
    assert lib.status() == 0
