"""4-bit weights: quantise, dequantise and the products against the definition in 64 bits.

The codes and scales are whole decisions of fp32 arithmetic, so they are compared bit by bit with the same arithmetic in numpy's
fp32. Products: fp16 times fp16 is exact in fp32; an instruction that adds 16 of them to a sum errs by at most 2^-22 of the magnitudes it
sees (truncated alignment), so K / 16 of them, a few more for the pieces of a split sum and one each for bias, residual and
epilogue err by (K / 16 + 24) 2^-22 sum |x w|; the result is rounded once to fp16, half a step 2^-11 (2^-25 where it is subnormal).
gelu_new has a slope of at most 1.13 and tanhf errs by 2 units of 2^-24.
"""
import numpy as np
import pytest

import gpt2_b200 as G

pytestmark = pytest.mark.gpu

PLACES = (0, 16, 4, 20, 8, 24, 12, 28)


def unpack(codes, K):
    """codes uint8 [N][K/2] -> whole numbers [N][K], in plain numpy."""
    words = codes.reshape(-1, K // 2).view(np.uint32)
    return np.stack([(words >> p) & 15 for p in PLACES], -1).reshape(-1, K).astype(np.int64)


def values(codes, scale, least, K, group):
    """What the codes stand for, fp16-rounded, in 64 bits."""
    q = unpack(codes, K)
    s = np.repeat(scale.T.astype(np.float64), group, 1)
    with np.errstate(over="ignore", invalid="ignore"):
        v = (q - 8) * s if least is None else q * s + np.repeat(least.T.astype(np.float64), group, 1)
        return v.astype(np.float16).astype(np.float64)


def down16(x):
    """fp32 >= 0 to fp16, towards zero."""
    h = x.astype(np.float16)
    return np.where(h.astype(np.float32) > x, (h.view(np.uint16) - 1).view(np.float16), h).astype(np.float16)


def quantised(w, group, least):
    """codes (whole numbers), scale and least of fp16 w, step by step in fp32."""
    x = w.astype(np.float32)
    x = np.where(np.isnan(x), np.float32(0), np.clip(x, -65504, 65504)).reshape(w.shape[0], -1, group)
    if least:
        low = x.min(-1)
        s = down16((x.max(-1) - low) / np.float32(15))
        y, first, last, zero = x - low[..., None], 0, 15, 0
    else:
        low = None
        s = down16(np.abs(x).max(-1) / np.float32(7))
        y, first, last, zero = x, -7, 7, 8
    s32 = s.astype(np.float32)[..., None]
    inv = np.where(s32 > 0, np.float32(1) / np.where(s32 > 0, s32, np.float32(1)), np.float32(0))
    code = np.clip(np.rint(y * inv), first, last) + zero
    return code.reshape(w.shape).astype(np.int64), s.T, None if low is None else low.astype(np.float16).T


def make(torch, N, K, group, least, seed):
    """A weight of random codes and scales, and its values."""
    rng = np.random.default_rng(seed)
    codes = rng.integers(0, 256, (N, K // 2), dtype=np.uint8)
    scale = (0.01 * np.exp(0.4 * rng.standard_normal((K // group, N)))).astype(np.float16)
    low = (-7.5 * scale.astype(np.float32) * (1 + 0.2 * rng.standard_normal(scale.shape))).astype(np.float16) if least else None
    d = [torch.from_numpy(a).cuda() if a is not None else None for a in (codes, scale, low)]
    return d, values(codes, scale, low, K, group)


def gelu(x):
    return 0.5 * x * (1 + np.tanh(np.sqrt(2 / np.pi) * (x + 0.044715 * x**3)))


def close(got, want, magnitude, K, gelu_too=False):
    err = np.abs(got.astype(np.float64) - want)
    acc = (K / 16 + 24) * 2.0**-22 * magnitude * (1.13 if gelu_too else 1.0) + (2.0**-22 * np.abs(want) if gelu_too else 0)
    tol = 2.0**-11 * np.abs(want) + 2.0**-25 + acc * (1 + 2.0**-10)
    bad = err > tol
    assert not bad.any(), (f"{int(bad.sum())} of {bad.size} off, worst {float((err / tol).max()):.2f} of the tolerance at "
                           f"{np.unravel_index(int((err / tol).argmax()), err.shape)}")


SHAPES = [(1, 32, 32), (1, 128, 128), (7, 64, 32), (33, 96, 32), (129, 160, 32), (100, 320, 64), (257, 768, 64), (130, 1408, 128), (64, 2080, 32), (1000, 256, 128)]


@pytest.mark.parametrize("least", [False, True])
@pytest.mark.parametrize("N,K,group", SHAPES)
def test_quantise_and_back(lib, cuda, N, K, group, least):
    torch = cuda
    rng = np.random.default_rng(N * K + group + least)
    w = (rng.standard_normal((N, K)) * np.exp(2 * rng.standard_normal((N, 1)))).astype(np.float16)
    w.reshape(-1)[rng.integers(0, N * K, 1 + N * K // 500)] *= 40
    w[N // 2] = 0                       # a row of zeros
    w.reshape(-1, group)[0] = -3.25     # a group of one value
    w.reshape(-1, group)[-1] = (rng.integers(-9, 9, group) * 2.0**-24).astype(np.float16)  # subnormal ones
    pad = torch.zeros(N, K + 24, dtype=torch.float16, device="cuda")
    pad[:, :K] = torch.from_numpy(w).cuda()
    q = G.W4Weight.pack(lib, torch, pad[:, :K], group, least)
    back = torch.full((N, K + 8), 7.0, dtype=torch.float16, device="cuda")
    q.dequantize(back[:, :K])
    code, scale, low = quantised(w, group, least)
    codes, got_scale = q.codes.cpu().numpy(), q.scale.cpu().numpy()
    assert np.array_equal(got_scale, scale)
    assert np.array_equal(unpack(codes, K), code)
    if least:
        assert np.array_equal(q.least.cpu().numpy(), low)
    got = back.cpu().numpy()
    assert (got[:, K:] == 7).all()
    assert np.array_equal(got[:, :K].astype(np.float64), values(codes, scale, low, K, group))
    # a code is at most half a step off, and at the ends what the scale lost by its rounding down: 15 (or 7) 2^-10 of it, and 2^-24
    step = np.repeat(scale.T.astype(np.float64), group, 1)
    ends = (15 if least else 7) * (2.0**-10 * step + 2.0**-24)
    assert (np.abs(got[:, :K].astype(np.float64) - w) <= 0.5 * step * (1 + 2.0**-10) + ends + 2.0**-11 * np.abs(w)).all()
    assert lib.status() == (0 if np.isfinite(w).all() else G.ST_W4_NONFINITE)


@pytest.mark.parametrize("least", [False, True])
def test_quantise_values_that_are_not_finite_and_the_types_ends(lib, cuda, least):
    torch = cuda
    w = np.zeros((5, 64), np.float16)
    w[0, :3] = (np.nan, 1, -1)
    w[1, :3] = (np.inf, -np.inf, 2)
    w[2, :2] = (65504, -65504)
    w[3] = np.nan
    w[4] = 65504
    q = G.W4Weight.pack(lib, torch, torch.from_numpy(w).cuda(), 32, least)
    assert lib.status() == G.ST_W4_NONFINITE
    back = torch.empty(5, 64, dtype=torch.float16, device="cuda")
    q.dequantize(back)
    code, scale, low = quantised(w, 32, least)
    got = back.cpu().numpy().astype(np.float64)
    assert np.isfinite(got).all()
    assert np.array_equal(unpack(q.codes.cpu().numpy(), 64), code)
    assert np.array_equal(got, values(q.codes.cpu().numpy(), scale, low, 64, 32))
    assert (got[3] == 0).all() and lib.status() == 0


LINEAR = [(1, 1, 32, 32), (1, 768, 768, 64), (2, 5, 64, 64), (3, 130, 96, 32), (5, 300, 1024, 128), (8, 2304, 768, 64), (9, 17, 4096, 128),
          (15, 999, 224, 32), (16, 256, 2048, 64), (17, 128, 160, 32), (31, 640, 1152, 128), (33, 700, 96, 32), (64, 2304, 768, 64), (65, 129, 320, 64),
          (100, 1111, 416, 32), (128, 768, 768, 64), (129, 260, 2080, 32), (200, 77, 32, 32), (256, 520, 1024, 128), (256, 1, 64, 64),
          (12, 4100, 1056, 32), (13, 2048, 2048, 128), (16, 2049, 2048, 64), (16, 100, 2080, 32), (16, 2304, 768, 64), (11, 9001, 96, 32),
          (13, 1100, 3776, 64), (10, 70, 4896, 32),
          # few rows of many features: every tile height, one and several tiles per CTA, whole rounds of the buffers and their ends
          (1, 7104, 6144, 128), (2, 4700, 1248, 32), (4, 2400, 8192, 64), (8, 9472, 1024, 64), (3, 16380, 352, 32), (5, 14000, 128, 64), (7, 40001, 192, 64),
          (1, 60000, 64, 32), (6, 2369, 5152, 32), (10, 4000, 1024, 128), (16, 2400, 1696, 32), (12, 16000, 256, 64), (9, 50000, 64, 32), (14, 30000, 128, 32)]


@pytest.mark.parametrize("epi", ["store", "gelu", "resid"])
@pytest.mark.parametrize("B,N,K,group", LINEAR)
def test_linear(lib, cuda, B, N, K, group, epi):
    torch = cuda
    least = (B + N + (epi == "gelu")) % 2 == 0
    d, v = make(torch, N, K, group, least, B * 1000 + N)
    w = G.W4Weight(lib, torch, *d)
    rng = np.random.default_rng(B + N + K)
    x = (rng.standard_normal((B, K)) * np.exp(rng.standard_normal(K))).astype(np.float16)
    bias = rng.standard_normal(N).astype(np.float16) if epi != "store" or N % 2 else None
    c0 = rng.standard_normal((B, N)).astype(np.float16)
    wide = torch.full((B, K + 40), float("nan"), dtype=torch.float16, device="cuda")  # rows among others
    wide[:, 8:8 + K] = torch.from_numpy(x).cuda()
    out = torch.full((B, N + 3), 5.0, dtype=torch.float16, device="cuda")
    out[:, :N] = torch.from_numpy(c0).cuda()
    w.linear(out[:, :N], wide[:, 8:8 + K], torch.from_numpy(bias).cuda() if bias is not None else None,
             {"store": G.LINEAR_STORE, "gelu": G.LINEAR_GELU, "resid": G.LINEAR_RESID}[epi])
    got = out.cpu().numpy()
    assert (got[:, N:] == 5).all()
    x64 = x.astype(np.float64)
    want, magnitude = x64 @ v.T, np.abs(x64) @ np.abs(v).T
    if bias is not None:
        want, magnitude = want + bias.astype(np.float64), magnitude + np.abs(bias.astype(np.float64))
    if epi == "gelu":
        want = gelu(want)
    if epi == "resid":
        want, magnitude = want + c0.astype(np.float64), magnitude + np.abs(c0.astype(np.float64))
    close(got[:, :N], want, magnitude, K, epi == "gelu")
    assert lib.status() == 0


@pytest.mark.parametrize("B,N,K,group", [(1, 7104, 16384, 128), (4, 40000, 2048, 32), (8, 50257, 768, 64), (2, 20001, 4096, 64), (15, 50257, 768, 64),
                                         (64, 9000, 8192, 128), (250, 20000, 2080, 32)])
def test_linear_of_many_tiles(lib, cuda, B, N, K, group):
    """Large weights, several tiles per CTA, against the values that dequantize gives (compared bit by bit above) in 64 bits."""
    torch = cuda
    g = torch.Generator(device="cuda")
    g.manual_seed(N + B)
    codes = torch.randint(0, 256, (N, K // 2), generator=g, device="cuda", dtype=torch.uint8)
    scale = (0.01 * torch.exp(0.5 * torch.randn(K // group, N, generator=g, device="cuda"))).half()
    least = (-7.5 * scale.float() * (1 + 0.2 * torch.randn(K // group, N, generator=g, device="cuda"))).half() if B % 2 == 0 else None
    w = G.W4Weight(lib, torch, codes, scale, least)
    v = torch.empty(N, K, dtype=torch.float16, device="cuda")
    w.dequantize(v)
    x = torch.randn(B, K, generator=g, device="cuda", dtype=torch.float16)
    out = torch.full((B, N), float("nan"), dtype=torch.float16, device="cuda")
    w.linear(out, x)
    want, magnitude = torch.empty(B, N, dtype=torch.float64, device="cuda"), torch.empty(B, N, dtype=torch.float64, device="cuda")
    for n in range(0, N, 4096):
        part = v[n:n + 4096].double().t()
        want[:, n:n + 4096], magnitude[:, n:n + 4096] = x.double() @ part, x.double().abs() @ part.abs()
    close(out.cpu().numpy(), want.cpu().numpy(), magnitude.cpu().numpy(), K)
    assert lib.status() == 0


@pytest.mark.parametrize("B", [1, 4, 16, 40, 256])
def test_linear_residual_of_its_own_and_repeated_calls(lib, cuda, B):
    torch = cuda
    d, v = make(torch, 300, 512, 64, True, B)
    w = G.W4Weight(lib, torch, *d)
    g = torch.Generator(device="cuda")
    g.manual_seed(B)
    x, r = (torch.randn(B, n, generator=g, device="cuda", dtype=torch.float16) for n in (512, 300))
    a, b, c = (torch.empty(B, 300, dtype=torch.float16, device="cuda") for _ in range(3))
    w.linear(a, x, None, G.LINEAR_RESID, r)
    b.copy_(r)
    w.linear(b, x, None, G.LINEAR_RESID)
    w.linear(c, x, None, G.LINEAR_RESID, r)
    assert torch.equal(a, b) and torch.equal(a, c)  # the same bits every time
    x64 = x.cpu().numpy().astype(np.float64)
    r64 = r.cpu().numpy().astype(np.float64)
    close(a.cpu().numpy(), x64 @ v.T + r64, np.abs(x64) @ np.abs(v).T + np.abs(r64), 512)


@pytest.mark.parametrize("B", [1, 16, 64, 256])
def test_a_row_does_not_touch_another(lib, cuda, B):
    """NaN and infinities in one row of x, or in one feature's scale, stay in its outputs."""
    torch = cuda
    N, K, group = 200, 256, 32
    d, v = make(torch, N, K, group, False, 7)
    x = np.random.default_rng(8).standard_normal((B, K)).astype(np.float16)
    row, feature = B // 2, 131
    bad = x.copy()
    bad[row, 77] = np.nan
    d[1][3, feature] = float("inf")
    out = torch.empty(B, N, dtype=torch.float16, device="cuda")
    G.W4Weight(lib, torch, *d).linear(out, torch.from_numpy(bad).cuda())
    got = out.cpu().numpy()
    assert np.isnan(got[row]).all()
    assert not np.isfinite(got[:, feature]).any()
    keep_b, keep_n = np.arange(B) != row, np.arange(N) != feature
    if B > 1:
        x64 = x[keep_b].astype(np.float64)
        close(got[keep_b][:, keep_n], x64 @ v[keep_n].T, np.abs(x64) @ np.abs(v[keep_n]).T, K)
    assert lib.status() == 0


@pytest.mark.parametrize("B", [1, 16, 64])
def test_captured_replayed_and_on_a_side_stream(lib, cuda, B):
    torch = cuda
    d, v = make(torch, 768, 768, 64, False, 3)
    w = G.W4Weight(lib, torch, *d)
    x, out = torch.randn(B, 768, device="cuda", dtype=torch.float16), torch.zeros(B, 768, device="cuda", dtype=torch.float16)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        w.linear(out, x, stream=st.cuda_stream)
    st.synchronize()
    first = out.clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=st):
        w.linear(out, x, stream=st.cuda_stream)
    y = torch.randn(B, 768, device="cuda", dtype=torch.float16)
    x0 = x.clone()
    for src, want in ((y, None), (x0, first)):
        x.copy_(src)
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        s64 = src.cpu().numpy().astype(np.float64)
        close(out.cpu().numpy(), s64 @ v.T, np.abs(s64) @ np.abs(v).T, 768)
        if want is not None:
            assert torch.equal(out, want)


def test_two_streams_at_once(lib, cuda):
    """Calls that run beside one another share nothing."""
    torch = cuda
    jobs = []
    for i, B in enumerate((1, 5, 64, 200)):
        d, v = make(torch, 1500, 1024, 128, i % 2 == 0, i)
        x = torch.randn(B, 1024, device="cuda", dtype=torch.float16)
        jobs.append((G.W4Weight(lib, torch, *d), v, x, torch.empty(B, 1500, device="cuda", dtype=torch.float16), torch.cuda.Stream()))
    torch.cuda.synchronize()
    for _ in range(10):
        for w, _, x, out, st in jobs:
            w.linear(out, x, stream=st.cuda_stream)
    torch.cuda.synchronize()
    for _, v, x, out, _ in jobs:
        x64 = x.cpu().numpy().astype(np.float64)
        close(out.cpu().numpy(), x64 @ v.T, np.abs(x64) @ np.abs(v).T, 1024)


@pytest.mark.parametrize("B", [12, 64, 200])
def test_beside_the_fp16_products(lib, cuda, B):
    """Both kinds of products hold tensor memory: on two streams at once each gives the bits that it gives alone."""
    torch = cuda
    d, _ = make(torch, 2304, 768, 64, False, B)
    w = G.W4Weight(lib, torch, *d)
    v = torch.empty(2304, 768, dtype=torch.float16, device="cuda")
    w.dequantize(v)
    x = torch.randn(B, 768, device="cuda", dtype=torch.float16)
    out = torch.empty(2, 2, B, 2304, device="cuda", dtype=torch.float16)
    one, two = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()

    def both(o, first, second, times):
        for _ in range(times):
            w.linear(o[0], x, stream=first)
            lib.check(lib.gpt2_b200_linear(o[1].data_ptr(), 2304, x.data_ptr(), 768, v.data_ptr(), None, B, 2304, 768, G.LINEAR_STORE, second), "linear")
        torch.cuda.synchronize()

    both(out[0], one.cuda_stream, one.cuda_stream, 1)
    both(out[1], one.cuda_stream, two.cuda_stream, 30)
    assert torch.equal(out[0], out[1])
    assert lib.status() == 0
