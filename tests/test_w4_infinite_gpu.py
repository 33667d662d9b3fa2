"""4-bit weights whose value, code times a finite scale, is beyond fp16. Tolerances: those of test_w4_gpu.py."""
import numpy as np
import pytest

import gpt2_b200 as G
from test_w4_gpu import close, unpack, values

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("least", [False, True])
@pytest.mark.parametrize("B,N,K,group", [(1, 40, 32, 32), (1, 300, 96, 32), (5, 2304, 768, 64), (3, 40, 2080, 32), (8, 5000, 224, 32), (12, 70, 1056, 32), (2, 200, 8192, 128),
                                         (17, 128, 160, 32), (64, 300, 1088, 64), (200, 77, 96, 32)])
def test_a_value_beyond_fp16_is_infinite(lib, cuda, B, N, K, group, least):
    """Finite scales may stand for an infinite weight; a product with numbers other than 0 is infinite then, whatever k the kernel pads."""
    torch = cuda
    rng = np.random.default_rng(B + N + K)
    codes = rng.integers(0, 256, (N, K // 2), dtype=np.uint8)
    scale = np.full((K // group, N), 0.01, np.float16)
    low = np.full((K // group, N), -0.07, np.float16) if least else None
    hot = rng.permutation(N)[:max(1, N // 7)]  # features with one group whose code 15 is too large, at its first, last or any k
    for i, n in enumerate(hot):
        g = (0, K // group - 1, int(rng.integers(0, K // group)))[i % 3]
        scale[g, n] = 10000 if i % 2 else 60000
    v = values(codes, scale, low, K, group)
    q = unpack(codes, K)
    x = (np.abs(rng.standard_normal((B, K))) + 0.01).astype(np.float16)  # of one sign: +inf never meets -inf
    # a symmetric group's codes below 8 would be -inf: those are made 8
    where = np.isneginf(v)
    if where.any():
        q[where] = 8
        words = np.zeros((N, K // 8), np.uint32)
        for i, place in enumerate((0, 16, 4, 20, 8, 24, 12, 28)):
            words |= q.reshape(N, K // 8, 8)[..., i].astype(np.uint32) << np.uint32(place)
        codes = words.view(np.uint8).reshape(N, K // 2)
        v = values(codes, scale, low, K, group)
    assert np.isposinf(v).any() and not np.isneginf(v).any()
    w = G.W4Weight(lib, torch, *(torch.from_numpy(a).cuda() if a is not None else None for a in (codes, scale, low)))
    out = torch.empty(B, N, dtype=torch.float16, device="cuda")
    w.linear(out, torch.from_numpy(x).cuda())
    got, over = out.cpu().numpy(), np.isposinf(v).any(1)
    assert np.isposinf(got[:, over]).all()
    cold = np.setdiff1d(np.arange(N), hot)
    x64 = x.astype(np.float64)
    close(got[:, cold], x64 @ v[cold].T, np.abs(x64) @ np.abs(v[cold]).T, K)
    assert lib.status() == 0
