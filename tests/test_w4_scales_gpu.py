"""Products whose scales lie on either side of 0.25, where the conversion of the codes changes its steps, negative and subnormal scales among
them. Tolerances: those of test_w4_gpu.py, which hold for any weights."""
import numpy as np
import pytest

import gpt2_b200 as G
from test_w4_gpu import close, values

pytestmark = pytest.mark.gpu

# both kernels; 8 and 16 warps, one and several tiles per CTA, whole rounds of the buffers, clusters, several column blocks
SHAPES = [(1, 33, 96, 32), (1, 700, 2080, 32), (1, 5000, 640, 128), (8, 2304, 768, 64), (7, 300, 4096, 128), (12, 260, 1056, 32), (16, 4000, 960, 64),
          (17, 128, 160, 32), (40, 300, 1024, 128), (64, 700, 2080, 32), (130, 257, 704, 64), (256, 520, 512, 128)]
NEAR = np.array([0x33FF, 0x3400], np.uint16).view(np.float16)  # the last below 0.25, and 0.25
KINDS = {"below": [0.1, NEAR[0], 2.0**-24, 5 * 2.0**-24, 0.2], "above": [NEAR[1], 0.26, 1, 30], "both": [0.02, NEAR[0], NEAR[1], 1, 30, 2.0**-20, 0],
         "signed": [-0.02, 0.02, -0.25, -3, -0.0, -(2.0**-24)]}


@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("least", [False, True])
@pytest.mark.parametrize("B,N,K,group", SHAPES)
def test_scales_on_either_side(lib, cuda, B, N, K, group, least, kind):
    torch = cuda
    rng = np.random.default_rng(B + N + K + least)
    scale = rng.choice(np.array(KINDS[kind], np.float16), (K // group, N))
    if kind == "both":  # one large scale in a warp's features is enough
        scale = np.where(rng.random(scale.shape) < 0.97, np.float16(0.02), scale)
    codes = rng.integers(0, 256, (N, K // 2), dtype=np.uint8)
    low = (-7.5 * scale.astype(np.float32) * (1 + 0.2 * rng.standard_normal(scale.shape))).astype(np.float16) if least else None
    w = G.W4Weight(lib, torch, *(torch.from_numpy(a).cuda() if a is not None else None for a in (codes, scale, low)))
    x = rng.standard_normal((B, K)).astype(np.float16)
    out = torch.full((B, N), float("nan"), dtype=torch.float16, device="cuda")
    w.linear(out, torch.from_numpy(x).cuda())
    v, x64 = values(codes, scale, low, K, group), x.astype(np.float64)
    assert np.isfinite(v).all()
    close(out.cpu().numpy(), x64 @ v.T, np.abs(x64) @ np.abs(v).T, K)
    assert lib.status() == 0
