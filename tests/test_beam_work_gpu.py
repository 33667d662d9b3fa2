"""Beam selection: one work area, sized for the largest call and zeroed once, serves calls of every smaller batch and width in
any order."""
import numpy as np
import pytest

from test_beam_gpu import check, select

pytestmark = pytest.mark.gpu
CALLS = [(64, 4), (128, 4), (1, 4), (128, 4), (16, 32), (512, 1), (3, 5), (128, 4), (70, 7), (16, 32), (256, 2), (512, 1)]


@pytest.mark.parametrize("V", [301, 20011])
@pytest.mark.parametrize("own_size", [False, True])
def test_one_work_area_serves_every_batch_and_width(cuda, lib, V, own_size):
    """Whether a call names the whole area or only what it needs of it."""
    torch = cuda
    rng = np.random.default_rng(V)
    area = torch.zeros(max(lib.gpt2_beam_work_bytes_b200(B, W) for B, W in CALLS), dtype=torch.uint8, device="cuda")
    for B, W in CALLS:
        x = (3.0 * rng.standard_normal((B * W, V))).astype(np.float16)
        score = (-20 * rng.random(B * W)).astype(np.float32)
        done = (rng.random(B * W) < 0.2).astype(np.int32)
        work = area[: lib.gpt2_beam_work_bytes_b200(B, W)] if own_size else area
        got = select(torch, lib, torch.from_numpy(x).cuda(), torch.from_numpy(score).cuda(), torch.from_numpy(done).cuda(), B, W, V - 1, work=work)
        check(x, score, done, B, W, V - 1, got)
    assert lib.status() == 0
