"""Packing a weight on another stream than torch's current one: what pack() allocates, and what it reads, is ordered on both."""
import pytest

import gpt2_b200 as G

pytestmark = pytest.mark.gpu
LONG = 200_000_000  # cycles: a tenth of a second, far longer than a call takes to be enqueued


def parts(q):
    return [t for t in (q.codes, q.scale, q.least) if t is not None]


@pytest.mark.parametrize("least", [False, True])
@pytest.mark.parametrize("side_is_current", [False, True])
def test_packed_behind_the_current_streams_work(lib, cuda, side_is_current, least):
    """The current stream is busy, and makes the weight when it gets there; the other one is idle."""
    torch = cuda
    src = torch.randn(300, 512, device="cuda", dtype=torch.float16)
    want = G.W4Weight.pack(lib, torch, src, 64, least)
    side, main = torch.cuda.Stream(), torch.cuda.current_stream()
    w = torch.zeros_like(src)
    torch.cuda.synchronize()
    with torch.cuda.stream(side if side_is_current else main):
        torch.cuda._sleep(LONG)
        w.copy_(src)
        q = G.W4Weight.pack(lib, torch, w, 64, least, 0 if side_is_current else side.cuda_stream)
    torch.cuda.synchronize()
    for got, ref in zip(parts(q), parts(want)):
        assert torch.equal(got, ref)


def test_a_weight_dropped_before_it_was_packed(lib, cuda):
    """The memory of a weight that is given up while its stream has yet to fill it goes to nobody else."""
    torch = cuda
    src = torch.randn(4096, 2048, device="cuda", dtype=torch.float16)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(LONG)
    shapes = [(t.shape, t.dtype) for t in parts(G.W4Weight.pack(lib, torch, src, 32, True, side.cuda_stream))]
    others = [torch.full(shape, 7, dtype=dtype, device="cuda") for shape, dtype in shapes]
    torch.cuda.synchronize()
    assert all(bool((t == 7).all()) for t in others)
