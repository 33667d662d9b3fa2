"""Attention over the 8-bit cache where a few keys outweigh a long rest: every key's share counts.

A softmax row is one dominant key, a long rest that is flat and many binary orders below it, and value blocks of very unlike
size. The rest's share of the output is what fewer bits for the probabilities would lose.

The tolerance is that of the fp64 tests of the attention."""
import math

import pytest

from test_kv8_gpu import check_attention, make

pytestmark = pytest.mark.gpu


def peaked(torch, lib, kind, rows, heads, group, Tq, dim, n, octaves, sink_v, big=(0, 0.0, 0.0), block=16, seed=0):
    """Rows of about n keys whose key 5 lies `octaves` binary orders above a flat rest, with values of sink_v in its block; big =
    (blocks, octaves, factor): so many blocks behind the first quarter have keys that many octaves above the rest, and
    values `factor` times the rest's, which are 0.5 to 1.5."""
    page = max(block, 32)
    lens = [n - 7 * (i % 5) for i in range(rows)]
    cache = make(torch, lib, rows, heads, dim, page, block, kind, n, layers=1, seed=seed, q_heads=heads * group, queries=Tq)
    g = torch.Generator().manual_seed(seed + 1)
    k = (0.1 * torch.randn(rows, n, heads, dim, generator=g)).cuda()
    v = (0.5 + torch.rand(rows, n, heads, dim, generator=g)).cuda()
    k[..., 0] = 0.0
    k[:, 5, :, 0] = octaves * math.log(2.0)
    v[:, 5 // block * block: 5 // block * block + block] *= sink_v
    at = n // 4 // block * block
    k[:, at: at + big[0] * block, :, 0] = big[1] * math.log(2.0)
    v[:, at: at + big[0] * block] *= big[2] if big[0] else 1.0
    k, v = (x.flatten(2).half()[None] for x in (k, v))
    cache.store(k, v, count=torch.tensor(lens, dtype=torch.int32, device="cuda"))
    cache.length.copy_(torch.tensor(lens, dtype=torch.int32))
    q = torch.zeros(rows, Tq, heads * group, dim, device="cuda")
    q[..., 0] = math.sqrt(dim)  # a key's score is its first element
    return cache, q.flatten(2).half(), lens


@pytest.mark.parametrize("octaves", [20.5, 21.4, 22.3])
@pytest.mark.parametrize("rows,heads,group,n", [(16, 12, 1, 12288), (2, 12, 4, 40000)])
def test_a_flat_rest_far_below_one_key_counts(cuda, lib, rows, heads, group, n, octaves):
    """Long int8 contexts: the tolerance of the fp64 tests holds where tens of thousands of keys lie near 2^-22 of the largest."""
    torch = cuda
    cache, q, lens = peaked(torch, lib, "int8", rows, heads, group, 1, 64, n, octaves, 1.0)
    out = torch.full_like(q, 9.0)
    cache.attend(out, q)
    check_attention(torch, cache, "int8", q, out, 0, lens, None)
    assert lib.status() == 0
