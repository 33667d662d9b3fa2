"""Attention over the 8-bit cache where a few keys outweigh a long rest: every key's share counts.

A softmax row is one dominant key, a long rest that is flat and many binary orders below it, and value blocks of very unlike
size. The rest's share of the output is what fewer bits for the probabilities would lose.

Tolerance, against fp64 on the same codes and scales. With w_k the softmax weights and v_k the values: scores and
exponentials give every w_k a relative error of rel = 2 (D + 8) 2^-24 terms + 2^-20 (terms: the largest sum of magnitudes of
a score's products), the sums over keys at most 2^-24 per step of 16 keys, 2^-14 for the up to 512 steps of a warp and their
merges; a probability that goes into the products in two fp16 parts next to the largest w_k s_k (s_k the
key's value scale) so far keeps 2^-34 of it, which with codes of at most qmax is 2^-33 qmax max(w_k s_k) per key; and one
rounding to fp16: 2^-11 |o|, 2^-25 at least."""
import math

import pytest

import gpt2_b200 as G
from test_kv8_gpu import check_attention, values

pytestmark = pytest.mark.gpu


def peaked(torch, lib, kind, rows, heads, group, Tq, dim, n, octaves, sink_v, big=(0, 0.0, 0.0), block=16, seed=0):
    """Rows of about n keys whose key 5 lies `octaves` binary orders above a flat rest, with values of sink_v in its block; big =
    (blocks, octaves, factor): so many blocks behind the first quarter have keys that many octaves above the rest, and
    values `factor` times the rest's, which are 0.5 to 1.5."""
    page = max(block, 32)
    lens = [n - 7 * (i % 5) for i in range(rows)]
    most = -(-n // page)
    cache = G.KV8Cache.create(lib, torch, rows, most, rows * most, 1, heads, dim, page, block, kind, heads * group, Tq)
    g = torch.Generator(device="cuda").manual_seed(seed)
    cache.table.copy_(torch.randperm(rows * most, generator=g, device="cuda").view(rows, most))
    k = 0.1 * torch.randn(rows, n, heads, dim, generator=g, device="cuda")
    v = 0.5 + torch.rand(rows, n, heads, dim, generator=g, device="cuda")
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


def check_shares(torch, cache, kind, q, out, lens, first=None):
    heads, dim, block = cache.c.nHead, cache.c.headDim, cache.c.block
    qmax = 127.0 if kind == "int8" else 448.0
    rows, Tq = q.shape[:2]
    Hq = q.shape[2] // dim
    for r in sorted({*range(0, rows, max(1, rows // 9)), rows - 1}):  # rows are alike but for their codes and lengths
        n, lo = lens[r], 0 if first is None else max(0, first[r])
        ids = cache.table[r, : -(-n // cache.c.page)].long()
        scale = cache.scale[ids, 0].double().repeat_interleave(block, -1)  # [page][2][head][position]
        kv = values(torch, cache.data[ids, 0], kind).double() * scale[..., None]
        k, v = (kv[:, i].transpose(0, 1).reshape(heads, -1, dim).repeat_interleave(Hq // heads, 0) for i in (0, 1))
        sv = scale[:, 1].transpose(0, 1).reshape(heads, -1).repeat_interleave(Hq // heads, 0)
        for t in range(Tq):
            end = n - Tq + t + 1
            qd = q[r, t].double().view(Hq, dim, 1)
            kk, vv, ss = k[:, lo:end], v[:, lo:end], sv[:, lo:end]
            w = torch.softmax((kk @ qd)[..., 0] / dim ** 0.5, -1)
            want = (w[:, None] @ vv)[:, 0]
            terms = (kk.abs() @ qd.abs())[..., 0].amax(-1) / dim ** 0.5
            rel = 2 * (dim + 8) * 2.0 ** -24 * terms + 2.0 ** -20 + 2.0 ** -14
            tol = rel[:, None] * (w[:, None] @ vv.abs())[:, 0] + (end - lo) * 2.0 ** -33 * qmax * (w * ss).amax(-1)[:, None] + 2.0 ** -11 * want.abs() + 2.0 ** -25
            err = (out[r, t].double().view(Hq, dim) - want).abs()
            assert bool((err <= tol).all()), f"row {r} query {t}: {float((err / tol).max()):.2f} of the tolerance, off by {float((err / want.abs().clamp(min=1e-30)).max()):.2g}"


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


SHAPES = [(1, 2, 1, 1, 16384), (3, 2, 4, 2, 9000), (16, 12, 1, 1, 4096), (2, 2, 3, 5, 3000), (60, 12, 1, 1, 900), (130, 12, 2, 1, 500), (44, 12, 1, 6, 400), (110, 12, 6, 1, 300), (44, 12, 6, 2, 400)]


@pytest.mark.parametrize("kind,dim", [("int8", 64), ("e4m3", 64), ("int8", 128), ("e4m3", 128)])
@pytest.mark.parametrize("rows,heads,group,Tq,n", SHAPES)
@pytest.mark.parametrize("octaves,sink_v,big", [(23.0, 1.0, (0, 0, 0)),            # a peaked row
                                                (23.0, 0.0, (0, 0, 0)),            # the dominant key's values are 0
                                                (30.0, 0.0, (0, 0, 0)),
                                                (60.0, 2.0 ** -20, (0, 0, 0)),     # no share left, small values
                                                (17.5, 1.0, (1, 1.0, 64.0)),       # larger values in a block of the rest
                                                (0.0, 1.0, (2, -80.0, 2.0 ** 14)), # a block nobody attends, of huge values
                                                (12.0, 2.0 ** -10, (1, -40.0, 2.0 ** 15))])
def test_shares_of_unlike_keys_and_values(cuda, lib, kind, dim, rows, heads, group, Tq, n, octaves, sink_v, big):
    torch = cuda
    cache, q, lens = peaked(torch, lib, kind, rows, heads, group, Tq, dim, n, octaves, sink_v, big)
    out = torch.full_like(q, 9.0)
    cache.attend(out, q)
    check_shares(torch, cache, kind, q, out, lens)
    first = [(r % 4) * 2 for r in range(rows)]  # windows that begin around the dominant key
    cache.attend(out, q, first=torch.tensor(first, dtype=torch.int32, device="cuda"))
    check_shares(torch, cache, kind, q, out, lens, first)
    assert lib.status() == 0
