"""Attention over the 8-bit cache with scores at the end of what fp16 queries and keys can reach: finite inputs give the
value of the key with the largest score.

Queries and keys have one element each that is not 0, of up to 65504, so a score is one product: its size in base 2 is up to
2^29, where neighbouring fp32 numbers lie 32 and more apart. The largest score is over 2^20 above the next, so its softmax weight is 1
whatever the rounding, and the output is its value: the sums' 2^-20 of it off at most, and rounded once to fp16 (2^-11, 2^-25 at least)."""
import pytest

import gpt2_b200 as G  # noqa: F401 - the library fixture loads it
from test_kv8_gpu import make, values

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind,dim", [("int8", 64), ("e4m3", 64), ("int8", 128), ("e4m3", 128)])
@pytest.mark.parametrize("rows,heads,group,Tq,n", [(1, 2, 1, 1, 700), (3, 2, 12, 1, 900), (60, 12, 1, 1, 200), (130, 12, 2, 1, 150), (44, 12, 6, 1, 130), (110, 12, 6, 2, 90)])
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_the_largest_score_wins(cuda, lib, kind, dim, rows, heads, group, Tq, n, sign):
    torch = cuda
    cache = make(torch, lib, rows, heads, dim, 32, 16, kind, n, layers=1, q_heads=heads * group, queries=Tq)
    g = torch.Generator().manual_seed(n)
    codes = torch.stack([torch.randperm(n, generator=g) for _ in range(rows)]) % 13 + 100  # 100 .. 112
    best = torch.stack([torch.randperm(n - Tq, generator=g)[:1] for _ in range(rows)])[:, 0]  # a key that every query sees
    codes[torch.arange(rows), best] = 127
    if sign < 0:
        codes = 227 - codes  # the same order of scores with a negative query
    k = torch.zeros(rows, n, heads, dim)
    if kind == "int8":
        x = codes * 512.0
    else:  # fewer bits: the best key alone at its end
        x = torch.where(codes == (127 if sign > 0 else 100), 65504.0 if sign > 0 else 2.0 ** 14, 2.0 ** 15)
    k[..., 3] = x[..., None]
    v = torch.randn(rows, n, heads, dim, generator=g)
    k, v = (t.flatten(2).half()[None].cuda() for t in (k, v))
    cache.store(k, v)
    cache.length.fill_(n)
    q = torch.zeros(rows, Tq, heads * group, dim)
    q[..., 3] = sign * 65504.0
    q = q.flatten(2).half().cuda()
    out = torch.full_like(q, 9.0)
    cache.attend(out, q)
    for r in range(rows):
        ids = cache.table[r].long()
        kv = values(torch, cache.data[ids, 0], kind) * cache.scale[ids, 0].repeat_interleave(16, -1)[..., None]
        kk, vv = (kv[:, i].transpose(0, 1).reshape(heads, -1, dim)[:, :n].double() for i in (0, 1))
        score = sign * 65504.0 * kk[..., 3] / dim ** 0.5
        top = score.topk(2, -1)
        assert bool((top.indices[:, 0].cpu() == best[r]).all()) and bool((top.values[:, 0] - top.values[:, 1] > 2.0 ** 20).all())
        want = vv[:, int(best[r])].repeat_interleave(group, 0).reshape(-1)
        err = (out[r].double() - want).abs()
        assert bool((err <= (2.0 ** -20 + 2.0 ** -11) * want.abs() + 2.0 ** -25).all()), f"row {r}: off by up to {float(err.max())}"
    assert lib.status() == 0
