"""The paged 8-bit cache on the GPU: store and load against the definition's arithmetic, attention against
fp64, the page operators against a row-by-row simulation, bad device-side state, streams and graphs.

Tolerances. Codes and scales are IEEE fp32 functions of the inputs: compared bit for bit. Attention: with
fp16 queries and 8-bit codes every product is exact in fp32, so a score's error is at most (D + 8) 2^-24
times the sum of its terms' magnitudes (summation, scaling), a probability's relative error twice that plus a
few ulp of exp2 and of the sums (2^-20), and the output adds one fp16 rounding (2^-11, or 2^-25 absolute below
the normal range)."""
import ctypes

import numpy as np
import pytest

import gpt2_b200 as G

pytestmark = pytest.mark.gpu
QMAX = {"int8": 127.0, "e4m3": 448.0}


def values(torch, codes, kind):
    return codes.view(torch.int8 if kind == "int8" else torch.float8_e4m3fn).float()


def encode(torch, x, kind):
    x = x.clamp(-QMAX[kind], QMAX[kind])
    if kind == "int8":
        return x.round().to(torch.int8).view(torch.uint8)
    return x.to(torch.float8_e4m3fn).view(torch.uint8)


def make(torch, lib, rows, heads, dim, page, block, kind, capacity, layers=2, spare=3, seed=0, q_heads=0, queries=1):
    """A cache with random content, every row's table filled with shuffled pages of its own."""
    g = torch.Generator().manual_seed(seed)
    most = -(-capacity // page)
    n = rows * most + spare
    data = torch.randint(0, 256, (n, layers, 2, heads, page, dim), generator=g).to(torch.uint8)  # NaN codes among e4m3's
    scale = torch.full((n, layers, 2, heads, page // block), float("nan"))
    table = torch.randperm(n, generator=g)[: rows * most].view(rows, most).to(torch.int32)
    ref = torch.bincount(table.flatten().long(), minlength=n).to(torch.int32)
    cuda = [t.cuda().contiguous() for t in (data, scale, ref, table, torch.zeros(rows, dtype=torch.int32))]
    return G.KV8Cache(lib, torch, *cuda, kind=kind, q_heads=q_heads, queries=queries)


def plain_store(torch, cache, kind, k, v, layer, lens, counts):
    """The definition, row by row and block by block, on CPU copies; returns (data, scale)."""
    data, scale, table = cache.data.cpu(), cache.scale.cpu(), cache.table.cpu()
    page, block, heads, dim = cache.c.page, cache.c.block, cache.c.nHead, cache.c.headDim
    for r, (pos, n) in enumerate(zip(lens, counts)):
        for b0 in range(pos // block * block, pos + n, block) if n else ():
            lo, hi = max(b0, pos), min(b0 + block, pos + n)
            p, at = int(table[r, b0 // page]), b0 % page
            for which, x in enumerate((k, v)):
                x = x[:, r, lo - pos: hi - pos].float().cpu().view(k.shape[0], hi - lo, heads, dim).transpose(1, 2)
                x = torch.where(x.isnan(), torch.zeros(()), x.clamp(-65504, 65504))
                ls = slice(layer, layer + k.shape[0])
                s_old = scale[p, ls, which, :, at // block] if b0 < pos else torch.zeros(k.shape[0], heads)
                s = torch.maximum(s_old, x.abs().amax((2, 3)) / QMAX[kind])
                inv = torch.where(s > 0, 1.0 / s, torch.zeros(()))[..., None, None]
                ratio = torch.where(s > 0, s_old / s, torch.zeros(()))[..., None, None]
                old = data[p, ls, which, :, at: at + lo - b0]
                moved = encode(torch, values(torch, old, kind) * ratio, kind)
                data[p, ls, which, :, at: at + lo - b0] = torch.where((s > s_old)[..., None, None], moved, old)
                data[p, ls, which, :, at + lo - b0: at + hi - b0] = encode(torch, x * inv, kind)
                scale[p, ls, which, :, at // block] = s
    return data, scale


SHAPES = [(16, 16, 64), (32, 16, 64), (64, 64, 128), (128, 32, 128), (128, 128, 64), (64, 16, 128), (32, 32, 64), (128, 128, 128)]


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("page,block,dim", SHAPES)
def test_store_is_the_definition_bit_for_bit(cuda, lib, kind, page, block, dim):
    """Prompts of several lengths (none, one, across blocks and pages), then appends of 1 and of 3 and 40 tokens
    whose values grow, so that older codes are rescaled; strided inputs; rows with nothing to store."""
    torch = cuda
    heads, layers, rows, cap = 3, 3, 5, 300
    cache = make(torch, lib, rows, heads, dim, page, block, kind, cap, layers=layers, seed=page + block + dim)
    g = torch.Generator().manual_seed(1)
    lens = [0] * rows
    for step, (T, counts) in enumerate([(177, [0, 1, 16, 177, 130]), (1, [1, 1, 0, 1, 1]), (3, [3, 2, 3, 0, 1]), (40, [40, 0, 40, 7, 33]), (1, None)]):
        wide = (torch.randn(layers, rows, T, 3 * heads * dim + 8, generator=g) * 2.0 ** step).half().cuda()
        E = heads * dim
        k, v = wide[:2, :, :, E: 2 * E], wide[:2, :, :, 2 * E: 3 * E]
        todo = counts if counts is not None else [T] * rows
        want = plain_store(torch, cache, kind, k, v, 1, lens, todo)
        cache.length.copy_(torch.tensor(lens, dtype=torch.int32))
        cache.store(k, v, layer=1, count=None if counts is None else torch.tensor(counts, dtype=torch.int32, device="cuda"))
        torch.cuda.synchronize()
        assert torch.equal(cache.data.cpu(), want[0]), f"codes after step {step}"
        assert torch.equal(cache.scale.cpu().view(torch.int32), want[1].view(torch.int32)), f"scales after step {step}"
        lens = [a + b for a, b in zip(lens, todo)]
    # and back: code * scale in fp32, rounded once; 0 outside the held positions
    cache.length.copy_(torch.tensor([n - 1 for n in lens], dtype=torch.int32))
    first = torch.tensor([-2, 0, 5, lens[3], 100], dtype=torch.int32)
    out = torch.full((2, 2, rows, 231, E), 7.0, dtype=torch.float16, device="cuda")
    cache.load(out[0], out[1], layer=1, first=first.cuda(), count=1)
    data, scale, table = (t.cpu() for t in (cache.data, cache.scale, cache.table))
    for r in range(rows):
        at = torch.arange(231) + int(first[r])
        ok = (at >= 0) & (at < lens[r])
        a = at.clamp(0, cap - 1)
        p = table[r, a // page].long()
        val = values(torch, data[p, :, :, :, a % page], kind) * scale[p, :, :, :, a % page // block][..., None]
        val = torch.where(ok[:, None, None, None, None], val, torch.zeros(())).half()[:, 1:3].permute(2, 1, 0, 3, 4).reshape(2, 2, 231, E)
        assert torch.equal(out[:, :, r].cpu(), val), f"load of row {r}"
    assert lib.status() == 0


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
def test_store_of_zeros_subnormals_and_non_finite_values(cuda, lib, kind):
    torch = cuda
    cache = make(torch, lib, 2, 2, 64, 16, 16, kind, 32, layers=1)
    x = torch.zeros(1, 2, 20, 128, dtype=torch.float16)
    x[0, 0, :, :64] = 6e-8  # the smallest subnormal in head 0, zeros in head 1
    x[0, 1, 3, 5], x[0, 1, 4, 70], x[0, 1, 5, 71] = float("nan"), float("inf"), float("-inf")
    x[0, 1, 17, 9] = 65504.0
    k = x.cuda()
    want = plain_store(torch, cache, kind, k, k, 0, [0, 0], [20, 20])
    cache.store(k, k)
    torch.cuda.synchronize()
    assert torch.equal(cache.data.cpu(), want[0])
    assert torch.equal(cache.scale.cpu().view(torch.int32), want[1].view(torch.int32))
    assert lib.status() == G.ST_KV8_NONFINITE
    cache.length.fill_(20)
    out = torch.empty(2, 1, 2, 20, 128, dtype=torch.float16, device="cuda")
    cache.load(out[0], out[1])
    assert bool(out.isfinite().all()) and float(out[0, 0, 1, 4, 70]) > 6e4 and float(out[0, 0, 0, 0, 0]) > 0


def filled(torch, lib, kind, rows, heads, dim, page, block, lens, q_heads, queries, seed, spread=1.0):
    """A cache whose positions 0..len-1 hold sensible codes and scales; everything behind them, and every
    scale of an unused block, stays as make() left it (NaN codes, NaN scales)."""
    cap = max(max(lens), 1)
    cache = make(torch, lib, rows, heads, dim, page, block, kind, cap, seed=seed, q_heads=q_heads, queries=queries)
    g = torch.Generator().manual_seed(seed + 1)
    T = max(max(lens), 1)
    k = (torch.randn(2, rows, T, heads * dim, generator=g) * spread).half().cuda()
    v = torch.randn(2, rows, T, heads * dim, generator=g).half().cuda()
    cache.store(k, v, count=torch.tensor(lens, dtype=torch.int32, device="cuda"))
    cache.length.copy_(torch.tensor(lens, dtype=torch.int32))
    return cache


def check_attention(torch, cache, kind, q, out, layer, lens, first, what=""):
    heads, dim, page, block = cache.c.nHead, cache.c.headDim, cache.c.page, cache.c.block
    rows, Tq = q.shape[:2]
    Hq = q.shape[2] // dim
    for r in range(rows):
        n = lens[r]
        got = out[r].double().view(Tq, Hq, dim)
        lo = max(0, first[r]) if first is not None else 0
        ids = cache.table[r, : -(-n // page)].long()
        kv = values(torch, cache.data[ids, layer], kind).double() * cache.scale[ids, layer].double().repeat_interleave(block, -1)[..., None]
        k, v = (kv[:, i].transpose(0, 1).reshape(heads, -1, dim).repeat_interleave(Hq // heads, 0) for i in (0, 1))
        for t in range(Tq):
            end = n - Tq + t + 1
            if end <= lo:
                assert bool((got[t] == 0).all()), f"{what}: row {r} query {t} sees no key"
                continue
            qd = q[r, t].double().view(Hq, dim, 1)
            kk, vv = k[:, lo:end], v[:, lo:end]
            w = torch.softmax((kk @ qd)[..., 0] / dim ** 0.5, -1)
            want = (w[:, None] @ vv)[:, 0]
            terms = (kk.abs() @ qd.abs())[..., 0].amax(-1) / dim ** 0.5  # the largest sum of magnitudes of a score
            rel = 2 * (dim + 8) * 2.0 ** -24 * terms + 2.0 ** -20
            tol = rel[:, None] * vv.abs().amax(1) + 2.0 ** -11 * want.abs() + 2.0 ** -25
            err = (got[t] - want).abs()
            assert bool((err <= tol).all()), f"{what}: row {r} query {t}: {float((err / tol).max()):.2f} of the tolerance"


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("page,block,dim", SHAPES)
@pytest.mark.parametrize("group,Tq", [(1, 1), (4, 1), (1, 3), (8, 5), (3, 33)])
def test_attention_matches_fp64(cuda, lib, kind, page, block, dim, group, Tq):
    """Lengths 0, 1, around tiles, blocks and pages, and long ones, in one call; garbage (NaN codes and scales)
    behind every length; more queries than keys in some rows."""
    torch = cuda
    heads, lens = 2, [0, 1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 129, 255, 700]
    rows = len(lens)
    cache = filled(torch, lib, kind, rows, heads, dim, page, block, lens, heads * group, Tq, seed=dim + page + group)
    g = torch.Generator().manual_seed(3)
    wide = torch.randn(rows, Tq, 3 * heads * group * dim, generator=g).half().cuda()
    q = wide[:, :, : heads * group * dim]
    out = torch.full((rows, Tq, heads * group * dim + 8), 9.0, dtype=torch.float16, device="cuda")
    cache.attend(out[:, :, :-8], q, layer=1)
    assert bool((out[:, :, -8:] == 9.0).all())
    check_attention(torch, cache, kind, q, out[:, :, :-8], 1, lens, None)
    first = [0, 0, 2, 15, 8, 16, -5, 32, 0, 63, 64, 100, 1, 254, 650]
    cache.attend(out[:, :, :-8], q, layer=0, first=torch.tensor(first, dtype=torch.int32, device="cuda"))
    check_attention(torch, cache, kind, q, out[:, :, :-8], 0, lens, first, "first")
    assert lib.status() == 0


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("rows,heads,group,Tq,n,dim", [(1, 1, 1, 1, 20000, 64), (1, 12, 1, 1, 1023, 64), (3, 4, 8, 2, 5000, 128),
                                                       (200, 12, 1, 1, 130, 64), (2, 2, 1, 300, 640, 64), (1, 2, 16, 1, 9000, 128)])
def test_attention_few_rows_many_rows_long_contexts(cuda, lib, kind, rows, heads, group, Tq, n, dim):
    """Shapes that split keys over CTAs, that do not, and many query rows; large scores (a peaked softmax)."""
    torch = cuda
    lens = [max(1, n - 37 * i) for i in range(rows)]
    cache = filled(torch, lib, kind, rows, heads, dim, 64, 32, lens, heads * group, Tq, seed=n, spread=3.0)
    g = torch.Generator().manual_seed(4)
    q = (2.0 * torch.randn(rows, Tq, heads * group * dim, generator=g)).half().cuda()
    out = torch.empty_like(q)
    cache.attend(out, q, layer=0)
    check_attention(torch, cache, kind, q, out, 0, lens, None)
    again = torch.empty_like(q)
    cache.attend(again, q, layer=0, max_len=max(lens))
    other = torch.empty_like(q)
    cache.attend(other, q, layer=0, max_len=max(lens))
    torch.cuda.synchronize()
    assert torch.equal(again, other)  # the same call twice: the same bits
    check_attention(torch, cache, kind, q, again, 0, lens, None, "max_len")
    assert lib.status() == 0


@pytest.mark.parametrize("kind,page,block,dim", [("int8", 16, 16, 64), ("e4m3", 32, 16, 64), ("int8", 64, 32, 128), ("e4m3", 128, 128, 128)])
@pytest.mark.parametrize("rows,group,Tq", [(114, 1, 1), (114, 2, 1), (114, 1, 2), (114, 3, 1), (51, 1, 1), (53, 2, 2), (114, 5, 1)])
def test_attention_of_rows_that_share_pages(cuda, lib, kind, page, block, dim, rows, group, Tq):
    """Many rows in neighbouring fours that hold no, some, most or all of their pages in common, of equal and unequal lengths
    (none among them, shorter than the shared part, more queries than keys), and a last group of fewer rows."""
    torch = cuda
    heads = 12
    rng = np.random.default_rng(dim + page)
    lens, share = [], []
    for b in range(0, rows, 4):
        kind_of = b // 4 % 6
        longest = int(rng.integers(130, 420))
        same = [0, 64, longest // page * page, longest // 2, longest, 200][kind_of]
        few = [longest, longest, longest, longest - 70, longest, longest]
        more = [int(rng.integers(0, longest + 1)) for _ in range(4)] if kind_of == 5 else [longest, few[kind_of], longest, longest]
        if kind_of == 0 and b % 24 == 0:
            more = [0, 1, 65, 2]
        lens += more
        share += [same] * 4
    lens, share = lens[:rows], share[:rows]
    cache = filled(torch, lib, kind, rows, heads, dim, page, block, lens, heads * group, Tq, seed=4)
    table = cache.table.cpu()
    for r in range(rows):
        first = r // 4 * 4
        n = share[r] // page
        full = [x // page for x in (lens[first], lens[r])]
        if r != first and n:
            table[r, : min(n, *full)] = table[first, : min(n, *full)]  # whole pages, filled in both
    cache.table.copy_(table)
    q = torch.randn(rows, Tq, heads * group * dim, device="cuda").half()
    out = torch.full_like(q, 9.0)
    cache.attend(out, q)
    check_attention(torch, cache, kind, q, out, 0, lens, None)
    before = out.clone()
    cache.length[5] = cache.c.maxPages * page + 1  # one row of a group is refused, the others stay
    cache.attend(out, q)
    assert lib.status() == G.ST_KV8_BAD_LEN
    assert bool((out[5] == 0).all())
    lens[5] = 0
    check_attention(torch, cache, kind, q, out, 0, lens, None, "refused row")
    assert torch.equal(out[8:], before[8:])


@pytest.mark.parametrize("kind,dim", [("int8", 64), ("e4m3", 64), ("int8", 128), ("e4m3", 128)])
@pytest.mark.parametrize("rows,heads,group,n", [(5, 3, 1, 200), (16, 6, 2, 700), (9, 3, 12, 300), (60, 12, 1, 300), (100, 12, 2, 150), (100, 12, 1, 500)])
def test_values_of_another_size_in_other_rows_and_heads(cuda, lib, kind, dim, rows, heads, group, n):
    """V's magnitude differs 2^20-fold from row to row and head to head: each keeps its own precision."""
    torch = cuda
    g = torch.Generator().manual_seed(n)
    lens = [n - 13 * i % n for i in range(rows)]
    cache = make(torch, lib, rows, heads, dim, 16, 16, kind, n, q_heads=heads * group)
    k, v = torch.randn(2, 2, rows, n, heads, dim, generator=g).unbind(0)
    v = v * 2.0 ** (torch.arange(rows)[:, None, None, None] * 7 + torch.arange(heads)[:, None] * 9).remainder(21).sub(10)
    k, v = (x.flatten(3).half().cuda() for x in (k, v))
    cache.store(k, v, count=torch.tensor(lens, dtype=torch.int32, device="cuda"))
    cache.length.copy_(torch.tensor(lens, dtype=torch.int32))
    q = torch.randn(rows, 1, heads * group * dim, generator=g).half().cuda()
    out = torch.full_like(q, 9.0)
    cache.attend(out, q)
    check_attention(torch, cache, kind, q, out, 0, lens, None)
    assert lib.status() == 0


@pytest.mark.parametrize("kind,dim,group,n,rows", [("int8", 64, 1, 200, 3), ("int8", 64, 1, 20000, 4), ("int8", 64, 1, 90, 400), ("int8", 64, 16, 90, 3),
                                                  ("int8", 128, 1, 90, 3), ("e4m3", 64, 1, 90, 3)])
def test_queries_that_are_not_finite_give_nan_in_their_head_alone(cuda, lib, kind, dim, group, n, rows):
    """And queries of zeros, of the smallest subnormals and of fp16's ends stay within the tolerance."""
    torch = cuda
    heads = 4
    lens = [n] * rows
    cache = filled(torch, lib, kind, rows, heads, dim, 32, 16, lens, heads * group, 1, seed=1)
    q = torch.randn(rows, 1, heads * group * dim, device="cuda").half()
    q[0, 0, 3], q[1, 0, dim * group + 5], q[2, 0, 2 * dim * group] = float("nan"), float("inf"), float("-inf")
    q[0, 0, dim * group: 2 * dim * group] = 0.0
    q[1, 0, :dim] = 6e-8
    q[2, 0, :dim] = 65504.0 * torch.sign(q[2, 0, :dim])
    out = torch.empty_like(q)
    cache.attend(out, q)
    view = out.view(rows, heads * group, dim)
    for r, h in ((0, 0), (1, group), (2, 2 * group)):
        assert bool(view[r, h].isnan().all())
        view[r, h] = 0
        q.view(rows, heads * group, dim)[r, h] = 0
    assert bool(out.isfinite().all())
    again = torch.empty_like(q)
    cache.attend(again, q)
    for r, h in ((0, 0), (1, group), (2, 2 * group)):
        view[r, h] = again.view(rows, heads * group, dim)[r, h]
    assert torch.equal(out, again)  # the other heads do not see them
    check_attention(torch, cache, kind, q, again, 0, lens, None)
    assert lib.status() == 0


def test_attention_counts_this_steps_tokens(cuda, lib):
    """count / d_count: keys stored in this step, before reorder() counts them in."""
    torch = cuda
    lens = [40, 0, 17]
    cache = filled(torch, lib, "int8", 3, 2, 64, 16, 16, [n + 1 for n in lens], 2, 1, seed=8)
    cache.length.copy_(torch.tensor(lens, dtype=torch.int32))
    q = torch.randn(3, 1, 128, device="cuda").half()
    out = torch.empty_like(q)
    cache.attend(out, q, count=1)
    check_attention(torch, cache, "int8", q, out, 0, [n + 1 for n in lens], None)
    some = torch.tensor([1, 0, 1], dtype=torch.int32, device="cuda")
    cache.attend(out, q, count=some)
    check_attention(torch, cache, "int8", q, out, 0, [41, 0, 18], None)
    assert lib.status() == 0


@pytest.mark.parametrize("kind,rows,dim", [("int8", 100, 64), ("e4m3", 41, 128)])
def test_attention_of_many_rows_counts_this_steps_tokens(cuda, lib, kind, rows, dim):
    """count / d_count and max_len with rows taken together, whose pages are all shared up to this step's token."""
    torch = cuda
    lens = [95 - r % 3 for r in range(rows)]
    cache = filled(torch, lib, kind, rows, 12, dim, 16, 16, [n + 1 for n in lens], 12, 1, seed=9)
    table = cache.table.cpu()
    for r in range(rows):
        table[r, :5] = table[r // 4 * 4, :5]
    cache.table.copy_(table)
    cache.length.copy_(torch.tensor(lens, dtype=torch.int32))
    q = torch.randn(rows, 1, 12 * dim, device="cuda").half()
    out = torch.empty_like(q)
    cache.attend(out, q, count=1, max_len=96)
    check_attention(torch, cache, kind, q, out, 0, [n + 1 for n in lens], None)
    some = [r % 2 for r in range(rows)]
    cache.attend(out, q, count=torch.tensor(some, dtype=torch.int32, device="cuda"))
    check_attention(torch, cache, kind, q, out, 0, [n + s for n, s in zip(lens, some)], None)
    assert lib.status() == 0


class Pages:
    """The page operators row by row, as the header defines them."""

    def __init__(self, rows, most, pages, page):
        self.table = [[-1] * most for _ in range(rows)]
        self.ref, self.len = [0] * pages, [0] * rows
        self.most, self.page = most, page

    def reorder(self, parent, advance, reserve):
        page, copies = self.page, []
        n0 = [n + advance for n in self.len]
        old = [list(t) for t in self.table]
        for t in old:
            for p in t:
                if p >= 0:
                    self.ref[p] -= 1
        for r, f in enumerate(parent):
            n = n0[f] if f >= 0 else 0
            held = -(-n // page)
            self.table[r] = (old[f][:held] if f >= 0 else []) + [-1] * (self.most - held)
            self.len[r] = n
            for p in self.table[r][:held]:
                self.ref[p] += 1
        free = [p for p, c in enumerate(self.ref) if c == 0]
        for r, n in enumerate(self.len):
            held = -(-n // page)
            if reserve and n % page and self.ref[self.table[r][held - 1]] > 1:
                src, p = self.table[r][held - 1], free.pop(0)
                self.ref[src] -= 1
                self.ref[p] = 1
                self.table[r][held - 1] = p
                copies.append((src, p, n % page))
            for i in range(held, -(-(n + reserve) // page)):
                p = free.pop(0)
                self.ref[p] = 1
                self.table[r][i] = p
        return copies

    def compact(self):
        live = sum(c > 0 for c in self.ref)
        dst = [p for p in range(live) if self.ref[p] == 0]
        src = [p for p in range(live, len(self.ref)) if self.ref[p] > 0]
        to = dict(zip(src, dst))
        for a, b in to.items():
            self.ref[b], self.ref[a] = self.ref[a], 0
        self.table = [[to.get(p, p) for p in t] for t in self.table]
        return live, to


@pytest.mark.parametrize("page,block,rows,most,pages,seed", [(16, 16, 6, 9, 60, 1), (32, 16, 1, 3, 5, 2), (64, 32, 33, 5, 200, 3),
                                                             (16, 16, 300, 4, 1300, 4), (128, 64, 4, 2, 2600, 5), (16, 16, 1024, 3, 3100, 6)])
def test_page_operators_match_the_row_by_row_definition(cuda, lib, page, block, rows, most, pages, seed):
    """Random walks of advance, fork, release, reserve and compact: tables, lengths, reference counts and every
    byte of every page against the simulation."""
    torch = cuda
    rng = np.random.default_rng(seed)
    cache = G.KV8Cache.create(lib, torch, rows, most, pages, layers=2, heads=2, dim=64, page=page, block=block)
    cache.data.copy_(torch.from_numpy(rng.integers(0, 256, tuple(cache.data.shape), dtype=np.uint8)))
    cache.scale.copy_(torch.from_numpy(rng.standard_normal(tuple(cache.scale.shape)).astype(np.float32)))
    data, scale = cache.data.cpu().clone(), cache.scale.cpu().clone()
    sim = Pages(rows, most, pages, page)
    room = 0
    for step in range(14):
        advance = int(rng.integers(0, room + 1)) if step else 0
        longest = max(sim.len) + advance
        room = min(int(rng.integers(0, 2 * page)), most * page - longest)
        if step == 3:
            room = 0
        parent = rng.integers(-1 if step % 3 == 2 else 0, rows, rows) if step % 4 else np.arange(rows)
        if step == 5:
            parent[:] = parent[0] if parent[0] >= 0 else 0  # every row continues the same one
        # rows that would share too little: keep within the pool
        keep = [list(t) for t in sim.table], list(sim.ref), list(sim.len)
        try:
            copies = sim.reorder(parent.tolist(), advance, room)
        except IndexError:
            sim.table, sim.ref, sim.len = keep
            parent[:], room = -1, 0
            copies = sim.reorder(parent.tolist(), advance, room)
        for a, b, n in copies:
            data[b, :, :, :, :n] = data[a, :, :, :, :n]
            nb = -(-n // block)
            scale[b, ..., :nb] = scale[a, ..., :nb]
        same = bool((parent == np.arange(rows)).all())
        cache.reorder(None if same else torch.from_numpy(parent.astype(np.int32)).cuda(), advance, room)
        if step % 5 == 4:
            live, to = sim.compact()
            n = torch.zeros(1, dtype=torch.int32, device="cuda")
            cache.compact(n)
            assert int(n) == live
            for a, b in to.items():
                data[b], scale[b] = data[a], scale[a]
        assert cache.length.tolist() == sim.len, f"step {step}"
        assert cache.table.tolist() == sim.table, f"step {step}"
        assert cache.ref.tolist() == sim.ref, f"step {step}"
        assert torch.equal(cache.data.cpu(), data) and torch.equal(cache.scale.cpu(), scale), f"step {step}"
    assert lib.status() == 0


def test_pinned_pages_are_copied_before_they_are_written_and_never_freed(cuda, lib):
    """A hold that the caller adds to ref: the page stays live when its rows go, and a row that continues in it
    gets a copy."""
    torch = cuda
    cache = G.KV8Cache.create(lib, torch, 2, 4, 8, layers=1, heads=1)
    cache.reorder(reserve=20)
    assert cache.table.tolist() == [[0, 1, -1, -1], [2, 3, -1, -1]]
    cache.ref[1] += 1
    cache.reorder(advance=20, reserve=1)  # row 0's last page is pinned: 20 % 16 positions continue in a copy
    assert cache.table.tolist() == [[0, 4, -1, -1], [2, 3, -1, -1]] and cache.ref.tolist() == [1, 1, 1, 1, 1, 0, 0, 0]
    cache.reorder(torch.tensor([-1, -1], dtype=torch.int32, device="cuda"))
    assert cache.ref.tolist() == [0, 1, 0, 0, 0, 0, 0, 0] and cache.length.tolist() == [0, 0]
    cache.reorder(reserve=1)
    assert cache.table[:, 0].tolist() == [0, 2]
    assert lib.status() == 0


def test_bad_device_state_sets_status_bits_and_nothing_is_read_out_of_range(cuda, lib):
    torch = cuda
    i32 = dict(dtype=torch.int32, device="cuda")
    cache = filled(torch, lib, "int8", 3, 2, 64, 16, 16, [40, 40, 40], 2, 1, seed=5)
    cap = cache.c.maxPages * 16
    q = torch.randn(3, 1, 128, device="cuda").half()
    out = torch.full_like(q, 9.0)
    k = torch.randn(1, 3, 4, 128, device="cuda").half()
    cache.length.copy_(torch.tensor([40, cap + 1, -3]))
    cache.attend(out, q)
    assert lib.status() == G.ST_KV8_BAD_LEN
    assert bool((out[1:] == 0).all()) and bool((out[0] != 0).any())
    before = cache.data.clone()
    cache.length.copy_(torch.tensor([cap - 3, cap, -1]))
    cache.store(k, k)  # no row has room for 4 more
    assert lib.status() == G.ST_KV8_BAD_LEN and torch.equal(cache.data, before)
    cache.length.fill_(40)
    cache.table[1, 1], cache.table[2, 2] = -1, 10 ** 6
    cache.attend(out, q)  # keys of entries that are no page are left out
    assert lib.status() == G.ST_KV8_BAD_PAGE and bool(out.isfinite().all())
    cache.load(torch.empty(1, 3, 48, 128, dtype=torch.float16, device="cuda"), torch.empty(1, 3, 48, 128, dtype=torch.float16, device="cuda"))
    assert lib.status() == G.ST_KV8_BAD_PAGE
    cache.length.copy_(torch.tensor([32, 20, 44]))
    cache.store(k, k, layer=1)
    assert lib.status() == G.ST_KV8_BAD_PAGE
    small = G.KV8Cache.create(lib, torch, 3, 2, 4, layers=1, heads=1)
    small.reorder(torch.tensor([7, 0, -2], **i32), reserve=1)
    assert lib.status() == G.ST_KV8_BAD_PARENT and small.table[:, 0].tolist() == [0, 1, 2]
    small.reorder(reserve=17)  # six pages wanted, four there
    assert lib.status() == G.ST_KV8_NO_PAGE
    assert small.table.tolist() == [[0, 1], [2, 3], [-1, -1]] and small.ref.tolist() == [1, 1, 1, 1]
    small.reorder(reserve=33)  # beyond the table row
    assert lib.status() == G.ST_KV8_NO_PAGE
    small.length.copy_(torch.tensor([40, -1, 0]))
    small.reorder()
    assert lib.status() & G.ST_KV8_BAD_LEN and small.length.tolist() == [32, 0, 0]
    lib.status()


def test_one_step_in_a_graph_on_a_side_stream(cuda, lib):
    """reorder, store and attend of a step captured on a stream of their own and replayed as the context grows."""
    torch = cuda
    rows, steps, E = 4, 37, 128
    g = torch.Generator().manual_seed(2)
    ks, vs, qs = (torch.randn(steps, rows, 1, E, generator=g).half().cuda() for _ in range(3))
    parents = torch.randint(0, rows, (steps, rows), generator=g).to(torch.int32).cuda()

    def new():
        return G.KV8Cache.create(lib, torch, rows, 3, 14, layers=1, heads=2)

    direct, outs = new(), []
    direct.reorder(reserve=1)
    for i in range(steps):
        out = torch.empty_like(qs[i])
        direct.store(ks[i][None], vs[i][None])
        direct.attend(out, qs[i], count=1)
        outs.append(out)
        direct.reorder(parents[i], advance=1, reserve=1)
    torch.cuda.synchronize()
    cache = new()
    k, v, q, out, par = ks[0].clone()[None], vs[0].clone()[None], qs[0].clone(), torch.empty_like(qs[0]), parents[0].clone()
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        cache.reorder(reserve=1, stream=st.cuda_stream)
        graph = torch.cuda.CUDAGraph()
        graph.capture_begin()
        cache.store(k, v, stream=st.cuda_stream)
        cache.attend(out, q, count=1, stream=st.cuda_stream)
        cache.reorder(par, advance=1, reserve=1, stream=st.cuda_stream)
        graph.capture_end()
        for i in range(steps):
            k.copy_(ks[i][None]), v.copy_(vs[i][None]), q.copy_(qs[i]), par.copy_(parents[i])
            graph.replay()
            assert torch.equal(out, outs[i]), f"step {i}"
    st.synchronize()
    assert torch.equal(cache.table, direct.table) and torch.equal(cache.ref, direct.ref) and torch.equal(cache.length, direct.length)
    assert lib.status() == 0


def test_alloc_and_free_in_c(cuda, lib):
    torch = cuda
    torch.cuda.synchronize()
    free0 = torch.cuda.mem_get_info()[0]
    c = G.GPT2KV8Cache()
    c.nPages, c.nRow, c.maxPages, c.nLayer, c.nHead, c.headDim, c.page, c.block, c.kind = 1000, 8, 64, 12, 12, 64, 16, 16, 0
    assert lib.gpt2_kv8_alloc_b200(ctypes.byref(c), 12, 1) == 0
    assert c.data and c.scale and c.ref and c.table and c.len and c.work and c.work_bytes
    assert free0 - torch.cuda.mem_get_info()[0] >= 1000 * 12 * 2 * 12 * 16 * 64
    lib.check(lib.gpt2_kv8_reorder_b200(ctypes.byref(c), None, 0, 1, None), "reorder")
    lib.gpt2_kv8_free_b200(ctypes.byref(c))
    assert not c.data and not c.work
    lib.gpt2_kv8_free_b200(ctypes.byref(c))
    lib.gpt2_kv8_free_b200(None)
    torch.cuda.synchronize()
    assert torch.cuda.mem_get_info()[0] >= free0 - (2 << 20)
    c.nPages = 2 ** 31 - 1
    assert lib.gpt2_kv8_alloc_b200(ctypes.byref(c), 12, 1) == 1 and not c.data
    c.nPages = 0
    assert lib.gpt2_kv8_alloc_b200(ctypes.byref(c), 12, 1) == 1
    assert lib.status() == 0


def test_addresses_beyond_32_bits(cuda, lib):
    """A pool of more than 2^32 code bytes: the last pages hold what is stored there."""
    torch = cuda
    pages = 2 ** 32 // (12 * 2 * 12 * 128 * 128) + 40
    cache = G.KV8Cache.create(lib, torch, 2, 12, pages, dim=128, page=128, block=64, q_heads=12)
    cache.table[0] = torch.arange(pages - 12, pages, dtype=torch.int32)
    cache.table[1] = torch.arange(12, dtype=torch.int32)
    k, v = (torch.randn(1, 2, 1500, 12 * 128, device="cuda").half() for _ in range(2))
    cache.store(k, v, layer=11)
    cache.length.fill_(1500)
    q = torch.randn(2, 1, 12 * 128, device="cuda").half()
    q[1] = q[0]
    out = torch.empty_like(q)
    cache.attend(out, q, layer=11)
    check_attention(torch, cache, "int8", q, out, 11, [1500, 1500], None)
    back = torch.empty_like(k)
    cache.load(back, torch.empty_like(v), layer=11)
    assert bool(((back - k).abs() <= cache.scale.max() * 0.51 + 1e-2).all())
    assert lib.status() == 0
