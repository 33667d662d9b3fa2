"""Attention over the 8-bit cache in every launch shape: 8 or 16 query rows, a one- or two-warp CTA per unit, equal pieces and
groups, with and without windows, among them the prompt form (more queries than a tile holds) over several rows. The tolerance is
that of the fp64 tests of the attention (tests/test_kv8_gpu.py)."""
import pytest

from test_kv8_gpu import check_attention, filled

pytestmark = pytest.mark.gpu


def plan(sms, rows, heads, group, Tq, windows):
    """Query rows per tile and warps of the launch, as the library chooses them."""
    R = group * Tq
    tile = 8 if R <= 8 else 16
    units = rows * -(-R // tile) * heads
    if units < 3 * sms:
        return tile, "pieces"
    one = units >= 8 * sms
    if R <= 4 and not windows:
        return tile, "groups of 4" if one and R <= 2 else "groups of 2"
    return tile, "one warp" if one else "two warps"


# rows, heads, query heads per head, queries, keys; the plan without and with windows on a GPU of 148 SMs
CASES = [(45, 12, 5, 1, 150, (8, "two warps"), (8, "two warps")), (45, 12, 1, 8, 150, (8, "two warps"), (8, "two warps")),
         (45, 12, 1, 1, 300, (8, "groups of 2"), (8, "two warps")), (45, 12, 2, 2, 200, (8, "groups of 2"), (8, "two warps")),
         (110, 12, 7, 1, 90, (8, "one warp"), (8, "one warp")), (110, 12, 1, 1, 300, (8, "groups of 4"), (8, "one warp")),
         (110, 12, 1, 3, 100, (8, "groups of 2"), (8, "one warp")),
         (45, 12, 12, 1, 150, (16, "two warps"), (16, "two warps")), (4, 12, 1, 160, 260, (16, "two warps"), (16, "two warps")),
         (110, 12, 3, 4, 70, (16, "one warp"), (16, "one warp")), (13, 12, 2, 70, 200, (16, "one warp"), (16, "one warp")),
         (9, 3, 4, 25, 300, (16, "pieces"), (16, "pieces"))]


@pytest.mark.parametrize("kind,page,block,dim", [("int8", 16, 16, 64), ("e4m3", 32, 16, 64), ("int8", 64, 32, 128), ("e4m3", 128, 64, 128)])
@pytest.mark.parametrize("rows,heads,group,Tq,n,whole,windowed", CASES)
def test_every_launch_shape(cuda, lib, kind, page, block, dim, rows, heads, group, Tq, n, whole, windowed):
    """Rows of no, one, few and many keys, fewer than queries among them; windows that begin before, in and behind a row."""
    torch = cuda
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    if sms == 148:  # the list above covers what it says
        assert plan(sms, rows, heads, group, Tq, False) == whole and plan(sms, rows, heads, group, Tq, True) == windowed
    lens = [(n - 29 * r) % (n + 1) if r % 9 else r // 9 % 4 for r in range(rows)]
    cache = filled(torch, lib, kind, rows, heads, dim, page, block, lens, heads * group, Tq, seed=rows + Tq)
    q = torch.randn(rows, Tq, heads * group * dim, device="cuda").half()
    out = torch.full_like(q, 9.0)
    cache.attend(out, q, layer=1)
    check_attention(torch, cache, kind, q, out, 1, lens, None)
    again = torch.full_like(q, 9.0)
    cache.attend(again, q, layer=1)
    assert torch.equal(out, again)
    first = [[0, -3, 1, lens[r] - 1, lens[r], lens[r] + 5, lens[r] // 2, lens[r] - 40][r % 8] for r in range(rows)]
    out.fill_(9.0)
    cache.attend(out, q, layer=1, first=torch.tensor(first, dtype=torch.int32, device="cuda"))
    check_attention(torch, cache, kind, q, out, 1, lens, first, "windows")
    assert lib.status() == 0


@pytest.mark.parametrize("kind,dim", [("int8", 64), ("e4m3", 128)])
@pytest.mark.parametrize("rows,heads,group,Tq,n", [(4, 3, 1, 3, 2), (45, 12, 5, 1, 40), (45, 12, 2, 2, 2), (110, 12, 4, 4, 30), (3, 2, 16, 2, 50)])
def test_queries_that_are_not_finite_next_to_ones_that_see_no_key(cuda, lib, kind, dim, rows, heads, group, Tq, n):
    """A query that sees no key gives 0, whatever is in it; one that is NaN gives NaN; the other rows' results stay within the tolerance."""
    torch = cuda
    lens = [n if r % 3 else min(n, 1) for r in range(rows)]
    cache = filled(torch, lib, kind, rows, heads, dim, 32, 16, lens, heads * group, Tq, seed=3)
    q = torch.randn(rows, Tq, heads * group * dim, device="cuda").half()
    odd = [r for r in range(rows) if r % 4 == 0]
    bad = q.clone()
    bad[odd, :, :dim] = float("nan")
    out = torch.full_like(q, 9.0)
    cache.attend(out, bad)
    for r in odd:
        for t in range(Tq):
            part = out[r, t, :dim]
            assert bool((part == 0).all() if lens[r] - Tq + t < 0 else part.isnan().all()), (r, t)
    clean = torch.full_like(q, 9.0)
    cache.attend(clean, q)
    mask = torch.zeros_like(q, dtype=torch.bool)
    mask[odd, :, :dim] = True
    check_attention(torch, cache, kind, q, torch.where(mask, clean, out), 0, lens, None)
    assert lib.status() == 0
