"""4-bit weights of one feature: the stride of a single row, or column, says nothing."""
import pytest

import gpt2_b200 as G

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("ld", [131, 1000])
def test_a_weight_of_one_feature(lib, cuda, ld):
    torch = cuda
    many = torch.randn(4 * ld + 128, device="cuda", dtype=torch.float16)
    row = many.as_strided((1, 128), (ld, 1))
    assert row.data_ptr() % 16 == 0
    q, want = G.W4Weight.pack(lib, torch, row, 32, True), G.W4Weight.pack(lib, torch, row.contiguous().clone(), 32, True)
    assert torch.equal(q.codes, want.codes) and torch.equal(q.scale, want.scale) and torch.equal(q.least, want.least)
    back = torch.full((4 * ld + 128,), 7.0, device="cuda", dtype=torch.float16)
    q.dequantize(back.as_strided((1, 128), (ld, 1)))
    assert bool((back[128:] == 7).all()) and float((back[:128] - many[:128]).abs().max()) < 0.5


@pytest.mark.parametrize("B", [1, 5, 40])
def test_outputs_of_one_feature(lib, cuda, B):
    torch = cuda
    q = G.W4Weight.pack(lib, torch, torch.randn(1, 64, device="cuda", dtype=torch.float16), 32)
    x = torch.randn(B, 64, device="cuda", dtype=torch.float16)
    want = torch.empty(B, 1, device="cuda", dtype=torch.float16)
    q.linear(want, x)
    out = torch.full((3 * B,), 7.0, device="cuda", dtype=torch.float16)
    q.linear(out.as_strided((B, 1), (3, 5)), x)
    assert torch.equal(out[::3], want[:, 0]) and bool((out.view(B, 3)[:, 1:] == 7).all())
