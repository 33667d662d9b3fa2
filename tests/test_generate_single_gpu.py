"""Generation of one sequence: the stride of a single row says nothing."""
import pytest

import gpt2_b200 as G

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("edited", [False, True])
def test_a_generation_of_one_sequence(lib, cuda, edited):
    torch = cuda
    w = G.ModelWeights(torch, "cuda", seed=3)
    bt = G.DecodeBatch(lib, w, torch.zeros(1, 12, 2, 12, 16, 64, dtype=torch.float16, device="cuda"))
    i32 = dict(dtype=torch.int32, device="cuda")
    edit = G.LogitsEdit(lib, torch, 1, G.VOCAB) if edited else None
    prompt, plen, steps = torch.tensor([[5, 6, 7]], **i32), torch.tensor([3], **i32), 6
    want, out = torch.zeros(1, steps + 1, **i32), torch.zeros(steps + 1, 1, **i32).t()
    assert out.stride() == (1, 1)
    bt.generate(prompt, plen, steps, want, edit=edit)
    bt.generate(prompt.t().contiguous().t(), plen, steps, out, edit=edit)
    torch.cuda.synchronize()
    assert torch.equal(out, want) and want[0, :3].tolist() == [5, 6, 7]
    bt.close()
    assert lib.status() == 0
