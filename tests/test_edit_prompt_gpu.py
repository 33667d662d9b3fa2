"""Generation with edited logits: positions of the prompt."""
import pytest

import gpt2_b200 as G

pytestmark = pytest.mark.gpu
V = G.VOCAB


@pytest.fixture(scope="module")
def weights(cuda):
    return G.ModelWeights(cuda, "cuda", seed=21, hf_init=False)


def batch(torch, lib, weights, B, max_t=32):
    return G.DecodeBatch(lib, weights, torch.zeros(B, 12, 2, 12, max_t, 64, dtype=torch.float16, device="cuda"))


@pytest.mark.parametrize("B", [1, 2, 70])
def test_prompt_positions_choose_nothing(cuda, lib, weights, B):
    """A mask that leaves nothing: a sequence still in its prompt reports nothing, the first choice behind it does."""
    torch = cuda
    steps = 9
    prompt = torch.randint(0, V, (B, steps + 1), dtype=torch.int32, device="cuda")
    plen = torch.full((B,), steps + 1, dtype=torch.int32, device="cuda")
    bt = batch(torch, lib, weights, B)
    out = torch.empty(B, steps + 1, dtype=torch.int32, device="cuda")
    edit = G.LogitsEdit(lib, torch, B, V, mask=torch.zeros(1, (V + 31) // 32, dtype=torch.int32, device="cuda"))
    bt.generate(prompt, plen, steps, out, edit=edit)
    torch.cuda.synchronize()
    assert torch.equal(out, prompt) and lib.status() == 0
    plen[B - 1] = steps  # the last step of the last sequence chooses
    bt.generate(prompt, plen, steps, out, edit=edit)
    torch.cuda.synchronize()
    prompt[B - 1, steps] = -1
    assert torch.equal(out, prompt) and lib.status() == G.ST_EDIT_NO_TOKEN
    bt.close()
