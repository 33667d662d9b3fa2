"""Greedy, attention-only and edited generations in turn on one batch."""
import pytest

import gpt2_b200 as G

pytestmark = pytest.mark.gpu
V = G.VOCAB


@pytest.fixture(scope="module")
def weights(cuda):
    return G.ModelWeights(cuda, "cuda", seed=21, hf_init=False)


def batch(torch, lib, weights, B, max_t=32):
    return G.DecodeBatch(lib, weights, torch.zeros(B, 12, 2, 12, max_t, 64, dtype=torch.float16, device="cuda"))


def ints(torch, *values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def test_greedy_attention_only_and_edited_in_turn(cuda, lib, weights):
    """Each kind writes where it was told to, whatever the others' graphs were captured with."""
    torch = cuda
    B, steps = 3, 8
    prompt, plen = torch.randint(1, V, (B, 4), dtype=torch.int32, device="cuda"), ints(torch, 4, 2, 1)
    bt = batch(torch, lib, weights, B)
    mask = torch.full((1, (V + 31) // 32), -1, dtype=torch.int32, device="cuda")
    edit = G.LogitsEdit(lib, torch, B, V, mask=mask, repetition=torch.full((B,), 1.3, device="cuda"))

    def run(kind, out, prompt=prompt):
        if kind == "attention":
            lib.check(lib.gpt2_b200_batch_generate(bt.h, prompt.data_ptr(), prompt.stride(0), plen.data_ptr(), steps, out.data_ptr(), out.stride(0),
                                                   G.GEN_ATTENTION_ONLY, None), "generate")
        else:
            bt.generate(prompt, plen, steps, out, edit=edit if kind == "edited" else None)
        torch.cuda.synchronize()

    def fresh(width=steps + 1):
        return torch.full((B, width), -9, dtype=torch.int32, device="cuda")

    want = {}
    for kind in ("greedy", "attention", "edited"):
        alone = batch(torch, lib, weights, B)
        bt, keep = alone, bt
        want[kind] = fresh()
        run(kind, want[kind])
        alone.close()
        bt = keep
    last = torch.minimum(torch.arange(1, steps + 1, device="cuda")[None], plen[:, None] - 1)  # the prompt, then its last token
    assert torch.equal(want["attention"][:, 1:], prompt.gather(1, last.long()))
    assert not torch.equal(want["greedy"], want["edited"])
    a, b, c, d = fresh(), fresh(), fresh(steps + 5), fresh()
    for order in ("greedy", "attention", "edited"), ("edited", "attention", "greedy"), ("attention", "edited", "attention"), ("greedy", "edited", "edited"):
        for kind, out in zip(order, (a, b, c)):
            everything = (a, b, c, d)
            for t in everything:
                t.fill_(-9)
            run(kind, out)
            assert torch.equal(out[:, :steps + 1], want[kind]) and bool((out[:, steps + 1:] == -9).all()), (order, kind)
            assert all(bool((t == -9).all()) for t in everything if t is not out)
        run(order[0], d)  # into another buffer, when the last kind captured its own
        assert torch.equal(d, want[order[0]])
        other = prompt.clone()
        run(order[1], d, other)
        assert torch.equal(d, want[order[1]])
    bt.close()
    assert lib.status() == 0
