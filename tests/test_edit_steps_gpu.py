"""A mask that changes with every token: steps and edits in turn, the mask renewed between them on the same stream."""
import pytest

import gpt2_b200 as G

pytestmark = pytest.mark.gpu
V = G.VOCAB


@pytest.mark.parametrize("B", [1, 3])
def test_a_mask_per_token(cuda, lib, B):
    """Each step allows one token per sequence, worked out on the device from the last one; the host waits for nothing."""
    torch = cuda
    w = G.ModelWeights(torch, "cuda", seed=5)
    bt = G.DecodeBatch(lib, w, torch.zeros(B, 12, 2, 12, 16, 64, dtype=torch.float16, device="cuda"))
    i32 = dict(dtype=torch.int32, device="cuda")
    st = torch.cuda.Stream()
    words, steps = (V + 31) // 32, 8
    mask, row = torch.zeros(B, words, **i32), torch.arange(B, device="cuda")
    edit = G.LogitsEdit(lib, torch, B, V, mask=mask)
    logits, tokens = torch.empty(B, V, dtype=torch.float16, device="cuda"), torch.zeros(B, steps + 1, **i32)
    tok, nxt, pos = torch.arange(7, 7 + B, **i32), torch.empty(B, **i32), torch.zeros(B, **i32)
    torch.cuda.synchronize()
    with torch.cuda.stream(st):
        tokens[:, 0] = tok
        for t in range(steps):
            allowed = (tok.long() * 31 + 17) % V
            mask.zero_()
            mask[row, allowed // 32] = (1 << (allowed % 32)).to(torch.int32)
            bt.step(tok, pos, logits, stream=st.cuda_stream)
            edit.apply(logits, logits, nxt, stream=st.cuda_stream)
            tok.copy_(nxt)
            pos += 1
            tokens[:, t + 1] = nxt
    st.synchronize()
    for b in range(B):
        want = 7 + b
        for got in tokens[b].tolist():
            assert got == want
            want = (want * 31 + 17) % V
    bt.close()
    assert lib.status() == 0
