"""The end of a beam search: the last step asks for no room behind it, so a table and a pool that hold n_steps positions
and no more are enough."""
import numpy as np
import pytest

import gpt2_b200 as G

pytestmark = pytest.mark.gpu


def pages_needed(plen, W, n_steps, page):
    """Per item: the prompt's whole pages once, then every beam's own; while the prompt lasts, a page for each empty row."""
    whole = min(int(plen), n_steps) // page
    return max(whole + W * (-(-n_steps // page) - whole), -(-min(int(plen), n_steps) // page) + W - 1)


@pytest.mark.parametrize("page,most,plens,W,kind", [(16, 2, [1, 7], 4, "int8"), (16, 4, [40, 3, 20], 3, "e4m3"), (32, 3, [50], 5, "int8"), (64, 1, [1], 1, "int8"), (16, 2, [32], 2, "int8"), (16, 1, [1], 2, "int8")])
def test_a_search_may_fill_its_table_and_its_pool(cuda, lib, page, most, plens, W, kind):
    torch = cuda
    w = G.ModelWeights(torch, "cuda", seed=5)
    B, n_steps = len(plens), most * page
    prompt = torch.from_numpy(np.random.default_rng(page).integers(0, G.VOCAB, (B, n_steps)).astype(np.int32)).cuda()
    d_plen = torch.tensor(plens, dtype=torch.int32, device="cuda")

    def search(pages):
        cache = G.KV8Cache.create(lib, torch, B * W, most, pages, page=page, block=16, kind=kind)
        beam = G.BeamDecoder(lib, w, cache, B, W)
        out = torch.full((B * W, n_steps + 1), -9, dtype=torch.int32, device="cuda")
        score = torch.empty(B * W, dtype=torch.float32, device="cuda")
        beam.generate(prompt, d_plen, n_steps, out, score)
        torch.cuda.synchronize()
        got = lib.status()
        kv = torch.empty(2, G.N_LAYER, B * W, n_steps, G.N_EMBD, dtype=torch.float16, device="cuda")
        cache.load(kv[0], kv[1])
        held = cache.length.clone()
        table, ref = cache.table.cpu(), cache.ref.cpu()
        assert torch.equal(torch.bincount(table[table >= 0].long(), minlength=ref.numel()).to(torch.int32), ref)
        beam.close()
        return out, score, kv, held, got, cache

    pages = sum(pages_needed(p, W, n_steps, page) for p in plens)
    wide = search(B * W * (most + 1))
    exact = search(pages)
    assert wide[4] == 0 and exact[4] == 0
    for a, b in zip(wide[:4], exact[:4]):
        assert torch.equal(a, b)
    full = exact[3] == n_steps
    assert bool(full.any())
    cache = exact[5]
    assert bool((cache.table[full] >= 0).all())  # no position of a finished hypothesis is lost
    assert lib.status() == 0
