"""What the entry points of 4-bit weights and of edited logits refuse, before any CUDA call, and what their Python wrappers refuse (no GPU
needed). Only refused calls appear here: an accepted one would launch on these made-up pointers."""
import ctypes

import pytest

import gpt2_b200 as G


def weight(**other):
    w = G.GPT2W4()
    for name, value in {**dict(codes=4096, scale=8192, least=None, N=64, K=256, group=64), **other}.items():
        setattr(w, name, value)
    return w


BAD = [dict(codes=None), dict(codes=4104), dict(scale=None), dict(scale=8193), dict(least=8193), dict(N=0), dict(N=-1), dict(N=2**30 + 1), dict(K=0), dict(K=32), dict(K=250),
       dict(K=2**24 + 64), dict(group=0), dict(group=16), dict(group=48), dict(group=256), dict(group=-64)]


@pytest.mark.parametrize("bad", BAD)
def test_every_call_refuses_a_bad_weight(lib, bad):
    p = ctypes.byref(weight(**bad))
    assert lib.gpt2_w4_quantize_b200(p, 16, 1 << 25, None) == G.EINVAL
    assert lib.gpt2_w4_dequantize_b200(16, 1 << 25, p, None) == G.EINVAL
    assert lib.gpt2_w4_linear_b200(16, 64, 16, 1 << 25, p, None, None, 0, 1, G.LINEAR_STORE, None) == G.EINVAL


def test_calls_refuse_bad_arguments(lib):
    p = ctypes.byref(weight())
    for call in (lambda W, ld: lib.gpt2_w4_quantize_b200(p, W, ld, None), lambda W, ld: lib.gpt2_w4_dequantize_b200(W, ld, p, None)):
        assert call(None, 256) == call(8, 256) == call(16, 248) == call(16, 257) == call(16, -256) == G.EINVAL
    assert lib.gpt2_w4_quantize_b200(None, 16, 256, None) == lib.gpt2_w4_dequantize_b200(16, 256, None, None) == G.EINVAL
    big = ctypes.byref(weight(N=2**30, K=2**24))  # more tiles than a grid has
    assert lib.gpt2_w4_quantize_b200(big, 16, 2**24, None) == G.EINVAL

    def linear(C=16, ldc=64, A=16, lda=256, w=p, bias=None, R=None, ldr=0, B=1, epi=G.LINEAR_STORE):
        return lib.gpt2_w4_linear_b200(C, ldc, A, lda, w, bias, R, ldr, B, epi, None)

    assert linear(C=None) == linear(C=17) == linear(ldc=63) == linear(A=None) == linear(A=24) == linear(lda=248) == linear(lda=260) == linear(w=None) == G.EINVAL
    assert linear(B=0) == linear(B=257) == linear(B=-1) == linear(epi=-1) == linear(epi=3) == linear(bias=17) == G.EINVAL
    assert linear(epi=G.LINEAR_RESID) == linear(epi=G.LINEAR_RESID, R=16, ldr=63) == linear(epi=G.LINEAR_RESID, R=17, ldr=64) == G.EINVAL


def edit(**other):
    e = G.GPT2LogitsEdit()
    for name, value in other.items():
        setattr(e, name, value)
    return e


GOOD = dict(history=16, history_stride=32, max_history=32, bias_token=16, bias=16, bias_stride=8, max_bias=8, mask=16, mask_stride=4, mask_rows=2)


@pytest.mark.parametrize("bad", [dict(history_stride=31), dict(history_stride=-1), dict(max_history=-1), dict(max_history=2**20, history_stride=2**20),
                                 dict(bias=None), dict(bias_stride=7), dict(bias_stride=-8), dict(max_bias=-1), dict(max_bias=1025, bias_stride=1025),
                                 dict(mask_stride=3), dict(mask_rows=0)] +
                         [{name: 18} for name in ("repetition", "frequency", "presence", "history", "length", "prompt", "bias_token", "bias", "n_bias", "mask", "mask_row")])
def test_the_edit_refuses_a_bad_descriptor(lib, bad):
    assert lib.gpt2_logits_edit_b200(16, 100, 4096, 100, 0, 2, 100, ctypes.byref(edit(**{**GOOD, **bad})), None, None) == G.EINVAL


def test_the_edit_refuses_bad_arguments(lib):
    e = edit(**GOOD)

    def call(out=16, ldo=100, x=4096, ld=100, kind=G.BEAM_HALF, rows=2, V=100, e=ctypes.byref(e), nxt=None):
        return lib.gpt2_logits_edit_b200(out, ldo, x, ld, kind, rows, V, e, nxt, None)

    assert call(out=None) == call(out=17) == call(x=None) == call(x=17) == call(kind=2) == call(kind=-1) == call(rows=0) == call(V=0) == call(e=None) == G.EINVAL
    assert call(ld=99) == call(ldo=99) == call(nxt=18) == call(kind=G.BEAM_FLOAT, out=18) == call(x=16, ldo=104) == call(rows=2**29) == G.EINVAL
    assert call(V=129, ld=129, ldo=129) == call(rows=3) == G.EINVAL  # a mask of 4 words, of 2 rows
    assert call(V=2**30 + 1, ld=2**31, ldo=2**31) == G.EINVAL


@pytest.fixture(scope="module")
def torch():
    import torch
    return torch


def test_weight_wrappers(lib, torch, monkeypatch):
    half = dict(dtype=torch.float16)
    codes, scale = torch.zeros(6, 64, dtype=torch.uint8), torch.zeros(2, 6, **half)
    for bad in ((codes.int(), scale), (codes[0], scale), (codes, scale.float()), (codes, scale.t()), (codes, scale[:, :5].contiguous()), (codes, torch.zeros(3, 6, **half)),
                (codes, torch.zeros(8, 6, **half)), (codes, torch.zeros(0, 6, **half)), (codes, scale, scale[:1]), (codes, scale, scale.float()),
                (codes[:, ::2], scale), (codes, scale.to("meta"))):
        with pytest.raises(ValueError):
            G.W4Weight(lib, torch, *bad)
    for K, group in ((100, 64), (128, 16), (0, 32)):
        with pytest.raises(ValueError):
            G.W4Weight.create(lib, torch, 4, K, group, device="cpu")
    w = G.W4Weight(lib, torch, codes, scale, scale.clone())
    made = []
    monkeypatch.setattr(w, "_linear", lambda *a: made.append(a) or 0)
    out, x = torch.zeros(3, 6, **half), torch.zeros(3, 128, **half)
    for bad in ((out.float(), x), (out, x.float()), (out[:2], x), (out[:, :5], x), (out, x[:, :64]), (out.t(), x), (torch.zeros(6, 3, **half).t(), x),
                (out, torch.zeros(128, 3, **half).t()), (out.to("meta"), x), (out, x.to("meta")), (out, x, torch.zeros(5, **half)), (out, x, torch.zeros(6)),
                (out, x, None, G.LINEAR_RESID, out[:2]), (out, x, None, G.LINEAR_RESID, out.float()), (out[0], x[0])):
        with pytest.raises(ValueError):
            w.linear(*bad)
    for bad in (torch.zeros(6, 127, **half), torch.zeros(5, 128, **half), torch.zeros(6, 128), torch.zeros(128, 6, **half).t(), torch.zeros(6, 128, device="meta", **half)):
        for call in (w.quantize, w.dequantize):
            with pytest.raises(ValueError):
                call(bad)
    assert not made
    w.linear(out, x), w.linear(out, x, torch.zeros(6, **half), G.LINEAR_RESID, out), w.linear(out[:1], x[:1], None, G.LINEAR_GELU)
    assert len(made) == 3 and made[2][1] == 6 and made[2][3] == 128


def test_edit_wrappers(lib, torch, monkeypatch):
    i32, rows, vocab = dict(dtype=torch.int32), 3, 100
    good = dict(repetition=torch.ones(3), history=torch.zeros(3, 8, **i32), length=torch.zeros(3, **i32), prompt=torch.zeros(3, **i32), bias_token=torch.zeros(3, 4, **i32),
                bias=torch.zeros(3, 4), n_bias=torch.zeros(3, **i32), mask=torch.zeros(2, 4, **i32), mask_row=torch.zeros(3, **i32))
    for bad in (dict(repetition=torch.ones(2)), dict(repetition=torch.ones(3, dtype=torch.float64)), dict(history=torch.zeros(3, 8)), dict(history=torch.zeros(2, 8, **i32)),
                dict(history=torch.zeros(8, 3, **i32).t()), dict(history=None), dict(length=torch.zeros(3)), dict(bias=None), dict(bias_token=None), dict(bias=torch.zeros(3, 5)),
                dict(bias=torch.zeros(3, 8)[:, :4]), dict(mask=torch.zeros(2, 3, **i32)), dict(mask=torch.zeros(2, 4)), dict(mask_row=None), dict(mask=None),
                dict(history=torch.zeros(20, **i32).as_strided((3, 8), (4, 1))), dict(mask=torch.zeros(1, 4, **i32).expand(2, 4)),
                dict(mask=torch.zeros(9, **i32).as_strided((2, 4), (2, 1))), dict(n_bias=torch.zeros(4, **i32)), dict(mask_row=torch.zeros(3, dtype=torch.int64)), dict(prompt=torch.zeros(3, device="meta", **i32))):
        with pytest.raises(ValueError):
            G.LogitsEdit(lib, torch, rows, vocab, **{**good, **bad})
    e = G.LogitsEdit(lib, torch, rows, vocab, **good)
    made = []
    monkeypatch.setattr(e, "_edit", lambda *a: made.append(a) or 0)
    x = torch.zeros(3, 100)
    for bad in ((x, x.double()), (x.half(), x), (x[:2], x[:2]), (x[:, :99], x[:, :99]), (x, torch.zeros(100, 3).t()), (x.to("meta"), x), (x.to("meta"), x.to("meta")),
                (x, x, torch.zeros(3)), (x, x, torch.zeros(2, **i32))):
        with pytest.raises(ValueError):
            e.apply(*bad)
    assert not made
    e.apply(x, x), e.apply(x.half(), x.half(), torch.zeros(3, **i32))
    assert len(made) == 2


def test_an_edit_over_tables_that_all_rows_share(lib, torch):
    i32 = dict(dtype=torch.int32)
    one = torch.zeros(1, 4, **i32)
    e = G.LogitsEdit(lib, torch, 3, 100, mask=one.expand(3, 4), history=one.expand(3, 4), bias_token=one.expand(3, 4), bias=torch.zeros(1, 4).expand(3, 4)).c
    assert (e.mask_rows, e.mask_stride, e.history_stride, e.max_history, e.bias_stride, e.max_bias) == (1, 4, 0, 4, 0, 4)
    e = G.LogitsEdit(lib, torch, 1, 100, mask=one, history=torch.zeros(4, 1, **i32).t()).c  # the stride of a single row says nothing
    assert (e.mask_rows, e.mask_stride, e.history_stride, e.max_history) == (1, 4, 4, 4)


def _weights():
    w = G.GPT2WeightsGPU()
    for name in ("data", "wte", "wpe", "lnf_g", "lnf_b"):
        setattr(w, name, 4096)
    for L in range(12):
        for name, _ in G.LAYER_TENSORS:
            setattr(w.layers[L], name, 4096 if not name.endswith("_w") else None)  # the matmuls' own weights are not needed
    return w


def _four_bits():
    q = G.GPT2W4Weights()
    for name, N, K in (("qkv", 2304, 768), ("attn_proj", 768, 768), ("fc", 4 * 768, 768), ("proj", 768, 4 * 768)):
        for L in range(12):
            getattr(q, name)[L] = weight(N=N, K=K)
    return q


def test_a_batch_refuses_4_bit_weights_of_another_shape(lib):
    h, w, kv = ctypes.c_void_p(), _weights(), G.cache_view(4096, 12, 32)
    create = lib.gpt2_b200_batch_create_w4

    def refused(q, w=w, kv=kv, B=1):
        h.value = 5
        return create(ctypes.byref(h), ctypes.byref(w), ctypes.byref(q) if q else None, ctypes.byref(kv), B) == G.EINVAL and not h.value

    assert refused(None)
    for name in ("qkv", "attn_proj", "fc", "proj"):
        for bad in (dict(N=767), dict(K=704), dict(codes=None), dict(scale=None), dict(codes=4104), dict(group=48)):
            q = _four_bits()
            good = getattr(q, name)[7]
            getattr(q, name)[7] = weight(**{**dict(N=good.N, K=good.K), **bad})
            assert refused(q), (name, bad)
    q = _four_bits()
    q.head = weight(N=50256, K=768)
    assert refused(q)
    bad = _weights()
    bad.layers[3].qkv_b = None
    assert refused(_four_bits(), w=bad) and refused(_four_bits(), B=0) and refused(_four_bits(), B=257)
    assert refused(_four_bits(), kv=G.cache_view(4096, 11, 32))
    assert create(None, ctypes.byref(w), ctypes.byref(_four_bits()), ctypes.byref(kv), 1) == G.EINVAL


def test_edited_generation_refuses_a_history_of_its_own(lib):
    gen = lib.gpt2_b200_batch_generate_edited
    for bad in (None, edit(history=16), edit(length=16), edit(prompt=16)):
        assert gen(16, 16, 4, 16, 3, 16, 4, ctypes.byref(bad) if bad else None, None) == G.EINVAL
    assert gen(None, 16, 4, 16, 3, 16, 4, ctypes.byref(edit()), None) == G.EINVAL
