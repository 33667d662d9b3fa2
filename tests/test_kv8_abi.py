"""What the 8-bit cache and beam selection entry points refuse, before any CUDA call (no GPU needed). Only
refused calls appear here: an accepted one would launch on these made-up pointers."""
import ctypes

import pytest

import gpt2_b200 as G


def cache(**other):
    c = G.GPT2KV8Cache()
    shape = dict(nPages=10, nRow=2, maxPages=4, nLayer=2, nHead=4, headDim=64, page=16, block=16, kind=0)
    for name, value in {**shape, **other}.items():
        setattr(c, name, value)
    for i, name in enumerate(("data", "scale", "ref", "table", "len", "work")):
        if name not in other:
            setattr(c, name, 4096 * (i + 1))
    return c


BAD_SHAPES = [dict(nPages=0), dict(nRow=0), dict(nRow=1025), dict(maxPages=0), dict(nLayer=0), dict(nHead=0), dict(headDim=32), dict(headDim=96),
              dict(page=8), dict(page=24), dict(page=256), dict(block=8), dict(block=32), dict(kind=2), dict(kind=-1), dict(maxPages=2 ** 30)]


@pytest.mark.parametrize("bad", BAD_SHAPES + [dict(data=0), dict(scale=8), dict(ref=None), dict(table=4), dict(len=2), dict(work=None), dict(work=8)])
def test_every_call_refuses_a_bad_descriptor(lib, bad):
    c = cache(**bad)
    c.work_bytes = 1 << 40
    p = ctypes.byref(c)
    assert lib.gpt2_kv8_store_b200(p, 0, 1, 16, 16, 0, 256, 256, None, 1, None) == G.EINVAL
    assert lib.gpt2_kv8_load_b200(p, 0, 1, 16, 16, 0, 256, 256, None, 1, None, 0, None) == G.EINVAL
    assert lib.gpt2_kv8_attend_b200(16, 256, 256, 16, 256, 256, p, 0, 4, 1, None, None, 0, 0, None) == G.EINVAL
    assert lib.gpt2_kv8_reorder_b200(p, None, 0, 1, None) == G.EINVAL
    assert lib.gpt2_kv8_compact_b200(p, None, None) == G.EINVAL
    assert lib.gpt2_kv8_reset_b200(p, None) == G.EINVAL
    if bad in BAD_SHAPES:
        assert lib.gpt2_kv8_work_bytes_b200(p, 4, 1) == 0
        assert lib.gpt2_kv8_alloc_b200(p, 4, 1) == 1 and not c.data


def test_null_descriptors(lib):
    assert lib.gpt2_kv8_store_b200(None, 0, 1, 16, 16, 0, 256, 256, None, 1, None) == G.EINVAL
    assert lib.gpt2_kv8_reorder_b200(None, None, 0, 1, None) == G.EINVAL
    assert lib.gpt2_kv8_work_bytes_b200(None, 4, 1) == 0
    assert lib.gpt2_kv8_alloc_b200(None, 4, 1) == 1
    assert lib.gpt2_kv8_reset_b200(None, None) == G.EINVAL
    lib.gpt2_kv8_free_b200(None)


def test_store_and_load_refuse_bad_arguments(lib):
    c = cache()
    p = ctypes.byref(c)
    for call, tail in ((lib.gpt2_kv8_store_b200, (None, 1, None)), (lib.gpt2_kv8_load_b200, (None, 1, None, 0, None))):
        assert call(p, -1, 1, 16, 16, 0, 256, 256, *tail) == G.EINVAL
        assert call(p, 1, 2, 16, 16, 0, 256, 256, *tail) == G.EINVAL       # layers 1..2 of 2
        assert call(p, 0, 0, 16, 16, 0, 256, 256, *tail) == G.EINVAL
        assert call(p, 0, 1, None, 16, 0, 256, 256, *tail) == G.EINVAL
        assert call(p, 0, 1, 16, 24, 0, 256, 256, *tail) == G.EINVAL       # misaligned
        assert call(p, 0, 1, 16, 16, 0, 257, 256, *tail) == G.EINVAL       # stride % 8
        assert call(p, 0, 1, 16, 16, 4, 256, 256, *tail) == G.EINVAL
    assert lib.gpt2_kv8_store_b200(p, 0, 1, 16, 16, 0, 256, 256, None, 65, None) == G.EINVAL  # beyond the table
    assert lib.gpt2_kv8_store_b200(p, 0, 1, 16, 16, 0, 256, 256, None, -1, None) == G.EINVAL
    assert lib.gpt2_kv8_store_b200(p, 0, 1, None, None, 0, 0, 0, None, 0, None) == G.OK       # no tokens: nothing to do
    assert lib.gpt2_kv8_load_b200(p, 0, 1, None, None, 0, 0, 0, None, 0, None, 0, None) == G.OK


def test_attend_refuses_bad_arguments(lib):
    c = cache()
    c.work_bytes = lib.gpt2_kv8_work_bytes_b200(ctypes.byref(c), 8, 1)
    p = ctypes.byref(c)
    attend = lib.gpt2_kv8_attend_b200

    def call(out=16, os=512, ot=512, q=16, qs=512, qt=512, L=0, Hq=8, Tq=1, first=None, dc=None, count=0, most=0):
        return attend(out, os, ot, q, qs, qt, p, L, Hq, Tq, first, dc, count, most, None)

    assert call(L=2) == call(L=-1) == call(Hq=0) == call(Hq=6) == call(Tq=-1) == call(count=-1) == G.EINVAL
    assert call(most=65) == call(most=-1) == call(out=None) == call(out=8) == call(q=None) == call(q=24) == G.EINVAL
    assert call(os=508) == call(ot=4) == call(qs=513) == call(qt=12) == G.EINVAL
    assert call(Tq=2) == call(Hq=16) == G.EINVAL  # more query rows than the work area was sized for
    assert call(Tq=0) == G.OK
    assert lib.gpt2_kv8_work_bytes_b200(p, 6, 1) == lib.gpt2_kv8_work_bytes_b200(p, 8, 0) == 0


def test_reorder_and_compact_refuse_bad_arguments(lib):
    c = cache()
    p = ctypes.byref(c)
    assert lib.gpt2_kv8_reorder_b200(p, None, 0, 1, None) == G.EINVAL  # no work area
    assert lib.gpt2_kv8_compact_b200(p, None, None) == G.EINVAL
    c.work_bytes = lib.gpt2_kv8_work_bytes_b200(p, 4, 1)
    assert lib.gpt2_kv8_reorder_b200(p, None, -1, 1, None) == G.EINVAL
    assert lib.gpt2_kv8_reorder_b200(p, None, 0, -1, None) == G.EINVAL


def test_beam_select_refuses_bad_arguments(lib):
    n = lib.gpt2_beam_work_bytes_b200(2, 4)
    assert n > 0
    assert lib.gpt2_beam_work_bytes_b200(0, 4) == lib.gpt2_beam_work_bytes_b200(2, 0) == lib.gpt2_beam_work_bytes_b200(2, 33) == 0

    def call(token=16, parent=16, new=16, logits=16, type=0, ld=100, score=16, B=2, W=4, V=100, eos=-1, work=256, size=n):
        return lib.gpt2_beam_select_b200(token, parent, new, None, logits, type, ld, score, None, B, W, V, eos, work, size, None)

    for bad in (dict(token=None), dict(parent=None), dict(new=None), dict(logits=None), dict(score=None), dict(work=None), dict(type=2), dict(ld=99), dict(B=-1),
                dict(W=0), dict(W=33), dict(V=0), dict(eos=100), dict(eos=-2), dict(size=n - 1), dict(V=2 ** 30, ld=2 ** 30)):
        assert call(**bad) == G.EINVAL, bad
    assert call(B=0) == G.OK


def test_python_wrappers_refuse_other_layouts(lib):
    import torch
    z = dict(dtype=torch.int32)
    ok = [torch.zeros(5, 1, 2, 2, 16, 64, dtype=torch.uint8), torch.zeros(5, 1, 2, 2, 1), torch.zeros(5, **z), torch.zeros(3, 2, **z), torch.zeros(3, **z)]
    c = G.KV8Cache(lib, torch, *ok)
    for i, bad in ((0, ok[0].to(torch.int8)), (1, ok[1].double()), (1, torch.zeros(5, 1, 2, 3, 1)), (2, torch.zeros(4, **z)), (3, torch.zeros(2, 3, **z).t()),
                   (4, torch.zeros(2, **z)), (0, torch.zeros(5, 1, 2, 2, 24, 64, dtype=torch.uint8))):
        with pytest.raises(ValueError):
            G.KV8Cache(lib, torch, *ok[:i], bad, *ok[i + 1:])
    k = torch.zeros(1, 3, 4, 128, dtype=torch.float16)
    for a, b in ((k, k[:, :, :, :64]), (k.float(), k.float()), (k[0], k[0]), (k[:, :2], k[:, :2]), (k.transpose(2, 3), k.transpose(2, 3)), (k, k.repeat(1, 1, 2, 1)[:, :, ::2])):
        with pytest.raises(ValueError):
            c.store(a, b)
        with pytest.raises(ValueError):
            c.load(a, b)
    for q in (k[0, :, :, :100], k[0].float(), k[0, :2], k):
        with pytest.raises(ValueError):
            c.attend(q, q)
    with pytest.raises(ValueError):
        lib.beam_select(ok[2], ok[2], ok[1], None, torch.zeros(4, 8).double(), ok[1], None, 2, 2, -1, ok[0])
