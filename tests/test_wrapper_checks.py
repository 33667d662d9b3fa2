"""What the Python wrappers of the 8-bit cache and of beam search refuse before a call: tensors whose type, number of elements, layout or
device is not what the library reads (no GPU needed: nothing here reaches a launch)."""
import types

import pytest

import gpt2_b200 as G


@pytest.fixture(scope="module")
def torch():
    import torch
    return torch


@pytest.fixture()
def calls(monkeypatch, lib, torch):
    """A cache of 3 rows on the CPU whose library calls are only counted, and the count."""
    made = []
    z = dict(dtype=torch.int32)
    cache = G.KV8Cache(lib, torch, torch.zeros(5, 1, 2, 2, 16, 64, dtype=torch.uint8), torch.zeros(5, 1, 2, 2, 1), torch.zeros(5, **z), torch.zeros(3, 2, **z), torch.zeros(3, **z))
    for name in ("_store", "_load", "_attend", "_reorder", "_compact"):
        monkeypatch.setattr(cache, name, lambda *a: made.append(a) or 0)
    return cache, made


def vectors(torch, n):
    """Of n int32: a good one, and every kind of bad one."""
    good = torch.zeros(n, dtype=torch.int32)
    bad = [good.long(), good.bool(), good.float(), good.to(torch.int16), torch.zeros(n - 1, dtype=torch.int32), torch.zeros(n + 1, dtype=torch.int32),
           torch.zeros(2 * n, dtype=torch.int32)[::2], torch.zeros(n, dtype=torch.int32, device="meta")]
    return good, bad


def test_counts_firsts_and_parents(calls, torch):
    cache, made = calls
    k = torch.zeros(1, 3, 4, 128, dtype=torch.float16)
    q = torch.zeros(3, 1, 128, dtype=torch.float16)
    good, bad = vectors(torch, 3)
    for b in bad:
        for call in (lambda: cache.store(k, k, count=b), lambda: cache.load(k, k, count=b), lambda: cache.load(k, k, first=b), lambda: cache.attend(q, q, count=b),
                     lambda: cache.attend(q, q, first=b), lambda: cache.reorder(b)):
            with pytest.raises(ValueError):
                call()
    for b in (torch.zeros(1), torch.zeros(2, dtype=torch.int32), torch.zeros(1, dtype=torch.int64)):
        with pytest.raises(ValueError):
            cache.compact(b)
    assert not made
    cache.store(k, k, count=good), cache.load(k, k, first=good, count=good), cache.load(k, k, count=2), cache.attend(q, q, first=good, count=good), cache.attend(q, q, count=1)
    cache.reorder(good), cache.reorder(), cache.compact(torch.zeros(1, dtype=torch.int32)), cache.compact(), cache.store(k, k)
    assert len(made) == 10


def test_rows_and_queries_of_another_device(calls, torch):
    cache, made = calls
    k, q = (torch.zeros(*s, dtype=torch.float16, device="meta") for s in ((1, 3, 4, 128), (3, 1, 128)))
    here_k, here_q = (torch.zeros(*s, dtype=torch.float16) for s in ((1, 3, 4, 128), (3, 1, 128)))
    for call in (lambda: cache.store(k, k), lambda: cache.store(here_k, k), lambda: cache.load(here_k, k), lambda: cache.load(k, here_k), lambda: cache.attend(here_q, q), lambda: cache.attend(q, here_q)):
        with pytest.raises(ValueError):
            call()
    assert not made


def test_a_cache_of_tensors_on_unlike_devices(lib, torch):
    z = dict(dtype=torch.int32)
    ok = [torch.zeros(5, 1, 2, 2, 16, 64, dtype=torch.uint8), torch.zeros(5, 1, 2, 2, 1), torch.zeros(5, **z), torch.zeros(3, 2, **z), torch.zeros(3, **z)]
    for i in range(1, 5):
        with pytest.raises(ValueError):
            G.KV8Cache(lib, torch, *ok[:i], ok[i].to("meta"), *ok[i + 1:])


def test_beam_select(monkeypatch, lib, torch):
    made = []
    monkeypatch.setattr(lib, "_beam_select", lambda *a: made.append(a) or 0)
    B, W, V = 2, 3, 11
    i32, f32 = torch.zeros(6, dtype=torch.int32), torch.zeros(6)
    good = dict(token=i32, parent=i32, new_score=f32, new_done=i32, logits=torch.zeros(6, V), score=f32, done=i32, B=B, W=W, eos=-1, work=torch.zeros(64, dtype=torch.uint8))
    _, bad = vectors(torch, 6)
    for name in ("token", "parent", "new_done", "done"):
        for b in bad:
            with pytest.raises(ValueError):
                lib.beam_select(**{**good, name: b})
    for name in ("new_score", "score"):
        for b in (f32.double(), f32.half(), i32, torch.zeros(5), torch.zeros(12)[::2], torch.zeros(6, device="meta")):
            with pytest.raises(ValueError):
                lib.beam_select(**{**good, name: b})
    for b in (torch.zeros(5, V), torch.zeros(7, V), torch.zeros(6, V).bfloat16(), torch.zeros(V, 6).t(), torch.zeros(6, V, device="meta"), torch.zeros(2, 3, V)):
        with pytest.raises(ValueError):
            lib.beam_select(**{**good, "logits": b})
    for b in (torch.zeros(64), torch.zeros(128, dtype=torch.uint8)[::2], torch.zeros(64, dtype=torch.uint8, device="meta")):
        with pytest.raises(ValueError):
            lib.beam_select(**{**good, "work": b})
    assert not made
    for other in ({}, dict(done=None), dict(new_done=None), dict(logits=torch.zeros(6, V + 3).half()[:, :V]), dict(score=f32.view(B, W), token=i32.view(B, W))):
        lib.beam_select(**{**good, **other})
    assert len(made) == 5 and made[0][9:13] == (B, W, V, -1)


def test_beam_decoder_generate(monkeypatch, lib, torch):
    made = []
    beam = G.BeamDecoder.__new__(G.BeamDecoder)
    beam.lib, beam.B, beam.W, beam.h = types.SimpleNamespace(gpt2_b200_beam_generate=lambda *a: made.append(a) or 0, check=lib.check), 2, 3, None
    beam.cache = types.SimpleNamespace(data=torch.zeros(1, dtype=torch.uint8))
    good = dict(prompt=torch.zeros(2, 5, dtype=torch.int32), prompt_len=torch.ones(2, dtype=torch.int32), n_steps=7, out=torch.zeros(6, 8, dtype=torch.int32), score=torch.zeros(6))
    for name, bads in dict(prompt=[torch.zeros(2, 5, dtype=torch.int64), torch.zeros(1, 5, dtype=torch.int32), torch.zeros(5, 2, dtype=torch.int32).t(), torch.zeros(10, dtype=torch.int32), torch.zeros(2, 0, dtype=torch.int32),
                                   torch.zeros(2, 5, dtype=torch.int32, device="meta")],
                           prompt_len=vectors(torch, 2)[1],
                           out=[torch.zeros(5, 8, dtype=torch.int32), torch.zeros(6, 8, dtype=torch.int64), torch.zeros(8, 6, dtype=torch.int32).t(), torch.zeros(6, 12, dtype=torch.int32)[:, :7], torch.zeros(6, 8, dtype=torch.int32, device="meta")],
                           score=[torch.zeros(5), torch.zeros(6).double(), torch.zeros(12)[::2]]).items():
        for b in bads:
            with pytest.raises(ValueError):
                beam.generate(**{**good, name: b})
    assert not made
    beam.generate(**good)
    beam.generate(**{**good, "score": None, "prompt": torch.zeros(2, 9, dtype=torch.int32)[:, :5], "out": torch.zeros(6, 20, dtype=torch.int32)[:, 3:15]})
    assert len(made) == 2
