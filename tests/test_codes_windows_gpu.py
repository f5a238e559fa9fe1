"""Portions over a window of a cache of codes (4 and 8 bits): what they read back is what they see."""
import dataclasses

import pytest
import torch

import test_cache_8bit_gpu as eight
from helpers import TOL, batch_index, rel_error
from test_cache_4bit_engine_gpu import prompt, registered, run
from test_cache_4bit_gpu import DEV, Cache, attend, attention_of, ops  # noqa: F401

pytestmark = pytest.mark.gpu


def kept_reads(ops, monkeypatch, name):
    """What a portion's read-backs returned, and how many requests each was of."""
    read, kept = getattr(ops, name), []

    def spy(*args, **kw):
        found = read(*args, **kw)
        kept.append(found)
        return found

    monkeypatch.setattr(ops, name, spy)
    return kept


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dim", [64, 128, 32])
@pytest.mark.parametrize("window", [1, 2, 64, 66, 100, 1000, 5000])
def test_a_windowed_portion_reads_what_it_sees(ops, monkeypatch, dtype, dim, window):
    """The runs that are made room for and written: those in the table, and at most one a request beside them."""
    held, lens = [3000, 40, 1200, 129], [70, 40, 1, 64]
    cache = Cache(held, 2, dim, 16)
    for brought in (lens, None):
        kept = kept_reads(ops, monkeypatch, "_read_4bit")
        out, want = attend(ops, cache, lens, 6, dtype, window=window, ctx_lens=held, **({"q_lens": brought} if brought else {}))
        assert rel_error(out, want) < TOL[dtype]
        for k, v, table, *_ in kept:
            seen = int((table >= 0).sum())
            extra = len(lens) if brought else sum((max(lens) - n + 63) // 64 + 1 for n in lens)
            assert k.shape[0] == v.shape[0] <= seen + extra
        assert len(kept) == 1
        monkeypatch.undo()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("told", [[3000, 40, 1200, 129], [3063, 90, 1263, 140], [3100, 3100, 3100, 3100]])
@pytest.mark.parametrize("window", [64, 100])
def test_windowed_portions_under_a_bound_of_their_contexts(ops, dtype, told, window):
    """Requests that hold less than the host says, wherever in a run of 64 their window begins."""
    held, lens = [3000, 40, 1200, 129], [70, 40, 1, 64]
    cache = Cache(held, 2, 64, 16)
    for kw in ({}, {"q_lens": lens}):
        out, want = attend(ops, cache, lens, 6, dtype, window=window, ctx_lens=told, **kw)
        assert rel_error(out, want) < TOL[dtype]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("window", [1, 66, 100, 1000])
def test_a_windowed_portion_over_the_8bit_cache_reads_what_it_sees(ops, monkeypatch, dtype, window):
    held, lens = [3000, 40, 1200, 129], [70, 40, 1, 64]
    cache = eight.Cache(held, 2, 64, 16, 1)
    kept = kept_reads(ops, monkeypatch, "_read_8bit")
    positions, seq, q_start, start_pos = batch_index(lens, [h - n for h, n in zip(held, lens)], DEV)
    q = (torch.randn(sum(lens), 6 * 64, generator=torch.Generator().manual_seed(11)) * 0.05).to(dtype)
    out = ops.attention_8bit(q.to(DEV), *cache.device(), cache.table.to(DEV), q_start, start_pos, positions, seq, 4, max(lens), max(held), 6, 2, 64, 0.125,
                             window=window, ctx_lens=held, q_lens=lens)
    ops.check_status()
    at, want = 0, []
    for r, n in enumerate(lens):
        want.append(attention_of(q[at:at + n].view(n, 6, 64), cache.values("k", r), cache.values("v", r), held[r] - n, 0.125, window, None))
        at += n
    assert rel_error(out, torch.cat(want).flatten(1)) < TOL[dtype]
    assert len(kept) == 1 and kept[0][0].shape[0] <= int((kept[0][2] >= 0).sum()) + len(lens)


@pytest.mark.parametrize("cache_dtype,read", [("uint4", "_read_4bit"), ("int8", "_read_8bit")])
def test_an_engines_windowed_portions_read_what_they_see(monkeypatch, cache_dtype, read):
    from aegean_tge_b200 import Engine, ops
    raw = registered(monkeypatch, "WindowedPortionForCausalLM",
                     lambda i, layer: dataclasses.replace(layer, mixer=dataclasses.replace(layer.mixer, params=dict(layer.mixer.params, window=100))))
    eng = Engine(random_config=raw, dtype="bfloat16", context=512, max_tokens=4096, page_size=16, cache_dtype=cache_dtype)
    each, kept = getattr(ops, read), []

    def spy(*args, **kw):
        kept.append(each(*args, **kw))
        return kept[-1]

    monkeypatch.setattr(ops, read, spy)
    run(eng, [400, 30], prompt(430))
    assert len(kept) == 4
    for k, _, table, *_ in kept:
        assert k.shape[0] <= int((table >= 0).sum()) + 1
    assert kept[-1][0].shape[0] <= 4                         # 30 behind 400 over a window of 100: 129 positions
    ops.check_status()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dim", [64, 128])
def test_portions_longer_than_the_host_says_are_reported(ops, dtype, dim):
    """Room is made for what the host says a request brings: more is a status and no output, never another request's keys."""
    held, lens = [900, 40], [300, 40]
    cache = Cache(held, 2, dim, 16)
    for q_lens in ([3, 40], [0, 0]):
        with pytest.raises(ops.DeviceStatusError):
            attend(ops, cache, lens, 6, dtype, window=10, ctx_lens=held, q_lens=q_lens)
    with pytest.raises(ops.KernelError):
        attend(ops, cache, lens, 6, dtype, window=10, ctx_lens=held, q_lens=[300])
    out, want = attend(ops, cache, lens, 6, dtype, window=10, ctx_lens=held, q_lens=lens)
    assert rel_error(out, want) < TOL[dtype]
