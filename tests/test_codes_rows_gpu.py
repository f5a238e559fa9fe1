"""Rows that lie as an inner buffer's do, single tokens beside portions, over caches of codes (4 and 8 bits)."""
import pytest
import torch

import test_cache_8bit_gpu as eight
from helpers import TOL, batch_index, rel_error
from test_cache_4bit_gpu import DEV, Cache, attention_of, ops  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("heads,kv,dim", [(6, 2, 128), (6, 2, 64), (4, 2, 32), (4, 2, 80)])
@pytest.mark.parametrize("lead,behind", [(0, 0), (1, 0), (0, 3), (2, 0), (8, 8)])
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("sink", [False, True])
def test_portions_behind_single_tokens(ops, monkeypatch, dtype, heads, kv, dim, lead, behind, bits, sink):
    """On odd elements, on even ones, on whole 16 bytes; on one stream and on two; whether the host tells of the single tokens or not."""
    held = [1, 5, 64, 65, 200, 17, 128, 90, 400, 33, 300, 270]
    lens = [1] * 10 + [70, 64]
    cache = Cache(held, kv, dim, 16) if bits == 4 else eight.Cache(held, kv, dim, 16, 1)
    call = ops.attention_4bit if bits == 4 else ops.attention_8bit
    positions, seq, q_start, start_pos = batch_index(lens, [h - n for h, n in zip(held, lens)], DEV)
    gen = torch.Generator().manual_seed(3)
    wide = (torch.randn(sum(lens), lead + heads * dim + behind, generator=gen) * (1.0 if bits == 4 else 0.02)).to(dtype)
    q = wide[:, lead:lead + heads * dim]
    sinks = torch.randn(heads, generator=gen) if sink else None
    want, at = [], 0
    for r, n in enumerate(lens):
        want.append(attention_of(q[at:at + n].reshape(n, heads, dim), cache.values("k", r), cache.values("v", r), held[r] - n, 0.1, 0, sinks))
        at += n
    want = torch.cat(want).flatten(1)
    on_device = wide.to(DEV)[:, lead:lead + heads * dim]
    for limit in (ops.BESIDE_8BIT_FLOPS, 0.0):
        monkeypatch.setattr(ops, "BESIDE_8BIT_FLOPS", limit)
        for told in (10, 9, 1, 0):
            out = torch.full((sum(lens), heads * dim + 3), 7.0, dtype=dtype, device=DEV)
            call(on_device, *cache.device(), cache.table.to(DEV), q_start, start_pos, positions, seq, 12, 70, 400, heads, kv, dim, 0.1, decode_prefix=told,
                 ctx_lens=held, sink=None if sinks is None else sinks.to(DEV), out=out[:, 3 if lead == 1 else 0:][:, :heads * dim])
            ops.check_status()
            found = out[:, 3 if lead == 1 else 0:][:, :heads * dim]
            assert rel_error(found, want) < TOL[dtype], (limit, told)
            assert (out[:, :3] == 7).all() if lead == 1 else (out[:, heads * dim:] == 7).all()
