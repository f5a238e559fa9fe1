"""The 4-bit cache at the ends of float32's range: norms, queries, sinks."""
import math

import pytest
import torch

import test_cache_8bit_gpu as eight
from helpers import TOL, batch_index, rel_error
from test_cache_4bit_gpu import DEV, Cache, attend, attention_of, ops, tables  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dim", [32, 64, 128, 256, 48])
def test_norms_of_large_rows(ops, dtype, dim):
    """A row times a power of two has the norm of the row, also where its squares are beyond float32: the same bits, in both kernels."""
    heads, kv, tokens = 2, 2, 9
    gen = torch.Generator().manual_seed(3)
    rows = torch.randn(tokens, 6 * dim, generator=gen).to(dtype).float().clamp(-4.0, 4.0)
    weight = (1.0 + 0.3 * torch.randn(dim, generator=gen)).to(DEV)
    positions, seq, _, _ = batch_index([tokens], [0], DEV)
    cache = Cache([tokens], kv, dim, 16)
    cos, sin = (t.to(DEV) for t in tables(64, dim))

    def stored(up, wide):
        x = rows.clone()
        x[:, :4 * dim] *= 2.0 ** up
        assert torch.isfinite(x).all()
        place = torch.zeros(tokens, 6 * dim + wide, dtype=dtype, device=DEV)
        place[:, wide:] = x.to(dtype)
        device = cache.device()
        q = ops.norm_rope_kv_store_4bit(place[:, wide:], cos, sin, dim, positions, seq, 1, cache.table.to(DEV), *device, heads, kv, dim,
                                        q_norm=weight, k_norm=weight, eps=2.0 ** -125)
        return [q, device[0], device[1], device[2].nan_to_num(0.0), device[3].nan_to_num(0.0)]

    want = stored(0, 0)
    x = rows[:, :2 * dim].double().view(tokens, 2, dim)
    norm = x / x.square().mean(-1, keepdim=True).sqrt() * weight.cpu().double()
    c, s = (t.cpu().double()[:tokens, None] for t in (cos, sin))
    lo, hi = norm[..., :dim // 2], norm[..., dim // 2:]
    turned = torch.cat([lo * c - hi * s, lo * s + hi * c], -1).flatten(1)
    assert rel_error(want[0], turned) < 2 * torch.finfo(dtype).eps + 2.0 ** -20
    for up in (-20, 40, 63, 64, 65, 100, 125):
        for wide in (0, 1):
            assert all(torch.equal(a, b) for a, b in zip(stored(up, wide), want)), (up, wide)
    ops.check_status()


def test_an_eps_that_float32_does_not_hold_is_refused(ops):
    cache = Cache([1], 1, 64, 16)
    positions, seq, _, _ = batch_index([1], [0], DEV)
    qkv, weight = torch.zeros(1, 3 * 64, device=DEV), torch.ones(64, device=DEV)
    store = lambda eps: ops.norm_rope_kv_store_4bit(qkv, None, None, 0, positions, seq, 1, cache.table.to(DEV), *cache.device(), 1, 1, 64, q_norm=weight, k_norm=weight, eps=eps)  # noqa: E731
    assert (store(1.2e-38) == 0).all()                       # a row of zeros
    for eps in (1e-39, 1e-50, 1e-300):
        with pytest.raises(ops.KernelError):
            store(eps)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dim", [64, 128, 256, 48])
@pytest.mark.parametrize("up", [112, 118, 120, 121, 122, 124])
def test_large_queries_over_small_keys(ops, dtype, dim, up):
    """Rows of queries up to the end of the range, over keys that make scores of ordinary size of them."""
    cache = Cache([300, 1, 90], 2, dim, 16)
    cache.pairs["k"] = (cache.pairs["k"].double() * 2.0 ** -up).bfloat16()
    out, want = attend(ops, cache, [1, 1, 1], 6, dtype, size=2.0 ** up, scale=0.09)
    assert rel_error(out, want) < TOL[dtype]


@pytest.mark.parametrize("heads,kv,dim", [(6, 2, 64), (8, 1, 128), (5, 1, 256), (24, 2, 128)])
@pytest.mark.parametrize("columns", [16, 130])
@pytest.mark.parametrize("size", [3.2e38, 2e36])
def test_large_queries_over_keys_of_ordinary_size(ops, heads, kv, dim, columns, size):
    """One head's queries near the end of bfloat16's range: its row is its best key's value, or NaN where float32 has no room for a score
    (in base-2 units); the others' rows are as they were."""
    cache = Cache([100, 1, 30], kv, dim, 64)
    wide = torch.full((3, columns), -1, dtype=torch.int32)
    wide[:, :cache.table.shape[1]] = cache.table
    positions, seq, q_start, start_pos = batch_index([1] * 3, [h - 1 for h in cache.held], DEV)
    q = torch.randn(3, heads, dim, generator=torch.Generator().manual_seed(5)).bfloat16()
    q[:, 1] = (q[:, 1].float() / q[:, 1].float().abs().amax(-1, keepdim=True) * size).bfloat16()
    assert torch.isfinite(q).all()
    scale = dim ** -0.5
    want = torch.cat([attention_of(q[r:r + 1], cache.values("k", r), cache.values("v", r), cache.held[r] - 1, scale, 0, None) for r in range(3)])
    room = []
    for r in range(3):
        scores = cache.values("k", r)[:, 0] @ q[r, 1].double()
        most = float(scores.abs().max()) * scale / math.log(2)
        assert not 3.4e38 < most < 3.41e38                  # (float32 ends between the two)
        room.append(most < 3.4e38)
        if r != 1:                  # the best key is best by far more than float32's sums are off
            best = scores.topk(2).values
            assert float(best[0] - best[1]) > 1e-3 * float(q[r, 1].double().abs().sum()) * 0.2
    assert all(room) or size > 1e38
    out = ops.attention_4bit(q.flatten(1).to(DEV), *cache.device(), wide.to(DEV), q_start, start_pos, positions, seq, 3, 1, 100, heads, kv, dim, scale)
    ops.check_status()
    out = out.view(3, heads, dim).cpu()
    for r in range(3):
        if not room[r]:
            assert torch.isnan(out[r, 1]).all()
            out[r, 1] = want[r, 1].to(out.dtype)
    assert rel_error(out, want) < TOL[torch.bfloat16]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dim,columns", [(64, 16), (64, 300), (128, 16), (128, 300), (80, 16)])
@pytest.mark.parametrize("bits", [4, 8])
def test_sinks_at_the_ends_of_the_range(ops, dtype, dim, columns, bits):
    """A sink of minus infinity is none, one far above every score leaves zeros; a row that sees nothing (its page is outside the pool, and
    reported) is zero under any."""
    heads, kv = 6, 2
    cache = Cache([100, 20, 5], kv, dim, 16) if bits == 4 else eight.Cache([100, 20, 5], kv, dim, 16, 1)
    table = torch.full((3, columns), -1, dtype=torch.int32)
    table[:, :cache.table.shape[1]] = cache.table
    table[2] = -1
    positions, seq, q_start, start_pos = batch_index([1] * 3, [99, 19, 4], DEV)
    q = (torch.randn(3, heads * dim, generator=torch.Generator().manual_seed(7)) * (1.0 if bits == 4 else 0.05)).to(dtype).to(DEV)
    call = ops.attention_4bit if bits == 4 else ops.attention_8bit

    def rows(sink):
        out = call(q, *cache.device(), table.to(DEV), q_start, start_pos, positions, seq, 3, 1, 100, heads, kv, dim, 0.1,
                   sink=None if sink is None else torch.tensor(sink, device=DEV))
        with pytest.raises(ops.DeviceStatusError):
            ops.check_status()
        return out.view(3, heads, dim)

    none = rows(None)
    assert (none[2] == 0).all() and torch.isfinite(none.float()).all()
    for sinks in ([-math.inf] * 6, [-3.4e38] * 6):
        assert torch.equal(rows(sinks), none)
    some = rows([math.inf, 3.4e38, 2.5e38, -math.inf, math.nan, 0.0])
    assert (some[:, :3] == 0).all() and torch.equal(some[:, 3], none[:, 3]) and torch.isnan(some[:, 4]).all()
    assert torch.isfinite(some[:, 5].float()).all() and (some[2, 5] == 0).all()


def test_a_window_beyond_whole_numbers_of_32_bits_is_refused(ops):
    cache = Cache([20], 2, 64, 16)
    positions, seq, q_start, start_pos = batch_index([1], [19], DEV)
    q = torch.zeros(1, 256, device=DEV)
    for window in (2 ** 31, 2 ** 32 + 5):
        with pytest.raises(ops.KernelError):
            ops.attention_4bit(q, *cache.device(), cache.table.to(DEV), q_start, start_pos, positions, seq, 1, 1, 20, 4, 2, 64, 0.1, window=window)
        with pytest.raises(ops.KernelError):
            ops.read_cache_4bit(*cache.device(), cache.table.to(DEV), q_start, start_pos, [20], 64, torch.float32, window=window)
    assert ops.attention_4bit(q, *cache.device(), cache.table.to(DEV), q_start, start_pos, positions, seq, 1, 1, 20, 4, 2, 64, 0.1, window=2 ** 31 - 1).shape == (1, 256)
    ops.check_status()
