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
