"""The 8-bit cache on the device against its definition in float64: store, reading back, attention, refusals."""
import math
import random

import pytest
import torch

from helpers import TOL, batch_index, rel_error
from plain import cache_8bit_plain as plain

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module")
def ops():
    from aegean_tge_b200 import ops as module
    module.core()
    return module


class Cache:
    """Random codes and scales of requests that hold ``held`` positions, on shuffled pages; what no request holds reads as NaN."""

    def __init__(self, held, kv_heads, dim, page, block, seed=0):
        gen = torch.Generator().manual_seed(seed)
        self.held, self.kv_heads, self.dim, self.page, self.block = held, kv_heads, dim, page, block
        need = [-(-n // page) for n in held]
        order = list(range(sum(need) + 3))
        random.Random(seed).shuffle(order)
        self.table = torch.full((len(held), max(max(need), 1)), -1, dtype=torch.int32)
        at = 0
        for r, n in enumerate(need):
            self.table[r, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
            at += n
        pages = len(order)
        self.codes = {n: (torch.randn(pages, kv_heads, page, dim, generator=gen) * 40).round().clamp(-127, 127).to(torch.int8) for n in "kv"}
        self.scales = {n: torch.full((pages, kv_heads, page // block), math.nan) for n in "kv"}
        for n in "kv":
            for r, count in enumerate(held):
                for b in range(-(-count // block)):
                    where = self.table[r, b * block // page]
                    self.scales[n][where, :, b * block % page // block] = 2.0 + torch.rand(kv_heads, generator=gen)

    def of(self, name, request, codes=None, scales=None):
        """(codes [held, kv, dim], scales [blocks, kv]) of one request."""
        codes, scales = (self.codes if codes is None else codes)[name].cpu(), (self.scales if scales is None else scales)[name].cpu()
        pos = torch.arange(self.held[request])
        where = self.table[request, pos // self.page].long()
        lead = pos[::self.block]
        return (codes[where, :, pos % self.page],
                scales[self.table[request, lead // self.page].long(), :, lead % self.page // self.block])

    def values(self, name, request, codes=None, scales=None):
        c, s = self.of(name, request, codes, scales)
        if not len(c):
            return torch.zeros(0, self.kv_heads, self.dim, dtype=torch.float64)
        return torch.stack([plain.values(c[:, h], s[:, h], self.block) for h in range(self.kv_heads)], 1)

    def device(self):
        return (self.codes["k"].to(DEV), self.codes["v"].to(DEV), self.scales["k"].to(DEV), self.scales["v"].to(DEV))


def tables(positions, rotary):
    angles = torch.arange(positions)[:, None].float() * (10000.0 ** (-torch.arange(0, rotary, 2).float() / max(rotary, 1)))
    return angles.cos(), angles.sin()


def store(ops, cache, qkv, starts, heads, rotary, cos, sin, lens, out=None):
    """Appends and compares scales, codes and rotated queries with the definition; returns the device's cache."""
    positions, seq, q_start, start_pos = batch_index(lens, starts, DEV)
    device = cache.device()
    kv, dim, block = cache.kv_heads, cache.dim, cache.block
    q = ops.rope_kv_store_8bit(qkv.to(DEV), cos.to(DEV) if rotary else None, sin.to(DEV) if rotary else None, rotary, positions, seq, q_start,
                               cache.table.to(DEV), *device, heads, kv, dim, out=out)
    after = {"k": device[0].cpu(), "v": device[1].cpu()}, {"k": device[2].cpu(), "v": device[3].cpu()}
    rows = qkv[:, :(heads + 2 * kv) * dim].double().view(len(qkv), heads + 2 * kv, dim)
    turned = torch.stack([plain.rotated(rows[t, :heads + kv], cos, sin, rotary, int(positions[t])) for t in range(len(qkv))])
    # one rounding to the output's type behind two products and a sum in float32
    assert rel_error(q, turned[:, :heads].flatten(1)) < (2 ** -8 if qkv.dtype == torch.bfloat16 else 3e-7)
    at = 0
    for r, (n, start) in enumerate(zip(lens, starts)):
        for name, new in (("k", turned[at:at + n, heads:]), ("v", rows[at:at + n, heads + kv:])):
            codes, scales = cache.of(name, r)
            got_codes, got_scales = cache.of(name, r, *after)
            for h in range(kv):
                want, wanted_scales = plain.append(codes[:, h].double(), scales[:, h].double(), new[:, h], start, block)
                s = got_scales[:, h].double()
                assert torch.equal(torch.isnan(s), torch.isnan(wanted_scales))
                fine = ~torch.isnan(s)
                # keys: products and a sum rounded in float32; values as they are
                assert ((s - wanted_scales).abs()[fine] <= 4e-7 * wanted_scales[fine]).all()
                off = (got_codes[:, h].double() - want).abs()
                # a code is the nearest whole number of a quotient that float32 knows to 127 * 2e-6 (a rotation that cancels
                # leaves an error relative to the block's largest, not to the number)
                assert not off.numel() or float(off.max()) <= 0.5 + 127 * 2e-6, (name, r, h, float(off.max()))
        at += n
    ops.check_status()
    return device, after


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("heads,kv,dim,rotary,page,block", [
    (28, 4, 128, 128, 64, 1), (40, 8, 128, 128, 16, 16), (12, 2, 128, 128, 32, 4), (4, 2, 64, 64, 64, 64), (3, 1, 16, 16, 8, 2),
    (5, 1, 256, 128, 64, 8), (6, 3, 80, 40, 16, 1), (2, 2, 10, 6, 4, 4), (2, 1, 33, 0, 64, 16)])
def test_store(ops, dtype, heads, kv, dim, rotary, page, block):
    lens, starts = [1, 1, 37, 5, 130, 64], [0, 77, 9, 3, 0, 64]
    cache = Cache([a + b for a, b in zip(lens, starts)], kv, dim, page, block)
    cos, sin = tables(300, rotary)
    gen = torch.Generator().manual_seed(3)
    qkv = torch.randn(sum(lens), (heads + 2 * kv) * dim + 16, generator=gen)          # the row goes on behind the values
    qkv[:, heads * dim] *= 20.0                                                       # scales that old blocks have to grow to
    qkv[7, (heads + kv) * dim:(heads + 2 * kv) * dim] = 0.0                           # a position of zeros
    store(ops, cache, qkv.to(dtype), starts, heads, rotary, cos, sin, lens)


@pytest.mark.parametrize("size", [1e-42, 1e-38, 1e-30, 1e30, 3e38])
@pytest.mark.parametrize("block", [1, 8])
def test_store_at_the_ends_of_the_range(ops, size, block):
    lens, starts = [3, 9], [5, 0]
    cache = Cache([8, 9], 2, 64, 16, block)
    cache.scales["k"] = torch.full_like(cache.scales["k"], size / 4)
    cache.scales["v"] = torch.full_like(cache.scales["v"], size * 0.3)
    gen = torch.Generator().manual_seed(4)
    qkv = ((torch.rand(12, 6 * 64, generator=gen).double() * 2 - 1) * size).float()
    store(ops, cache, qkv, starts, 2, 0, None, None, lens)


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("block", [1, 4])
def test_store_of_values_that_are_not_finite(ops, bad, block):
    """Their block reads as NaN, its neighbours do not; begun anew, the block forgets it."""
    lens, starts = [6, 7], [2, 0]
    cache = Cache([8, 7], 2, 64, 8, block)
    qkv = torch.randn(13, 6 * 64, generator=torch.Generator().manual_seed(5))
    qkv[3, 2 * 64 + 5] = bad              # a key of head 0 at position 5 of request 0
    qkv[8, 5 * 64 + 9] = bad              # a value of head 1 at position 2 of request 1
    device, _ = store(ops, cache, qkv, starts, 2, 0, None, None, lens)
    assert int(torch.isnan(device[2][cache.table[0, 0].item()]).sum()) == 1
    clean = torch.randn(7, 6 * 64, generator=torch.Generator().manual_seed(6))
    positions, seq, q_start, _ = batch_index([7], [0], DEV)
    ops.rope_kv_store_8bit(clean.to(DEV), None, None, 0, positions, seq, q_start, cache.table[1:].to(DEV), *device, 2, 2, 64)
    assert torch.isfinite(device[3][cache.table[1, 0].item(), :, :-(-7 // block)]).all()


def test_store_rows_of_an_inner_buffer(ops):
    """Odd row strides, starts that are no multiple of 16 bytes, an output inside a wider buffer; neighbours stay as they are."""
    heads, kv, dim = 4, 2, 64
    cache = Cache([40, 3], kv, dim, 16, 1)
    cos, sin = tables(64, dim)
    gen = torch.Generator().manual_seed(8)
    for dtype in (torch.bfloat16, torch.float32):
        for lead, width in ((1, 8 * 64 + 3), (8, 8 * 64 + 8), (0, 8 * 64 + 1)):
            rows = torch.randn(43, width, generator=gen).to(dtype).to(DEV)
            before = rows.clone()
            wide = torch.full((43, heads * dim + 5), 7.0, dtype=dtype, device=DEV)
            view = rows[:, lead:lead + 8 * 64] if width - lead >= 8 * 64 else rows
            store(ops, cache, view.cpu(), [0, 0], heads, dim, cos, sin, [40, 3], out=wide[:, 3:3 + heads * dim])
            assert (wide[:, :3] == 7).all() and (wide[:, 3 + heads * dim:] == 7).all()
            positions, seq, q_start, _ = batch_index([40, 3], [0, 0], DEV)
            d1, d2 = cache.device(), cache.device()
            a = ops.rope_kv_store_8bit(view, cos.to(DEV), sin.to(DEV), dim, positions, seq, q_start, cache.table.to(DEV), *d1, heads, kv, dim)
            b = ops.rope_kv_store_8bit(view.contiguous(), cos.to(DEV), sin.to(DEV), dim, positions, seq, q_start, cache.table.to(DEV), *d2, heads, kv, dim)
            assert torch.equal(a, b) and torch.equal(d1[0], d2[0]) and torch.equal(d1[1], d2[1])
            assert torch.equal(rows, before)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_entries_do_not_depend_on_the_cut_with_blocks_of_one(ops, dtype):
    heads, kv, dim, n = 4, 2, 128, 150
    cos, sin = tables(n, dim)
    qkv = torch.randn(n, 8 * dim, generator=torch.Generator().manual_seed(9)).to(dtype).to(DEV)
    found = []
    for cuts in ([150], [1] * 150, [64, 1, 85], [7, 63, 80]):
        cache = Cache([n], kv, dim, 16, 1)
        device, at, q = cache.device(), 0, []
        for count in cuts:
            positions, seq, q_start, _ = batch_index([count], [at], DEV)
            q.append(ops.rope_kv_store_8bit(qkv[at:at + count], cos.to(DEV), sin.to(DEV), dim, positions, seq, q_start, cache.table.to(DEV), *device, heads, kv, dim))
            at += count
        found.append([torch.cat(q)] + list(device[:2]) + [s.nan_to_num(0.0) for s in device[2:]])
    for other in found[1:]:
        assert all(torch.equal(a, b) for a, b in zip(found[0], other))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kv,dim,page,block,window", [(4, 128, 64, 1, 0), (2, 128, 16, 16, 100), (1, 16, 8, 2, 0), (3, 80, 4, 4, 70), (2, 33, 64, 64, 1), (1, 256, 32, 1, 0)])
def test_read_back(ops, dtype, kv, dim, page, block, window):
    held, lens = [1, 64, 65, 200, 0, 130] + [3] * 40, [1, 1, 65, 20, 0, 2] + [1] * 40
    cache = Cache(held, kv, dim, page, block)
    _, _, q_start, start_pos = batch_index(lens, [h - n for h, n in zip(held, lens)], DEV)
    for first in (0, 2, 44):
        k, v, table = ops.read_cache_8bit(*cache.device(), cache.table.to(DEV), q_start, start_pos, held, dtype, window=window, first_seq=first)
        for got, name in ((k, "k"), (v, "v")):
            for r in range(first, len(held)):
                seen = max(held[r] - lens[r] - window + 1, 0) // 64 if window else 0
                runs = table[r - first].tolist()
                want = cache.values(name, r)
                for i, run in enumerate(runs):
                    if i < seen or i >= -(-held[r] // 64):
                        assert run == -1
                        continue
                    part = got[run].transpose(0, 1).double().cpu()
                    n = min(64, held[r] - i * 64)
                    # one rounding to the output's type, two in float32 before it
                    assert rel_error(part[:n], want[i * 64:i * 64 + n]) < (2 ** -8 if dtype == torch.bfloat16 else 3e-7)
                    assert (part[n:] == 0).all()
    ops.check_status()


# ---------------------------------------------------------------------------
def attend(ops, cache, lens, heads, dtype, window=0, sink=False, scale=None, **kw):
    starts = [h - n for h, n in zip(cache.held, lens)]
    positions, seq, q_start, start_pos = batch_index(lens, starts, DEV)
    gen = torch.Generator().manual_seed(11)
    q = (torch.randn(sum(lens), heads * cache.dim, generator=gen) * 1.5).to(dtype)
    sinks = torch.randn(heads, generator=gen) if sink else None
    scale = cache.dim ** -0.5 if scale is None else scale
    out = ops.attention_8bit(q.to(DEV), *cache.device(), cache.table.to(DEV), q_start, start_pos, positions, seq, len(lens), max(lens), max(cache.held),
                             heads, cache.kv_heads, cache.dim, scale, window=window, sink=None if sinks is None else sinks.to(DEV), **kw)
    want, at = [], 0
    for r, n in enumerate(lens):
        want.append(plain.attend(q[at:at + n].view(n, heads, cache.dim), cache.values("k", r), cache.values("v", r), starts[r], scale, window, sinks))
        at += n
    ops.check_status()
    return out, torch.cat(want).flatten(1)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("heads,kv,dim", [(28, 4, 128), (40, 8, 128), (12, 2, 128), (14, 2, 64), (4, 2, 16), (3, 1, 32), (16, 1, 128), (33, 3, 128),
                                          (40, 2, 64), (6, 2, 80), (2, 2, 256), (4, 1, 33)])
def test_single_tokens(ops, dtype, heads, kv, dim):
    cache = Cache([1, 2, 7, 15, 16, 17, 63, 64, 65, 127, 128, 129, 300, 1000], kv, dim, 64, 1)
    out, want = attend(ops, cache, [1] * 14, heads, dtype)
    assert rel_error(out, want) < TOL[dtype]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("page,block", [(64, 64), (64, 4), (32, 1), (16, 16), (16, 2), (8, 8), (4, 1), (1, 1)])
@pytest.mark.parametrize("window,sink", [(0, False), (0, True), (1, False), (50, True), (128, False)])
def test_single_tokens_on_pages_blocks_windows(ops, dtype, page, block, window, sink):
    cache = Cache([1, 33, 64, 100, 513], 2, 128, page, block)
    out, want = attend(ops, cache, [1] * 5, 14, dtype, window=window, sink=sink)
    assert rel_error(out, want) < TOL[dtype]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("heads,kv,dim,page,block", [(28, 4, 128, 64, 1), (12, 2, 128, 16, 16), (4, 2, 16, 32, 4), (3, 1, 32, 8, 1), (6, 2, 80, 64, 2), (2, 1, 256, 64, 1)])
@pytest.mark.parametrize("window,sink", [(0, False), (33, True)])
def test_portions(ops, dtype, heads, kv, dim, page, block, window, sink):
    cache = Cache([40, 2, 65, 200, 129], kv, dim, page, block)
    out, want = attend(ops, cache, [40, 2, 64, 5, 1], heads, dtype, window=window, sink=sink)
    assert rel_error(out, want) < TOL[dtype]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("singles,told", [(9, 9), (9, 8), (2, 2), (9, 0)])
@pytest.mark.parametrize("window", [0, 40])
def test_single_tokens_beside_portions(ops, dtype, singles, told, window):
    """However many of the single tokens the caller tells of, and whether it tells the contexts."""
    held = [1, 5, 64, 65, 200, 17, 128, 90, 400][:singles] + [100, 70]
    cache = Cache(held, 2, 128, 16, 1)
    for ctx in (None, held):
        out, want = attend(ops, cache, [1] * singles + [30, 70], 14, dtype, window=window, decode_prefix=told, ctx_lens=ctx)
        assert rel_error(out, want) < TOL[dtype]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_peaked_and_shifted_scores(ops, dtype):
    """Scores in the hundreds: sums that start far below their maximum, and rows that are one key."""
    cache = Cache([700, 64, 1], 2, 128, 64, 1)
    for scale in (20.0, 1e-8):
        out, want = attend(ops, cache, [1, 1, 1], 8, dtype, scale=scale)
        # a score of some thousands is known to 2^-24 of the sum of its products' magnitudes
        assert rel_error(out, want) < (TOL[dtype] if dtype == torch.bfloat16 or scale < 1 else 2e-3)


def test_one_request_among_many_lengths(ops):
    cache = Cache([1 + 7 * i % 90 for i in range(300)], 2, 64, 16, 1)
    out, want = attend(ops, cache, [1] * 300, 8, torch.bfloat16)
    assert rel_error(out, want) < TOL[torch.bfloat16]


def test_long_contexts(ops):
    """Against float64 on the device: 40,000 positions, offsets of entries beyond 2^31 bytes."""
    kv, dim, heads, page = 2, 128, 8, 64
    pages = 2 ** 31 // (kv * page * dim) + 700
    codes = torch.empty(pages, kv, page, dim, dtype=torch.int8, device=DEV).random_(-127, 128)
    scales = torch.rand(pages, kv, page, device=DEV) + 1.0
    held = [40000, 39, 3000]
    table = torch.full((3, 625), -1, dtype=torch.int32)
    table[0, :625] = torch.arange(pages - 1, pages - 626, -1)
    table[1, :1] = 5
    table[2, :47] = torch.arange(pages - 700, pages - 653)
    q = torch.randn(3, heads * dim, device=DEV).bfloat16()
    positions, seq, q_start, start_pos = batch_index([1, 1, 1], [n - 1 for n in held], DEV)
    out = ops.attention_8bit(q, codes, codes, scales, scales, table.to(DEV), q_start, start_pos, positions, seq, 3, 1, 40000, heads, kv, dim, 0.05)
    for r, n in enumerate(held):
        pos = torch.arange(n, device=DEV)
        where = table[r].to(DEV)[pos // page].long()
        k = codes[where, :, pos % page].double() * scales[where, :, pos % page].double()[..., None] / 127
        p = torch.softmax(torch.einsum("kgd,ckd->kgc", q[r].double().view(kv, 4, dim), k) * 0.05, -1)
        assert rel_error(out[r], torch.einsum("kgc,ckd->kgd", p, k).flatten()) < TOL[torch.bfloat16]
    ops.check_status()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_block_that_reads_as_nan_reaches_only_who_sees_it(ops, dtype):
    cache = Cache([100, 100, 100], 2, 128, 16, 1)
    cache.scales["v"][cache.table[0, 2].item(), 1, 3] = math.nan           # position 35 of request 0, head 1
    cache.scales["k"][cache.table[1, 1].item(), 0, 0] = math.nan           # position 16 of request 1, head 0
    lens, heads = [1, 1, 1], 8
    positions, seq, q_start, start_pos = batch_index(lens, [99] * 3, DEV)
    q = torch.randn(3, heads * 128, generator=torch.Generator().manual_seed(1)).to(dtype).to(DEV)
    for window in (0, 64):
        out = ops.attention_8bit(q, *cache.device(), cache.table.to(DEV), q_start, start_pos, positions, seq, 3, 1, 100, heads, 2, 128, 0.09, window=window)
        nan = torch.isnan(out.view(3, heads, 128)).all(-1).cpu()
        some = torch.isnan(out.view(3, heads, 128)).any(-1).cpu()
        want = torch.zeros(3, heads, dtype=torch.bool)
        if not window:
            want[0, 4:], want[1, :4] = True, True
        assert torch.equal(nan, want) and torch.equal(some, want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("lens", [[1, 1], [3, 20]])
def test_pages_outside_the_pool_are_reported_not_read(ops, dtype, lens):
    cache = Cache([50, 80], 2, 128, 16, 1)
    table = cache.table.clone()
    table[0] = torch.tensor([-1, 9999, -7, 10 ** 6, -1])
    positions, seq, q_start, start_pos = batch_index(lens, [50 - lens[0], 80 - lens[1]], DEV)
    q = torch.randn(sum(lens), 8 * 128).to(dtype).to(DEV)
    args = (q_start, start_pos, positions, seq, 2, max(lens), 80, 8, 2, 128, 0.1)
    good = ops.attention_8bit(q, *cache.device(), cache.table.to(DEV), *args)
    ops.check_status()
    out = ops.attention_8bit(q, *cache.device(), table.to(DEV), *args)
    with pytest.raises(ops.DeviceStatusError):
        ops.check_status()
    assert (out[:lens[0]] == 0).all() and torch.equal(out[lens[0]:], good[lens[0]:])
    device = cache.device()
    before = [t.clone() for t in device]
    ops.rope_kv_store_8bit(torch.randn(lens[0], 12 * 128).to(dtype).to(DEV), None, None, 0, positions[:lens[0]], seq[:lens[0]], q_start[:2].clone(), table.to(DEV), *device, 8, 2, 128)
    with pytest.raises(ops.DeviceStatusError):
        ops.check_status()
    assert all(torch.equal(a.nan_to_num(0) if a.is_floating_point() else a, b.nan_to_num(0) if b.is_floating_point() else b) for a, b in zip(before, device))


def test_positions_outside_the_tables_are_reported(ops):
    cache = Cache([70], 2, 64, 16, 1)
    cos, sin = tables(50, 64)
    positions, seq, q_start, _ = batch_index([1], [60], DEV)
    device = cache.device()
    ops.rope_kv_store_8bit(torch.randn(1, 6 * 64).to(DEV), cos.to(DEV), sin.to(DEV), 64, positions, seq, q_start, cache.table.to(DEV), *device, 2, 2, 64)
    with pytest.raises(ops.DeviceStatusError):
        ops.check_status()
    assert torch.equal(device[0].cpu(), cache.codes["k"])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_on_a_stream_of_its_own_and_again(ops, dtype):
    """On another stream than the default, with rows of an inner buffer: the same bits."""
    cache = Cache([200, 65, 3, 90], 2, 128, 64, 1)
    lens = [1, 1, 1, 1]
    positions, seq, q_start, start_pos = batch_index(lens, [h - 1 for h in cache.held], DEV)
    wide = torch.randn(4, 8 * 128 + 24, generator=torch.Generator().manual_seed(2)).to(dtype).to(DEV)
    device, table = cache.device(), cache.table.to(DEV)
    args = (*device, table, q_start, start_pos, positions, seq, 4, 1, 200, 8, 2, 128, 0.1)
    first = ops.attention_8bit(wide[:, 8:8 + 1024].contiguous(), *args)
    odd = ops.attention_8bit(wide[:, 8:8 + 1024], *args)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        again = ops.attention_8bit(wide[:, 8:8 + 1024], *args)
    side.synchronize()
    assert torch.equal(first, odd) and torch.equal(first, again)
    into = torch.zeros(4, 1024 + 8, dtype=dtype, device=DEV)
    ops.attention_8bit(wide[:, 8:8 + 1024], *args, out=into[:, 8:])
    assert torch.equal(into[:, 8:], first) and (into[:, :8] == 0).all()
    # rows that start on odd elements
    odd_rows = torch.zeros(4, 1024 + 1, dtype=dtype, device=DEV)
    odd_rows[:, 1:] = wide[:, 8:8 + 1024]
    assert rel_error(ops.attention_8bit(odd_rows[:, 1:], *args), first) < TOL[dtype]


def test_nothing_to_do(ops):
    cache = Cache([5], 2, 64, 16, 1)
    empty = lambda *shape: torch.empty(shape, dtype=torch.bfloat16, device=DEV)  # noqa: E731
    none = torch.empty(0, dtype=torch.int32, device=DEV)
    start = torch.zeros(1, dtype=torch.int32, device=DEV)
    assert ops.rope_kv_store_8bit(empty(0, 6 * 64), None, None, 0, none, none, start, cache.table.to(DEV), *cache.device(), 2, 2, 64).shape == (0, 128)
    assert ops.attention_8bit(empty(0, 128), *cache.device(), cache.table.to(DEV), start, none, none, none, 0, 0, 0, 2, 2, 64, 0.1).shape == (0, 128)
    k, _v, table = ops.read_cache_8bit(*cache.device(), cache.table.to(DEV), start, none, [], torch.bfloat16)
    assert k.shape == (0, 2, 64, 64) and table.shape == (0, 0)


def test_refusals(ops):
    cache = Cache([20], 2, 64, 16, 1)
    kp, vp, ks, vs = cache.device()
    table = cache.table.to(DEV)
    positions, seq, q_start, start_pos = batch_index([1], [19], DEV)
    q = torch.zeros(1, 4 * 64, dtype=torch.bfloat16, device=DEV)
    qkv = torch.zeros(1, 8 * 64, dtype=torch.bfloat16, device=DEV)

    def attention(q=q, kp=kp, vp=vp, ks=ks, vs=vs, table=table, q_start=q_start, positions=positions, seqs=1, heads=4, kv=2, dim=64, **kw):
        return ops.attention_8bit(q, kp, vp, ks, vs, table, q_start, start_pos, positions, seq, seqs, 1, 20, heads, kv, dim, 0.1, **kw)

    def stored(qkv=qkv, kp=kp, vp=vp, ks=ks, vs=vs, rotary=0, cos=None, sin=None, positions=positions, **kw):
        return ops.rope_kv_store_8bit(qkv, cos, sin, rotary, positions, seq, q_start, table, kp, vp, ks, vs, 4, 2, 64, **kw)

    attention(), stored()
    wrong = [
        lambda: attention(q=q.half()), lambda: attention(q=q.cpu()), lambda: attention(kp=kp.float()), lambda: attention(kp=kp[:, :1]),
        lambda: attention(vp=vp[:1]), lambda: attention(ks=ks.double()), lambda: attention(ks=ks[:, :, :5].contiguous()),
        lambda: attention(vs=vs[:, :, :8].contiguous()), lambda: attention(ks=ks[:, :, :0], vs=vs[:, :, :0]), lambda: attention(heads=5), lambda: attention(heads=8),
        lambda: attention(seqs=2), lambda: attention(positions=positions.long()), lambda: attention(q_start=q_start[:1]), lambda: attention(ctx_lens=[20, 20]),
        lambda: attention(sink=torch.zeros(3, device=DEV)), lambda: attention(window=-1), lambda: attention(decode_prefix=2),
        lambda: attention(out=torch.zeros(1, 5, dtype=torch.bfloat16, device=DEV)), lambda: attention(out=torch.zeros(1, 256, device=DEV)),
        lambda: attention(dim=32), lambda: attention(table=table.long()),
        lambda: stored(qkv=qkv[:, :7 * 64]), lambda: stored(qkv=qkv.int()), lambda: stored(rotary=64), lambda: stored(rotary=3, cos=torch.zeros(30, 1, device=DEV), sin=torch.zeros(30, 1, device=DEV)),
        lambda: stored(rotary=66, cos=torch.zeros(30, 33, device=DEV), sin=torch.zeros(30, 33, device=DEV)), lambda: stored(kp=kp.to(torch.uint8)),
        lambda: stored(positions=positions[:0]), lambda: stored(out=torch.zeros(1, 5, dtype=torch.bfloat16, device=DEV)), lambda: stored(ks=ks.transpose(1, 2)),
        lambda: ops.read_cache_8bit(kp, vp, ks, vs, table, q_start, start_pos, [20], torch.float16),
        lambda: ops.read_cache_8bit(kp, vp, ks, vs, table, q_start, start_pos, [20, 20], torch.float32),
    ]
    for call in wrong:
        with pytest.raises((ops.KernelError, AttributeError, TypeError)):
            call()
    three = torch.zeros(4, 2, 3, 64, dtype=torch.int8, device=DEV), torch.zeros(4, 2, 1, device=DEV)      # a block of three
    with pytest.raises(ops.KernelError):
        attention(kp=three[0], vp=three[0], ks=three[1], vs=three[1])
    wide = torch.zeros(4, 2, 16, 320, dtype=torch.int8, device=DEV), torch.zeros(4, 2, 16, device=DEV)
    with pytest.raises(ops.KernelError):
        attention(q=torch.zeros(1, 4 * 320, device=DEV), kp=wide[0], vp=wide[0], ks=wide[1], vs=wide[1], dim=320)
    ops.check_status()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("heads,kv,dim", [(14, 2, 128), (6, 2, 32)])
def test_side_by_side_is_the_same(ops, monkeypatch, dtype, heads, kv, dim):
    """Single tokens beside portions on two streams: the bits of one, from any stream, time and again; head sizes that only the portions'
    kernels take as well."""
    held = [1, 5, 64, 65, 200, 17, 128, 90, 400, 33, 300, 270]
    lens = [1] * 10 + [200, 64]
    cache = Cache(held, kv, dim, 16, 1)
    want, _ = attend(ops, cache, lens, heads, dtype, decode_prefix=10, ctx_lens=held)
    monkeypatch.setattr(ops, "BESIDE_8BIT_FLOPS", 0.0)
    for _ in range(4):
        got, _ = attend(ops, cache, lens, heads, dtype, decode_prefix=10, ctx_lens=held)
        assert torch.equal(got, want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got, _ = attend(ops, cache, lens, heads, dtype, decode_prefix=10, ctx_lens=held)
    side.synchronize()
    if dim == 128:
        assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("heads,kv,dim", [(14, 2, 128), (6, 2, 64), (6, 2, 32), (4, 2, 80), (2, 2, 256)])
@pytest.mark.parametrize("window", [0, 50])
def test_a_block_that_reads_as_nan_in_a_portion(ops, dtype, heads, kv, dim, window):
    """Rows in front of it, rows behind its window and other requests do not see it, in whatever tile of keys it lies."""
    held, lens = [300, 150, 70], [300, 90, 6]
    cache = Cache(held, kv, dim, 16, 1)
    bad = {0: (170, "v"), 1: (63, "k"), 2: (66, "v")}
    for request, (pos, name) in bad.items():
        cache.scales[name][cache.table[request, pos // 16].item(), 1, pos % 16] = math.nan
    positions, seq, q_start, start_pos = batch_index(lens, [h - n for h, n in zip(held, lens)], DEV)
    q = torch.randn(sum(lens), heads * dim, generator=torch.Generator().manual_seed(1)).to(dtype).to(DEV)
    out = ops.attention_8bit(q, *cache.device(), cache.table.to(DEV), q_start, start_pos, positions, seq, 3, 300, 300, heads, kv, dim, 0.09, window=window, ctx_lens=held)
    nan = torch.isnan(out.view(-1, heads, dim)).cpu()
    want, at = torch.zeros(sum(lens), heads, dtype=torch.bool), 0
    for r, n in enumerate(lens):
        for i in range(n):
            pos = held[r] - n + i
            sees = bad[r][0] <= pos and (not window or bad[r][0] > pos - window)
            want[at + i, heads // kv:2 * (heads // kv)] = sees
        at += n
    assert torch.equal(nan.all(-1), want) and torch.equal(nan.any(-1), want)


@pytest.mark.parametrize("splits", [128, 192])
def test_portions_whose_keys_are_cut(ops, monkeypatch, splits):
    """The runs of keys that a short portion deep in a long context is cut into, and their merging."""
    monkeypatch.setattr(ops, "choose_attention_split", lambda *a, **k: splits)
    cache = Cache([700, 64, 1000], 2, 128, 64, 1)
    out, want = attend(ops, cache, [9, 64, 30], 14, torch.bfloat16, ctx_lens=[700, 64, 1000], sink=True)
    assert rel_error(out, want) < TOL[torch.bfloat16]


@pytest.mark.parametrize("heads,kv,dim", [(14, 2, 128), (6, 2, 64)])
@pytest.mark.parametrize("window", [0, 70])
def test_portions_over_scales_far_apart(ops, heads, kv, dim, window, first=(0, 30, -30, 0, 5, 60, -60, 1, 0, -1)):
    """Values whose size changes by up to 2^120 from one run of 64 positions to the next, keys by 2^3; queries of 2^60 over keys of 2^-60."""
    held, lens = [640, 150, 130], [600, 150, 6]
    cache = Cache(held, kv, dim, 64, 1)
    for r, (size, sizes) in enumerate(zip((60, 0, -60), (first, [-40, 20, 0], [1, 0, -100]))):
        for run, f in enumerate(sizes):
            where = cache.table[r, run].item()
            cache.scales["v"][where] *= 2.0 ** f
            cache.scales["k"][where] *= 2.0 ** (run % 4 - size)
    positions, seq, q_start, start_pos = batch_index(lens, [h - n for h, n in zip(held, lens)], DEV)
    q = torch.randn(sum(lens), heads * dim, generator=torch.Generator().manual_seed(2))
    q = (q * 2.0 ** torch.tensor([60.0, 0, -60]).repeat_interleave(torch.tensor(lens))[:, None]).bfloat16()
    out = ops.attention_8bit(q.to(DEV), *cache.device(), cache.table.to(DEV), q_start, start_pos, positions, seq, 3, 600, 640, heads, kv, dim, 0.02,
                             window=window, ctx_lens=held)
    ops.check_status()
    at = 0
    for r, n in enumerate(lens):
        k, v, rows = cache.values("k", r), cache.values("v", r), q[at:at + n].view(n, heads, dim)
        want = plain.attend(rows, k, v, held[r] - n, 0.02, window, None)
        # a row and head's error against the largest sum of probabilities times magnitudes: each product's roundings are of its own size
        size = plain.attend(rows, k, v.abs(), held[r] - n, 0.02, window, None).amax(-1)
        error = (out[at:at + n].cpu().double().view(n, heads, dim) - want).abs().amax(-1)
        assert float((error / size).max()) < 2 ** -7
        at += n


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("heads,kv,dim", [(8, 1, 128), (14, 2, 64), (5, 1, 256), (24, 2, 128)])
@pytest.mark.parametrize("columns", [16, 33, 64, 66, 128, 130])
@pytest.mark.parametrize("window,sink", [(0, True), (70, False)])
def test_single_tokens_under_every_bound(ops, dtype, heads, kv, dim, columns, window, sink):
    """The bound of the contexts (the block table's columns, of 64 positions here) decides how a unit's keys are shared out: clusters of 8 and 16
    blocks, runs; requests of one position, of less than a slice to a block, of more."""
    cache = Cache([1, 17, 1000, 130, 64], kv, dim, 64, 1)
    wide = torch.full((5, columns), -1, dtype=torch.int32)
    wide[:, :cache.table.shape[1]] = cache.table
    cache.table = wide
    out, want = attend(ops, cache, [1] * 5, heads, dtype, window=window, sink=sink)
    assert rel_error(out, want) < TOL[dtype]


@pytest.mark.parametrize("columns", [16, 66, 130])
def test_a_page_outside_the_pool_under_every_bound(ops, columns):
    """A unit whose keys are partly or wholly outside the pool: reported, unread, zero where nothing is seen."""
    cache = Cache([40, 300], 1, 128, 64, 1)
    wide = torch.full((2, columns), -1, dtype=torch.int32)
    wide[1, :5] = cache.table[1, :5]
    positions, seq, q_start, start_pos = batch_index([1, 1], [39, 299], DEV)
    q = torch.randn(2, 8 * 128, device=DEV).bfloat16()
    out = ops.attention_8bit(q, *cache.device(), wide.to(DEV), q_start, start_pos, positions, seq, 2, 1, 300, 8, 1, 128, 0.09)
    with pytest.raises(ops.DeviceStatusError, match="page"):
        ops.check_status()
    assert (out[0] == 0).all()
    want = plain.attend(q[1:].cpu().view(1, 8, 128), cache.values("k", 1), cache.values("v", 1), 299, 0.09, 0, None)
    assert rel_error(out[1:], want.flatten(1)) < TOL[torch.bfloat16]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("lens", [[1, 0, 1, 0], [0, 1, 1, 0], [0, 0, 1, 0], [3, 0, 70, 0]])
@pytest.mark.parametrize("columns", [16, 130])
@pytest.mark.parametrize("block", [1, 16])
def test_requests_that_bring_nothing(ops, dtype, lens, columns, block):
    """In front of, between and behind others, with and without a context of their own: no row is theirs, nothing of theirs changes."""
    heads, kv, dim = 6, 2, 128
    cache = Cache([100, 64, 80, 0], kv, dim, 16, block)
    wide = torch.full((4, 4 * columns), -1, dtype=torch.int32)
    wide[:, :cache.table.shape[1]] = cache.table
    cache.table = wide
    starts = [h - n for h, n in zip(cache.held, lens)]
    cos, sin = tables(100, dim)
    qkv = torch.randn(sum(lens), (heads + 2 * kv) * dim, generator=torch.Generator().manual_seed(3)).to(dtype)
    _, after = store(ops, cache, qkv, starts, heads, dim, cos, sin, lens)
    for r in (r for r in range(4) if lens[r] == 0):
        for name in "kv":
            assert all(torch.equal(a, b) for a, b in zip(cache.of(name, r), cache.of(name, r, *after)))
    out, want = attend(ops, cache, lens, heads, dtype, ctx_lens=cache.held)
    assert rel_error(out, want) < TOL[dtype]
    positions, seq, q_start, start_pos = batch_index(lens, starts, DEV)
    k, _, table = ops.read_cache_8bit(*cache.device(), cache.table.to(DEV), q_start, start_pos, cache.held, torch.float32)
    ops.check_status()
    assert [(row >= 0).sum().item() for row in table] == [2, 1, 2, 0] and k.shape[0] == 5


def test_attention_over_a_cache_that_was_read_back(ops):
    """The read-back's block table right in front of an attention kernel, which looks tables up ahead of its wait: many runs, time and again."""
    heads, kv, dim = 6, 2, 128
    held = [4000, 900, 64, 2000] * 4
    cache = Cache(held, kv, dim, 64, 1)
    positions, seq, q_start, start_pos = batch_index([1] * 16, [h - 1 for h in held], DEV)
    q = torch.randn(16, heads * dim, generator=torch.Generator().manual_seed(5)).bfloat16().to(DEV)
    device, table = cache.device(), cache.table.to(DEV)
    want = ops.attention_8bit(q, *device, table, q_start, start_pos, positions, seq, 16, 1, 4000, heads, kv, dim, 0.05)
    for _ in range(20):
        k, v, runs = ops.read_cache_8bit(*device, table, q_start, start_pos, held, torch.bfloat16)
        out = ops.attention(q, k, v, runs, q_start, start_pos, positions, seq, 16, 1, 4000, heads, kv, dim, 0.05)
        runs.fill_(-1)
        assert rel_error(out, want) < TOL[torch.bfloat16]
    ops.check_status()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("lens", [[1, 1, 1], [40, 1, 70]])
@pytest.mark.parametrize("values,keys", [(1e-35, 1.0), (1e35, 1.0), (1.0, 1e-25), (1e-32, 1e25)])
def test_attention_at_the_ends_of_the_range(ops, dtype, lens, values, keys):
    """Values of very small and large scales; keys of them under queries that make up for it."""
    heads, kv, dim = 6, 2, 128
    cache = Cache([300, 1, 90], kv, dim, 64, 1)
    cache.scales["v"] *= values
    cache.scales["k"] *= keys
    positions, seq, q_start, start_pos = batch_index(lens, [h - n for h, n in zip(cache.held, lens)], DEV)
    q = (torch.randn(sum(lens), heads * dim, generator=torch.Generator().manual_seed(9)) * (0.5 / keys)).to(dtype)
    out = ops.attention_8bit(q.to(DEV), *cache.device(), cache.table.to(DEV), q_start, start_pos, positions, seq, 3, max(lens), 300, heads, kv, dim, 0.09)
    ops.check_status()
    want, at = [], 0
    for r, n in enumerate(lens):
        want.append(plain.attend(q[at:at + n].view(n, heads, dim), cache.values("k", r), cache.values("v", r), cache.held[r] - n, 0.09, 0, None))
        at += n
    want = torch.cat(want).flatten(1)
    assert rel_error(out.cpu().double() / values, want / values) < TOL[dtype]


@pytest.mark.parametrize("first", [(100, 20, -60, -100, 40, 100, 10, -70, 0, 90), (-100, -20, 60, 110, 30, -50, -110, 0, 80, -80)])
@pytest.mark.parametrize("window", [0, 70, 200])
def test_portions_over_scales_that_fall_and_rise(ops, window, first):
    """By 2^80 and more from run to run, several times in a row."""
    test_portions_over_scales_far_apart(ops, 14, 2, 128, window, first)


def released(cache, lens, window):
    """The cache's table as its manager leaves it over a window: pages wholly behind the first query's window are given back."""
    table = cache.table.clone()
    for r, (held, n) in enumerate(zip(cache.held, lens)):
        table[r, :max(held - n - window + 1, 0) // cache.page] = -1
    return table


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("heads,kv,dim", [(14, 2, 128), (6, 2, 64), (4, 2, 80), (2, 1, 256)])
@pytest.mark.parametrize("page,window", [(16, 100), (32, 33), (16, 1)])
def test_windows_over_released_pages(ops, dtype, heads, kv, dim, page, window):
    """Pages behind the window are nobody's: not read, and no fault of the call's.  One that a query sees is."""
    lens = [70, 1, 30, 65, 40, 2]
    cache = Cache([200, 150, 290, 65, 350, 131], kv, dim, page, 1)
    cache.table = released(cache, lens, window)
    out, want = attend(ops, cache, lens, heads, dtype, window=window, ctx_lens=cache.held)
    assert rel_error(out, want) < TOL[dtype]
    positions, seq, q_start, start_pos = batch_index(lens, [h - n for h, n in zip(cache.held, lens)], DEV)
    ops.read_cache_8bit(*cache.device(), cache.table.to(DEV), q_start, start_pos, cache.held, dtype, window=window)
    ops.check_status()
    missing = cache.table.clone()
    missing[4, (350 - 40 - window + 1) // page] = -1
    with pytest.raises(ops.DeviceStatusError, match="page"):
        ops.read_cache_8bit(*cache.device(), missing.to(DEV), q_start, start_pos, cache.held, dtype, window=window)
        ops.check_status()


def known_rows(q, k, v, start, scale, window):
    """[new, heads]: rows whose result float16's rounding of keys (2^-12 of each product, and half of that again for the sums) does not decide: neither the
    probabilities nor their products with the values' magnitudes."""
    new, heads = q.shape[:2]
    out = torch.zeros(new, heads, dtype=torch.bool)
    for h in range(heads):
        kvh = h // (heads // k.shape[1])
        s, off = (torch.einsum("id,jd->ij", f(q[:, h].double()), f(k[:, kvh].double())) * scale for f in (lambda x: x, torch.abs))
        pos, key = start + torch.arange(new)[:, None], torch.arange(len(k))
        s = s.masked_fill((key > pos) | (key <= pos - (window or 1 << 30)), -math.inf)
        top = s.argmax(-1, keepdim=True)
        weight = torch.maximum(torch.log_softmax(s, -1), torch.log_softmax(s + v[:, kvh].abs().amax(-1).log(), -1))
        off = off * 2.0 ** -11
        moved = torch.exp((weight + torch.log(torch.expm1((2 * (off + off.gather(1, top))).clamp_max(700)))).scatter(1, top, -math.inf)).sum(-1)
        out[:, h] = moved < 2 ** -8
    return out


def row_errors(out, q, cache, lens, heads, scale, window=0, known=None):
    """Of every row and head the error over the sum of its probabilities times magnitudes of values, the largest number's; with ``known`` (the least
    share of such rows) only of rows whose scores float16 keys tell."""
    worst, at = 0.0, 0
    for r, n in enumerate(lens):
        k, v, rows = cache.values("k", r), cache.values("v", r), q[at:at + n].view(n, heads, cache.dim)
        want = plain.attend(rows, k, v, cache.held[r] - n, scale, window, None)
        size = plain.attend(rows, k, v.abs(), cache.held[r] - n, scale, window, None).amax(-1)
        got = out[at:at + n].cpu().double().view(n, heads, cache.dim)
        assert torch.isfinite(got).all()
        error = (got - want).abs().amax(-1) / size
        if known is not None:
            told = known_rows(rows, k, v, cache.held[r] - n, scale, window)
            assert float(told.double().mean()) >= known
            error = error[told]
        worst = max(worst, float(error.max()))
        at += n
    return worst


def portions_of(ops, cache, lens, heads, q, scale, window=0):
    positions, seq, q_start, start_pos = batch_index(lens, [h - n for h, n in zip(cache.held, lens)], DEV)
    out = ops.attention_8bit(q.to(DEV), *cache.device(), cache.table.to(DEV), q_start, start_pos, positions, seq, len(lens), max(lens), max(cache.held),
                             heads, cache.kv_heads, cache.dim, scale, window=window, ctx_lens=cache.held)
    ops.check_status()
    return out


@pytest.mark.parametrize("heads,kv,dim", [(14, 2, 128), (6, 2, 64)])
@pytest.mark.parametrize("powers", [(-70, 70, -70), (-100, 100, 0), (100, -100, 100), (0, 115, -115), (-120, 120, -120)])
@pytest.mark.parametrize("window", [0, 70])
def test_portions_over_scales_that_jump_inside_a_block_of_queries(ops, heads, kv, dim, powers, window):
    """Values whose size changes by up to 2^240 where one run of 64 positions ends and the next begins: rows that see the next run and rows that do not
    lie in one block of queries."""
    held = lens = [192, 100]
    cache = Cache(held, kv, dim, 64, 1)
    for r in range(2):
        for run in range(cache.table.shape[1]):
            if cache.table[r, run] >= 0:
                cache.scales["v"][cache.table[r, run].item()] *= 2.0 ** powers[run]
    q = (torch.randn(sum(lens), heads * dim, generator=torch.Generator().manual_seed(4))).bfloat16()
    out = portions_of(ops, cache, lens, heads, q, 0.02, window)
    assert row_errors(out, q, cache, lens, heads, 0.02, window) < 2 ** -7


@pytest.mark.parametrize("far", [60, 100, 200, 400])
@pytest.mark.parametrize("base,power", [(0, 20), (0, 60), (0, 120), (-110, 230)])
@pytest.mark.parametrize("order", [(0, 1), (1, 0)])
def test_portions_that_hardly_weigh_a_run_of_large_values(ops, far, base, power, order):
    """A run whose values are 2^120 the others' size and more, and whose scores lie far below theirs."""
    heads, kv, dim, held = 4, 2, 128, [128]
    cache = Cache(held, kv, dim, 64, 1)
    codes = torch.randint(-127, 128, (dim,), generator=torch.Generator().manual_seed(3)).to(torch.int8)
    near, away = (cache.table[0, i].item() for i in order)
    cache.codes["k"][near], cache.codes["k"][away] = codes, -codes
    cache.scales["k"].fill_(1.0)
    cache.scales["v"][near] *= 2.0 ** base
    cache.scales["v"][away] *= 2.0 ** (base + power)
    q = (codes.float() / 127).repeat(128, heads, 1).flatten(1).bfloat16()
    scale = far / 2 * math.log(2) / float((codes.float() / 127).pow(2).sum())            # scores of far / 2 and its negative, in powers of two
    out = portions_of(ops, cache, held, heads, q, scale)
    assert row_errors(out, q, cache, held, heads, scale) < 2 ** -7


@pytest.mark.parametrize("window", [0, 40])
@pytest.mark.parametrize("keys,queries,scale", [(-90, -90, 0.09), (-120, -60, 0.09), (-60, -120, 0.09), (-120, 118, 2.0), (-128, 118, 300.0)])
def test_portions_of_queries_and_keys_at_the_ends_of_the_range(ops, window, keys, queries, scale):
    """Scores that float32 has no number for are zeros: every key weighs the same, and masked ones nothing.  Queries whose product with the scale alone
    float32 has no number for."""
    heads, kv, dim, held = 6, 2, 128, [150]
    cache = Cache(held, kv, dim, 64, 1)
    cache.scales["k"] *= 2.0 ** keys
    q = (torch.randn(150, heads * dim, generator=torch.Generator().manual_seed(6)) * 2.0 ** queries).bfloat16()
    out = portions_of(ops, cache, held, heads, q, scale, window)
    assert row_errors(out, q, cache, held, heads, scale, window) < 2 ** -7


# A row and head's error: the result, the probabilities and the entries are rounded to 2^-9, 2^-12 and 2^-12, a score of some tens is known to 2^-12 of it.
@pytest.mark.parametrize("heads,kv,dim", [(14, 2, 128), (6, 2, 64)])
@pytest.mark.parametrize("block", [1, 4])
@pytest.mark.parametrize("keys,values", [(0, 8), (0, 14), (0, 20), (20, 0), (12, 12), (0, -20), (-20, -9), (0, 100), (-30, 60), (50, 90)])
@pytest.mark.parametrize("window", [0, 70])
def test_portions_over_scales_far_apart_inside_a_run(ops, heads, kv, dim, block, keys, values, window):
    """One block of positions whose keys and values are 2^20 (more, less) the others' size: rows in front of it, behind it and behind its window."""
    held, lens = [200, 150, 130], [200, 90, 6]
    cache = Cache(held, kv, dim, 64, block)
    for name, power in (("k", keys), ("v", values)):
        cache.scales[name] *= 2.0 ** (-max(power, 0) / 2)
        for r, pos in enumerate((41, 70, 127)):
            cache.scales[name][cache.table[r, pos // 64].item(), :, pos % 64 // block] *= 2.0 ** power
    q = (torch.randn(sum(lens), heads * dim, generator=torch.Generator().manual_seed(2)) * 2.0 ** (max(keys, 0) / 2)).bfloat16()
    out = portions_of(ops, cache, lens, heads, q, 0.02, window)
    assert row_errors(out, q, cache, lens, heads, 0.02, window, known=0.5 if keys > 0 else None) < 2 ** -7


@pytest.mark.parametrize("dim", [128, 64])
@pytest.mark.parametrize("small", [-10, -20, -40])
def test_portions_whose_rows_look_at_a_small_value(ops, dim, small):
    """Nearly all of a row's weight is on one position whose value is far smaller than its neighbours'."""
    heads, kv, held = 4, 2, [130]
    cache = Cache(held, kv, dim, 64, 1)
    for page, slot in ((0, 20), (1, 3)):
        cache.scales["v"][cache.table[0, page].item(), :, slot] *= 2.0 ** small
    q = torch.zeros(130, heads, dim)
    for i in range(130):
        pos = 67 if i >= 67 else 20
        q[i] = cache.values("k", 0)[pos].float().repeat_interleave(heads // kv, 0)
    q = q.flatten(1).bfloat16()
    scale = 60.0 / float(q.float().view(130, heads, dim).pow(2).sum(-1).min())
    out = portions_of(ops, cache, held, heads, q, scale)
    assert row_errors(out, q, cache, held, heads, scale) < 2 ** -7


@pytest.mark.parametrize("heads,kv,dim", [(14, 2, 128), (6, 2, 64)])
@pytest.mark.parametrize("window", [0, 50])
def test_a_run_of_scales_far_apart_with_blocks_of_zeros_and_nan(ops, heads, kv, dim, window):
    """Positions that are zero weigh as such, positions that read as NaN reach only who sees them, in runs whose scales lie far apart too."""
    held = lens = [190, 100]
    cache = Cache(held, kv, dim, 16, 1)

    def at(name, request, pos):
        return cache.scales[name][cache.table[request, pos // 16].item(), :, pos % 16]

    for r in range(2):
        at("v", r, 30).mul_(2.0 ** 30)
        at("k", r, 31).mul_(2.0 ** -30)
        at("v", r, 70).mul_(2.0 ** -30)
        for pos in (5, 33, 71):
            at("v", r, pos).zero_()
            at("k", r, pos + 1).zero_()
    positions, seq, q_start, start_pos = batch_index(lens, [0, 0], DEV)
    q = torch.randn(290, heads * dim, generator=torch.Generator().manual_seed(8)).bfloat16()
    assert row_errors(portions_of(ops, cache, lens, heads, q, 0.05, window), q, cache, lens, heads, 0.05, window) < 2 ** -7
    bad = {0: (62, "k"), 1: (40, "v")}
    for r, (pos, name) in bad.items():
        at(name, r, pos)[1] = math.nan
    out = portions_of(ops, cache, lens, heads, q, 0.05, window)
    nan, want = torch.isnan(out.view(-1, heads, dim)).cpu(), torch.zeros(290, heads, dtype=torch.bool)
    for r, first in ((0, 0), (1, 190)):
        for i in range(held[r]):
            want[first + i, heads // kv:] = bad[r][0] <= i and (not window or bad[r][0] > i - window)
    assert torch.equal(nan.all(-1), want) and torch.equal(nan.any(-1), want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("requests,kv,dim,columns,held", [(3, 2, 128, 2, 300), (40, 2, 128, 2, 300), (3, 1, 128, 130, 8330), (3, 2, 80, 2, 300), (2, 1, 256, 1, 65)])
@pytest.mark.parametrize("window", [0, 50])
def test_single_tokens_beyond_their_block_table_are_reported(ops, dtype, requests, kv, dim, columns, held, window):
    """A context that the table has no room for, and one that starts in front of position 0: as faults, whatever kernel serves them."""
    heads = 4 * kv
    cache = Cache([held] + [60] * (requests - 1), kv, dim, 64, 1)
    device, short = cache.device(), cache.table[:, :columns].contiguous().to(DEV)
    q = torch.randn(requests, heads * dim, generator=torch.Generator().manual_seed(1)).to(dtype).to(DEV)

    def call(starts, table):
        positions, seq, q_start, start_pos = batch_index([1] * requests, starts, DEV)
        return ops.attention_8bit(q, *device, table, q_start, start_pos, positions, seq, requests, 1, held, heads, kv, dim, 0.09, window=window)

    good = call([n - 1 for n in cache.held], cache.table.to(DEV))
    ops.check_status()
    out = call([n - 1 for n in cache.held], short)
    with pytest.raises(ops.DeviceStatusError, match="page"):
        ops.check_status()
    assert rel_error(out[1:], good[1:]) < TOL[dtype]
    out = call([-1] + [n - 1 for n in cache.held[1:]], cache.table.to(DEV))
    with pytest.raises(ops.DeviceStatusError, match="row"):
        ops.check_status()
    assert (out[0] == 0).all() and rel_error(out[1:], good[1:]) < TOL[dtype]
    call([columns * 64 - 1] + [n - 1 for n in cache.held[1:]], short)           # the last position that the table has room for
    ops.check_status()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("heads,kv,dim,page", [(6, 2, 32, 16), (6, 2, 80, 16), (14, 2, 128, 8)])
@pytest.mark.parametrize("singles", [1, 9])
def test_a_portion_goes_the_same_way_beside_single_tokens(ops, dtype, heads, kv, dim, page, singles):
    """Caches that the single tokens' kernel does not take: the bits of both parts on their own."""
    held = [40 + 3 * i for i in range(singles)] + [100, 70]
    lens = [1] * singles + [64, 70]
    cache = Cache(held, kv, dim, page, 1)
    positions, seq, q_start, start_pos = batch_index(lens, [h - n for h, n in zip(held, lens)], DEV)
    q = torch.randn(sum(lens), heads * dim, generator=torch.Generator().manual_seed(5)).to(dtype).to(DEV)
    device, table = cache.device(), cache.table.to(DEV)
    rest = (heads, kv, dim, dim ** -0.5)
    both = ops.attention_8bit(q, *device, table, q_start, start_pos, positions, seq, len(lens), 70, max(held), *rest, decode_prefix=singles, ctx_lens=held)
    first = ops.attention_8bit(q[:singles], *device, table, q_start, start_pos, positions, seq, singles, 1, max(held), *rest, ctx_lens=held[:singles])
    second = ops.attention_8bit(q[singles:], *device, table[singles:].contiguous(), q_start[singles:] - singles, start_pos[singles:].clone(),
                                positions[singles:].clone(), seq[singles:] - singles, 2, 70, 100, *rest, ctx_lens=held[singles:])
    ops.check_status()
    assert torch.equal(both[:singles], first) and torch.equal(both[singles:], second)


class Refusing:
    """The kernels' library, with one entry that refuses."""

    def __init__(self, lib, name):
        self._lib, self._name = lib, name

    def __getattr__(self, name):
        return (lambda *args: -1) if name == self._name else getattr(self._lib, name)


def test_side_by_side_joins_its_stream_when_a_part_is_refused(ops, monkeypatch):
    """What the second stream still uses is the caller's again once the call has raised: the caller's stream waits for it."""
    held, lens, heads = [1, 5, 64, 65, 200, 17, 128, 90, 400, 200], [1] * 9 + [100], 14
    cache = Cache(held, 2, 128, 16, 1)
    want, _ = attend(ops, cache, lens, heads, torch.bfloat16, decode_prefix=9, ctx_lens=held)
    monkeypatch.setattr(ops, "BESIDE_8BIT_FLOPS", 0.0)
    waits, wait_stream = [], torch.cuda.Stream.wait_stream
    monkeypatch.setattr(torch.cuda.Stream, "wait_stream", lambda self, other: (waits.append((self, other)), wait_stream(self, other))[1])
    lib = ops.core()
    main, side = torch.cuda.current_stream(), ops._side_stream()
    for refused in ("tge_attention_8bit_decode", "tge_read_8bit"):
        waits.clear()
        with monkeypatch.context() as patch:
            patch.setattr(ops, "core", lambda: Refusing(lib, refused))
            with pytest.raises(ops.KernelError):
                attend(ops, cache, lens, heads, torch.bfloat16, decode_prefix=9, ctx_lens=held)
        assert waits[0] == (side, main) and waits[-1] == (main, side)
    got, _ = attend(ops, cache, lens, heads, torch.bfloat16, decode_prefix=9, ctx_lens=held)
    assert torch.equal(got, want)


def test_a_read_back_is_planned_by_a_kernel_of_its_own(ops):
    """Its block table is there before the kernel that reads entries lets the next one start; requests that hold nothing have a plan too."""
    cache = Cache([130, 0, 40], 2, 64, 16, 1)
    _, _, q_start, start_pos = batch_index([1, 0, 1], [129, 0, 39], DEV)
    device, table = cache.device(), cache.table.to(DEV)
    before = ops.launches
    k, _v, runs = ops.read_cache_8bit(*device, table, q_start, start_pos, cache.held, torch.bfloat16)
    assert ops.launches - before == 2 and k.shape[0] == 4 and runs.tolist() == [[0, 1, 2], [-1, -1, -1], [3, -1, -1]]
    many = [i * 37 % 300 for i in range(600)]                     # more requests than the plan takes at a time
    lens = [min(n, 2) for n in many]
    cache = Cache(many, 1, 64, 16, 1)
    _, _, q_start, start_pos = batch_index(lens, [h - n for h, n in zip(many, lens)], DEV)
    for window, first in ((0, 0), (70, 5)):
        found = ops.read_cache_8bit(*cache.device(), cache.table.to(DEV), q_start, start_pos, many, torch.bfloat16, window=window, first_seq=first)[2].tolist()
        at = 0
        for held, n, row in zip(many[first:], lens[first:], found):
            seen = max(held - n - window + 1, 0) // 64 if window else 0
            count = max(-(-held // 64) - seen, 0)
            assert row == [-1] * seen + list(range(at, at + count)) + [-1] * (len(row) - seen - count)
            at += count
    _, _, q_start, start_pos = batch_index([1, 0, 1], [129, 0, 39], DEV)
    starts = torch.full((2,), -7, dtype=torch.int32, device=DEV)
    before = ops.launches
    found = ops._read_8bit((device[0].shape[0], 16, 1), *device, table, q_start, start_pos, [130, 0], torch.bfloat16, 0, 1, starts)
    assert ops.launches - before == 1 and found[0].shape[0] == 0 and starts.tolist() == [0, 0]
    ops.check_status()


def test_pages_of_one_call_leave_no_tensor_maps_behind(ops):
    """Portions that go over bfloat16 pages of the call's own, of other sizes every time."""
    for heads, kv, dim, odd in ((2, 1, 256, 0), (6, 2, 128, 1)):
        lib = ops.attention_lib(dim)
        before = lib.tge_attention_mma_kept_maps()
        for held in (70, 200, 330, 500):
            cache = Cache([held, 90], kv, dim, 16, 1)
            q = torch.randn(100, heads * dim + 2 * odd, generator=torch.Generator().manual_seed(held)).bfloat16()
            positions, seq, q_start, start_pos = batch_index([40, 60], [held - 40, 30], DEV)
            rows = q.to(DEV)[:, 2 * odd:]                       # rows that do not lie on 16 bytes
            out = ops.attention_8bit(rows, *cache.device(), cache.table.to(DEV), q_start, start_pos, positions, seq, 2, 60, held, heads, kv, dim, 0.09, ctx_lens=[held, 90])
            want = [plain.attend(q[a:b, 2 * odd:].reshape(b - a, heads, dim), cache.values("k", r), cache.values("v", r), s, 0.09, 0, None)
                    for r, (a, b, s) in enumerate(((0, 40, held - 40), (40, 100, 30)))]
            assert rel_error(out, torch.cat(want).flatten(1)) < TOL[torch.bfloat16]
        assert lib.tge_attention_mma_kept_maps() == before
    ops.check_status()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dim", [128, 64, 256, 80])
@pytest.mark.parametrize("small", [-10, -25, -40, -100])
@pytest.mark.parametrize("columns", [5, 130])
def test_single_tokens_that_look_at_a_small_value(ops, dtype, dim, small, columns):
    """Nearly all of a token's weight is on one position whose value is far smaller than what else it sees, early, late or alone in its slice."""
    heads, kv, held, looks = 4, 2, [300, 300, 40, 17], (3, 280, 20, 16)
    cache = Cache(held, kv, dim, 64, 1)
    wide = torch.full((4, columns), -1, dtype=torch.int32)
    wide[:, :cache.table.shape[1]] = cache.table
    cache.table = wide
    q = torch.stack([cache.values("k", r)[pos].float().repeat_interleave(heads // kv, 0) for r, pos in enumerate(looks)])
    for r, pos in enumerate(looks):
        cache.scales["v"][cache.table[r, pos // 64].item(), :, pos % 64] *= 2.0 ** small
    scale = 100.0 / float(q.pow(2).sum(-1).min())
    q = q.flatten(1).to(dtype)
    positions, seq, q_start, start_pos = batch_index([1] * 4, [h - 1 for h in held], DEV)
    out = ops.attention_8bit(q.to(DEV), *cache.device(), cache.table.to(DEV), q_start, start_pos, positions, seq, 4, 1, 300, heads, kv, dim, scale)
    ops.check_status()
    # float32: a score of some hundreds is known to 2^-22 of it
    assert row_errors(out, q, cache, [1] * 4, heads, scale) < (2 ** -7 if dtype == torch.bfloat16 else 2 ** -12)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("far", [60, 100, 400])
@pytest.mark.parametrize("base,power", [(0, 20), (0, 60), (0, 120), (-110, 230)])
@pytest.mark.parametrize("order", [(0, 1, 2), (1, 0, 2), (2, 1, 0), (1, 2, 0)])
def test_single_tokens_that_hardly_weigh_large_values(ops, dtype, far, base, power, order):
    """Pages whose values are 2^120 the others' size and more, and whose scores lie far below theirs, in front of them and behind them."""
    heads, kv, dim, held = 4, 2, 128, [192]
    cache = Cache(held, kv, dim, 64, 1)
    codes = torch.randint(-127, 128, (dim,), generator=torch.Generator().manual_seed(3)).to(torch.int8)
    near, away, middle = (cache.table[0, i].item() for i in order)
    cache.codes["k"][near], cache.codes["k"][away], cache.codes["k"][middle] = codes, -codes, 0
    cache.scales["k"].fill_(1.0)
    cache.scales["v"][[near, middle]] *= 2.0 ** base
    cache.scales["v"][away] *= 2.0 ** (base + power)
    q = (codes.float() / 127).repeat(1, heads, 1).flatten(1).to(dtype)
    scale = far / 2 * math.log(2) / float((codes.float() / 127).pow(2).sum())            # scores of far / 2, its negative and 0, in powers of two
    positions, seq, q_start, start_pos = batch_index([1], [191], DEV)
    out = ops.attention_8bit(q.to(DEV), *cache.device(), cache.table.to(DEV), q_start, start_pos, positions, seq, 1, 1, 192, heads, kv, dim, scale)
    ops.check_status()
    assert row_errors(out, q, cache, [1], heads, scale) < (2 ** -7 if dtype == torch.bfloat16 else 2 ** -12)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dim", [128, 80])
@pytest.mark.parametrize("lens", [[1, 0], [1, 0, 0], [0, 0]])
@pytest.mark.parametrize("window", [0, 20])
def test_requests_behind_single_tokens_that_neither_bring_nor_hold(ops, dtype, dim, lens, window):
    """Under a bound of their lengths that would let them bring more."""
    held = [50] * lens[0] + [0] * (len(lens) - lens[0])
    cache = Cache(held, 2, dim, 16, 1)
    for prefix in (0, lens[0]):
        positions, seq, q_start, start_pos = batch_index(lens, [h - n for h, n in zip(held, lens)], DEV)
        q = torch.randn(sum(lens), 4 * dim, generator=torch.Generator().manual_seed(1)).to(dtype)
        out = ops.attention_8bit(q.to(DEV), *cache.device(), cache.table.to(DEV), q_start, start_pos, positions, seq, len(lens), 7, 50, 4, 2, dim, 0.1,
                                 window=window, decode_prefix=prefix, ctx_lens=held)
        ops.check_status()
        assert out.shape == q.shape
        if lens[0]:
            want = plain.attend(q.view(1, 4, dim), cache.values("k", 0), cache.values("v", 0), 49, 0.1, window, None)
            assert rel_error(out, want.flatten(1)) < TOL[dtype]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("heads,kv,dim", [(14, 2, 128), (6, 2, 64), (4, 2, 80), (2, 1, 256), (6, 2, 32)])
@pytest.mark.parametrize("told", [[90, 200], [3000, 40], [0, 200], [64, 64]])
def test_contexts_longer_than_the_host_was_told_are_reported(ops, dtype, heads, kv, dim, told):
    """Memory that is sized by the host's numbers is not run over; the next step is right again."""
    held, lens = [3000, 200], [40, 70]
    cache = Cache(held, kv, dim, 16, 1)
    positions, seq, q_start, start_pos = batch_index(lens, [h - n for h, n in zip(held, lens)], DEV)
    q = torch.randn(sum(lens), heads * dim, generator=torch.Generator().manual_seed(1)).to(dtype).to(DEV)
    args = (q, *cache.device(), cache.table.to(DEV), q_start, start_pos, positions, seq, 2, 70)
    want = ops.attention_8bit(*args, 3000, heads, kv, dim, 0.09, ctx_lens=held)
    ops.check_status()
    out = ops.attention_8bit(*args, max(told), heads, kv, dim, 0.09, ctx_lens=told)
    if dtype == torch.float32 and dim in (80, 256):              # the kernel that walks the keys row by row needs no such numbers
        assert torch.equal(out, want)
    else:
        with pytest.raises(ops.DeviceStatusError, match="row"):
            ops.check_status()
        with pytest.raises(ops.KernelError):
            ops.attention_8bit(*args, 0, heads, kv, dim, 0.09, ctx_lens=[0, 0])
    assert torch.equal(ops.attention_8bit(*args, 3000, heads, kv, dim, 0.09, ctx_lens=held), want)
    ops.check_status()


@pytest.mark.parametrize("heads,kv,dim", [(14, 2, 128), (6, 2, 64)])
@pytest.mark.parametrize("powers", [(-60, 100), (0, 110), (-110, 110)])
@pytest.mark.parametrize("zeros", [1, 3, 64])
def test_portions_whose_rows_see_only_zeros_of_a_run_of_large_values(ops, heads, kv, dim, powers, zeros):
    """Values of zero in front of ones 2^110 the run before's size: the rows that see no more of the run than zeros keep what they have."""
    held = [160]
    cache = Cache(held, kv, dim, 64, 1)
    for run in range(3):
        cache.scales["v"][cache.table[0, run].item()] *= 2.0 ** powers[min(run, 1)]
    cache.scales["v"][cache.table[0, 1].item(), :, :zeros] = 0.0
    q = torch.randn(160, heads * dim, generator=torch.Generator().manual_seed(4)).bfloat16()
    out = portions_of(ops, cache, held, heads, q, 0.02)
    assert row_errors(out, q, cache, held, heads, 0.02) < 2 ** -7
