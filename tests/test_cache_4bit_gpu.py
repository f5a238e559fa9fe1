"""The 4-bit cache on the device against its definition: store with norm and rotation, reading back, attention, refusals."""
import math
import random

import pytest
import torch

from helpers import TOL, batch_index, rel_error
from plain import cache_4bit_plain as plain
from plain import cache_8bit_plain

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
attention_of = cache_8bit_plain.attend


@pytest.fixture(scope="module")
def ops():
    from aegean_tge_b200 import ops as module
    module.core()
    return module


class Cache:
    """Random codes, steps and bases of requests that hold ``held`` positions, on shuffled pages; what no request holds reads as NaN."""

    def __init__(self, held, kv_heads, dim, page, seed=0):
        gen = torch.Generator().manual_seed(seed)
        self.held, self.kv_heads, self.dim, self.page, self.groups = held, kv_heads, dim, page, -(-dim // 32)
        need = [-(-n // page) for n in held]
        order = list(range(sum(need) + 3))
        random.Random(seed).shuffle(order)
        self.table = torch.full((len(held), max(max(need), 1)), -1, dtype=torch.int32)
        at = 0
        for r, n in enumerate(need):
            self.table[r, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
            at += n
        self.pages = len(order)
        self.codes = {n: torch.randint(0, 256, (self.pages, kv_heads, page, 16 * self.groups), generator=gen).to(torch.uint8) for n in "kv"}
        self.pairs = {n: torch.full((self.pages, kv_heads, page, 2 * self.groups), math.nan).bfloat16() for n in "kv"}
        for n in "kv":
            for r, count in enumerate(held):
                pos = torch.arange(count)
                pairs = torch.rand(count, kv_heads, self.groups, 2, generator=gen)
                pairs[..., 0] = 0.1 + 0.2 * pairs[..., 0]
                pairs[..., 1] = 0.8 * pairs[..., 1] - 0.4
                self.pairs[n][self.table[r, pos // page].long(), :, pos % page] = pairs.flatten(2).bfloat16()

    def scaled(self, name, request, positions, by):
        """Steps and bases of some of a request's positions times a power of two."""
        for pos in positions:
            self.pairs[name][self.table[request, pos // self.page].item(), :, pos % self.page] *= by

    def of(self, name, request, codes=None, pairs=None):
        """(units [held, kv, 16 groups], pairs [held, kv, 2 groups]) of one request."""
        codes, pairs = (self.codes if codes is None else codes)[name].cpu(), (self.pairs if pairs is None else pairs)[name].cpu()
        pos = torch.arange(self.held[request])
        where = self.table[request, pos // self.page].long()
        return codes[where, :, pos % self.page], pairs[where, :, pos % self.page]

    def values(self, name, request):
        return plain.values(*self.of(name, request), self.dim)

    def device(self):
        return tuple(t.to(DEV) for t in (self.codes["k"], self.codes["v"], self.pairs["k"], self.pairs["v"]))


def tables(positions, rotary):
    angles = torch.arange(positions)[:, None].float() * (10000.0 ** (-torch.arange(0, rotary, 2).float() / max(rotary, 1)))
    return angles.cos(), angles.sin()


def store(ops, cache, qkv, starts, heads, rotary, lens, pairs=False, norms=None, out=None, positions=300):
    """Appends and compares queries, codes, steps and bases with the definition; returns the device's cache and what it holds."""
    at, seq, q_start, _ = batch_index(lens, starts, DEV)
    device = cache.device()
    kv, dim = cache.kv_heads, cache.dim
    cos, sin = tables(positions, rotary)
    q_norm, k_norm = norms or (None, None)
    up = lambda t: None if t is None else t.to(DEV)  # noqa: E731
    q = ops.norm_rope_kv_store_4bit(qkv.to(DEV), up(cos) if rotary else None, up(sin) if rotary else None, rotary, at, seq, len(lens), cache.table.to(DEV),
                                    *device, heads, kv, dim, q_norm=up(q_norm), k_norm=up(k_norm), eps=1e-6, pairs=pairs, out=out)
    ops.check_status()
    codes, steps = {"k": device[0].cpu(), "v": device[1].cpu()}, {"k": device[2].cpu(), "v": device[3].cpu()}
    rows = qkv[:, :(heads + 2 * kv) * dim].float().view(len(qkv), heads + 2 * kv, dim)
    row = 0
    wanted = []
    for r, (n, start) in enumerate(zip(lens, starts)):
        got = {name: cache.of(name, r, codes, steps) for name in "kv"}
        before = {name: cache.of(name, r) for name in "kv"}
        for i in range(n):
            qs, ks, vs = rows[row, :heads], rows[row, heads:heads + kv], rows[row, heads + kv:]
            if q_norm is not None:
                qs = plain.normalised(qs, q_norm, 1e-6)
            if k_norm is not None:
                ks = plain.normalised(ks, k_norm, 1e-6)
            if rotary:
                qs, ks = (plain.turned(x, cos, sin, rotary, start + i, pairs) for x in (qs, ks))
            wanted.append(qs.flatten())
            for name, x in (("k", ks), ("v", vs)):
                units, of = got[name][0][start + i], got[name][1][start + i].float()
                for h in range(kv):
                    want, wanted_steps, wanted_bases = plain.entry(x[h])
                    assert torch.equal(of[h].view(-1, 2).nan_to_num(-7.0), torch.tensor([wanted_steps, wanted_bases]).t().nan_to_num(-7.0)), (r, i, name, h)
                    if want is None:
                        assert torch.isnan(of[h]).all()
                        continue
                    assert plain.unpack(units[h], dim).tolist() == want, (r, i, name, h)
                    # half a step off at most, and what 24 bits make of the division and of the base
                    off = (plain.values(units[h], got[name][1][start + i][h], dim) - x[h].double()).abs()
                    step = torch.tensor(wanted_steps).double().repeat_interleave(32)[:dim]
                    assert bool((off <= step * (0.5 + 16 * 2.0 ** -23) + 2.0 ** -23 * x[h].abs().double() + 1e-44).all())
            row += 1
        for name in "kv":           # what was there stays
            assert torch.equal(got[name][0][:start], before[name][0][:start]) and torch.equal(got[name][1][:start], before[name][1][:start])
            assert torch.equal(got[name][0][start + n:], before[name][0][start + n:])
    if wanted:
        # the same float32 numbers, rounded once
        assert torch.equal(q.cpu(), torch.stack(wanted).to(qkv.dtype))
    return device, (codes, steps)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("heads,kv,dim,rotary,page", [
    (28, 4, 128, 128, 64), (40, 8, 128, 128, 16), (4, 2, 64, 64, 64), (3, 1, 16, 16, 8), (5, 1, 32, 32, 64), (3, 2, 256, 256, 32), (5, 1, 256, 128, 64),
    (6, 3, 80, 40, 16), (2, 2, 10, 6, 4), (2, 1, 33, 0, 64), (6, 2, 64, 0, 16), (2, 1, 128, 48, 16)])
@pytest.mark.parametrize("normed,pairs", [(False, False), (True, False), (True, True), (False, True)])
def test_store(ops, dtype, heads, kv, dim, rotary, page, normed, pairs):
    lens, starts = [1, 1, 17, 5, 3], [0, 77, 9, 3, 62]
    cache = Cache([a + b for a, b in zip(lens, starts)], kv, dim, page)
    gen = torch.Generator().manual_seed(3)
    qkv = torch.randn(sum(lens), (heads + 2 * kv) * dim + 16, generator=gen)          # the row goes on behind the values
    qkv[:, heads * dim] *= 20.0                                                       # a number that stands out
    qkv[7, (heads + kv) * dim:(heads + 2 * kv) * dim] = 0.0                           # a position of zeros
    qkv[8, heads * dim:(heads + 2 * kv) * dim] = 1.7                                  # one of equal numbers
    qkv[9, heads * dim:(heads + 2 * kv) * dim] += 100.0                               # one far from zero
    norms = tuple(1.0 + 0.3 * torch.randn(dim, generator=gen) for _ in range(2)) if normed else None
    store(ops, cache, qkv.to(dtype), starts, heads, rotary, lens, pairs, norms)


def test_store_with_one_of_the_norms(ops):
    for dim in (64, 48):
        for norms in ((None, torch.full((dim,), 0.5)), (torch.full((dim,), 0.5), None)):
            cache = Cache([9, 3], 2, dim, 16)
            store(ops, cache, torch.randn(12, 6 * dim, generator=torch.Generator().manual_seed(1)).bfloat16(), [0, 0], 2, dim, [9, 3], False, norms)


@pytest.mark.parametrize("size", [1e-44, 1e-42, 1e-38, 1e-30, 1e20, 7.9e28, 8e28, 3e38])
@pytest.mark.parametrize("dim", [64, 48])
def test_store_at_the_ends_of_the_range(ops, size, dim):
    """Down to float32's smallest numbers; from 2^96 (7.92e28) on entries read as NaN."""
    lens, starts = [3, 9], [5, 0]
    cache = Cache([8, 9], 2, dim, 16)
    gen = torch.Generator().manual_seed(4)
    qkv = ((torch.rand(12, 6 * dim, generator=gen).double() * 2 - 1) * size).float()
    qkv[2, 2 * dim:] = size
    _, (_, pairs) = store(ops, cache, qkv, starts, 2, 0, lens)
    assert bool(torch.isnan(pairs["k"][cache.table[0, 0].item(), 0, 7]).all()) == (size >= 2.0 ** 96)


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("dim", [128, 40])
def test_store_of_values_that_are_not_finite(ops, bad, dim):
    """All of the entry reads as NaN, its neighbours do not; stored anew it forgets it."""
    lens, starts = [6, 7], [2, 0]
    cache = Cache([8, 7], 2, dim, 8)
    qkv = torch.randn(13, 6 * dim, generator=torch.Generator().manual_seed(5))
    qkv[3, 2 * dim + 5] = bad             # a key of head 0 at position 5 of request 0
    qkv[8, 5 * dim + 39] = bad            # a value of head 1 at position 2 of request 1
    device, (_, pairs) = store(ops, cache, qkv, starts, 2, 0, lens)
    for name, r, pos, head in (("k", 0, 5, 0), ("v", 1, 2, 1)):
        nan = torch.isnan(pairs[name][cache.table[r, 0].item()])
        assert bool(nan[head, pos].all()) and not nan[1 - head].any(-1)[:7].any()
    clean = torch.randn(7, 6 * dim, generator=torch.Generator().manual_seed(6))
    positions, seq, _, _ = batch_index([7], [0], DEV)
    ops.norm_rope_kv_store_4bit(clean.to(DEV), None, None, 0, positions, seq, 1, cache.table[1:].to(DEV), *device, 2, 2, dim)
    assert torch.isfinite(device[3][cache.table[1, 0].item(), :, :7].float()).all()


def test_store_rows_of_an_inner_buffer(ops):
    """Odd row strides, starts that are no multiple of 16 bytes, an output inside a wider buffer; neighbours stay as they are."""
    heads, kv, dim = 4, 2, 64
    cache = Cache([40, 3], kv, dim, 16)
    gen = torch.Generator().manual_seed(8)
    norms = (torch.ones(dim), torch.full((dim,), 2.0))
    for dtype in (torch.bfloat16, torch.float32):
        for lead, width in ((1, 8 * 64 + 3), (8, 8 * 64 + 8), (0, 8 * 64 + 1)):
            rows = torch.randn(43, width, generator=gen).to(dtype).to(DEV)
            before = rows.clone()
            wide = torch.full((43, heads * dim + 5), 7.0, dtype=dtype, device=DEV)
            view = rows[:, lead:lead + 8 * 64] if width - lead >= 8 * 64 else rows
            positions, seq, _, _ = batch_index([40, 3], [0, 0], DEV)
            cos, sin = (t.to(DEV) for t in tables(64, dim))
            d1, d2 = cache.device(), cache.device()
            args = (cos, sin, dim, positions, seq, 2, cache.table.to(DEV))
            kw = {"q_norm": norms[0].to(DEV), "k_norm": norms[1].to(DEV)}
            a = ops.norm_rope_kv_store_4bit(view, *args, *d1, heads, kv, dim, out=wide[:, 3:3 + heads * dim], **kw)
            b = ops.norm_rope_kv_store_4bit(view.contiguous(), *args, *d2, heads, kv, dim, **kw)
            assert torch.equal(a, b) and all(torch.equal(x.nan_to_num(0.0) if x.is_floating_point() else x, y.nan_to_num(0.0) if y.is_floating_point() else y)
                                             for x, y in zip(d1, d2))
            assert torch.equal(rows, before)
            assert (wide[:, :3] == 7).all() and (wide[:, 3 + heads * dim:] == 7).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("size", [1.0, 1e-35, 1e-24, 1e25])
def test_codes_of_both_kernels(ops, dtype, size):
    """A million numbers, many of them halfway between two codes, by the kernel that divides (rows on odd elements) and the one that has the quotients
    by parts: the same bits."""
    tokens, heads, kv, dim = 512, 1, 8, 128
    gen = torch.Generator().manual_seed(4)
    rows = torch.randn(tokens, (heads + 2 * kv) * dim, generator=gen)
    grid = torch.randint(-60, 60, rows.shape, generator=gen) / 16.0                 # sums and halves of few bits: ties are common
    rows[::2] = grid[::2]
    rows = (rows.double() * size).to(dtype).to(DEV)
    wide = torch.zeros(tokens, rows.shape[1] + 1, dtype=dtype, device=DEV)
    wide[:, 1:] = rows
    cache = Cache([tokens], kv, dim, 64)
    positions, seq, _, _ = batch_index([tokens], [0], DEV)
    weight = (1.0 + 0.3 * torch.randn(dim, generator=gen)).to(DEV)
    for norm in (None, weight):
        found = []
        for x in (rows, wide[:, 1:]):
            device = cache.device()
            found.append([ops.norm_rope_kv_store_4bit(x, None, None, 0, positions, seq, 1, cache.table.to(DEV), *device, heads, kv, dim, q_norm=norm, k_norm=norm), *device])
        assert all(torch.equal(a.nan_to_num(0.0) if a.is_floating_point() else a, b.nan_to_num(0.0) if b.is_floating_point() else b) for a, b in zip(*found))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_norms_of_rows_that_are_not_finite(ops, dtype):
    """A number that is not finite makes its row's queries and its entry what the formula makes of them, in both kernels; nobody else's."""
    heads, kv, dim = 2, 2, 64
    weight = torch.ones(dim, device=DEV)
    for bad in (math.nan, math.inf):
        rows = torch.randn(3, 6 * dim, generator=torch.Generator().manual_seed(2))
        rows[1, 5] = rows[1, (heads + 1) * dim + 7] = bad
        rows[2, :dim] = 0.0
        wide = torch.zeros(3, 6 * dim + 1, dtype=dtype, device=DEV)
        wide[:, 1:] = rows.to(dtype)
        positions, seq, _, _ = batch_index([3], [0], DEV)
        for x in (rows.to(dtype).to(DEV), wide[:, 1:]):
            cache = Cache([3], kv, dim, 16)
            device = cache.device()
            q = ops.norm_rope_kv_store_4bit(x, None, None, 0, positions, seq, 1, cache.table.to(DEV), *device, heads, kv, dim, q_norm=weight, k_norm=weight).cpu().float()
            want = plain.normalised(rows.to(dtype).float()[:, :2 * dim].reshape(3, 2, dim), torch.ones(dim), 1e-6).flatten(1).to(dtype).float()
            assert torch.equal(torch.isnan(q), torch.isnan(want)) and torch.equal(q.nan_to_num(9.0), want.nan_to_num(9.0))
            nan = torch.isnan(device[2][cache.table[0, 0].item(), :, :3].float()).all(-1).cpu()
            assert nan.tolist() == [[False, False, False], [False, True, False]]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_entries_do_not_depend_on_the_cut(ops, dtype):
    heads, kv, dim, n = 4, 2, 128, 150
    cos, sin = (t.to(DEV) for t in tables(n, dim))
    qkv = torch.randn(n, 8 * dim, generator=torch.Generator().manual_seed(9)).to(dtype).to(DEV)
    weight = torch.rand(dim, generator=torch.Generator().manual_seed(1)).to(DEV)
    found = []
    for cuts in ([150], [1] * 150, [64, 1, 85], [7, 63, 80]):
        cache = Cache([n], kv, dim, 16)
        device, at, q = cache.device(), 0, []
        for count in cuts:
            positions, seq, _, _ = batch_index([count], [at], DEV)
            q.append(ops.norm_rope_kv_store_4bit(qkv[at:at + count], cos, sin, dim, positions, seq, 1, cache.table.to(DEV), *device, heads, kv, dim,
                                                 q_norm=weight, k_norm=weight))
            at += count
        found.append([torch.cat(q)] + list(device[:2]) + [s.nan_to_num(0.0) for s in device[2:]])
    for other in found[1:]:
        assert all(torch.equal(a, b) for a, b in zip(found[0], other))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kv,dim,page,window", [(4, 128, 64, 0), (2, 128, 16, 100), (1, 16, 8, 0), (3, 80, 4, 70), (2, 33, 64, 1), (1, 256, 32, 0),
                                                (2, 64, 16, 1), (1, 32, 16, 65), (2, 128, 48, 0)])
def test_read_back(ops, dtype, kv, dim, page, window):
    held, lens = [1, 64, 65, 200, 0, 130] + [3] * 40, [1, 1, 65, 20, 0, 2] + [1] * 40
    cache = Cache(held, kv, dim, page)
    _, _, q_start, start_pos = batch_index(lens, [h - n for h, n in zip(held, lens)], DEV)
    for first in (0, 2, 44):
        for told in (None, lens):
            k, v, table = ops.read_cache_4bit(*cache.device(), cache.table.to(DEV), q_start, start_pos, held, dim, dtype, window=window, first_seq=first, q_lens=told)
            if told is not None:
                assert k.shape[0] == int((table >= 0).sum())
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
                        # a step times a code is exact in float32, the sum with the base rounded once, and once more to the output's type
                        assert torch.equal(part[:n], want[i * 64:i * 64 + n].float().to(dtype).double())
                        assert (part[n:] == 0).all()
    ops.check_status()


# ---------------------------------------------------------------------------
def attend(ops, cache, lens, heads, dtype, window=0, sink=False, scale=None, size=1.5, **kw):
    starts = [h - n for h, n in zip(cache.held, lens)]
    positions, seq, q_start, start_pos = batch_index(lens, starts, DEV)
    gen = torch.Generator().manual_seed(11)
    q = (torch.randn(sum(lens), heads * cache.dim, generator=gen) * size).to(dtype)
    sinks = torch.randn(heads, generator=gen) if sink else None
    scale = cache.dim ** -0.5 if scale is None else scale
    out = ops.attention_4bit(q.to(DEV), *cache.device(), cache.table.to(DEV), q_start, start_pos, positions, seq, len(lens), max(lens), max(cache.held),
                             heads, cache.kv_heads, cache.dim, scale, window=window, sink=None if sinks is None else sinks.to(DEV), **kw)
    want, at = [], 0
    for r, n in enumerate(lens):
        want.append(attention_of(q[at:at + n].view(n, heads, cache.dim), cache.values("k", r), cache.values("v", r), starts[r], scale, window, sinks))
        at += n
    ops.check_status()
    return out, torch.cat(want).flatten(1)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("heads,kv,dim", [(28, 4, 128), (40, 8, 128), (12, 2, 128), (14, 2, 64), (4, 2, 16), (3, 1, 32), (16, 1, 128), (33, 3, 128),
                                          (40, 2, 64), (6, 2, 80), (2, 2, 256), (4, 1, 33)])
def test_single_tokens(ops, dtype, heads, kv, dim):
    cache = Cache([1, 2, 7, 15, 16, 17, 63, 64, 65, 127, 128, 129, 300, 1000], kv, dim, 64)
    out, want = attend(ops, cache, [1] * 14, heads, dtype)
    assert rel_error(out, want) < TOL[dtype]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("page", [64, 32, 16, 8, 48, 1])
@pytest.mark.parametrize("window,sink", [(0, False), (0, True), (1, False), (50, True), (128, False)])
def test_single_tokens_on_pages_and_windows(ops, dtype, page, window, sink):
    cache = Cache([1, 33, 64, 100, 513], 2, 128, page)
    out, want = attend(ops, cache, [1] * 5, 14, dtype, window=window, sink=sink)
    assert rel_error(out, want) < TOL[dtype]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("heads,kv,dim", [(8, 1, 128), (14, 2, 64), (5, 1, 256), (24, 2, 128), (20, 2, 64)])
@pytest.mark.parametrize("columns", [16, 33, 64, 66, 128, 130])
@pytest.mark.parametrize("window,sink", [(0, True), (70, False)])
def test_single_tokens_under_every_bound(ops, dtype, heads, kv, dim, columns, window, sink):
    """The bound of the contexts (the block table's columns, of 64 positions here) decides how a unit's keys are shared out: clusters of 8 and 16
    blocks, runs; requests of one position, of less than a slice to a block, of more."""
    cache = Cache([1, 17, 1000, 130, 64], kv, dim, 64)
    wide = torch.full((5, columns), -1, dtype=torch.int32)
    wide[:, :cache.table.shape[1]] = cache.table
    cache.table = wide
    out, want = attend(ops, cache, [1] * 5, heads, dtype, window=window, sink=sink)
    assert rel_error(out, want) < TOL[dtype]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("heads,kv,dim,page", [(28, 4, 128, 64), (12, 2, 128, 16), (14, 2, 64, 32), (4, 2, 16, 32), (3, 1, 32, 8), (6, 2, 80, 64), (2, 1, 256, 64)])
@pytest.mark.parametrize("window,sink", [(0, False), (33, True)])
def test_portions(ops, dtype, heads, kv, dim, page, window, sink):
    cache = Cache([40, 2, 65, 200, 129], kv, dim, page)
    out, want = attend(ops, cache, [40, 2, 64, 5, 1], heads, dtype, window=window, sink=sink)
    assert rel_error(out, want) < TOL[dtype]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("singles,told", [(9, 9), (9, 8), (2, 2), (9, 0)])
@pytest.mark.parametrize("window", [0, 40])
def test_single_tokens_beside_portions(ops, dtype, singles, told, window):
    """However many of the single tokens the caller tells of, and whether it tells the contexts."""
    held = [1, 5, 64, 65, 200, 17, 128, 90, 400][:singles] + [100, 70]
    cache = Cache(held, 2, 128, 16)
    for ctx in (None, held):
        out, want = attend(ops, cache, [1] * singles + [30, 70], 14, dtype, window=window, decode_prefix=told, ctx_lens=ctx)
        assert rel_error(out, want) < TOL[dtype]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_peaked_and_shifted_scores(ops, dtype, dim):
    """Scores in the hundreds: sums that start far below their maximum, and rows that are one key."""
    cache = Cache([700, 64, 1], 2, dim, 64)
    for scale in (20.0, 1e-8):
        out, want = attend(ops, cache, [1, 1, 1], 8, dtype, scale=scale)
        # A score is a sum of dim products of some 1.5 x 1; scaled by 20 times log2 e, the sum's roundings (2^-24 of its largest partial sum, and for
        # bfloat16 of codes raised by 136: sums of some 136 step sum|q| = 136 x 0.2 x 1.2 dim) are up to dim x 1.5 x 29 x 2^-24 = 3.3e-4 x dim / 128 of a
        # probability for float32 and dim x 33 x 29 x 2^-24 = 7e-3 x dim / 128 for bfloat16, several of them
        assert rel_error(out, want) < (TOL[dtype] if scale < 1 else 2e-3 if dtype == torch.float32 else 4e-2)


def test_one_request_among_many_lengths(ops):
    cache = Cache([1 + 7 * i % 90 for i in range(300)], 2, 64, 16)
    out, want = attend(ops, cache, [1] * 300, 8, torch.bfloat16)
    assert rel_error(out, want) < TOL[torch.bfloat16]


def test_long_contexts(ops):
    """Against float64 on the device: 40,000 positions, offsets of entries beyond 2^31 bytes."""
    kv, dim, heads, page = 2, 128, 8, 64
    pages = 2 ** 32 // (kv * page * dim) + 700
    codes = torch.empty(pages, kv, page, dim // 2, dtype=torch.uint8, device=DEV).random_(0, 256)
    pairs = (torch.rand(pages, kv, page, dim // 16, device=DEV) * 0.2 + 0.1).bfloat16()
    held = [40000, 39, 3000]
    table = torch.full((3, 625), -1, dtype=torch.int32)
    table[0, :625] = torch.arange(pages - 1, pages - 626, -1)
    table[1, :1] = 5
    table[2, :47] = torch.arange(pages - 700, pages - 653)
    q = torch.randn(3, heads * dim, device=DEV).bfloat16()
    positions, seq, q_start, start_pos = batch_index([1, 1, 1], [n - 1 for n in held], DEV)
    out = ops.attention_4bit(q, codes, codes, pairs, pairs, table.to(DEV), q_start, start_pos, positions, seq, 3, 1, 40000, heads, kv, dim, 0.05)
    read, _, runs = ops.read_cache_4bit(codes, codes, pairs, pairs, table.to(DEV), q_start, start_pos, held, dim, torch.float32)
    for r, n in enumerate(held):
        pos = torch.arange(n)
        where = table[r][pos // page].long()
        k = plain.values(codes[where.to(DEV), :, (pos % page).to(DEV)].cpu(), pairs[where.to(DEV), :, (pos % page).to(DEV)].cpu(), dim)
        got = read[runs[r, :-(-n // 64)].long()].transpose(1, 2).flatten(0, 1)[:n]
        assert rel_error(got, k) < 2.0 ** -23
        k = k.to(DEV)
        p = torch.softmax(torch.einsum("kgd,ckd->kgc", q[r].double().view(kv, 4, dim), k) * 0.05, -1)
        assert rel_error(out[r], torch.einsum("kgc,ckd->kgd", p, k).flatten()) < TOL[torch.bfloat16]
    ops.check_status()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dim", [64, 128, 256, 48])
def test_an_entry_that_reads_as_nan_reaches_only_who_sees_it(ops, dtype, dim):
    cache = Cache([100, 100, 100], 2, dim, 16)
    cache.pairs["v"][cache.table[0, 2].item(), 1, 3] = math.nan           # position 35 of request 0, head 1
    cache.pairs["k"][cache.table[1, 1].item(), 0, 0] = math.nan           # position 16 of request 1, head 0
    lens, heads = [1, 1, 1], 8
    positions, seq, q_start, start_pos = batch_index(lens, [99] * 3, DEV)
    q = torch.randn(3, heads * dim, generator=torch.Generator().manual_seed(1)).to(dtype).to(DEV)
    for window in (0, 64):
        out = ops.attention_4bit(q, *cache.device(), cache.table.to(DEV), q_start, start_pos, positions, seq, 3, 1, 100, heads, 2, dim, 0.09, window=window)
        nan = torch.isnan(out.view(3, heads, dim)).all(-1).cpu()
        some = torch.isnan(out.view(3, heads, dim)).any(-1).cpu()
        want = torch.zeros(3, heads, dtype=torch.bool)
        if not window:
            want[0, 4:], want[1, :4] = True, True
        assert torch.equal(nan, want) and torch.equal(some, want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_queries_that_are_not_finite(ops, dtype):
    """Their own head's row of output, no other."""
    cache = Cache([100, 70], 2, 128, 16)
    positions, seq, q_start, start_pos = batch_index([1, 1], [99, 69], DEV)
    q = torch.randn(2, 8 * 128, generator=torch.Generator().manual_seed(1)).to(dtype).to(DEV)
    args = (*cache.device(), cache.table.to(DEV), q_start, start_pos, positions, seq, 2, 1, 100, 8, 2, 128, 0.09)
    good = ops.attention_4bit(q, *args).view(2, 8, 128)
    for bad in (math.nan, math.inf, -math.inf):
        q2 = q.clone()
        q2[0, 3 * 128 + 77] = bad
        out = ops.attention_4bit(q2, *args).view(2, 8, 128)
        assert torch.isnan(out[0, 3]).all()
        out[0, 3] = good[0, 3]
        assert rel_error(out, good) < TOL[dtype]          # (which references the running maxima had may change with it)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("heads,kv,dim", [(14, 2, 128), (6, 2, 64), (6, 2, 32), (4, 2, 80), (2, 2, 256)])
@pytest.mark.parametrize("window", [0, 50])
def test_an_entry_that_reads_as_nan_in_a_portion(ops, dtype, heads, kv, dim, window):
    """Rows in front of it, rows behind its window and other requests do not see it, in whatever tile of keys it lies."""
    held, lens = [300, 150, 70], [300, 90, 6]
    cache = Cache(held, kv, dim, 16)
    bad = {0: (170, "v"), 1: (63, "k"), 2: (66, "v")}
    for request, (pos, name) in bad.items():
        cache.pairs[name][cache.table[request, pos // 16].item(), 1, pos % 16] = math.nan
    positions, seq, q_start, start_pos = batch_index(lens, [h - n for h, n in zip(held, lens)], DEV)
    q = torch.randn(sum(lens), heads * dim, generator=torch.Generator().manual_seed(1)).to(dtype).to(DEV)
    out = ops.attention_4bit(q, *cache.device(), cache.table.to(DEV), q_start, start_pos, positions, seq, 3, 300, 300, heads, kv, dim, 0.09, window=window, ctx_lens=held)
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
    cache = Cache([700, 64, 1000], 2, 128, 64)
    out, want = attend(ops, cache, [9, 64, 30], 14, torch.bfloat16, ctx_lens=[700, 64, 1000], sink=True)
    assert rel_error(out, want) < TOL[torch.bfloat16]


@pytest.mark.parametrize("heads,kv,dim", [(14, 2, 128), (6, 2, 64)])
@pytest.mark.parametrize("window", [0, 70])
@pytest.mark.parametrize("first,each", [((0, 30, -30, 0, 5, 60, -60, 1, 0, -1), 64), ((-90, -20, 60, 50, 30, -50, -90, 0, 50, -50), 64),
                                        ((0, 20, 0, -20, 3, 40, -40, 0, 17, 1) * 7, 9)])
def test_portions_over_entries_far_apart(ops, heads, kv, dim, window, first, each):
    """Values whose size changes by up to 2^150 from one run of positions to the next, keys by 2^3; queries of 2^60 over keys of 2^-60."""
    held, lens = [640, 150, 130], [600, 150, 6]
    cache = Cache(held, kv, dim, 64)
    for r, (size, sizes) in enumerate(zip((60, 0, -60), (first, [-40, 20, 0], [1, 0, -90]))):
        for run, f in enumerate(sizes):
            here = range(run * (each if r == 0 else 64), min((run + 1) * (each if r == 0 else 64), held[r]))
            cache.scaled("v", r, here, 2.0 ** f)
            cache.scaled("k", r, here, 2.0 ** (run % 4 - size))
    positions, seq, q_start, start_pos = batch_index(lens, [h - n for h, n in zip(held, lens)], DEV)
    q = torch.randn(sum(lens), heads * dim, generator=torch.Generator().manual_seed(2))
    q = (q * 2.0 ** torch.tensor([60.0, 0, -60]).repeat_interleave(torch.tensor(lens))[:, None]).bfloat16()
    out = ops.attention_4bit(q.to(DEV), *cache.device(), cache.table.to(DEV), q_start, start_pos, positions, seq, 3, 600, 640, heads, kv, dim, 0.02,
                             window=window, ctx_lens=held)
    ops.check_status()
    at = 0
    for r, n in enumerate(lens):
        k, v, rows = cache.values("k", r), cache.values("v", r), q[at:at + n].view(n, heads, dim)
        want = attention_of(rows, k, v, held[r] - n, 0.02, window, None)
        # a row and head's error against the largest sum of probabilities times magnitudes: each product's roundings are of its own size
        size = attention_of(rows, k, v.abs(), held[r] - n, 0.02, window, None).amax(-1)
        error = (out[at:at + n].cpu().double().view(n, heads, dim) - want).abs().amax(-1)
        assert float((error / size).max()) < 2 ** -7
        at += n


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("heads,kv,dim", [(6, 2, 128), (6, 2, 64), (2, 1, 256)])
@pytest.mark.parametrize("lens", [[1, 1, 1], [40, 1, 70]])
def test_entries_of_zeros_and_of_equal_numbers(ops, dtype, heads, kv, dim, lens):
    """Steps of zero; values of zero that a row sees alone beside large ones that it does not."""
    cache = Cache([300, 1, 90], kv, dim, 64)
    cache.scaled("v", 0, range(0, 250), 0.0)
    cache.scaled("v", 0, range(250, 300), 2.0 ** 40)
    for r, n in enumerate(cache.held):
        for pos in range(0, n, 3):
            cache.pairs["k"][cache.table[r, pos // 64].item(), :, pos % 64, ::2] = 0.0
    for window in (0, 20):
        out, want = attend(ops, cache, lens, heads, dtype, window=window)
        assert rel_error(out, want) < TOL[dtype]
        out, want = attend(ops, cache, lens, heads, dtype, window=window, scale=8.0)
        zero = (want == 0).all(-1)
        assert (out.cpu()[zero] == 0).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("lens", [[1, 1, 1], [40, 1, 70]])
@pytest.mark.parametrize("values,keys", [(1e-35, 1.0), (1e28, 1.0), (1.0, 1e-25), (1e-32, 1e25)])
@pytest.mark.parametrize("dim", [128, 64])
def test_attention_at_the_ends_of_the_range(ops, dtype, lens, values, keys, dim):
    """Values of very small and large steps; keys of them under queries that make up for it."""
    heads, kv = 6, 2
    cache = Cache([300, 1, 90], kv, dim, 64)
    cache.pairs["v"] = (cache.pairs["v"].double() * values).bfloat16()
    cache.pairs["k"] = (cache.pairs["k"].double() * keys).bfloat16()
    out, want = attend(ops, cache, lens, heads, dtype, size=0.5 / keys, scale=0.09)
    assert rel_error(out.cpu().double() / values, want / values) < TOL[dtype]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_groups_of_very_different_sizes_in_single_tokens(ops, dtype, dim):
    """A group 2^30 larger than its neighbours takes nothing from them: every group's numbers against their own."""
    cache = Cache([700, 65, 9], 2, dim, 64)
    cache.pairs["v"][..., :2] *= 2.0 ** 30
    out, want = attend(ops, cache, [1, 1, 1], 6, dtype)
    out, want = (x.view(3, 6, dim) for x in (out, want))
    assert rel_error(out[..., :32], want[..., :32]) < TOL[dtype] and rel_error(out[..., 32:], want[..., 32:]) < TOL[dtype]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("lens", [[1, 1], [3, 20]])
def test_pages_outside_the_pool_are_reported_not_read(ops, dtype, lens):
    cache = Cache([50, 80], 2, 128, 16)
    table = cache.table.clone()
    table[0] = torch.tensor([-1, 9999, -7, 10 ** 6, -1])
    positions, seq, q_start, start_pos = batch_index(lens, [50 - lens[0], 80 - lens[1]], DEV)
    q = torch.randn(sum(lens), 8 * 128).to(dtype).to(DEV)
    args = (q_start, start_pos, positions, seq, 2, max(lens), 80, 8, 2, 128, 0.1)
    good = ops.attention_4bit(q, *cache.device(), cache.table.to(DEV), *args)
    ops.check_status()
    out = ops.attention_4bit(q, *cache.device(), table.to(DEV), *args)
    with pytest.raises(ops.DeviceStatusError):
        ops.check_status()
    assert (out[:lens[0]] == 0).all() and torch.equal(out[lens[0]:], good[lens[0]:])
    for dim in (128, 80):
        cache = Cache([50, 80], 2, dim, 16)
        device = cache.device()
        before = [t.clone() for t in device]
        ops.norm_rope_kv_store_4bit(torch.randn(lens[0], 12 * dim).to(dtype).to(DEV), None, None, 0, positions[:lens[0]], seq[:lens[0]], 1, table.to(DEV),
                                    *device, 8, 2, dim)
        with pytest.raises(ops.DeviceStatusError):
            ops.check_status()
        assert all(torch.equal(a.nan_to_num(0) if a.is_floating_point() else a, b.nan_to_num(0) if b.is_floating_point() else b) for a, b in zip(before, device))


@pytest.mark.parametrize("columns", [16, 66, 130])
def test_a_page_outside_the_pool_under_every_bound(ops, columns):
    """A unit whose keys are partly or wholly outside the pool: reported, unread, zero where nothing is seen."""
    cache = Cache([40, 300], 1, 128, 64)
    wide = torch.full((2, columns), -1, dtype=torch.int32)
    wide[1, :5] = cache.table[1, :5]
    positions, seq, q_start, start_pos = batch_index([1, 1], [39, 299], DEV)
    q = torch.randn(2, 8 * 128, device=DEV).bfloat16()
    out = ops.attention_4bit(q, *cache.device(), wide.to(DEV), q_start, start_pos, positions, seq, 2, 1, 300, 8, 1, 128, 0.09)
    with pytest.raises(ops.DeviceStatusError, match="page"):
        ops.check_status()
    assert (out[0] == 0).all()
    want = attention_of(q[1:].cpu().view(1, 8, 128), cache.values("k", 1), cache.values("v", 1), 299, 0.09, 0, None)
    assert rel_error(out[1:], want.flatten(1)) < TOL[torch.bfloat16]


@pytest.mark.parametrize("start", [-1, 80, 1000])
def test_positions_that_are_none(ops, start):
    """Single tokens at positions in front of all, or behind what the block table has room for: reported, their neighbours served."""
    cache = Cache([50, 60], 2, 128, 16)
    cache.table = torch.cat([cache.table, torch.full((2, 5 - cache.table.shape[1]), -1, dtype=torch.int32)], 1) if cache.table.shape[1] < 5 else cache.table[:, :5].contiguous()
    positions, seq, q_start, start_pos = batch_index([1, 1], [49, 59], DEV)
    q = torch.randn(2, 8 * 128, device=DEV).bfloat16()
    good = ops.attention_4bit(q, *cache.device(), cache.table.to(DEV), q_start, start_pos, positions, seq, 2, 1, 60, 8, 2, 128, 0.09)
    start_pos[0] = start
    out = ops.attention_4bit(q, *cache.device(), cache.table.to(DEV), q_start, start_pos, positions, seq, 2, 1, 60, 8, 2, 128, 0.09)
    with pytest.raises(ops.DeviceStatusError):
        ops.check_status()
    assert torch.equal(out[1], good[1])


def test_positions_outside_the_tables_are_reported(ops):
    for dim in (64, 48):
        cache = Cache([70], 2, dim, 16)
        cos, sin = tables(50, dim)
        positions, seq, _, _ = batch_index([1], [60], DEV)
        device = cache.device()
        ops.norm_rope_kv_store_4bit(torch.randn(1, 6 * dim).to(DEV), cos.to(DEV), sin.to(DEV), dim, positions, seq, 1, cache.table.to(DEV), *device, 2, 2, dim)
        with pytest.raises(ops.DeviceStatusError):
            ops.check_status()
        assert torch.equal(device[0].cpu(), cache.codes["k"])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("lens", [[1, 0, 1, 0], [0, 1, 1, 0], [0, 0, 1, 0], [3, 0, 70, 0]])
@pytest.mark.parametrize("columns", [16, 130])
def test_requests_that_bring_nothing(ops, dtype, lens, columns):
    """In front of, between and behind others, with and without a context of their own: no row is theirs, nothing of theirs changes."""
    heads, kv, dim = 6, 2, 128
    cache = Cache([100, 64, 80, 0], kv, dim, 16)
    wide = torch.full((4, 4 * columns), -1, dtype=torch.int32)
    wide[:, :cache.table.shape[1]] = cache.table
    cache.table = wide
    starts = [h - n for h, n in zip(cache.held, lens)]
    qkv = torch.randn(sum(lens), (heads + 2 * kv) * dim, generator=torch.Generator().manual_seed(3)).to(dtype)
    store(ops, cache, qkv, starts, heads, dim, lens)
    out, want = attend(ops, cache, lens, heads, dtype, ctx_lens=cache.held)
    assert rel_error(out, want) < TOL[dtype]
    positions, seq, q_start, start_pos = batch_index(lens, starts, DEV)
    k, _, table = ops.read_cache_4bit(*cache.device(), cache.table.to(DEV), q_start, start_pos, cache.held, dim, torch.float32)
    ops.check_status()
    assert [(row >= 0).sum().item() for row in table] == [2, 1, 2, 0] and k.shape[0] == 5


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
    cache = Cache([200, 150, 290, 65, 350, 131], kv, dim, page)
    cache.table = released(cache, lens, window)
    out, want = attend(ops, cache, lens, heads, dtype, window=window, ctx_lens=cache.held)
    assert rel_error(out, want) < TOL[dtype]
    positions, seq, q_start, start_pos = batch_index(lens, [h - n for h, n in zip(cache.held, lens)], DEV)
    ops.read_cache_4bit(*cache.device(), cache.table.to(DEV), q_start, start_pos, cache.held, dim, dtype, window=window)
    ops.check_status()
    missing = cache.table.clone()
    missing[4, (350 - 40 - window + 1) // page] = -1
    with pytest.raises(ops.DeviceStatusError, match="page"):
        ops.read_cache_4bit(*cache.device(), missing.to(DEV), q_start, start_pos, cache.held, dim, dtype, window=window)
        ops.check_status()


def test_contexts_beyond_the_hosts_numbers_are_reported(ops):
    """A portion whose request holds more than the call was told: reported, not run over; a read-back of fewer runs than there are too."""
    held, lens, heads, kv, dim = [3000, 90], [60, 20], 14, 2, 128
    cache = Cache(held, kv, dim, 64)
    positions, seq, q_start, start_pos = batch_index(lens, [h - n for h, n in zip(held, lens)], DEV)
    q = torch.randn(80, heads * dim, device=DEV).bfloat16()
    args = (q, *cache.device(), cache.table.to(DEV), q_start, start_pos, positions, seq, 2, 60)
    want = ops.attention_4bit(*args, 3000, heads, kv, dim, 0.09, ctx_lens=held)
    ops.check_status()
    for told in ([64, 90], [2900, 90], [2999, 0]):
        ops.attention_4bit(*args, max(told), heads, kv, dim, 0.09, ctx_lens=told)
        if sum(-(-n // 64) for n in told) < 49:
            with pytest.raises(ops.DeviceStatusError):
                ops.check_status()
        ops.read_cache_4bit(*cache.device(), cache.table.to(DEV), q_start, start_pos, told, dim, torch.bfloat16)
        if sum(-(-n // 64) for n in told) < 49:
            with pytest.raises(ops.DeviceStatusError):
                ops.check_status()
    assert torch.equal(ops.attention_4bit(*args, 3000, heads, kv, dim, 0.09, ctx_lens=held), want)
    ops.check_status()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_on_a_stream_of_its_own_and_again(ops, dtype):
    """On another stream than the default, with rows of an inner buffer: the same bits."""
    cache = Cache([200, 65, 3, 90], 2, 128, 64)
    lens = [1, 1, 1, 1]
    positions, seq, q_start, start_pos = batch_index(lens, [h - 1 for h in cache.held], DEV)
    wide = torch.randn(4, 8 * 128 + 24, generator=torch.Generator().manual_seed(2)).to(dtype).to(DEV)
    device, table = cache.device(), cache.table.to(DEV)
    args = (*device, table, q_start, start_pos, positions, seq, 4, 1, 200, 8, 2, 128, 0.1)
    first = ops.attention_4bit(wide[:, 8:8 + 1024].contiguous(), *args)
    odd = ops.attention_4bit(wide[:, 8:8 + 1024], *args)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        again = ops.attention_4bit(wide[:, 8:8 + 1024], *args)
    side.synchronize()
    assert torch.equal(first, odd) and torch.equal(first, again)
    into = torch.zeros(4, 1024 + 8, dtype=dtype, device=DEV)
    ops.attention_4bit(wide[:, 8:8 + 1024], *args, out=into[:, 8:])
    assert torch.equal(into[:, 8:], first) and (into[:, :8] == 0).all()
    # rows that start on odd elements
    odd_rows = torch.zeros(4, 1024 + 1, dtype=dtype, device=DEV)
    odd_rows[:, 1:] = wide[:, 8:8 + 1024]
    assert torch.equal(ops.attention_4bit(odd_rows[:, 1:], *args), first)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("heads,kv,dim", [(14, 2, 128), (6, 2, 32)])
def test_side_by_side_is_the_same(ops, monkeypatch, dtype, heads, kv, dim):
    """Single tokens beside portions on two streams: the bits of one, time and again; head sizes that only the portions' kernels take as well."""
    held = [1, 5, 64, 65, 200, 17, 128, 90, 400, 33, 300, 270]
    lens = [1] * 10 + [200, 64]
    cache = Cache(held, kv, dim, 16)
    want, _ = attend(ops, cache, lens, heads, dtype, decode_prefix=10, ctx_lens=held)
    monkeypatch.setattr(ops, "BESIDE_8BIT_FLOPS", 0.0)
    for _ in range(4):
        got, _ = attend(ops, cache, lens, heads, dtype, decode_prefix=10, ctx_lens=held)
        assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("columns", [16, 130])
def test_captured_store_and_attention(ops, dtype, columns):
    """A decode step as a graph holds it, replayed as the contexts grow, beside another graph of the same calls: the bits of eager calls."""
    heads, kv, dim, steps = 8, 2, 128, 5
    cache = Cache([70 + steps, 15 + steps, 200 + steps], kv, dim, 64)
    wide = torch.full((3, columns), -1, dtype=torch.int32)
    wide[:, :cache.table.shape[1]] = cache.table
    table = wide.to(DEV)
    cos, sin = (t.to(DEV) for t in tables(300, dim))
    weight = torch.rand(dim, generator=torch.Generator().manual_seed(2)).to(DEV)
    rows = torch.randn(steps, 3, 12 * dim, generator=torch.Generator().manual_seed(1)).to(dtype).to(DEV)
    qkv = torch.zeros_like(rows[0])
    starts = [70, 15, 200]
    positions, seq, q_start, start_pos = batch_index([1, 1, 1], starts, DEV)

    def step(device, out=None):
        q = ops.norm_rope_kv_store_4bit(qkv, cos, sin, dim, positions, seq, 3, table, *device, heads, kv, dim, q_norm=weight, k_norm=weight)
        return ops.attention_4bit(q, *device, table, q_start, start_pos, positions, seq, 3, 1, columns * 64, heads, kv, dim, 0.09, out=out)

    def at(i):
        qkv.copy_(rows[i])
        positions.copy_(torch.tensor([s + i for s in starts], dtype=torch.int32))
        start_pos.copy_(positions)

    eager, want = cache.device(), []
    for i in range(steps):
        at(i)
        want.append(step(eager))
    graphs = []
    at(0)
    for _ in range(2):
        device, out = cache.device(), torch.empty(3, heads * dim, dtype=dtype, device=DEV)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(device, out)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step(device, out)
        graphs.append((graph, device, out))
    for i in range(steps):
        at(i)
        for graph, _, _ in graphs:
            graph.replay()
        for _, device, out in graphs:
            assert torch.equal(out, want[i])
    for _, device, _ in graphs:
        assert all(torch.equal(a.nan_to_num(0) if a.is_floating_point() else a, b.nan_to_num(0) if b.is_floating_point() else b) for a, b in zip(device, eager))
    ops.check_status()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("heads,kv,dim,page", [(14, 2, 128, 64), (6, 2, 64, 16), (4, 2, 80, 16)])
def test_together(ops, dtype, heads, kv, dim, page):
    """A prompt in two portions beside another request, single tokens behind them: what attention over the bfloat16 rows' own entries gives, in 64 bits."""
    cache = Cache([150, 90], kv, dim, page)
    device = cache.device()
    cos, sin = tables(200, dim)
    gen = torch.Generator().manual_seed(7)
    weight = 1.0 + 0.2 * torch.randn(dim, generator=gen)
    qkv = torch.randn(240, (heads + 2 * kv) * dim, generator=gen).to(dtype)
    rows = {0: qkv[:150], 1: qkv[150:]}
    at = [0, 0]
    got = [[], []]
    for lens in ([100, 20], [47, 69], [1, 1], [1, 0], [1, 0]):
        positions, seq, q_start, start_pos = batch_index(lens, at, DEV)
        step = torch.cat([rows[r][at[r]:at[r] + n] for r, n in enumerate(lens)]).to(DEV)
        held = [a + n for a, n in zip(at, lens)]
        q = ops.norm_rope_kv_store_4bit(step, cos.to(DEV), sin.to(DEV), dim, positions, seq, 2, cache.table.to(DEV), *device, heads, kv, dim,
                                        q_norm=weight.to(DEV), k_norm=weight.to(DEV))
        out = ops.attention_4bit(q, *device, cache.table.to(DEV), q_start, start_pos, positions, seq, 2, max(lens), max(held), heads, kv, dim, dim ** -0.5, ctx_lens=held)
        for r, part in enumerate(out.split(lens)):
            got[r].append(part.cpu())
        at = held
    ops.check_status()
    cache.codes, cache.pairs = {"k": device[0].cpu(), "v": device[1].cpu()}, {"k": device[2].cpu(), "v": device[3].cpu()}
    for r in range(2):
        x = rows[r].float().view(len(rows[r]), heads + 2 * kv, dim)
        q = torch.stack([plain.turned(plain.normalised(x[i, :heads], weight, 1e-6), cos, sin, dim, i, False) for i in range(len(x))]).to(dtype)
        want = attention_of(q, cache.values("k", r)[:len(x)], cache.values("v", r)[:len(x)], 0, dim ** -0.5, 0, None)
        assert rel_error(torch.cat(got[r])[:len(x)], want.flatten(1)) < TOL[dtype]
        # and no further from attention over the rows themselves than steps of a fifteenth of a group's span explain: a standard normal group spans some 4.2,
        # so values are off by a step over sqrt(12), 0.08, before they are averaged, and scores by 0.08 x sqrt(dim) x dim^-0.5 x |q|
        k = torch.stack([plain.turned(plain.normalised(x[i, heads:heads + kv], weight, 1e-6), cos, sin, dim, i, False) for i in range(len(x))])
        free = attention_of(q, k, x[:, heads + kv:], 0, dim ** -0.5, 0, None)
        assert float((want - free).pow(2).mean().sqrt()) < 0.2 * float(free.pow(2).mean().sqrt())


def test_nothing_to_do(ops):
    cache = Cache([5], 2, 64, 16)
    empty = lambda *shape: torch.empty(shape, dtype=torch.bfloat16, device=DEV)  # noqa: E731
    none = torch.empty(0, dtype=torch.int32, device=DEV)
    start = torch.zeros(1, dtype=torch.int32, device=DEV)
    assert ops.norm_rope_kv_store_4bit(empty(0, 6 * 64), None, None, 0, none, none, 0, cache.table.to(DEV), *cache.device(), 2, 2, 64).shape == (0, 128)
    assert ops.attention_4bit(empty(0, 128), *cache.device(), cache.table.to(DEV), start, none, none, none, 0, 0, 0, 2, 2, 64, 0.1).shape == (0, 128)
    k, _v, table = ops.read_cache_4bit(*cache.device(), cache.table.to(DEV), start, none, [], 64, torch.bfloat16)
    assert k.shape == (0, 2, 64, 64) and table.shape == (0, 0)


def test_refusals(ops):
    cache = Cache([20], 2, 64, 16)
    kp, vp, kg, vg = cache.device()
    table = cache.table.to(DEV)
    positions, seq, q_start, start_pos = batch_index([1], [19], DEV)
    q = torch.zeros(1, 4 * 64, dtype=torch.bfloat16, device=DEV)
    qkv = torch.zeros(1, 8 * 64, dtype=torch.bfloat16, device=DEV)

    def attention(q=q, kp=kp, vp=vp, kg=kg, vg=vg, table=table, q_start=q_start, positions=positions, seqs=1, heads=4, kv=2, dim=64, **kw):
        return ops.attention_4bit(q, kp, vp, kg, vg, table, q_start, start_pos, positions, seq, seqs, 1, 20, heads, kv, dim, 0.1, **kw)

    def stored(qkv=qkv, kp=kp, vp=vp, kg=kg, vg=vg, rotary=0, cos=None, sin=None, positions=positions, seqs=1, heads=4, kv=2, dim=64, **kw):
        return ops.norm_rope_kv_store_4bit(qkv, cos, sin, rotary, positions, seq, seqs, table, kp, vp, kg, vg, heads, kv, dim, **kw)

    def read(ctx=(20,), dim=64, dtype=torch.float32, **kw):
        return ops.read_cache_4bit(kp, vp, kg, vg, table, q_start, start_pos, list(ctx), dim, dtype, **kw)

    attention(), stored(), read()
    angles = lambda n: {"cos": torch.zeros(30, n, device=DEV), "sin": torch.zeros(30, n, device=DEV)}  # noqa: E731
    wrong = [
        lambda: attention(q=q.half()), lambda: attention(q=q.cpu()), lambda: attention(kp=kp.float()), lambda: attention(kp=kp[:, :1]),
        lambda: attention(vp=vp[:1]), lambda: attention(kg=kg.float()), lambda: attention(kg=kg[..., :2].contiguous()), lambda: attention(vg=vg[:, :, :8].contiguous()),
        lambda: attention(heads=5), lambda: attention(heads=8), lambda: attention(seqs=2), lambda: attention(positions=positions.long()),
        lambda: attention(q_start=q_start[:1]), lambda: attention(ctx_lens=[20, 20]), lambda: attention(sink=torch.zeros(3, device=DEV)),
        lambda: attention(window=-1), lambda: attention(decode_prefix=2), lambda: attention(out=torch.zeros(1, 5, dtype=torch.bfloat16, device=DEV)),
        lambda: attention(out=torch.zeros(1, 256, device=DEV)), lambda: attention(dim=32), lambda: attention(table=table.long()), lambda: attention(kp=kp.cpu()),
        lambda: stored(qkv=qkv[:, :7 * 64]), lambda: stored(qkv=qkv.int()), lambda: stored(rotary=64), lambda: stored(rotary=3, **angles(1)),
        lambda: stored(rotary=66, **angles(33)), lambda: stored(rotary=-2, **angles(1)), lambda: stored(kp=kp.to(torch.int8)), lambda: stored(positions=positions[:0]),
        lambda: stored(out=torch.zeros(1, 5, dtype=torch.bfloat16, device=DEV)), lambda: stored(kg=kg.transpose(1, 2)), lambda: stored(seqs=2),
        lambda: stored(q_norm=torch.ones(32, device=DEV)), lambda: stored(k_norm=torch.ones(64, device=DEV).double()), lambda: stored(heads=0),
        lambda: stored(k_norm=torch.ones(64, device=DEV), eps=-1.0), lambda: stored(q_norm=torch.ones(64, device=DEV), eps=0.0), lambda: stored(k_norm=torch.ones(64, device=DEV), eps=math.nan),
        lambda: read(dtype=torch.float16), lambda: read(ctx=(20, 20)), lambda: read(dim=128), lambda: read(window=-1), lambda: read(first_seq=2), lambda: read(q_lens=[1, 1]),
    ]
    for i, call in enumerate(wrong):
        with pytest.raises((ops.KernelError, AttributeError, TypeError)):
            call()
            pytest.fail(f"call {i} was taken")
    wide = torch.zeros(4, 2, 16, 160, dtype=torch.uint8, device=DEV), torch.zeros(4, 2, 16, 20, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(ops.KernelError):
        attention(q=torch.zeros(1, 4 * 320, device=DEV), kp=wide[0], vp=wide[0], kg=wide[1], vg=wide[1], dim=320)
    ops.check_status()


class Elsewhere(torch.Tensor):
    """A tensor that says that it is on the device behind its own."""

    def get_device(self):
        return super().get_device() + 1


@pytest.mark.parametrize("which", range(8))
def test_tensors_of_another_device_are_refused(ops, which):
    cache = Cache([20], 2, 64, 16)
    held, table = cache.device(), cache.table.to(DEV)
    positions, seq, q_start, start_pos = batch_index([1], [19], DEV)
    q, qkv = torch.zeros(1, 256, dtype=torch.bfloat16, device=DEV), torch.zeros(1, 512, dtype=torch.bfloat16, device=DEV)
    weight, sink, angles = torch.ones(64, device=DEV), torch.zeros(4, device=DEV), torch.zeros(30, 32, device=DEV)

    def at(place, tensor):
        return tensor.as_subclass(Elsewhere) if place == which else tensor

    with pytest.raises(ops.KernelError):
        ops.attention_4bit(at(0, q), *held, table, at(1, q_start), at(2, start_pos), at(3, positions), at(4, seq), 1, 1, 20, 4, 2, 64, 0.1,
                           sink=at(5, sink), out=at(6, torch.empty_like(q)), **({"ctx_lens": [20, 20]} if which == 7 else {}))
    with pytest.raises(ops.KernelError):
        ops.norm_rope_kv_store_4bit(at(0, qkv), at(1, angles), at(2, angles), 64, at(3, positions), at(4, seq), 1, table, *held, 4, 2, 64,
                                    q_norm=at(5, weight), k_norm=weight, out=at(6, torch.empty_like(q)), eps=0.0 if which == 7 else 1e-6)
    with pytest.raises(ops.KernelError):
        ops.read_cache_4bit(*held, table, at(0, q_start), at(1, start_pos), [-64] if which in (2, 4, 6) else [20], 64, torch.float32,
                            window=8, q_lens=[-300] if which in (3, 5, 7) else [1])
    ops.check_status()
