"""How far single tokens over the 4-bit cache may be from float64, number by number."""
import pytest
import torch

from helpers import batch_index
from plain import cache_4bit_plain as plain
from test_cache_4bit_gpu import DEV, Cache, ops  # noqa: F401

pytestmark = pytest.mark.gpu


def bounds_of(cache, r, q, scale):
    """(attention in float64, a bound of what bfloat16 single tokens may be off), [heads, dim] both, of request r's last token.

    out = sum p v / sum p, v = base + (c - 8) step.  Probabilities go into the products as bfloat16, alone (beside the bases) and times the steps, each 2^-8 of
    itself off at most (half of bfloat16's eps); the sum of probabilities is of the numbers before that rounding.  With A = sum p (|base| + |c - 8| step) / sum p
    that is 2^-8 A, and the result's rounding 2^-8 |out| once more (1 + 2^-7: of what is off already).
    Scores: queries are exact in float16 (none is below 2^-27 of its row's largest), steps and bases are as they are held, a group's queries' sum is in
    three parts of eight bits, all that float32 has.  The bases' products are exact; a tensor core step adds the parts of two groups that count here (the others' are
    small), each cut 2^-24 below the largest at most: 2^-22 B, B = scale max |base sum q|, twice that with the second step.  The codes' products of a group
    are added by two such steps and the groups by a chain of eight additions at most, each 2^-23 of S = scale sum 15 step |q| off at most, sixteen of
    them with those inside a step: 2^-19 S.  Every p is a factor of 1 +- (2^-19 S + 2^-21 B) off (the largest over the positions), twice that with
    the denominator's.
    2^-18 A: the exponentials (2^-22) and float32 sums of up to some hundred terms.
    """
    pairs = cache.of("k", r)[1].double()
    group, dim = q.shape[0] // cache.kv_heads, cache.dim
    j = torch.arange(dim) // 32
    k, v = cache.values("k", r), cache.values("v", r)
    codes, of = plain.unpack(cache.of("v", r)[0], dim), cache.of("v", r)[1].double()
    parts = of[..., 2 * j + 1].abs() + (codes - 8).abs().double() * of[..., 2 * j]
    out, bound = [], []
    for h in range(q.shape[0]):
        x, g = q[h].double(), h // group
        p = torch.softmax(k[:, g] @ x * scale, 0)
        a, s = p @ parts[:, g], 15 * scale * float((pairs[:, g, 2 * j] @ x.abs()).max())
        b = scale * float((pairs[:, g, 1::2] * x.view(-1, 32).sum(-1)).abs().max())
        out.append(p @ v[:, g])
        bound.append((2.0 ** -8 * a + 2.0 ** -8 * out[-1].abs()) * (1 + 2.0 ** -7) + (2.0 ** -18 * s + 2.0 ** -20 * b + 2.0 ** -18) * a)
    return torch.stack(out), torch.stack(bound)


@pytest.mark.parametrize("heads,kv,dim", [(40, 8, 128), (14, 2, 64), (8, 2, 256), (24, 2, 128)])
@pytest.mark.parametrize("scale", [0.09, 20.0])
@pytest.mark.parametrize("columns", [1, 130])
def test_single_tokens_number_by_number(ops, heads, kv, dim, scale, columns):
    """Few positions, where roundings do not cancel: a bit of the probabilities less is seen here."""
    cache = Cache([2, 3, 2, 4, 2, 5, 3, 2, 17, 40], kv, dim, 64)
    wide = torch.full((10, columns), -1, dtype=torch.int32)
    wide[:, :1] = cache.table
    positions, seq, q_start, start_pos = batch_index([1] * 10, [h - 1 for h in cache.held], DEV)
    q = torch.randn(10, heads, dim, generator=torch.Generator().manual_seed(9)).bfloat16()
    out = ops.attention_4bit(q.flatten(1).to(DEV), *cache.device(), wide.to(DEV), q_start, start_pos, positions, seq, 10, 1, 64, heads, kv, dim, scale)
    ops.check_status()
    for r in range(10):
        want, bound = bounds_of(cache, r, q[r], scale)
        off = (out[r].view(heads, dim).cpu().double() - want).abs()
        assert bool((off <= bound).all()), (r, float((off / bound).max()))


SCALE = 0.02


def opposing(cache, heads, seed=13):
    """Large bases of keys whose sums cancel: a position's bases b and -3 b (of either sign) in a head's first two groups, queries of a head's first group that are three times
    those of its second (six bits, so that three times them are bfloat16 too; their sum has some 20).  Scores are then the steps' and the other groups' alone."""
    gen = torch.Generator().manual_seed(seed)
    q = torch.randn(len(cache.held), heads, cache.dim, generator=gen)
    shape = (len(cache.held), heads, 32)
    low = torch.randint(33, 63, shape, generator=gen) * 2.0 ** torch.randint(-19, -5, shape, generator=gen).float()
    q[..., 32:64] = low * torch.where(torch.rand(shape, generator=gen) < 0.3, -1.0, 1.0)
    q[..., :32] = 3 * q[..., 32:64]
    assert torch.equal(q[..., :64], q[..., :64].bfloat16().float()) and float(q[..., :32].abs().sum(-1).max()) < 32       # sums of 24 bits at most
    for r, n in enumerate(cache.held):
        pos = torch.arange(n)
        where = cache.table[r, pos // cache.page].long()
        b = (56 + torch.randint(0, 8, (n, cache.kv_heads), generator=gen)) * 2.0 ** 14 * torch.where(torch.rand(n, cache.kv_heads, generator=gen) < 0.5, -1.0, 1.0)
        pairs = cache.pairs["k"][where, :, pos % cache.page]
        pairs[..., 1], pairs[..., 3] = b.bfloat16(), (-3 * b).bfloat16()
        cache.pairs["k"][where, :, pos % cache.page] = pairs
    return q.bfloat16()


@pytest.mark.parametrize("heads,kv,dim", [(10, 2, 128), (6, 2, 64), (5, 1, 256)])
@pytest.mark.parametrize("columns", [1, 130])
def test_bases_that_cancel(ops, heads, kv, dim, columns):
    """The sums of a group's queries have all their bits: bases of up to 3 x 2^20 cancel to nothing."""
    cache = Cache([40, 3, 64, 17], kv, dim, 64)
    q = opposing(cache, heads)
    wide = torch.full((4, columns), -1, dtype=torch.int32)
    wide[:, :1] = cache.table
    positions, seq, q_start, start_pos = batch_index([1] * 4, [h - 1 for h in cache.held], DEV)
    out = ops.attention_4bit(q.flatten(1).to(DEV), *cache.device(), wide.to(DEV), q_start, start_pos, positions, seq, 4, 1, 64, heads, kv, dim, SCALE)
    ops.check_status()
    for r in range(4):
        want, bound = bounds_of(cache, r, q[r], SCALE)
        off = (out[r].view(heads, dim).cpu().double() - want).abs()
        assert bool((off <= bound).all()), (r, float((off / bound).max()))
