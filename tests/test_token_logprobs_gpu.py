"""Log probabilities of given tokens on the device against their definition in float64."""
import math

import pytest
import torch

from plain import cache_8bit_plain as plain

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module")
def ops():
    from aegean_tge_b200 import ops as module
    module.core()
    return module


def close(got, want):
    """A logit less its row's maximum and the logarithm of a sum: a few roundings of float32 at the size of what is subtracted."""
    got, want = float(got), float(want)
    if math.isnan(want) or math.isinf(want):
        return math.isnan(got) if math.isnan(want) else got == want
    return abs(got - want) <= 2e-6 * (8 + abs(want))


def check(ops, logits, tokens, top):
    found = [t.cpu() for t in ops.token_logprobs(logits.to(DEV), torch.tensor(tokens, dtype=torch.int32, device=DEV), top=top)]
    ops.check_status()
    for r, token in enumerate(tokens):
        lp, entropy, rank, ids, lps = plain.token_logprobs(logits[r].double().tolist(), token, top)
        assert close(found[0][r], lp), (r, float(found[0][r]), lp)
        assert close(found[1][r], entropy), (r, float(found[1][r]), entropy)
        assert int(found[2][r]) == rank
        assert found[3][r].tolist() == ids
        assert all(close(a, b) for a, b in zip(found[4][r].tolist(), lps))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,vocab,top", [(1, 1, 1), (1, 1, 0), (3, 2, 2), (2, 31, 5), (4, 32, 32), (2, 33, 32), (5, 257, 20), (3, 1000, 0), (2, 4096, 20), (2, 16384, 8),
                                            (2, 16385, 32), (1, 50257, 20), (3, 152064, 20), (1, 152063, 1), (300, 997, 5)])
def test_random_rows(ops, dtype, rows, vocab, top):
    gen = torch.Generator().manual_seed(rows + vocab)
    logits = (torch.randn(rows, vocab, generator=gen) * 3).to(dtype)
    tokens = torch.randint(0, vocab, (rows,), generator=gen).tolist()
    tokens[0], tokens[-1] = vocab - 1, int(logits[-1].float().argmax())
    check(ops, logits, tokens, top)


@pytest.mark.parametrize("vocab", [40, 5000, 70000])
def test_rows_that_are_hard_to_choose_from(ops, vocab):
    """Equal logits, rising and falling ones, two values, zeros of both signs, one that stands out, masks of all but a few."""
    n = torch.arange(vocab, dtype=torch.float32)
    rows = [torch.zeros(vocab), n / 100, -n / 100, (n % 2), (n % 7 == 3).float() * 50 - 1e30, torch.where(n % 2 == 0, 0.0, -0.0),
            torch.full((vocab,), -math.inf).index_fill(0, torch.tensor([7, 3, vocab - 1]), 2.0),
            torch.full((vocab,), -math.inf).index_fill(0, torch.tensor([vocab // 2]), -3e38),
            torch.where(n >= vocab - 10, n, torch.full_like(n, -3.4e38)), torch.full((vocab,), 3e38), (n - vocab) * 1e-30]
    logits = torch.stack(rows)
    for dtype in (torch.float32, torch.bfloat16):
        for top in (1, 20, 32):
            check(ops, logits.to(dtype), [(13 * r) % vocab for r in range(len(rows))], top)


@pytest.mark.parametrize("vocab", [40, 9000, 70000])
def test_rows_without_a_distribution(ops, vocab):
    gen = torch.Generator().manual_seed(1)
    logits = torch.randn(6, vocab, generator=gen)
    logits[0, 17] = math.nan
    logits[1, vocab - 1] = math.inf
    logits[2] = -math.inf
    logits[3] = math.nan
    logits[4, 3::2] = -math.nan
    check(ops, logits, [17, 5, 0, 9, 2, 11], 12)


def test_inner_rows_and_odd_strides(ops):
    gen = torch.Generator().manual_seed(2)
    for dtype in (torch.float32, torch.bfloat16):
        for lead in (0, 1, 3, 4, 8):
            wide = torch.randn(4, 5003, generator=gen).to(dtype)
            inner = wide.to(DEV)[:, lead:lead + 4990]
            whole = [t.cpu() for t in ops.token_logprobs(inner.contiguous(), torch.tensor([0, 1, 4989, 77], dtype=torch.int32, device=DEV), top=9)]
            found = [t.cpu() for t in ops.token_logprobs(inner, torch.tensor([0, 1, 4989, 77], dtype=torch.int32, device=DEV), top=9)]
            check(ops, wide[:, lead:lead + 4990], [0, 1, 4989, 77], 9)
            assert torch.equal(whole[2], found[2]) and torch.equal(whole[3], found[3])
            for a, b in zip(whole, found):
                assert torch.allclose(a.double(), b.double(), rtol=2e-6, atol=2e-5)


def test_the_same_twice_and_on_another_stream(ops):
    logits = torch.randn(5, 152064, device=DEV)
    tokens = torch.tensor([1, 2, 3, 4, 152063], dtype=torch.int32, device=DEV)
    first = ops.token_logprobs(logits, tokens, top=20)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        again = ops.token_logprobs(logits, tokens, top=20)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_a_token_outside_the_vocabulary_is_reported(ops):
    logits = torch.randn(3, 500, device=DEV)
    lp, entropy, rank, ids, _ = ops.token_logprobs(logits, torch.tensor([500, 2, -1], dtype=torch.int32, device=DEV), top=3)
    with pytest.raises(ops.DeviceStatusError):
        ops.check_status()
    assert torch.isnan(lp[0]) and torch.isnan(lp[2]) and torch.isfinite(lp[1]) and rank.tolist()[::2] == [-1, -1]
    assert torch.isfinite(entropy).all() and torch.equal(ids[:, 0].long(), logits.argmax(-1))


def test_refusals(ops):
    logits = torch.zeros(2, 50, device=DEV)
    tokens = torch.zeros(2, dtype=torch.int32, device=DEV)
    assert ops.token_logprobs(logits[:0], tokens[:0], top=3)[3].shape == (0, 3)
    for call in (lambda: ops.token_logprobs(logits.half(), tokens), lambda: ops.token_logprobs(logits.cpu(), tokens), lambda: ops.token_logprobs(logits, tokens.long()),
                 lambda: ops.token_logprobs(logits, tokens[:1]), lambda: ops.token_logprobs(logits, tokens, top=33), lambda: ops.token_logprobs(logits[:, :10], tokens, top=11),
                 lambda: ops.token_logprobs(logits, tokens, top=-1), lambda: ops.token_logprobs(logits.t(), tokens), lambda: ops.token_logprobs(logits[0], tokens)):
        with pytest.raises(ops.KernelError):
            call()
    ops.check_status()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,vocab,top", [(20, 40001, 32), (70, 33333, 5), (17, 100003, 0), (100, 50000, 20), (80, 70001, 32), (16, 16500, 1), (1, 12289, 32)])
def test_rows_cut_every_way(ops, dtype, rows, vocab, top):
    """Chunks that a cluster of 8 or 16 blocks joins, chunks that a second kernel joins, of odd vocabularies."""
    gen = torch.Generator().manual_seed(rows)
    logits = torch.randn(rows, vocab, generator=gen).to(dtype)
    logits[0, :vocab // 2] = -math.inf
    logits[-1] = torch.arange(vocab).to(dtype) / vocab
    check(ops, logits, torch.randint(0, vocab, (rows,), generator=gen).tolist(), top)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,vocab", [(1, 152064), (16, 152064), (64, 152064), (17, 100003), (600, 20001)])
def test_ranks_of_tokens_that_cannot_come(ops, dtype, rows, vocab):
    """Rows of -inf but for a few: a token of -inf comes behind those and the -inf of lower index, whatever chunks a row is cut into."""
    there = [7, vocab // 3, vocab // 2 + 1, vocab - 1]
    borders = [b for blocks in (8, 16) for chunk in [-(-(-(-vocab // blocks)) // 64) * 64] for b in range(chunk, vocab, chunk)]
    masked = sorted({t for b in [0, 100, 4096, 8192, vocab - 2, *borders] for t in (b - 1, b, b + 1, b + 2500) if 0 <= t < vocab} - set(there))
    logits = torch.full((rows, vocab), -math.inf, device=DEV)
    logits[:, there] = torch.tensor([2.0, -3e38, 0.5, -40.0], device=DEV)
    logits = logits.to(dtype)
    for first in range(0, len(masked), rows):
        tokens = [masked[(first + r) % len(masked)] for r in range(rows)]
        lp, _, rank, _, _ = ops.token_logprobs(logits, torch.tensor(tokens, dtype=torch.int32, device=DEV), top=0)
        assert (lp == -math.inf).all()
        assert rank.tolist() == [len(there) + t - sum(i < t for i in there) for t in tokens]
    ops.check_status()
