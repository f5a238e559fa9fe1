"""What the host works out for attention over a cache of codes."""
import pytest
import torch


def test_scratch_sizes_are_kept_by_device(monkeypatch):
    """The library's answer depends on the device's number of SMs: one of another device is asked for anew."""
    from aegean_tge_b200 import ops
    asked, device = [], [0]

    def ask(*sizes):
        asked.append((device[0], sizes))
        return 100 * (device[0] + 1)

    ask.__name__ = "tge_of_a_test"
    monkeypatch.setattr(ops, "_codes_floats", {})
    monkeypatch.setattr(ops, "_current_device", lambda: device[0])
    for here, want in ((0, 100), (1, 200), (0, 100), (1, 200)):
        device[0] = here
        assert ops._decode_floats(ask, 1, 8, 28) == want
    assert asked == [(0, (1, 8, 28)), (1, (1, 8, 28))]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("singles", [0, 2, 9])
def test_portions_behind_single_tokens_are_counted_from_their_own_first_request(monkeypatch, dtype, singles):
    """The tables and first tokens that a read-back makes begin with the portions' first request, and so do the requests that rows name: the attention kernel
    for rows on odd elements looks them up there."""
    from aegean_tge_b200 import ops
    lens, dim, heads = [1] * singles + [3, 2], 64, 4
    seqs, tokens, calls = len(lens), sum(lens), []
    seq = torch.tensor([r for r, n in enumerate(lens) for _ in range(n)], dtype=torch.int32)
    rows = torch.zeros(tokens, heads * dim + 1, dtype=dtype)
    q, out = rows[:, 1:], torch.zeros(tokens, heads * dim, dtype=dtype)
    positions, start_pos = torch.arange(tokens, dtype=torch.int32), torch.arange(seqs, dtype=torch.int32)
    monkeypatch.setattr(ops, "core", lambda: None)
    monkeypatch.setattr(ops, "mma_attention_supports", lambda *args: True)
    monkeypatch.setattr(ops, "attention", lambda *args, **kw: calls.append((args, kw)))
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)

    def read_as(kind, first, starts):
        assert (kind, first, starts.numel()) == (dtype, singles, 3)
        return "k", "v", "table"

    ops._attend_codes(q, out, q.stride(0), out.stride(0), torch.zeros(seqs + 1, dtype=torch.int32), start_pos, positions, seq, seqs, 3, heads, 2, dim, 0.1, 0,
                      None, [100] * seqs, singles, singles > 0, lambda: singles, None, read_as)
    (found_q, k, v, table, starts, found_start, found_positions, found_seq, count, *_), kw = calls[0]
    assert (k, v, table, count) == ("k", "v", "table", 2) and found_q.shape[0] == kw["out"].shape[0] == 5
    assert found_start.tolist() == [singles, singles + 1] and found_positions.tolist() == list(range(singles, singles + 5))
    assert found_seq.tolist() == [0, 0, 0, 1, 1] and found_seq.dtype == torch.int32
