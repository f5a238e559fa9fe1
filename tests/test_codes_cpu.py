"""What the host works out for attention over a cache of codes."""


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
