"""The listing of a step's kernels, on the host: what the profiler hands over in part is asked for again, and never listed."""
from types import SimpleNamespace

import pytest
import torch

from aegean_tge_b200 import bench_tools

KERNELS = 5


class Engine:
    def __init__(self):
        self.ops = SimpleNamespace(launches=0)
        self.spec = SimpleNamespace(vocab_size=100)
        self.model = SimpleNamespace(env=SimpleNamespace(ops=self.ops))
        self.runner = self
        self.live = set()

    def step(self, portions):
        self.live |= {p.request for p in portions}
        self.ops.launches += KERNELS

    def finish(self, name):
        self.live.discard(name)


@pytest.fixture
def handed(monkeypatch):
    """How many records each profile hands over, the last number for all that follow; the pauses that were made."""
    made = SimpleNamespace(counts=[KERNELS], profiles=0, pauses=[])

    class Profile:
        def __init__(self, activities):
            self.count = made.counts[min(made.profiles, len(made.counts) - 1)]
            made.profiles += 1

        def __enter__(self):
            return self

        def __exit__(self, *what):
            return False

        def events(self):
            return [SimpleNamespace(time_range=SimpleNamespace(start=10.0 * i), device_time_total=4.0, name=f"kernel_{i}(int)") for i in range(self.count)]

    monkeypatch.setattr(torch.profiler, "profile", Profile)
    monkeypatch.setattr(torch.cuda, "synchronize", lambda *a: None)
    monkeypatch.setattr(bench_tools.time, "sleep", made.pauses.append)
    return made


def test_a_whole_listing_is_taken_at_once(handed):
    engine = Engine()
    rows = bench_tools.step_timeline(engine, 1, 20, prefill=True)
    assert [r["kernel"] for r in rows[:-1]] == [f"kernel_{i}" for i in range(KERNELS)] and rows[-1]["launches"] == KERNELS
    assert handed.profiles == 1 and not engine.live


def test_a_part_is_asked_for_again(handed):
    handed.counts = [2, 0, 4, 1, 3, KERNELS]
    rows = bench_tools.step_timeline(Engine(), 1, 20, prefill=True)
    assert rows[-1]["launches"] == KERNELS and handed.profiles == 6
    assert sorted(handed.pauses) == handed.pauses and handed.pauses[-1] > 0


def test_a_part_is_never_listed(handed, monkeypatch):
    handed.counts = [KERNELS - 1]
    monkeypatch.setattr(bench_tools, "fill_cache", lambda engine, batch, length, prefix: [f"{prefix}{i}" for i in range(batch)])
    for prefill in (True, False):
        engine = Engine()
        with pytest.raises(RuntimeError, match="profiler"):
            bench_tools.step_timeline(engine, 2, 20, prefill=prefill)
        assert not engine.live


def test_a_step_in_front_takes_what_the_profiler_drops_first(handed, monkeypatch):
    """A profiler that never has the first kernels of its window: the step in front is what it drops, and what is left of that is not listed."""
    engine, clock, dropped = Engine(), SimpleNamespace(now=0.0, kernels=[]), 3

    class Profile:
        def __init__(self, activities):
            clock.kernels = []

        def __enter__(self):
            return self

        def __exit__(self, *what):
            return False

        def events(self):
            return [SimpleNamespace(time_range=SimpleNamespace(start=at), device_time_total=4.0, name=f"kernel_{i % KERNELS}(int)")
                    for i, at in enumerate(clock.kernels) if i >= dropped]

    def step(portions):
        engine.ops.launches += KERNELS
        for _ in range(KERNELS):
            clock.kernels.append(clock.now)
            clock.now += 5.0

    def sleep(seconds):
        clock.now += 1e6 * seconds

    monkeypatch.setattr(engine, "step", step, raising=False)
    monkeypatch.setattr(torch.profiler, "profile", Profile)
    monkeypatch.setattr(bench_tools.time, "sleep", sleep)
    rows = bench_tools.step_timeline(engine, 1, 20, prefill=True)
    assert sorted(r["kernel"] for r in rows[:-1]) == [f"kernel_{i}" for i in range(KERNELS)] and rows[-1]["launches"] == KERNELS
    assert all(r["launches"] == 1 for r in rows[:-1]) and rows[-1]["us"] == 24.0
