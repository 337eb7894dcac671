"""Requests behind a common prefix over an engine that is not there: what their results say of it when a run is cancelled, and caches
that do not hold a request beside the prefix."""
from types import SimpleNamespace

import numpy as np
import pytest

from quicknn_b200.engine import llm as module
from quicknn_b200.sampling import GenerationOptions


class FakeEngine:
    """Slots and lengths without a model."""

    def __init__(self, max_batch):
        self.cache = SimpleNamespace(max_tokens=64 * 64)
        self.max_seq, self.device = 512, "cpu"
        self.model = SimpleNamespace(spec=SimpleNamespace(embedding=SimpleNamespace(vocab_size=100)))
        self.free, self.prefixes_run = list(range(max_batch)), 0

    def new_sequence(self):
        return self.free.pop()

    def fork(self, slots):
        return [self.free.pop() for _ in slots]

    def release(self, slot):
        assert slot not in self.free
        self.free.append(slot)

    def step(self, entries, want):
        self.prefixes_run += 1


@pytest.fixture
def fake(monkeypatch):
    monkeypatch.setattr(module._PrefixBackend, "_start", lambda self, first, prompts, new: np.full(len(prompts), 7))
    monkeypatch.setattr(module._PrefixBackend, "advance", lambda self, keep: np.full(len(keep), 7))
    me = module.LLM.__new__(module.LLM)
    me.engine, me.max_batch, me.run_ahead = FakeEngine(3), 3, True
    me._sampler = lambda options: None
    return me


@pytest.mark.parametrize("n", [2, 7])
@pytest.mark.parametrize("probes,started", [(0, 0), (1, 2), (2, 2), (100, 7)])
def test_requests_that_were_not_started_reused_nothing(fake, n, probes, started):
    """``probes``: how often the caller says to go on.  Seven requests run two at a time: the prefix keeps one of the three sequences."""
    asked = []

    def should_cancel():
        asked.append(1)
        return len(asked) > probes

    got = fake.generate([[1, 2]] * n, GenerationOptions.greedy(1), prefix=[5] * 30, should_cancel=should_cancel, stop_ids=[])
    assert [r.reused_tokens for r in got] == [30] * min(started, n) + [0] * (n - min(started, n))
    assert all(r.prompt_tokens == 32 for r in got)
    assert sorted(fake.engine.free) == [0, 1, 2] and fake.engine.prefixes_run == (1 if started else 0)


def test_without_a_prefix_nothing_is_reused(fake, monkeypatch):
    monkeypatch.setattr(module._Backend, "_start", lambda self, first, prompts, new: np.full(len(prompts), 7))
    got = fake.generate([[1, 2]] * 2, GenerationOptions.greedy(1), stop_ids=[])
    assert [r.reused_tokens for r in got] == [0, 0]


@pytest.mark.parametrize("max_tokens,max_batch,runs", [(512, 3, 3), (576, 3, 1), (1024, 3, 1), (4096, 2, 1)])
def test_a_request_that_has_no_room_beside_the_prefix_runs_without_it(fake, max_tokens, max_batch, runs):
    """Each request may grow to 512 positions, the prefix takes a page of 64.  A cache that holds a request alone runs the prefix for every
    batch; one that holds both runs it once."""
    fake.engine.cache.max_tokens, fake.max_batch = max_tokens, max_batch
    got = fake.generate([[1, 2]] * 3, GenerationOptions.greedy(480), prefix=[5] * 30, stop_ids=[7])
    assert [r.finish_reason for r in got] == ["eos"] * 3 and [r.reused_tokens for r in got] == [30] * 3
    assert fake.engine.prefixes_run == runs and sorted(fake.engine.free) == [0, 1, 2]
