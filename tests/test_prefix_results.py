"""What the results of requests behind a common prefix say of it when a run is cancelled, over an engine that is not there."""
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
