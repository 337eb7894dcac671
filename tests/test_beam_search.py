"""Beam search's decisions on the host, with a language model that is a table: against a plain search and against all replies there are."""
import itertools
import math

import numpy as np
import pytest

from quicknn_b200.engine.beam import BeamBackend, beam_search
from quicknn_b200.engine.generate import CONTEXT_FULL, EOS, MAX_TOKENS, PromptError
from quicknn_b200.sampling import BeamOptions, OptionsError


class Toy(BeamBackend):
    """Log-probabilities of the next token drawn from the tokens so far; keeps the books that the engine's backend keeps."""

    def __init__(self, vocab=7, beams=3, take=6, max_batch=12, max_seq=64, max_tokens=1 << 20, seed=0):
        self.vocab_size, self.beams, self.take, self.max_batch, self.max_seq, self.max_tokens, self.seed = vocab, beams, take, max_batch, max_seq, max_tokens, seed
        self.rows, self.finished = [], 0

    def logp(self, seq):
        z = np.random.default_rng([self.seed] + [int(t) for t in seq]).normal(size=self.vocab_size) * 2
        return z - math.log(np.exp(z).sum())

    def _best(self, rows, scores):
        total = np.array([s + self.logp(r) for r, s in zip(rows, scores)])
        flat = total.reshape(-1)
        order = np.lexsort((np.arange(flat.size), -flat))[:self.take]
        out = np.full(self.take, -np.inf), np.full(self.take, -1), np.full(self.take, -1)
        n = int(np.isfinite(flat[order]).sum())
        out[0][:n], out[1][:n], out[2][:n] = flat[order][:n], order[:n] // self.vocab_size, order[:n] % self.vocab_size
        return out

    def begin(self, prompts):
        assert not self.rows and len(prompts) * self.beams <= self.max_batch
        self.rows = [[list(p)] for p in prompts]
        return [np.stack(x) for x in zip(*[self._best(r, [0.0]) for r in self.rows])]

    def advance(self, keep, parents, tokens, scores):
        assert parents.shape == tokens.shape == scores.shape == (len(keep), self.beams)
        self.rows = [[self.rows[r][int(p)] + [int(t)] for p, t in zip(parents[i], tokens[i])] for i, r in enumerate(keep)]
        return [np.stack(x) for x in zip(*[self._best(r, scores[i]) for i, r in enumerate(self.rows)])]

    def finish(self):
        self.rows, self.finished = [], self.finished + 1


def plain(toy, prompt, o, stop, room):
    """The same search, written down once more as lists."""
    limit = min(o.max_new_tokens, room)
    open_, done = [([], 0.0)], []
    norm = lambda lp, n: lp / n ** o.length_penalty  # noqa: E731
    for length in range(1, limit + 1):
        cand = sorted(((-(lp + v), b, t) for b, (seq, lp) in enumerate(open_) for t, v in enumerate(toy.logp(list(prompt) + seq))))
        nxt = []
        for rank, (neg, b, t) in enumerate(cand[:toy.take]):
            if len(nxt) == o.beams:
                break
            if t in stop:
                if rank < o.beams:
                    done.append((norm(-neg, length), open_[b][0], EOS))
            else:
                nxt.append((open_[b][0] + [t], -neg))
        done = sorted(done, key=lambda d: -d[0])[:o.beams]
        open_ = nxt
        if len(done) == o.beams and (o.early_stopping or not open_ or norm(open_[0][1], length) <= done[-1][0]):
            if length < limit:
                return done
        if not open_:
            return done
    reason = CONTEXT_FULL if room <= o.max_new_tokens else MAX_TOKENS
    return sorted(done + [(norm(lp, limit), seq, reason) for seq, lp in open_], key=lambda d: -d[0])[:o.beams]


@pytest.mark.parametrize("beams,penalty,early,n", [(1, 1.0, False, 5), (3, 1.0, False, 8), (3, 0.0, True, 8), (4, 2.0, False, 6), (2, -0.5, False, 9), (3, 1.0, True, 1)])
@pytest.mark.parametrize("stop", [(), (2,), (0, 5)])
@pytest.mark.parametrize("seed", range(5))
def test_against_a_plain_search(beams, penalty, early, n, stop, seed):
    o = BeamOptions(beams=beams, max_new_tokens=n, length_penalty=penalty, early_stopping=early, replies=beams)
    toy = Toy(beams=beams, take=o.take(len(stop)), seed=seed)
    prompts = [[1], [3, 4], [5, 1, 1], [2, 2], [6]]
    got = beam_search(toy, prompts, o, stop)
    assert [r.index for r in got] == list(range(5)) and toy.finished >= 1 and not toy.rows
    for r, p in zip(got, prompts):
        want = plain(toy, p, o, stop, toy.max_seq - len(p))
        assert [(h.tokens, h.finish_reason) for h in r.replies] == [(w[1], w[2]) for w in want]
        assert np.allclose([h.score for h in r.replies], [w[0] for w in want], atol=1e-5)
        assert r.prompt_tokens == len(p)


def test_as_many_beams_as_replies_there_are_finds_the_best():
    toy = Toy(vocab=3, beams=9, take=9, seed=4)
    o = BeamOptions(beams=9, max_new_tokens=3, length_penalty=0.0, replies=9)
    got = beam_search(toy, [[1, 2]], o)[0]
    best = max(itertools.product(range(3), repeat=3), key=lambda s: sum(toy.logp([1, 2] + list(s[:i]))[t] for i, t in enumerate(s)))
    assert got.replies[0].tokens == list(best)


def test_context_and_rows():
    toy = Toy(beams=2, take=4, max_seq=6)
    o = BeamOptions(beams=2, max_new_tokens=50, replies=2)
    got = beam_search(toy, [[1, 2, 3, 4], [1]], o)
    assert [len(h.tokens) for h in got[0].replies] == [2, 2] and {h.finish_reason for r in got for h in r.replies} == {CONTEXT_FULL}
    assert len(got[1].replies[0].tokens) == 5


def test_fewer_continuations_than_beams():
    toy = Toy(vocab=2, beams=4, take=8)
    got = beam_search(toy, [[1]], BeamOptions(beams=4, max_new_tokens=3, replies=4), [0])
    assert got[0].replies and all(0 not in h.tokens for h in got[0].replies)


def test_refusals():
    for bad in (dict(beams=0), dict(beams=65), dict(max_new_tokens=0), dict(length_penalty=float("nan")), dict(replies=0), dict(beams=2, replies=3)):
        with pytest.raises(OptionsError):
            BeamOptions(**bad).validate()
    with pytest.raises(OptionsError):
        beam_search(Toy(), [[1]], BeamOptions(beams=33, replies=1), [0])             # 66 continuations a step
    o = BeamOptions(beams=3, max_new_tokens=4)
    for prompts in ([[]], [[1], [9]], [[1] * 64], [[-1]]):
        with pytest.raises(PromptError):
            beam_search(Toy(), prompts, o)
    with pytest.raises(PromptError):
        beam_search(Toy(max_batch=2), [[1]], o)
    with pytest.raises(PromptError):
        beam_search(Toy(max_tokens=128), [[1]], o)                                   # three beams hold three pages
    toy = Toy(max_tokens=3 * 64)
    assert len(beam_search(toy, [[1], [2]], o)) == 2 and toy.finished == 2           # one request at a time


def test_launches_of_the_selection_are_counted_as_they_are():
    """one kernel where a request has few logits, else two, none without a request"""
    from quicknn_b200.kernels import lib
    kernels = lib.load().qnn_beam_select_kernels
    assert [kernels(*sizes) for sizes in ((1, 4, 1000, 8), (16, 4, 1000, 8), (1, 1, 3000, 8), (1, 11, 515, 22), (1, 64, 130, 64))] == [1] * 5
    assert [kernels(*sizes) for sizes in ((1, 8, 256000, 16), (16, 5, 255029, 10), (1, 1, 16384, 2), (1, 8, 16383, 16))] == [2] * 4
    assert kernels(0, 4, 1000, 8) == 0


@pytest.mark.parametrize("penalty", [33, 200.0, -200.0, 10 ** 400, float("inf"), float("nan"), "1"])
def test_length_penalties_whose_powers_are_no_numbers_are_refused(penalty):
    """200 ** 200.0 overflows and a score over 200 ** -200.0 divides by zero: in the middle of a search"""
    with pytest.raises(OptionsError):
        BeamOptions(length_penalty=penalty).validate()
    BeamOptions(length_penalty=32).validate()
    BeamOptions(length_penalty=-32.0).validate()
    assert 0 < (2 ** 31) ** 32.0 < float("inf") and (2 ** 31) ** -32.0 > 0
