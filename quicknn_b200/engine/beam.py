"""Beam search: the decisions on the host, over a small backend interface (so that they can be tested without a GPU).

Every request keeps ``beams`` rows of the batch.  A step gives its best continuations over all of its beams (best first); walking
down that list, a stop token among the first ``beams`` ends a reply (the stop token itself is not part of it), every other token
opens a hypothesis of the next step until there are ``beams`` of them.  A request whose search is over gives its rows back.
"""
from __future__ import annotations

import dataclasses
from typing import List, Optional, Sequence, Tuple

import numpy as np
import torch

from ..cache.pages import PAGE
from ..sampling.beam import BeamOptions, BeamSelector, check_beams
from .generate import CONTEXT_FULL, EOS, MAX_TOKENS, PromptError


@dataclasses.dataclass
class BeamReply:
    tokens: List[int]
    score: float                       # sum of log-probabilities over length ** length_penalty
    logprob: float                     # the sum
    finish_reason: str


@dataclasses.dataclass
class BeamResult:
    index: int
    prompt_tokens: int
    replies: List[BeamReply] = dataclasses.field(default_factory=list)      # best first


class BeamBackend:
    """What the search needs from the engine.  Rows are counted over all live requests, ``beams`` for each, in order."""

    max_batch: int
    max_tokens: int
    max_seq: int
    vocab_size: int

    def begin(self, prompts: Sequence[Sequence[int]]):
        """Run the prompts; (scores, beams, tokens) [requests, take] of the best first tokens."""
        raise NotImplementedError

    def advance(self, keep: Sequence[int], parents: np.ndarray, tokens: np.ndarray, scores: np.ndarray):
        """Drop the requests that are not in ``keep``; row (r, b) of the next step goes on from beam ``parents[r, b]`` of request
        ``keep[r]`` with ``tokens[r, b]`` at the score ``scores[r, b]`` (-inf: a row that is not there); returns as ``begin``."""
        raise NotImplementedError

    def finish(self) -> None:
        raise NotImplementedError


class _Search:
    """One request's hypotheses."""

    def __init__(self, index: int, prompt_len: int, limit: int, full: bool, options: BeamOptions):
        self.index, self.prompt_len, self.limit, self.options = index, prompt_len, limit, options
        self.reason_at_limit = CONTEXT_FULL if full else MAX_TOKENS
        self.open: List[List[int]] = [[]]
        self.done: List[BeamReply] = []

    def _score(self, logprob: float, length: int) -> float:
        return logprob / max(length, 1) ** self.options.length_penalty

    def _end(self, tokens: List[int], logprob: float, length: int, reason: str) -> None:
        self.done.append(BeamReply(tokens, self._score(logprob, length), logprob, reason))
        self.done.sort(key=lambda r: -r.score)                   # stable: earlier ones first among equals
        del self.done[self.options.beams:]

    def step(self, scores, beams, tokens, stop) -> Optional[List[Tuple[int, int, float]]]:
        """One step's continuations, best first; the hypotheses that go on as (beam, token, score), or None when the search is over."""
        W = self.options.beams
        nxt: List[Tuple[int, int, float]] = []
        for rank, (s, b, t) in enumerate(zip(scores, beams, tokens)):
            if t < 0 or len(nxt) == W:
                break
            if int(t) in stop:
                if rank < W:
                    self._end(list(self.open[int(b)]), float(s), len(self.open[int(b)]) + 1, EOS)
                continue
            nxt.append((int(b), int(t), float(s)))
        self.open = [self.open[b] + [t] for b, t, _ in nxt]
        length = len(self.open[0]) if nxt else 0
        over = not nxt or length >= self.limit
        if not over and len(self.done) >= W:
            over = self.options.early_stopping or self._score(nxt[0][2], length) <= self.done[-1].score
        if over:
            if length >= self.limit or not self.done:            # (without any continuation the prompt's replies are what there is)
                for (_, _, s), seq in zip(nxt, self.open):
                    self._end(seq, s, len(seq), self.reason_at_limit)
            return None
        return nxt


def beam_search(backend: BeamBackend, prompts: Sequence[Sequence[int]], options: BeamOptions, stop_ids: Sequence[int] = ()) -> List[BeamResult]:
    check_beams(options, stop_ids)
    stop = set(int(s) for s in stop_ids)
    W = options.beams
    if W > backend.max_batch:
        raise PromptError(f"{W} beams do not fit a batch of {backend.max_batch}")
    for i, p in enumerate(prompts):
        a = np.asarray(p, dtype=np.int64).reshape(-1)
        if not a.size:
            raise PromptError(f"request {i}: an empty prompt")
        if a.size >= backend.max_seq:
            raise PromptError(f"request {i}: the prompt of {a.size} tokens fills the context of {backend.max_seq}")
        if int(a.min()) < 0 or int(a.max()) >= backend.vocab_size:
            raise PromptError(f"request {i}: token id {int(a[(a < 0) | (a >= backend.vocab_size)][0])} is outside the vocabulary")
    results = [BeamResult(i, len(p)) for i, p in enumerate(prompts)]
    # batches in order; a request needs room for its beams at their longest, the prompt counted for each of them (a page that
    # beams still share is a page to spare)
    batches: List[List[int]] = []
    held = 0
    for i, p in enumerate(prompts):
        limit = min(options.max_new_tokens, backend.max_seq - len(p))
        need = W * ((len(p) + limit + PAGE - 1) // PAGE * PAGE)
        if need > backend.max_tokens:
            raise PromptError(f"request {i}: {W} beams of {len(p) + limit} tokens do not fit a cache of {backend.max_tokens}")
        if not batches or (len(batches[-1]) + 1) * W > backend.max_batch or held + need > backend.max_tokens:
            batches.append([])
            held = 0
        batches[-1].append(i)
        held += need
    for batch in batches:
        live: List[_Search] = []
        for i in batch:
            n, room = len(prompts[i]), backend.max_seq - len(prompts[i])
            live.append(_Search(i, n, min(options.max_new_tokens, room), room <= options.max_new_tokens, options))
        searches = list(live)
        try:
            got = backend.begin([prompts[i] for i in batch])
            while True:
                keep, rows = [], []
                for r, s in enumerate(live):
                    nxt = s.step(got[0][r], got[1][r], got[2][r], stop)
                    if nxt is not None:
                        keep.append(r)
                        rows.append(nxt + [(0, 0, float("-inf"))] * (W - len(nxt)))
                if not keep:
                    break
                live = [live[r] for r in keep]
                cols = list(zip(*[zip(*row) for row in rows]))
                got = backend.advance(keep, np.asarray(cols[0], np.int64), np.asarray(cols[1], np.int32), np.asarray(cols[2], np.float32))
        finally:
            backend.finish()
        for s in searches:
            results[s.index].replies = s.done[:options.replies]
    return results


class EngineBeams(BeamBackend):
    """The engine behind the search.  A row's sequence is a slot; of the beams that go on from one sequence the first keeps its slot,
    the others fork it (``Engine.fork``: its pages together with it, its states copied), and slots that nobody goes on from are given back
    before.  The selection runs inside the decode step's graph."""

    def __init__(self, engine, selector: BeamSelector, max_batch: int):
        self.engine, self.selector, self.max_batch = engine, selector, max_batch
        self.max_tokens, self.max_seq = engine.cache.max_tokens, engine.max_seq
        self.vocab_size = engine.model.spec.embedding.vocab_size
        self.beams = selector.beams
        self.slots: List[List[int]] = []
        self.decode_steps = 0
        self._tokens = torch.zeros(selector.requests * selector.beams, dtype=torch.int32, device=engine.device)

    def begin(self, prompts):
        eng = self.engine
        for _ in prompts:
            self.slots.append([eng.new_sequence()])
        logits = eng.step([(s[0], p) for s, p in zip(self.slots, prompts)], "last")
        self.selector(logits, beams=1, scores=torch.zeros(len(prompts), dtype=torch.float32, device=eng.device))
        return self.selector.collect(len(prompts))

    def advance(self, keep, parents, tokens, scores):
        eng = self.engine
        kept = set(keep)
        for r, slots in enumerate(self.slots):
            if r not in kept:
                for s in slots:
                    eng.release(s)
        old = [self.slots[r] for r in keep]
        self.slots = list(old)
        # Of a sequence's successors the first keeps the slot, the others fork it.  Sequences without one are given back first: their
        # slots are what the forks get.  `self.slots` names what is held at any time, so that `finish` can give it back.
        sources: List[int] = []
        for i, slots in enumerate(old):
            taken = set()
            for p in parents[i]:
                s = slots[int(p)]
                if s in taken:
                    sources.append(s)
                taken.add(s)
            for s in slots:
                if s not in taken:
                    eng.release(s)
            old[i] = [s if s in taken else -1 for s in slots]
            self.slots[i] = sorted(taken)
        made = iter(eng.fork(sources))
        for i, slots in enumerate(old):
            row, taken = [], set()
            for p in parents[i]:
                s = slots[int(p)]
                row.append(next(made) if s in taken else s)
                taken.add(s)
            self.slots[i] = row
        rows = [s for slots in self.slots for s in slots]
        n = len(rows)
        up = eng.cache.uploader
        up.send(self.selector.scores[:n], np.ascontiguousarray(scores.reshape(-1), np.float32))
        up.send(self._tokens[:n], np.ascontiguousarray(tokens.reshape(-1), np.int32))
        eng.decode(rows, self._tokens[:n], tail=self.selector)
        self.decode_steps += 1
        return self.selector.collect(len(keep))

    def finish(self) -> None:
        for slots in self.slots:
            for s in slots:
                self.engine.release(s)
        self.slots = []
