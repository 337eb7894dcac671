"""Options of beam search and the device-side selection of continuations (see csrc/beam_select.cu)."""
from __future__ import annotations

import dataclasses
from typing import List, Optional, Sequence

import numpy as np
import torch

from ..kernels import ops
from ..kernels.lib import KernelError, NonFiniteLogits
from .options import OptionsError


@dataclasses.dataclass
class BeamOptions:
    """``beams`` hypotheses go on side by side; a reply's score is the sum of the log-probabilities of its tokens, the stop token
    included, over (their number) ** ``length_penalty``.  ``early_stopping``: a request is over once ``beams`` replies have ended; without it
    it goes on while its best open hypothesis, scored at its present length, beats the worst of these.  ``replies`` of them come back."""

    beams: int = 4
    max_new_tokens: int = 256
    length_penalty: float = 1.0
    early_stopping: bool = False
    replies: int = 1

    def problems(self) -> List[str]:
        p: List[str] = []
        if not 1 <= self.beams <= ops.BEAM_MOST:
            p.append(f"beams must be in 1..{ops.BEAM_MOST}")
        if self.max_new_tokens < 1:
            p.append("max_new_tokens must be >= 1")
        # (lengths to the power of more than 32 either way leave the range of a float)
        if not isinstance(self.length_penalty, (int, float)) or not abs(self.length_penalty) <= 32:
            p.append("length_penalty must be in -32..32")
        if not 1 <= self.replies <= max(self.beams, 1):
            p.append("replies must be in 1..beams")
        return p

    def validate(self) -> None:
        p = self.problems()
        if p:
            raise OptionsError("invalid beam search options: " + "; ".join(p))

    def take(self, n_stops: int) -> int:
        """Continuations to ask for per request: enough that ``beams`` of them are no stop token."""
        n = self.beams * (1 + n_stops)
        if n > ops.BEAM_MOST:
            raise OptionsError(f"{self.beams} beams and {n_stops} stop ids need {n} continuations a step, at most {ops.BEAM_MOST} are selected")
        return n


class BeamSelector:
    """The best continuations of up to ``requests`` requests of ``beams`` beams: called on a step's logits (as a decode step's tail, inside
    its graph), it leaves scores, beams and tokens in buffers of its own, which ``collect`` brings to the host in one copy."""

    def __init__(self, vocab_size: int, requests: int, beams: int, take: int, device):
        self.vocab, self.requests, self.beams, self.take, self.device = vocab_size, requests, beams, take, device
        self.scores = torch.zeros(requests * beams, dtype=torch.float32, device=device)
        self._all = torch.zeros(3 * requests * take + 1, dtype=torch.int32, device=device)
        self.flag = self._all[-1:]
        self.scratch = torch.empty(ops.beam_select_scratch_bytes(requests * beams, vocab_size, take), dtype=torch.uint8, device=device)
        self._pinned: Optional[torch.Tensor] = None

    def __call__(self, logits: torch.Tensor, beams: Optional[int] = None, scores: Optional[torch.Tensor] = None) -> torch.Tensor:
        """``logits`` [requests * beams, vocab]; returns the tokens [requests, take].  ``beams``: 1 for the first step, whose requests have
        one row each (``scores`` then are those rows')."""
        W = self.beams if beams is None else beams
        Q = logits.shape[0] // W
        if Q > self.requests or Q * W != logits.shape[0]:
            raise ValueError(f"the selector was built for {self.requests} requests of {self.beams} beams, the step has {logits.shape[0]} rows")
        n = self.requests * self.take
        out = [self._all[i * n:i * n + Q * self.take].view(Q, self.take) for i in range(3)]
        out[0] = out[0].view(torch.float32)
        ops.beam_select(logits, self.scores[:Q * W] if scores is None else scores, W, self.take, self.scratch, tuple(out), self.flag,
                        ops.status_words(self.device)[0:1])
        return out[2]

    def collect(self, requests: int):
        """(scores, beams, tokens) of the first ``requests`` requests as host arrays; waits for the device."""
        if self._pinned is None:
            self._pinned = torch.empty(self._all.numel(), dtype=torch.int32, pin_memory=True)
        self._pinned.copy_(self._all, non_blocking=True)
        torch.cuda.current_stream(self.device).synchronize()
        a = self._pinned.numpy()
        word = int(a[-1])
        if word:
            self.flag.zero_()
            if word & 2:
                ops.status_words(self.device)[0:1].zero_()
                raise KernelError(ops.wait_status_message(word >> 8))
            raise NonFiniteLogits("the model produced non-finite logits")
        s, b, t = (x[:requests * self.take].reshape(requests, self.take).copy() for x in a[:-1].reshape(3, -1))
        return s.view(np.float32), b, t


def check_beams(options: BeamOptions, stop_ids: Sequence[int]) -> int:
    """Validate and return the number of continuations per request."""
    options.validate()
    return options.take(len(set(int(s) for s in stop_ids)))
