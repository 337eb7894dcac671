"""Words that kernels set or read are looked at before a launch takes their address."""
import pytest
import torch

from quicknn_b200.kernels import lib, ops


class Word:
    """Stands for a tensor on a device."""

    def __init__(self, dtype=torch.int32, n=1, device=0):
        self.is_cuda, self.dtype, self.n, self.shape, self.device = True, dtype, n, (n,), f"cuda:{device}"

    def numel(self):
        return self.n

    def get_device(self):
        return int(self.device[5:])


def test_words():
    ops._req_word(None, "word", 0)
    ops._req_word(Word(), "word", 0)
    ops._req_word(Word(n=3, device=2), "word", 2)
    with pytest.raises(lib.KernelError):
        ops._req_word(torch.zeros(1, dtype=torch.int32), "word", 0)
    for dtype in (torch.int64, torch.float32, torch.uint8):
        with pytest.raises(TypeError):
            ops._req_word(Word(dtype), "word", 0)
    for w in (Word(n=0), Word(device=1)):
        with pytest.raises(ValueError):
            ops._req_word(w, "word", 0)


WRONG = [(lambda: torch.zeros(1, dtype=torch.int32), lib.KernelError), (lambda: torch.zeros(1, dtype=torch.int64, device="cuda:0"), TypeError),
         (lambda: torch.zeros(0, dtype=torch.int32, device="cuda:0"), ValueError)]


@pytest.mark.gpu
@pytest.mark.parametrize("make,error", WRONG)
def test_beam_selection(make, error):
    logits, scores = torch.zeros(2, 50, device="cuda:0"), torch.zeros(2, device="cuda:0")
    scratch = torch.empty(ops.beam_select_scratch_bytes(2, 50, 4), dtype=torch.uint8, device="cuda:0")
    for word in ("error_flag", "status"):
        with pytest.raises(error):
            ops.beam_select(logits, scores, 2, 4, scratch, **{word: make()})


@pytest.mark.gpu
@pytest.mark.parametrize("make,error", WRONG)
def test_sampling(make, error):
    logits, rng = torch.zeros(2, 50, device="cuda:0"), torch.ones(2, dtype=torch.int32, device="cuda:0")
    out, cand = torch.zeros(2, dtype=torch.int32, device="cuda:0"), torch.zeros(2, 4, 2, device="cuda:0")
    scratch = torch.empty(ops.sample_scratch_bytes(2, 50, 4), dtype=torch.uint8, device="cuda:0")
    for words in ((make(), None), (None, make())):
        with pytest.raises(error):
            ops.sample(logits, 4, 1.0, 1.0, 1.0, rng, None, None, scratch, out, *words)
        with pytest.raises(error):
            ops.sample_candidates(cand, 2, 4, 50, 4, 1.0, 1.0, rng, None, None, out, *words)
    with pytest.raises(error):
        ops.head_argmax(torch.zeros(2, 64, dtype=torch.bfloat16, device="cuda:0"), torch.zeros(32, 64, dtype=torch.bfloat16, device="cuda:0"), None,
                        torch.zeros(2 * ops.head_candidates(32) * 2, device="cuda:0"), make())
