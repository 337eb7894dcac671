"""A key that holds a NaN makes every row that sees it NaN, in the heads that read it, and changes nothing else."""
import pytest
import torch

from quicknn_b200.kernels import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
NQ, NKV = 4, 2


def prompt(lens, hd, cap, nan_at=None):
    """Prompt attention of sequences of these lengths; ``nan_at``: a row of the step whose key of kv head 0 holds a NaN."""
    T = sum(lens)
    qkv = torch.randn((T, NQ + 2 * NKV, hd), device=DEV, generator=torch.Generator(device=DEV).manual_seed(hd)).bfloat16()
    if nan_at is not None:
        qkv[nan_at, NQ, 3] = float("nan")
    row0 = torch.tensor([sum(lens[:i]) for i in range(len(lens))], dtype=torch.int32, device=DEV)
    ln = torch.tensor(lens, dtype=torch.int32, device=DEV)
    pos = torch.cat([torch.arange(n) for n in lens]).to(DEV, torch.int32)
    out = ops.attn_prefill(qkv.view(T, -1), NQ, NKV, hd, pos, row0.repeat_interleave(ln), hd ** -0.5, cap, None, row0, ln, max(lens))
    ops.raise_on_status(torch.device(DEV))
    return out.view(T, NQ, hd)


def check_prompt(lens, hd, cap, places):
    clean = prompt(lens, hd, cap)
    assert torch.isfinite(clean).all()
    for at in places:
        got = prompt(lens, hd, cap, at)
        end = next(sum(lens[:i + 1]) for i in range(len(lens)) if at < sum(lens[:i + 1]))
        assert torch.isnan(got[at:end, :NQ // NKV]).all(), at
        got[at:end, :NQ // NKV] = clean[at:end, :NQ // NKV]
        assert torch.equal(got, clean), at


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_prompt_whose_tiles_two_blocks_share(hd):
    # one prompt of enough keys: its query tiles are walked by pairs of blocks, one of which sees the NaN
    check_prompt([1500], hd, None, (0, 70, 130, 200, 390, 777, 1300, 1499))


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_prompts_of_single_blocks(hd):
    check_prompt([130, 1, 300], hd, None, (0, 5, 129, 130, 131, 300, 430))
