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


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("cap", [50.0, 90.0])
def test_prompts_with_a_softcap(hd, cap):
    """with a softcap up to 70 the columns of a tile take their exponentials in two ways, four neighbours each"""
    check_prompt([130, 1, 300], hd, cap, tuple(range(8)) + (64, 70, 129, 130, 131 + 66, 300, 430))
    check_prompt([1500], hd, cap, (0, 65, 129, 130, 197, 390, 1300, 1499))


@pytest.mark.parametrize("nq,nkv,hd", [(8, 4, 256), (8, 2, 128), (16, 2, 64)])
@pytest.mark.parametrize("cap", [None, 50.0, 90.0])
@pytest.mark.parametrize("keys", [1, 1 << 20])
def test_rows_that_share_pages(nq, nkv, hd, cap, keys):
    """by the kernel of few rows and that of many (which the bound of the keys chooses)"""
    from test_gpu_shared_attention import BF, Batch
    b = Batch([(0, 192, [193 + i for i in range(40)])], nq, nkv, hd, BF, alone=[77], seed=hd)
    clean = b.run(hd ** -0.5, cap, (2, 1), keys=keys).view(b.B, nq, hd)
    assert torch.isfinite(clean).all()
    for at in tuple(range(8)) + (63, 64, 70, 127, 128, 191):
        page, cell = int(b.table[b.slots[0], at // 64]), at % 64
        held = b.k[page, 1, cell, 5].clone()
        b.k[page, 1, cell, 5] = float("nan")
        got = b.run(hd ** -0.5, cap, (2, 1), keys=keys).view(b.B, nq, hd)
        b.k[page, 1, cell, 5] = held
        mine = slice(nq // nkv, 2 * (nq // nkv))
        assert torch.isnan(got[:40, mine]).all(), at
        got[:40, mine] = clean[:40, mine]
        assert torch.equal(got, clean), at


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("pages", [3, 5])
def test_pages_whose_scores_are_all_minus_infinity(hd, pages):
    """Keys of the first pages score -inf for every query: they have no weight.  The last page, which has no neighbour, is the first with a
    maximum, a low one."""
    from test_gpu_shared_attention import BF, Batch
    n = pages * 64
    b = Batch([(0, n, [n + 1 + i for i in range(20)])], 8, 4, hd, BF, seed=pages)
    q = b.qkv[:, :8 * hd].view(b.B, 8, hd)
    q[:, :, 0] = 2.0
    table = torch.from_numpy(b.table[b.slots[0]].astype("int64")).to(DEV)
    for k in b.k_of:
        k[:n - 64, :, 0] = float("-inf")
        k[n - 64:, :, 0] = -200.0
    pos = torch.arange(n, device=DEV)
    b.k[table[pos // 64], :, pos % 64] = b.k_of[0][:n]
    for r in range(b.B):                                             # the rows' own keys score low as well
        own = torch.arange(n, b.lens[r], device=DEV)
        t = torch.from_numpy(b.table[b.slots[r]].astype("int64")).to(DEV)
        b.k[t[own // 64], :, own % 64] = b.k_of[r][n:]
    got = {keys: b.run(0.5, None, (1, 1), keys=keys) for keys in (1, 1 << 20)}
    for keys, o in got.items():
        assert torch.isfinite(o).all(), keys
        for r in range(b.B):
            k, v = b.k_of[r][n - 64:].double(), b.v_of[r][n - 64:].double()
            s = torch.einsum("khd,pkd->khp", q[r].double().view(4, 2, hd), k) * 0.5
            want = torch.einsum("khp,pkd->khd", torch.softmax(s, -1), v).reshape(-1)
            # as in the tests of this attention: bfloat16 weights, exponents of up to 200 in float32, the result's rounding
            size = torch.einsum("khp,pkd->khd", torch.softmax(s, -1), v.abs()).reshape(-1)
            tol = (2.0 ** -8 + (hd * 400 * 0.5 + 4 * 250) * 2.0 ** -23 + 2.0 ** -19) * size + 2.0 ** -8 * want.abs()
            assert ((o[r].double() - want).abs() <= tol).all(), (keys, r)
