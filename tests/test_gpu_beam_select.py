"""Beam search's selection, against log softmax in 64 bits and a sort; ties, dead beams, logits that are not finite, few continuations."""
import numpy as np
import pytest
import torch

from quicknn_b200.kernels import lib, ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def select(logits, scores, beams, take, **kw):
    scratch = torch.full((ops.beam_select_scratch_bytes(logits.shape[0], logits.shape[1], take) // 4,), float("nan"), device=DEV)
    return [t.cpu().numpy() for t in ops.beam_select(logits, scores, beams, take, scratch, **kw)]


def wanted(logits, scores, beams, take):
    x = logits.double().cpu().numpy()
    ok = np.isfinite(x)
    x = np.where(ok, x, -np.inf)
    t = scores.double().cpu().numpy()
    with np.errstate(all="ignore"):
        m = x.max(1, keepdims=True)
        lse = m + np.log(np.exp(x - m).sum(1, keepdims=True))
        total = np.where(ok & np.isfinite(t)[:, None], t[:, None] + (x - lse), -np.inf)
    Q, V = len(x) // beams, x.shape[1]
    out = []
    for q in range(Q):
        flat = total[q * beams:(q + 1) * beams].reshape(-1)
        order = np.lexsort((np.arange(flat.size), -flat))[:take]
        s = np.full(take, -np.inf)
        b, v = np.full(take, -1), np.full(take, -1)
        n = int(np.isfinite(flat[order]).sum())
        s[:n], b[:n], v[:n] = flat[order][:n], order[:n] // V, order[:n] % V
        out.append((s, b, v))
    return [np.stack(z) for z in zip(*out)]


def check(logits, scores, beams, take, **kw):
    got, want = select(logits, scores, beams, take, **kw), wanted(logits, scores, beams, take)
    assert np.array_equal(got[1], want[1]) and np.array_equal(got[2], want[2])
    n = np.isfinite(want[0])
    assert np.array_equal(np.isneginf(got[0]), ~n)
    # sums of float32 exponentials (2 ulp each, then a tree of at most 4 + 5 additions) move a score by less than 2^-20, its rounding by 2^-24
    assert (np.abs(got[0][n] - want[0][n]) <= 2.0 ** -20 + 2.0 ** -24 * np.abs(want[0][n])).all()


def data(Q, W, V, seed=0, spread=4.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (spread * torch.randn(Q * W, V, device=DEV, generator=g),
            (-10 * torch.rand(Q, W, device=DEV, generator=g)).sort(1, descending=True).values.reshape(-1).contiguous())


@pytest.mark.parametrize("Q,W,V,take", [(1, 1, 1, 1), (1, 2, 3, 4), (1, 4, 1000, 8), (3, 5, 301, 10), (2, 8, 512, 16), (1, 8, 16383, 16), (2, 3, 16384, 6),
                                        (5, 4, 32003, 8), (1, 8, 256000, 16), (2, 32, 5000, 64), (1, 16, 255029, 64), (7, 1, 130, 64), (1, 3, 20, 64)])
def test_against_a_sort(Q, W, V, take):
    check(*data(Q, W, V, Q + W + V), W, take)


@pytest.mark.parametrize("Q,W,V,take", [(2, 11, 515, 22), (3, 15, 537, 30), (1, 10, 1015, 20), (2, 14, 418, 28), (1, 64, 130, 64), (2, 6, 349, 12), (1, 17, 900, 64),
                                        (4, 9, 1653, 18), (1, 8, 99521, 16), (9, 17, 16384, 17)])
@pytest.mark.parametrize("spread", [0.01, 4.0])
def test_many_beams(Q, W, V, take, spread):
    """few segments for the continuations that are wanted; beams whose every continuation is better than another's best"""
    check(*data(Q, W, V, Q + W + V, spread), W, take)


def test_scratch_of_many_rows_serves_fewer():
    V, most = 65537, 64
    scratch = torch.empty(ops.beam_select_scratch_bytes(most, V, 8), dtype=torch.uint8, device=DEV)
    for Q in (16, 9, 8, 4, 1):
        logits, scores = data(Q, 4, V, Q)
        got, want = ops.beam_select(logits, scores, 4, 8, scratch), wanted(logits, scores, 4, 8)
        assert np.array_equal(got[1].cpu().numpy(), want[1]) and np.array_equal(got[2].cpu().numpy(), want[2])


def test_rows_off_sixteen_bytes():
    for V in (257, 16387, 255029):
        flat = torch.randn(4 * V + 5, device=DEV, generator=torch.Generator(device=DEV).manual_seed(V))
        for off in range(4):
            x = flat[off:off + 4 * V].view(4, V)
            x[:, 0] += 9 * (off % 2)                                # the first and the last of a row among the best
            x[:, V - 1] += 9
            check(x, torch.tensor([-1.0, -1.5, -1.2, -3.0], device=DEV), 2, 6)


def test_equal_scores_go_to_the_lowest_beam_and_token():
    logits, scores = data(2, 4, 3000, 1)
    logits = logits.round()                                         # many equal ones
    scores[:] = -1.0
    logits[1] = logits[0]                                           # beams with the same continuations
    logits[6] = logits[5]
    check(logits, scores, 4, 40)


@pytest.mark.parametrize("V", [900, 40000])
def test_more_equal_scores_than_the_list_holds(V):
    logits = torch.zeros(2 * 4, V, device=DEV)
    scores = torch.tensor([-1.0, -1.0, -1.0, -2.0] * 2, device=DEV)
    check(logits, scores, 4, 32)
    logits[0, V - 1] = 5.0
    logits[5, 17] = 0.5
    check(logits, scores, 4, 32)


def test_beams_that_are_not_there():
    logits, scores = data(3, 4, 700, 2)
    scores[1:4] = float("-inf")                                     # the first step of a request: one beam
    scores[4:8] = float("-inf")                                     # nothing at all
    scores[9] = float("nan")
    scores[10] = float("inf")
    check(logits, scores, 4, 8)


def test_logits_that_are_not_finite():
    logits, scores = data(2, 2, 5000, 3)
    flag = torch.zeros(1, dtype=torch.int32, device=DEV)
    check(logits, scores, 2, 6, error_flag=flag)
    assert flag.item() == 0
    logits[0, :] = float("-inf")                                    # a beam without continuations
    logits[1, 5:] = float("nan")
    logits[3, 77] = float("inf")
    check(logits, scores, 2, 6, error_flag=flag)
    assert flag.item() == 1


def test_status_joins_the_error_word():
    logits, scores = data(1, 2, 50)
    flag = torch.zeros(1, dtype=torch.int32, device=DEV)
    check(logits, scores, 2, 4, error_flag=flag, status=torch.tensor([5], dtype=torch.int32, device=DEV))
    assert flag.item() == 2 | (5 << 8)


def test_far_scores():
    logits, scores = data(1, 4, 2000, 5, spread=40.0)
    scores = torch.tensor([-1e6, -1000.0, -3e38, -1000.5], device=DEV)
    got, want = select(logits, scores, 4, 8), wanted(logits, scores, 4, 8)
    assert np.array_equal(got[1], want[1]) and np.array_equal(got[2], want[2])


def test_captured_and_replayed_with_new_values():
    logits, scores = data(2, 4, 20000, 6)
    scratch = torch.empty(ops.beam_select_scratch_bytes(8, 20000, 8), dtype=torch.uint8, device=DEV)
    ops.beam_select(logits, scores, 4, 8, scratch)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = ops.beam_select(logits, scores, 4, 8, scratch)
    for seed in (7, 8):
        a, b = data(2, 4, 20000, seed)
        logits.copy_(a)
        scores.copy_(b)
        g.replay()
        torch.cuda.synchronize()
        want = wanted(logits, scores, 4, 8)
        assert np.array_equal(out[1].cpu().numpy(), want[1]) and np.array_equal(out[2].cpu().numpy(), want[2])


def test_refusals():
    logits, scores = data(2, 3, 100)
    scratch = torch.empty(ops.beam_select_scratch_bytes(6, 100, 4), dtype=torch.uint8, device=DEV)
    for args in ((logits, scores, 4, 4, scratch), (logits, scores[:5], 3, 4, scratch), (logits, scores, 3, 0, scratch), (logits, scores, 3, 65, scratch),
                 (logits, scores, 3, 4, scratch[:-8]), (logits, scores, 0, 4, scratch)):
        with pytest.raises(ValueError):
            ops.beam_select(*args)
    with pytest.raises(TypeError):
        ops.beam_select(logits.bfloat16(), scores, 3, 4, scratch)
    with pytest.raises(lib.KernelError):
        ops.beam_select(logits.cpu(), scores, 3, 4, scratch)
    out = (torch.empty(2, 4, device=DEV), torch.empty(2, 4, dtype=torch.int32, device=DEV), torch.empty(2, 5, dtype=torch.int32, device=DEV))
    with pytest.raises(ValueError):
        ops.beam_select(logits, scores, 3, 4, scratch, out=out)


@pytest.mark.parametrize("level", [0.1, 10.0, 12.0, 30.0, -4.7])
@pytest.mark.parametrize("W,V,take", [(1, 3000, 8), (1, 4000, 64), (4, 900, 32), (3, 700, 24), (1, 40000, 8)])
def test_one_value_everywhere(level, W, V, take):
    """the threshold and the segments' best scores are the same number, however it is rounded"""
    logits = torch.full((2 * W, V), level, device=DEV)
    check(logits, torch.tensor([-0.3 * b for b in range(W)] * 2, device=DEV), W, take)


@pytest.mark.parametrize("level", [0.1, 10.0, 30.0, 4096.0])
def test_thousands_of_logits_a_few_steps_apart(level):
    """all within what the limit of the short list allows for roundings, so they do not fit it"""
    V = 3000
    g = torch.Generator().manual_seed(int(level))
    base = torch.tensor(level).view(torch.int32) + torch.randint(0, 5, (2, V), generator=g, dtype=torch.int32)
    check(base.view(torch.float32).to(DEV), torch.zeros(2, device=DEV), 1, 16)


@pytest.mark.parametrize("far,spread", [(4096.0, 0.03), (20000.0, 0.03), (1e6, 0.3)])
@pytest.mark.parametrize("scores", [(0.0, 0.0), (-5.0, -5.003)])
def test_beams_whose_logits_lie_apart(far, spread, scores):
    """Beam 0's logits stand far above beam 1's; their continuations score alike.  Where two beams' scores are closer than what the sums of
    exponentials may be off by (2^-20 each), their order is open, and the draw says nothing."""
    said = 0
    for seed in range(60):
        x = spread * torch.randn(2, 400, generator=torch.Generator().manual_seed(seed))
        x[0] += far
        t = torch.tensor(scores)
        s, b, _ = (a[0] for a in wanted(x, t, 2, 9))
        if any(b[i] != b[i + 1] and s[i] - s[i + 1] < 2.0 ** -18 for i in range(8)):
            continue
        said += 1
        check(x.to(DEV), t.to(DEV), 2, 8)
    assert said > 40


@pytest.mark.parametrize("W,V,take", [(1, 3000, 8), (3, 300, 12), (2, 20000, 16)])
def test_fewer_continuations_than_wanted(W, V, take):
    logits, scores = data(2, W, V, 7)
    logits[:, 3:] = float("-inf")
    logits[W:, 1:] = float("-inf")
    check(logits, scores, W, take)
