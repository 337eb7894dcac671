"""Copies of states and pages: the bits of plain indexing; what is not named stays."""
import pytest
import torch

from quicknn_b200.kernels import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("shapes", [[((3, 5), torch.float32)], [((2, 128, 256), torch.float32), ((3, 2304), torch.bfloat16)], [((1,), torch.uint8), ((7,), torch.bfloat16), ((), torch.float32)],
                                    [((4097,), torch.float32)], [((33, 3), torch.bfloat16)] * 70, [((0,), torch.float32), ((5,), torch.int32)]])
@pytest.mark.parametrize("src,dst", [([0], [1]), ([2, 2, 5], [1, 0, 7]), ([8], [0])])
def test_states(shapes, src, dst):
    g = torch.Generator(device=DEV).manual_seed(1)
    ts = [(torch.randn((9,) + s, device=DEV, generator=g) * 50).to(dt) for s, dt in shapes]
    want = [t.clone() for t in ts]
    for w in want:
        w[dst] = w[src]
    ops.copy_slots(ts, src, dst)
    assert all(torch.equal(a, b) for a, b in zip(ts, want))


def test_more_pairs_than_a_launch_takes():
    t = torch.randn(600, 10, device=DEV)
    src, dst = list(range(300)), list(range(300, 600))
    want = t.clone()
    want[dst] = want[src]
    ops.copy_slots([t], src, dst)
    assert torch.equal(t, want)


def test_tensors_that_start_off_sixteen_bytes():
    flat = torch.randn(4 * 33 + 1, device=DEV)
    t = flat[1:].view(4, 33)
    want = t.clone()
    want[3] = want[0]
    ops.copy_slots([t], [0], [3])
    assert torch.equal(t, want)


def test_far_rows_of_large_tensors():
    t = torch.zeros(3, (1 << 30) + 8, dtype=torch.uint8, device=DEV)           # offsets beyond 31 bits
    t[0, -5:] = 7
    ops.copy_slots([t], [0], [2])
    assert t[2, -5:].tolist() == [7] * 5 and not t[1].any()


@pytest.mark.parametrize("lines,pages,heads,dim,dtype", [(2, 9, 4, 256, torch.bfloat16), (1, 9, 1, 24, torch.float32), (3, 9, 2, 8, torch.bfloat16), (1, 9, 3, 5, torch.bfloat16)])
@pytest.mark.parametrize("src,dst,used", [([1], [2], [64]), ([3, 3, 3], [1, 8, 2], [1, 0, 63]), ([8, 1], [4, 5], [17, 33])])
def test_pages(lines, pages, heads, dim, dtype, src, dst, used):
    g = torch.Generator(device=DEV).manual_seed(2)
    k, v = (torch.randn((lines, pages, heads, 64, dim), device=DEV, generator=g).to(dtype) for _ in range(2))
    wk, wv = k.clone(), v.clone()
    for w in (wk, wv):
        for s, d, u in zip(src, dst, used):
            w[:, d, :, :u] = w[:, s, :, :u]
    ops.copy_pages(k, v, src, dst, used)
    assert torch.equal(k, wk) and torch.equal(v, wv)
    wk = k.clone()
    for s, d, u in zip(src, dst, used):
        wk[:, d, :, :u] = wk[:, s, :, :u]
    ops.copy_pages(k, k, src, dst, used)                              # a line without values
    assert torch.equal(k, wk)


def test_more_pages_than_a_launch_takes():
    k, v = torch.randn(1, 400, 2, 64, 16, device=DEV), torch.randn(1, 400, 2, 64, 16, device=DEV)
    src, dst = [1] * 200, list(range(150, 350))
    wk = k.clone()
    wk[:, dst, :, :9] = wk[:, src, :, :9]
    ops.copy_pages(k, v, src, dst, [9] * 200)
    assert torch.equal(k, wk)


def test_nothing_to_copy():
    ops.copy_slots([torch.ones(2, 2, device=DEV)], [], [])
    ops.copy_pages(torch.ones(1, 2, 1, 64, 8, device=DEV), torch.ones(1, 2, 1, 64, 8, device=DEV), [], [], [])
