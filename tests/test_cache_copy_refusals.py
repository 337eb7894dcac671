"""Moves that the copies refuse: decided on the host, before anything is launched."""
import pytest
import torch

from quicknn_b200.kernels import lib, ops


@pytest.mark.parametrize("src,dst", [([0], [0]), ([0, 1], [2, 2]), ([0, 2], [2, 3]), ([0], [4]), ([4], [0]), ([-1], [0]), ([0], [-1]), ([0, 1], [2]), ([], [1])])
def test_states(src, dst):
    with pytest.raises(ValueError):
        ops.copy_slots([torch.zeros(4, 3), torch.zeros(5, 2)], src, dst)


def test_states_in_host_memory():
    with pytest.raises(lib.KernelError):
        ops.copy_slots([torch.zeros(4, 3)], [0], [1])


def test_pages_in_host_memory():
    with pytest.raises(lib.KernelError):
        ops.copy_pages(torch.zeros(1, 4, 1, 64, 8), torch.zeros(1, 4, 1, 64, 8), [1], [2], [3])


@pytest.mark.parametrize("src,dst,used", [([1], [2], [1, 2]), ([1, 2], [3], [1, 1])])
def test_lists_of_unequal_lengths(src, dst, used):
    with pytest.raises((ValueError, lib.KernelError)):
        ops.copy_pages(torch.zeros(1, 4, 1, 64, 8), torch.zeros(1, 4, 1, 64, 8), src, dst, used)


@pytest.mark.parametrize("src,dst", [([0], [2]), ([1], [0]), ([1], [4]), ([1], [1]), ([1, 2], [3, 3])])
def test_moves_of_pages(src, dst):
    with pytest.raises(ValueError):
        ops._check_moves(src, dst, 1, 4, "copy_pages")
