"""Sizes that 32 bits do not hold, and tensors to fill that lie in one another, are refused before a launch: on the host, by tensors without memory."""

from __future__ import annotations

from types import SimpleNamespace

import pytest
import torch

from llmserve_amd.kernels import HipKernels, KernelError


@pytest.fixture
def library():
    """The checks of a library whose device is the host, with no kernels behind them."""
    k = object.__new__(HipKernels)
    k.device, k._pinned_stream = SimpleNamespace(index=-1), 0
    k._library_of = lambda module: pytest.fail(f"{module} was asked to launch")
    return k


def indices(*shape, stride=None):
    if stride is None:
        return torch.empty(shape, dtype=torch.int32, device="meta")
    return torch.empty_strided(shape, stride, dtype=torch.int32, device="meta")


def filled(tokens, width, groups=2, mapping_stride=None, compact_stride=None):
    mapping = indices(groups, tokens, stride=(mapping_stride or tokens, 1))
    return indices(tokens), indices(tokens), indices(3), indices(2), mapping, indices(groups, 2, width, stride=(compact_stride or 2 * width, width, 1))


@pytest.mark.parametrize("strides", [{"mapping_stride": 1 << 31}, {"mapping_stride": (1 << 32) + 5}, {"compact_stride": 1 << 31}, {"compact_stride": (1 << 33) + 6}, {"mapping_stride": 4}, {"compact_stride": 5}])
def test_groups_of_arrays_that_lie_too_far_apart_or_in_one_another(library, strides):
    tables, short = indices(2, 4, 8), indices(2)
    with pytest.raises(KernelError):
        library.place_tokens(tables, short, short, short, 16, 5, 3, out=filled(5, 3, **strides))


@pytest.mark.parametrize("page_size", [0, -1, 1 << 31, (1 << 32) + 16])
def test_page_sizes(library, page_size):
    tables, short = indices(2, 4, 8), indices(2)
    with pytest.raises(KernelError):
        library.place_tokens(tables, short, short, short, page_size, 5, 3, out=filled(5, 3))


@pytest.mark.parametrize("shape", [(0, 4, 8), (65, 1, 1), (2, 0, 8), (2, 4, 0), (1, (1 << 32) + 4, 1), (1, 4, (1 << 32) + 8)])
def test_tables(library, shape):
    short = indices(2)
    with pytest.raises(KernelError):
        library.place_tokens(indices(*shape), short, short, short, 16, 5, 3, out=filled(5, 3, shape[0]))
