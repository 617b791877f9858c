"""Attention over pages in 4 bits where results could depend on how walks are cut: values that are no number behind weights of zero, scores that overflow."""

from __future__ import annotations

import pytest
import torch

from tests.packed_cases import assert_near, expected_of, packed_case

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16]
WAYS = [(0, 0, 0), (1, 1, 0), (0, 0, 4), (1, 1, 4), (0, 0, 8), (1, 1, 8)]


@pytest.fixture(scope="module")
def kernels():
    from llmserve_amd.kernels import HipKernels

    return {dtype: HipKernels(dtype) for dtype in DTYPES}


def force(monkeypatch, k, way):
    """Walks in the given way: least units of walks of few and of many columns (0: whole), and 4: tiles shared (bfloat16), 8: few columns with many."""
    monkeypatch.setattr(type(k), "_packed_way", staticmethod(lambda *given: (*way[:2], way[2] if way[2] == 8 or k.dtype == torch.bfloat16 else 0)))


def check(k, lengths, counts, heads, kv_heads, dim, page, scale, **more):
    batch, cell, layout, qkv, found = packed_case(k, lengths, counts, heads, kv_heads, dim, page, **more)
    got = k.paged_attention(qkv, layout, batch, cell, scale, None)
    largest = torch.cat([v.nan_to_num().abs().amax().expand(c, 1) for (_, _, v), c in zip(found, counts)])
    want = expected_of(found, lengths, counts, scale, None)
    assert_near(got, want, largest, k.dtype)
    return want


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("way", WAYS)
@pytest.mark.parametrize("place", [40, 900])
def test_no_numbers_behind_weights_of_zero(kernels, dtype, way, place, monkeypatch):
    """One key far ahead of all others, so that parts without it count for exactly 0: a value that is no number there still makes its block no number."""
    def change(index, rows):  # [length, 2 q heads | key | value, of 64]
        rows[:, :128] = 1.0
        rows[place, 128:192] = 100.0
        rows[500, 192 + 40] = float("nan")  # the value's second block

    force(monkeypatch, kernels[dtype], way)
    want = check(kernels[dtype], [1000, 1000], [1, 40], 2, 1, 64, 16, 1.0, change=change, seed=place)
    blocks = torch.isnan(want).view(41, 2, 2, 32)
    assert bool(blocks[:, :, 1].all()) and not blocks[:, :, 0].any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("way", WAYS)
@pytest.mark.parametrize("dim", [64, 96])
def test_scores_below_all_floats(kernels, dtype, way, dim, monkeypatch):
    """Keys whose scores are below the smallest float32 have no weight, also where a wave's first keys are all such."""
    def change(index, rows):  # [length, query | key | value]
        rows[:, :dim] = 0.0
        rows[:, 0] = 2.0 ** 126
        rows[:, dim] = 0.0
        rows[:64, dim:2 * dim] = 0.0
        rows[:64, dim] = -2.0 ** 10

    force(monkeypatch, kernels[dtype], way)
    want = check(kernels[dtype], [200, 600], [1, 40], 1, 1, dim, 16, 1.0, change=change, seed=dim)
    assert not torch.isnan(want).any()
