"""Attention over pages in 4 bits, key by key and column by column: rows that tell which keys were counted, and random rows bounded by each element's own column, every way of walking,
beside requests that only pad the step (as a captured step has them)."""

from __future__ import annotations

import dataclasses
import functools

import pytest
import torch

from tests.packed_cases import packed_case

pytestmark = pytest.mark.gpu

WAYS = [(0, 0, 0), (1, 1, 0), (4, 8, 0), (0, 0, 4), (1, 1, 4), (0, 0, 8), (1, 1, 8)]
SHAPES = [(12, 2, 128, 16), (6, 2, 96, 24), (7, 1, 64, 8), (34, 2, 32, 16), (3, 1, 192, 40), (4, 2, 256, 16), (5, 1, 160, 16), (2, 1, 224, 8)]
LENGTHS, COUNTS = [1300, 1, 530, 777, 40, 0, 260, 1025], [1, 1, 1, 45, 40, 0, 2, 70]


@functools.lru_cache(maxsize=None)
def library(dtype):
    from llmserve_amd.kernels import HipKernels

    return HipKernels(dtype)


def force(monkeypatch, k, way):
    """Walks in the given way: least units of walks of few and of many columns (0: whole), and 4: tiles shared (bfloat16), 8: few columns with many."""
    monkeypatch.setattr(type(k), "_packed_way", staticmethod(lambda *given: (*way[:2], way[2] if way[2] == 8 or k.dtype == torch.bfloat16 else 0)))


def oracle(q, keys, values, scale, window, first_position):
    """(softmax(q k^T scale) v, the same over |v|, the largest sum of |q| |k| scale) in float64: [n, heads * D], [n, heads * D], a number."""
    n, heads, dim = q.shape
    if n == 0:
        return q.flatten(1), q.flatten(1), 0.0
    group = heads // keys.shape[1]
    position, key = first_position + torch.arange(n)[:, None], torch.arange(keys.shape[0])
    seen = (key <= position) & (key > position - (window or 1 << 40))
    out, size, largest = torch.empty_like(q), torch.empty_like(q), 0.0
    for h in range(heads):
        k, v = keys[:, h // group], values[:, h // group]
        scores = (q[:, h] @ k.T * scale).masked_fill(~seen, -torch.inf)
        weights = torch.softmax(scores, -1)
        out[:, h], size[:, h] = weights @ v, weights @ v.abs()
        largest = max(largest, float((q[:, h].abs() @ k.T.abs()).max()) * scale)
    return out.flatten(1), size.flatten(1), largest


def equal_scores(heads, kv_heads, dim):
    """All visible keys have the same weight, and a value is 1 in one of its elements: a result's element counts the keys of that element."""
    def change(index, rows):
        first = (heads + kv_heads) * dim
        rows[:, :heads * dim] = 0.0
        rows[:, first:first + kv_heads * dim] = 0.0
        at = torch.arange(rows.shape[0])
        for h in range(kv_heads):
            rows[at, first + h * dim + (11 * at + h) % dim] = 1.0
    return change


def picked_keys(heads, kv_heads, dim):
    """A query picks every key whose one element is its own, and a value tells which of those the key is."""
    def change(index, rows):
        rows[:, :(heads + 2 * kv_heads) * dim] = 0.0
        at = torch.arange(rows.shape[0])
        for h in range(heads):
            rows[at, h * dim + (3 * at + 7 * h) % dim] = 32.0
        for h in range(kv_heads):
            rows[at, (heads + h) * dim + (at + 5 * h) % dim] = 1.0
            rows[at, (heads + kv_heads + h) * dim + (11 * (at // dim) + h) % dim] = 1.0
    return change


def random_rows(heads, kv_heads, dim):
    """Channels of one size."""
    def change(index, rows):
        rows.copy_(torch.randn(rows.shape, generator=torch.Generator().manual_seed(index)))
    return change


@functools.lru_cache(maxsize=None)
def case(kind, dtype, shape, window):
    heads, kv_heads, dim, page = shape
    scale = 1.0 if kind is picked_keys else dim ** -0.5
    batch, cell, layout, qkv, found = packed_case(library(dtype), LENGTHS, COUNTS, heads, kv_heads, dim, page, window=window, padded=3, change=kind(heads, kv_heads, dim))
    parts = [oracle(q, k, v, scale, window, length - count) for (q, k, v), length, count in zip(found, LENGTHS, COUNTS)]
    # two requests that pad the step: nine tokens on a context of one token, so that most of their positions are negative, and none; both in page 0
    tokens, group = sum(COUNTS), batch.groups[0]
    more = lambda tensor, *values: torch.cat([tensor, torch.tensor(values, dtype=torch.int32, device="cuda")])
    batch = dataclasses.replace(
        batch, num_tokens=tokens + 9, query_start=more(batch.query_start, tokens + 9, tokens + 9), context_lengths=more(batch.context_lengths, 1, 1), scratch={}, padded_to=(tokens + 9, len(LENGTHS) + 2),
        groups=[dataclasses.replace(group, block_tables=torch.cat([group.block_tables, torch.zeros_like(group.block_tables[:2])]), slot_mapping=more(group.slot_mapping, *[-1] * 9))],
    )
    return batch, cell, layout, torch.cat([qkv, qkv[:9]]), scale, torch.cat([p[0] for p in parts]), torch.cat([p[1] for p in parts]), max(p[2] for p in parts)


def run(monkeypatch, kind, dtype, shape, way, window=None):
    k = library(dtype)
    force(monkeypatch, k, way)
    batch, cell, layout, qkv, scale, want, size, largest = case(kind, dtype, shape, window)
    got = k.paged_attention(qkv, layout, dataclasses.replace(batch, scratch={}), cell, scale, window)
    return got[:want.shape[0]].double().cpu(), want, size, largest


def assert_within(got, want, allowed):
    off = (got - want).abs()
    worst = int((off - allowed).argmax())
    assert bool((off <= allowed).all()), f"row {worst // want.shape[1]}, element {worst % want.shape[1]}: {got.flatten()[worst]} for {want.flatten()[worst]}"


# Weights are 1 exactly, their sums whole numbers, so a result is off by a reciprocal's rounding, a product's (2^-24 of itself each) and, in bfloat16, half a step of 2^-7.  A key
# too many or too few of at most 1,300 / 32 that an element counts is a fortieth of it.
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("way", WAYS)
@pytest.mark.parametrize("window", [None, 65, 300])
@pytest.mark.parametrize("shape", SHAPES)
def test_every_key_counts_once(monkeypatch, dtype, way, window, shape):
    got, want, _, _ = run(monkeypatch, equal_scores, dtype, shape, way, window)
    assert_within(got, want, (2.0 ** -22 + (2.0 ** -8 if dtype == torch.bfloat16 else 0.0)) * want)


# Scores are 32 or 0: log2 of the weights is off by a rounding of 32 log2 e < 2^6, of 2^-24 each, in the score's product and the reference's, so weights by 2^-16 at most (in bfloat16 they
# round to 1 then, or by half a step of those that count 2^-46); results as above.
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("way", WAYS)
@pytest.mark.parametrize("shape", SHAPES)
def test_keys_are_told_apart(monkeypatch, dtype, way, shape):
    got, want, _, _ = run(monkeypatch, picked_keys, dtype, shape, way)
    assert_within(got, want, (2.0 ** -15 + (2.0 ** -8 if dtype == torch.bfloat16 else 0.0)) * want + 2.0 ** -30)


# A score is a sum of D products in float32: off by at most D 2^-24 of the sum of their sizes, and a weight by that (twice: its own and the sum's).  In bfloat16 a weight is rounded by half a step,
# 2^-8 of itself, which counts twice the same way, and the result once more.  Float32's three terms and its sums stay within 2^-18.
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("way", WAYS)
@pytest.mark.parametrize("window", [None, 300])
@pytest.mark.parametrize("shape", SHAPES)
def test_random_rows_column_by_column(monkeypatch, dtype, way, window, shape):
    got, want, size, largest = run(monkeypatch, random_rows, dtype, shape, way, window)
    weights = 2.0 * shape[2] * 2.0 ** -24 * largest + 2.0 ** -18 + (2.0 ** -7 if dtype == torch.bfloat16 else 0.0)
    assert_within(got, want, weights * size + (2.0 ** -8 * want.abs() if dtype == torch.bfloat16 else 0.0))
