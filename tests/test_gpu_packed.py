"""Keys and values in 4 bits on the GPU: rows packed into pages and read back, attention over the pages, and a step's index arrays made on the device."""

from __future__ import annotations

import math
import types

import pytest
import torch

from tests.packed_cases import assert_near, expected_of, kept, packed_case

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16]


@pytest.fixture(scope="module")
def kernels():
    from llmserve_amd.kernels import HipKernels

    return {dtype: HipKernels(dtype) for dtype in DTYPES}


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def group_of(page, slots):
    from llmserve_amd.engine.batch import GroupBatch

    return types.SimpleNamespace(groups=[GroupBatch(page, ints([[0]]), ints(slots), 1)])


def same(got, want):
    torch.testing.assert_close(got.double().cpu(), want.double().cpu(), atol=0, rtol=0, equal_nan=True)


# ---------------------------------------------------------------------------- store and read back


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,kv_heads,dim,page,tokens,spare", [(4, 2, 32, 8, 1, 0), (12, 2, 128, 16, 37, 0), (3, 3, 96, 24, 65, 5), (8, 1, 256, 64, 9, 8), (2, 2, 160, 16, 130, 0), (7, 7, 64, 8, 301, 3)])
def test_rows_packed_and_read_back(kernels, dtype, heads, kv_heads, dim, page, tokens, spare):
    """Every row that is stored reads back as its definition says, through the kernel and through the host's read path; nothing else in the pages changes."""
    from llmserve_amd.cache import CacheCell
    from llmserve_amd.parts import HeadLayout, PackedKeyValue

    k, generator = kernels[dtype], torch.Generator().manual_seed(dim)
    layout, need = HeadLayout(heads, kv_heads, dim, (heads + 2 * kv_heads) * dim + spare), PackedKeyValue(kv_heads, dim)
    pages = -(-tokens // page) + 2
    storage = torch.full((pages, kv_heads, need.page_bytes(page)), 255, dtype=torch.uint8, device="cuda")
    cell = CacheCell(need, fields={"packed": storage}, group=0)
    rows = torch.randn((tokens, layout.stride), generator=generator) * torch.exp(6 * torch.randn((tokens, layout.stride), generator=generator))
    rows[0] = 0.0
    rows[tokens // 2, heads * dim:] = torch.tensor([3.4e38, -1e-45, 1.75, 0.25, 1.2e-38])[torch.arange(layout.stride - heads * dim) % 5]
    rows = rows.to(dtype)
    rows[:, layout.width:] = math.nan  # what lies behind the heads is nobody's
    slots = torch.randperm(pages * page, generator=generator)[:tokens]
    given = slots.tolist()
    given[tokens // 3] = -1 if tokens > 1 else given[0]
    k.store_packed(rows.cuda(), layout, group_of(page, given), cell)
    want = kept(rows[:, heads * dim:layout.width].double().view(tokens, 2 * kv_heads, dim))
    asked = [s if s >= 0 else -7 for s in given] + [pages * page]
    keys, values = k.packed_rows(cell, ints(asked), page)
    stored = torch.tensor([s >= 0 for s in given])
    want[~stored] = 0.0
    assert keys.dtype == dtype
    same(keys[:tokens], want[:, :kv_heads])
    same(values[:tokens], want[:, kv_heads:])
    assert not keys[tokens].any() and not values[tokens].any()
    seen = torch.zeros((pages, page), dtype=torch.bool)
    for p in range(pages):
        host = need.token_rows({"packed": storage[p].cpu()}, page)
        for offset in range(page):
            where = [i for i, s in enumerate(given) if s == p * page + offset]
            if where:
                same(host["keys"][offset], want[where[0], :kv_heads])
                same(host["values"][offset], want[where[0], kv_heads:])
            else:
                assert torch.isnan(host["keys"][offset]).all() and torch.isnan(host["values"][offset]).all()
            seen[p, offset] = bool(where)
    assert int(seen.sum()) == int(stored.sum())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("begins", [0, 3, 7])
@pytest.mark.parametrize("tokens", [2600, 2601, 4093])
def test_many_rows_packed_and_read_back(kernels, dtype, begins, tokens):
    """Portions of two requests, from anywhere in a page, with rows that are stored nowhere among them, and slots in no order at the end."""
    from llmserve_amd.cache import CacheCell
    from llmserve_amd.parts import HeadLayout, PackedKeyValue

    k, page, kv_heads, dim = kernels[dtype], 24, 3, 96
    layout, need, generator = HeadLayout(5, kv_heads, dim, 11 * dim + 8), PackedKeyValue(kv_heads, dim), torch.Generator().manual_seed(tokens + begins)
    pages = tokens // page + 40
    cell = CacheCell(need, fields={"packed": torch.full((pages, kv_heads, need.page_bytes(page)), 255, dtype=torch.uint8, device="cuda")}, group=0)
    order = torch.randperm(pages, generator=generator)
    place = lambda first, positions: order[first + positions // page] * page + positions % page
    one, other = begins + torch.arange(tokens // 2), 5 + torch.arange(tokens - tokens // 2 - 60)
    given = torch.cat([place(0, one), place(tokens // 2 // page + 3, other), place(pages - 10, torch.randperm(200, generator=generator)[:60])])
    given[[9, 10, 700, tokens - 1]] = torch.tensor([-1, pages * page, -5, -1])
    rows = (torch.randn((tokens, layout.stride), generator=generator) * 3).to(dtype)
    rows[33, 6 * dim] = math.inf
    k.store_packed(rows.cuda(), layout, group_of(page, given.tolist()), cell)
    keys, values = k.packed_rows(cell, given.int().cuda(), page)
    want = kept(rows[:, 5 * dim:11 * dim].double().view(tokens, 2 * kv_heads, dim))
    want[(given < 0) | (given >= pages * page)] = 0.0
    same(keys, want[:, :kv_heads])
    same(values, want[:, kv_heads:])
    untouched = torch.ones(pages * page, dtype=torch.bool)
    untouched[given[(given >= 0) & (given < pages * page)]] = False
    assert all(torch.isnan(x).all() for x in k.packed_rows(cell, untouched.nonzero().flatten().int().cuda(), page))


@pytest.mark.parametrize("dtype", DTYPES)
def test_blocks_that_are_no_numbers(kernels, dtype):
    """An infinity or a NaN makes its own block of 32 read as NaN and no other; the page's other tokens stay as they were."""
    from llmserve_amd.cache import CacheCell
    from llmserve_amd.parts import HeadLayout, PackedKeyValue

    k, need, layout = kernels[dtype], PackedKeyValue(1, 64), HeadLayout(1, 1, 64)
    cell = CacheCell(need, fields={"packed": torch.zeros((1, 1, need.page_bytes(8)), dtype=torch.uint8, device="cuda")}, group=0)
    rows = torch.randn((8, 192)).to(dtype)
    rows[2, 64 + 40], rows[5, 128 + 3], rows[6, 64] = math.nan, -math.inf, math.inf
    k.store_packed(rows.cuda(), layout, group_of(8, list(range(8))), cell)
    keys, values = k.packed_rows(cell, ints(list(range(8))), 8)
    want = kept(rows[:, 64:].double().view(8, 2, 64))
    assert torch.isnan(want).sum() == 96
    same(torch.stack((keys, values), 1).squeeze(2), want)


def test_rounding_at_every_border(kernels):
    """Halfway cases go to the even code, what is larger than 6 of its unit stays 6, and a block's unit changes at a significand of 1.75."""
    from llmserve_amd.cache import CacheCell
    from llmserve_amd.parts import HeadLayout, PackedKeyValue

    k, need, layout = kernels[torch.float32], PackedKeyValue(1, 32), HeadLayout(1, 1, 32)
    borders = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0]
    row = [s * b * (1 + e * 2.0 ** -23) for b in borders for s in (1, -1) for e in (-1, 0)] + [4.0, 6.0, 6.9, 6.99]
    rows = torch.tensor(row).repeat(6, 3).view(6, 96)
    rows[1] *= 2.0 ** 100
    rows[2] *= 2.0 ** -120
    rows[3, 31::32] = 7.0
    rows[4, 31::32] = torch.nextafter(torch.tensor(7.0), torch.tensor(0.0))
    rows[5, 31::32] = 7.99
    cell = CacheCell(need, fields={"packed": torch.zeros((1, 1, need.page_bytes(8)), dtype=torch.uint8, device="cuda")}, group=0)
    k.store_packed(rows.cuda(), layout, group_of(8, list(range(6))), cell)
    keys, values = k.packed_rows(cell, ints(list(range(6))), 8)
    want = kept(rows[:, 32:].double().view(6, 2, 32))
    same(torch.stack((keys, values), 1).squeeze(2), want)


# ---------------------------------------------------------------------------- attention

SHAPES = [  # heads, kv heads, dim, page
    (12, 2, 128, 16),
    (4, 4, 32, 8),
    (28, 4, 128, 24),
    (9, 3, 96, 16),
    (40, 8, 64, 64),
    (6, 2, 160, 16),
    (5, 1, 192, 8),
    (2, 1, 224, 40),
    (16, 2, 256, 16),
    (34, 1, 64, 16),  # more query heads a kv head than a tile of sixteen
]


def run_case(k, lengths, counts, heads, kv_heads, dim, page, *, window=None, scale=None, **more):
    scale = scale or dim ** -0.5
    batch, cell, layout, qkv, found = packed_case(k, lengths, counts, heads, kv_heads, dim, page, window=window, **more)
    got = k.paged_attention(qkv, layout, batch, cell, scale, window)
    want = expected_of(found, lengths, counts, scale, window)
    largest = torch.cat([v.nan_to_num().abs().amax().expand(c, 1) if v.numel() else v.new_zeros((c, 1)) for (_, _, v), c in zip(found, counts)])
    assert got.dtype == k.dtype
    assert_near(got, want, largest, k.dtype)
    return batch, cell, layout, qkv, got


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,kv_heads,dim,page", SHAPES)
def test_single_tokens_at_page_edges(kernels, dtype, heads, kv_heads, dim, page):
    lengths = [1, page - 1, page, page + 1, 31, 32, 33, 5 * page + 3, 150, 2]
    run_case(kernels[dtype], lengths, [1] * len(lengths), heads, kv_heads, dim, page, seed=dim)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,kv_heads,dim,page", SHAPES)
def test_portions_beside_single_tokens(kernels, dtype, heads, kv_heads, dim, page):
    lengths = [1, page + 1, 77, 2 * page, 5 * page + 3, 150, 3]
    counts = [1, 1, 77, 2, 2 * page + 2, 33, 3]
    run_case(kernels[dtype], lengths, counts, heads, kv_heads, dim, page, seed=dim + 1)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("window", [1, 2, 31, 32, 33, 100])
def test_windows(kernels, dtype, window):
    lengths, counts = [1, 40, 70, 141, 300, 90], [1, 1, 1, 1, 1, 60]
    run_case(kernels[dtype], lengths, counts, 6, 2, 64, 8, window=window, seed=window)


@pytest.mark.parametrize("dtype", DTYPES)
def test_requests_without_tokens_and_rows_behind_the_last(kernels, dtype):
    """A request that brings no token writes nothing, wherever it stands; rows behind the last request's keep what they held."""
    k = kernels[dtype]
    lengths, counts = [0, 20, 5, 60, 7], [0, 1, 0, 13, 0]
    batch, cell, layout, qkv, found = packed_case(k, lengths, counts, 4, 2, 64, 8)
    rows = torch.cat([qkv, qkv[:3]])
    out = torch.full((17, 4 * 64 + 8), 7.0, dtype=dtype, device="cuda")
    got = k.paged_attention(rows, layout, batch, cell, 0.125, None, out=out)
    assert got is out and bool((out[14:] == 7).all()) and bool((out[:, 256:] == 7).all())
    assert_near(out[:14, :256], expected_of(found, lengths, counts, 0.125, None), max(v.abs().max() for _, _, v in found if v.numel()), dtype)
    alone = packed_case(k, [3], [0], 4, 2, 64, 8)
    assert k.paged_attention(alone[3], alone[2], alone[0], alone[1], 0.125, None).shape == (0, 256)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("counts", [[1, 1], [40, 1], [3, 70]])
def test_no_numbers_reach_only_the_queries_that_see_them(kernels, dtype, counts):
    """A NaN key makes every query that sees it NaN, a NaN value the dimensions of its block; a query that does not see them is as without them."""
    def change(index, rows):  # [length, 4 q heads | 2 k heads | 2 v heads of 64]
        if index == 0:
            rows[90, 4 * 64 + 5] = math.nan  # a key of kv head 0, seen by queries from 90 on
            rows[80, 6 * 64 + 64 + 40] = math.inf  # a value of kv head 1, second block
        else:
            rows[3, 6 * 64 + 1] = math.nan  # before the window of most

    run_case(kernels[dtype], [100, 75], counts, 4, 2, 64, 8, window=60, change=change, seed=3)


@pytest.mark.parametrize("dtype", DTYPES)
def test_scores_far_apart(kernels, dtype):
    """Scores of several hundred: one key takes all the weight, and the largest comes late, early, and in between."""
    for place in (0, 37, 130, 199):
        def change(index, rows):
            rows[:, :64] *= 0.2
            rows[place, 64:128] = 100.0 * torch.sign(rows[199, :64])

        run_case(kernels[dtype], [200, 200], [1, 30], 1, 1, 64, 16, scale=1.0, change=change, seed=place)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lengths,counts,window", [([5000, 1, 700], [1, 1, 1], None), ([3000], [2], None), ([2500, 40], [20, 1], None), ([4100], [1], 1500), ([2050, 2050], [150, 1], 999)])
def test_long_contexts(kernels, dtype, lengths, counts, window):
    """Keys split over workgroups and joined."""
    run_case(kernels[dtype], lengths, counts, 4, 2, 64, 16, window=window, seed=lengths[0])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("first", [1, 3])
def test_rows_that_begin_anywhere(kernels, dtype, first):
    """Rows of an odd width, from an odd element on, and results into rows of an odd width."""
    k = kernels[dtype]
    lengths, counts = [50, 9], [1, 9]
    batch, cell, layout, qkv, found = packed_case(k, lengths, counts, 2, 1, 64, 8, row_stride=4 * 64 + 5)
    held = torch.zeros(qkv.numel() + 8, dtype=dtype, device="cuda")
    rows = held[first:first + qkv.numel()].view_as(qkv)
    rows.copy_(qkv)
    out = torch.zeros(10 * 131 + 8, dtype=dtype, device="cuda")[first:first + 10 * 131].view(10, 131)
    k.paged_attention(rows, layout, batch, cell, 0.125, None, out=out)
    assert_near(out[:, :128], expected_of(found, lengths, counts, 0.125, None), max(v.abs().max() for _, _, v in found), dtype)
    assert not out[:, 128:].any()


# ---------------------------------------------------------------------------- index arrays


def plain_places(tables, slots, starts, counts, page, tokens, width):
    groups, rows, blocks = len(tables), len(tables[0]), len(tables[0][0])
    positions, sequence, ends, contexts = [], [], [0], []
    mapping, compact = [[] for _ in range(groups)], [[] for _ in range(groups)]
    for b, (slot, start, count) in enumerate(zip(slots, starts, counts)):
        real = 0 <= slot < rows
        for i in range(count):
            p = start + i if real else 0
            positions.append(p)
            sequence.append(b)
            for g in range(groups):
                held = tables[g][slot][p // page] if real and p // page < blocks else -1
                mapping[g].append(-1 if held < 0 else held * page + p % page)
        ends.append(min(ends[-1] + count, tokens))
        contexts.append(start + count if real else 1)
        for g in range(groups):
            row = [tables[g][slot][j] if j < min(blocks, -(-(start + count) // page)) else -1 for j in range(width)] if real else [0] * width
            compact[g].append(row)
    missing = tokens - len(positions)
    positions, sequence = positions[:tokens] + [0] * missing, sequence[:tokens] + [len(slots) - 1] * missing
    return positions, sequence, ends, contexts, [m[:tokens] + [-1] * missing for m in mapping], compact


@pytest.mark.parametrize("requests,groups,page,most,spare", [(1, 1, 16, 1, 0), (1, 2, 8, 700, 0), (3, 1, 16, 300, 5), (64, 2, 16, 1, 0), (130, 3, 24, 9, 41), (257, 1, 1, 4, 0), (1500, 1, 16, 3, 7), (4096, 1, 64, 1, 0)])
def test_index_arrays_from_lengths(kernels, requests, groups, page, most, spare):
    generator = torch.Generator().manual_seed(requests)
    draw = lambda low, high: int(torch.randint(low, high, (1,), generator=generator))
    rows, blocks = requests + 3, 40
    tables = torch.randint(0, 1 << 20, (groups, rows, blocks), generator=generator, dtype=torch.int32)
    tables[torch.rand(tables.shape, generator=generator) < 0.05] = -1
    order = torch.randperm(rows, generator=generator)[:requests].tolist()
    slots = [s if draw(0, 10) else (-1 if draw(0, 2) else rows) for s in order]
    counts = [draw(0, most + 1) if most > 1 else 1 for _ in range(requests)]
    starts = [draw(0, max(1, blocks * page - c + 9)) for c in counts]  # (some run past their tables' last block)
    tokens, width = sum(counts) + spare, draw(1, blocks + 4)
    k = kernels[torch.bfloat16]
    got = k.place_tokens(tables.cuda(), ints(slots), ints(starts), ints(counts), page, tokens, width)
    want = plain_places(tables.tolist(), slots, starts, counts, page, tokens, width)
    for g, w in zip(got, want):
        assert g.dtype == torch.int32 and g.tolist() == w
    if tokens > 2:  # more tokens than there is room for: the last ones are left out
        short = k.place_tokens(tables.cuda(), ints(slots), ints(starts), ints(counts), page, tokens - 2, width)
        want = plain_places(tables.tolist(), slots, starts, counts, page, tokens - 2, width)
        for g, w in zip(short, want):
            assert g.tolist() == w


def test_index_arrays_into_given_tensors(kernels):
    """Into views of one array, as a captured step reads them, and no byte beside them."""
    k = kernels[torch.float32]
    tables = torch.arange(2 * 4 * 6, dtype=torch.int32, device="cuda").view(2, 4, 6)
    held = torch.full((200,), 99, dtype=torch.int32, device="cuda")
    out = (held[1:6], held[7:12], held[13:16], held[20:22], held[30:].as_strided((2, 5), (40, 1)), held[40:].as_strided((2, 2, 3), (40, 3, 1)))
    arguments = tables, ints([3, 1]), ints([10, 0]), ints([1, 4]), 4, 5, 3
    got, want = k.place_tokens(*arguments, out=out), k.place_tokens(*arguments)
    for g, w in zip(got, want):
        assert torch.equal(g, w)
    touched = torch.zeros(200, dtype=torch.bool)
    for a, n in ((1, 5), (7, 5), (13, 3), (20, 2), (30, 5), (70, 5), (40, 6), (80, 6)):
        touched[a:a + n] = True
    assert bool((held.cpu()[~touched] == 99).all())


def test_a_step_without_tokens(kernels):
    got = kernels[torch.bfloat16].place_tokens(ints([[[4, -1]]]), ints([0]), ints([3]), ints([0]), 8, 0, 2)
    assert [g.tolist() for g in got] == [[], [], [0, 0], [3], [[]], [[[4, -1]]]]
