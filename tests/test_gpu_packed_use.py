"""Caches in 4 bits as they are used: what the operators refuse, walks taken whole and cut, other streams, captured steps, the operators together, whole models."""

from __future__ import annotations

import dataclasses

import pytest
import torch

from llmserve_amd import CacheConfig, ModelRunner, StepEntry
from llmserve_amd.cache import CacheCell
from llmserve_amd.parts import HeadLayout, PackedKeyValue
from tests.packed_cases import assert_near, expected_of, kept, packed_case
from tests.plain import qwen2_plain as plain
from tests.tiny import BF16_LARGEST, BF16_MEAN, LONG, LOUD, TINY_B, random_tokens

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16]


@pytest.fixture(scope="module")
def kernels():
    from llmserve_amd.kernels import HipKernels

    return {dtype: HipKernels(dtype) for dtype in DTYPES}


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def largest_of(found, counts):
    return torch.cat([v.nan_to_num().abs().amax().expand(c, 1) if v.numel() else v.new_zeros((c, 1)) for (_, _, v), c in zip(found, counts)])


# ---------------------------------------------------------------------------- refusals (all found on the host, before a launch)


def test_refusals(kernels):
    from llmserve_amd.kernels import KernelError

    k = kernels[torch.bfloat16]
    batch, cell, layout, qkv, _ = packed_case(k, [20, 9], [1, 3], 4, 2, 64, 16)
    group = batch.groups[0]
    attend = lambda rows=qkv, shape=layout, step=batch, of=cell, scale=0.125, window=None, **more: k.paged_attention(rows, shape, step, of, scale, window, **more)
    store = lambda rows=qkv, shape=layout, step=batch, of=cell: k.store_packed(rows, shape, step, of)
    with_group = lambda **changes: dataclasses.replace(batch, groups=[dataclasses.replace(group, **changes)], scratch={})
    plain_cell = CacheCell(PackedKeyValue(2, 64), fields={"keys": torch.zeros(1, device="cuda"), "values": torch.zeros(1, device="cuda")}, group=0)
    wrong_pages = [
        CacheCell(cell.need, fields={"packed": cell.packed[:, :1]}, group=0),  # a head too few
        CacheCell(cell.need, fields={"packed": cell.packed[..., :-16]}, group=0),
        CacheCell(cell.need, fields={"packed": cell.packed.to(torch.int8)}, group=0),
        CacheCell(cell.need, fields={"packed": cell.packed.cpu()}, group=0),
        CacheCell(PackedKeyValue(2, 32), fields={"packed": cell.packed}, group=0),
        CacheCell(cell.need, fields={"packed": torch.zeros((4, 2, 2 * cell.packed.shape[2]), dtype=torch.uint8, device="cuda")[..., ::2]}, group=0),  # not contiguous
    ]
    refused = [
        *[lambda of=of: attend(of=of) for of in wrong_pages],
        *[lambda of=of: store(of=of) for of in wrong_pages],
        lambda: store(of=plain_cell),
        lambda: store(of=CacheCell(cell.need, writable=False, fields=cell.fields, group=0)),
        *[lambda rows=rows: attend(rows) for rows in (qkv[:, :-8], qkv.half(), qkv.cpu(), qkv[None])],
        *[lambda rows=rows: store(rows) for rows in (qkv[:, :-8], qkv.half(), qkv.cpu())],
        lambda: store(step=with_group(slot_mapping=group.slot_mapping[:-1])),
        lambda: store(step=with_group(slot_mapping=group.slot_mapping.long())),
        lambda: store(step=with_group(slot_mapping=group.slot_mapping.cpu())),
        lambda: store(step=with_group(page_size=8)),
        lambda: attend(step=with_group(block_tables=group.block_tables[:1])),
        lambda: attend(step=with_group(block_tables=group.block_tables.long())),
        lambda: attend(step=with_group(block_tables=group.block_tables.cpu())),
        lambda: attend(step=dataclasses.replace(batch, query_start=batch.query_start[:-1], scratch={})),
        lambda: attend(step=dataclasses.replace(batch, context_lengths=batch.context_lengths.long(), scratch={})),
        *[lambda scale=scale: attend(scale=scale) for scale in (0.0, -1.0, float("nan"))],
        lambda: k.rotate_and_store(qkv, layout, dataclasses.replace(batch, scratch={}, computed={}), cell, torch.ones(16, device="cuda"), "half"),  # angles of half the pairs
        lambda: k.rotate_and_store(qkv, layout, dataclasses.replace(batch, positions=batch.positions[:2], scratch={}, computed={}), cell, torch.ones(32, device="cuda"), "half"),
        lambda: attend(window=-3),
        lambda: attend(out=torch.empty((4, 256), dtype=torch.bfloat16)),
        lambda: attend(out=torch.empty((4, 256), device="cuda")),
        lambda: attend(out=torch.empty((4, 255), dtype=torch.bfloat16, device="cuda")),
        lambda: attend(soft_cap=30.0),
        lambda: attend(sinks=torch.zeros(4, device="cuda")),
        lambda: attend(keep_first=4),
        lambda: attend(chunk=16),
        *[lambda slots=slots: k.packed_rows(cell, slots, 16) for slots in (ints([0]).long(), torch.zeros(3, dtype=torch.int32), ints([[0, 1]]))],
        lambda: k.packed_rows(cell, ints([0]), 12),
        lambda: k.packed_rows(plain_cell, ints([0]), 16),
    ]
    before, held = qkv.clone(), cell.packed.clone()
    for index, call in enumerate(refused):
        with pytest.raises(KernelError):
            call()
            pytest.fail(f"call {index} was taken")
    assert torch.equal(qkv, before) and torch.equal(cell.packed, held)


def test_refusals_of_index_arrays(kernels):
    from llmserve_amd.kernels import KernelError

    k = kernels[torch.bfloat16]
    tables, slots, starts, counts = torch.zeros((1, 4, 8), dtype=torch.int32, device="cuda"), ints([0, 2]), ints([3, 0]), ints([1, 5])
    made = k.place_tokens(tables, slots, starts, counts, 16, 6, 8)
    for change in ({0: tables.long()}, {0: tables[0]}, {0: tables.cpu()}, {0: tables[..., ::2]}, {1: slots.long()}, {1: slots.cpu()}, {2: starts[:1]}, {3: counts.float()}, {4: 0}, {4: -16},
                   {5: -1}, {5: 1 << 30}, {6: 0}, {6: -1}, {1: slots[:0], 2: starts[:0], 3: counts[:0]}):
        arguments = [tables, slots, starts, counts, 16, 6, 8]
        for at, value in change.items():
            arguments[at] = value
        with pytest.raises(KernelError):
            k.place_tokens(*arguments)
    many = torch.zeros(4097, dtype=torch.int32, device="cuda")
    with pytest.raises(KernelError):
        k.place_tokens(tables, many, many, many, 16, 6, 8)
    for index in range(6):
        for wrong in (made[index].long(), made[index].cpu(), made[index].flatten()[:-1]):
            with pytest.raises(KernelError):
                k.place_tokens(tables, slots, starts, counts, 16, 6, 8, out=(*made[:index], wrong, *made[index + 1:]))
    with pytest.raises(KernelError):
        k.place_tokens(tables, slots, starts, counts, 16, 6, 8, out=made[:5])


# ---------------------------------------------------------------------------- whole and cut


def force(monkeypatch, k, least):
    """Walks in the given way (4: tiles shared where they can be, 8: few columns with many where a step has both, or many)."""
    monkeypatch.setattr(type(k), "_packed_way", staticmethod(lambda *given: (*least[:2], least[2] if least[2] == 8 or k.dtype == torch.bfloat16 else 0)))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("least", [(0, 0, 0), (1, 0, 0), (0, 1, 0), (1, 1, 0), (4, 8, 0), (3, 40, 0), (0, 0, 4), (1, 1, 4), (0, 8, 4), (4, 33, 4), (0, 0, 8), (1, 1, 8)])
@pytest.mark.parametrize("heads,kv_heads,dim,page,window", [(12, 2, 128, 16, None), (6, 2, 96, 24, 300), (7, 1, 64, 8, None), (34, 2, 32, 16, None), (3, 1, 192, 40, 65), (4, 2, 256, 16, None), (5, 1, 160, 16, None), (2, 1, 224, 8, None)])
def test_walks_whole_and_cut_anywhere(kernels, dtype, least, heads, kv_heads, dim, page, window, monkeypatch):
    k = kernels[dtype]
    lengths, counts = [1300, 1, 530, 777, 40, 0, 260, 1025], [1, 1, 1, 45, 40, 0, 2, 70]
    force(monkeypatch, k, least)
    batch, cell, layout, qkv, found = packed_case(k, lengths, counts, heads, kv_heads, dim, page, seed=dim)
    got = k.paged_attention(qkv, layout, batch, cell, dim ** -0.5, window)
    assert_near(got, expected_of(found, lengths, counts, dim ** -0.5, window), largest_of(found, counts), dtype)
    assert torch.equal(got, k.paged_attention(qkv, layout, batch, cell, dim ** -0.5, window))  # sums in one order


WAYS = [(0, 0, 0), (1, 1, 0), (0, 0, 4), (1, 1, 4), (0, 0, 8)]


def check(k, lengths, counts, heads, kv_heads, dim, page, scale, window=None, **more):
    batch, cell, layout, qkv, found = packed_case(k, lengths, counts, heads, kv_heads, dim, page, window=window, **more)
    got = k.paged_attention(qkv, layout, batch, cell, scale, window)
    assert_near(got, expected_of(found, lengths, counts, scale, window), largest_of(found, counts), k.dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("way", WAYS)
@pytest.mark.parametrize("counts", [[1, 1], [40, 1], [3, 70]])
def test_no_numbers_each_way(kernels, dtype, way, counts, monkeypatch):
    def change(index, rows):  # [length, 4 q heads | 2 k heads | 2 v heads of 64]
        if index == 0:
            rows[90, 4 * 64 + 5] = float("nan")  # a key of kv head 0, seen by queries from 90 on
            rows[80, 6 * 64 + 64 + 40] = float("inf")  # a value of kv head 1, second block
        else:
            rows[3, 6 * 64 + 1] = float("nan")  # before the window of most

    force(monkeypatch, kernels[dtype], way)
    check(kernels[dtype], [100, 75], counts, 4, 2, 64, 8, 0.125, 60, change=change, seed=3)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("way", WAYS)
@pytest.mark.parametrize("window", [1, 31, 33, 64, 65, 200])
def test_windows_each_way(kernels, dtype, way, window, monkeypatch):
    force(monkeypatch, kernels[dtype], way)
    check(kernels[dtype], [1, 40, 70, 341, 600, 290], [1, 1, 30, 141, 1, 200], 6, 2, 64, 8, 0.125, window, seed=window)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("way", WAYS)
@pytest.mark.parametrize("place", [0, 37, 130, 199])
def test_scores_far_apart_each_way(kernels, dtype, way, place, monkeypatch):
    def change(index, rows):
        rows[:, :64] *= 0.2
        rows[place, 64:128] = 100.0 * torch.sign(rows[199, :64])

    force(monkeypatch, kernels[dtype], way)
    check(kernels[dtype], [200, 200], [1, 30], 1, 1, 64, 16, 1.0, change=change, seed=place)


@pytest.mark.parametrize("way", WAYS)
def test_rows_of_nobody_and_rows_anywhere_each_way(kernels, way, monkeypatch):
    """Requests without tokens, rows behind the last request's, rows of an odd width from an odd element on, results into rows of an odd width."""
    k = kernels[torch.bfloat16]
    force(monkeypatch, k, way)
    lengths, counts = [0, 20, 5, 260, 7], [0, 1, 0, 133, 0]
    batch, cell, layout, qkv, found = packed_case(k, lengths, counts, 4, 2, 64, 8, row_stride=8 * 64 + 5)
    rows = torch.zeros(137 * layout.stride + 8, dtype=qkv.dtype, device="cuda")[3:3 + 137 * layout.stride].view(137, layout.stride)
    rows[:134].copy_(qkv)
    out = torch.full((137 * 263 + 8,), 7.0, dtype=qkv.dtype, device="cuda")[1:1 + 137 * 263].view(137, 263)
    assert k.paged_attention(rows, layout, batch, cell, 0.125, None, out=out) is out
    assert bool((out[134:] == 7).all()) and bool((out[:, 256:] == 7).all())
    assert_near(out[:134, :256], expected_of(found, lengths, counts, 0.125, None), max(v.abs().max() for _, _, v in found if v.numel()), k.dtype)


@pytest.mark.parametrize("way", WAYS)
def test_a_cache_beyond_32_bits(kernels, way, monkeypatch):
    """Pages that begin behind the first 4 GiB."""
    k, page, heads, kv_heads, dim = kernels[torch.bfloat16], 64, 4, 2, 128
    force(monkeypatch, k, way)
    lengths, counts = [700, 40, 300], [1, 1, 150]
    batch, cell, layout, qkv, found = packed_case(k, lengths, counts, heads, kv_heads, dim, page, spare=0)
    first = (1 << 32) // cell.packed[0].numel() + 1
    wide = torch.empty((first + cell.packed.shape[0], *cell.packed.shape[1:]), dtype=torch.uint8, device="cuda")
    wide[0] = 255
    far = CacheCell(cell.need, fields={"packed": wide}, group=0)
    tables = batch.groups[0].block_tables
    step = dataclasses.replace(batch, groups=[dataclasses.replace(batch.groups[0], block_tables=torch.where(tables >= 0, tables + first, tables),
                                                                  slot_mapping=batch.groups[0].slot_mapping + first * page)], scratch={})
    wide[first:] = cell.packed
    every = torch.arange(first * page, (first + 3) * page, dtype=torch.int32, device="cuda")
    for mine, theirs in zip(k.packed_rows(far, every, page), k.packed_rows(cell, every - first * page, page)):
        torch.testing.assert_close(mine, theirs, atol=0, rtol=0, equal_nan=True)
    k.store_packed(qkv, layout, step, far)
    assert torch.equal(wide[first:], cell.packed)  # (the step's rows were there already)
    got = k.paged_attention(qkv, layout, step, far, dim ** -0.5, None)
    assert torch.equal(got, k.paged_attention(qkv, layout, batch, cell, dim ** -0.5, None))
    assert_near(got, expected_of(found, lengths, counts, dim ** -0.5, None), largest_of(found, counts), k.dtype)


@pytest.mark.parametrize("page", [128, 1024, 1000])
@pytest.mark.parametrize("way", WAYS)
def test_large_pages(kernels, page, way, monkeypatch):
    force(monkeypatch, kernels[torch.bfloat16], way)
    check(kernels[torch.bfloat16], [page + 1, 2 * page - 1, 70], [1, 100, 70], 4, 2, 64, page, 0.125)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("least", [None, (1, 0, 0), (0, 0, 4), (0, 0, 8)])
@pytest.mark.parametrize("requests", [300, 700])
def test_many_requests(kernels, dtype, least, requests, monkeypatch):
    """More requests than a workgroup has threads for (256 over many columns, 512 over few), portions among them (which are then never cut)."""
    k = kernels[dtype]
    lengths = [1 + (index * 37) % 90 for index in range(requests)]
    counts = [1 if index % 50 else min(length, 30) for index, length in enumerate(lengths)]
    if least is not None:
        force(monkeypatch, k, least)
    batch, cell, layout, qkv, found = packed_case(k, lengths, counts, 4, 2, 64, 8)
    got = k.paged_attention(qkv, layout, batch, cell, 0.125, None)
    assert_near(got, expected_of(found, lengths, counts, 0.125, None), largest_of(found, counts), dtype)


def test_which_way_walks_go():
    """Few workgroups and long walks are cut, walks enough to fill the chip are not; tiles are shared where columns are many."""
    from types import SimpleNamespace

    from llmserve_amd.engine.batch import SequenceChunk
    from llmserve_amd.kernels import HipKernels

    def way(chunks, heads, kv_heads, window=0, shares=True, padded_to=None):
        batch = SimpleNamespace(max_context_length=max(start + count for start, count in chunks), max_query_length=max(count for _, count in chunks), padded_to=padded_to, scratch={}, context_lengths=torch.zeros(len(chunks)),
                                chunks=[SequenceChunk(str(i), i, start, count) for i, (start, count) in enumerate(chunks)])
        walks = HipKernels._packed_walks(batch, heads // kv_heads, window)
        assert walks == HipKernels._packed_walks(batch, heads // kv_heads, window)
        return walks[0], *HipKernels._packed_way(walks, len(chunks), heads // kv_heads, kv_heads, shares)

    assert way([(639, 1)], 12, 2) == (1, 0, 0, 0)
    assert way([(29999, 1)] * 8, 40, 8) == (1, 4, 0, 0) and way([(29999, 1)] * 8, 40, 8, 512) == (1, 0, 0, 0)
    assert way([(0, 2047)], 12, 2) == (2, 0, 0, 0)
    assert way([(30000, 128)], 12, 2) == (2, 0, 8, 0) and way([(30000, 128)], 12, 2, 512) == (2, 0, 0, 0)
    assert way([(30000, 2048)], 12, 2) == (2, 0, 8, 4) and not way([(30000, 2048)], 12, 2, shares=False)[3]
    assert way([(0, 8192)], 40, 8) == (2, 0, 0, 4)
    assert way([(600, 1)] * 31 + [(300, 256)], 28, 4) == (3, 0, 0, 8)  # the single tokens go with the portion
    assert way([(20000, 1)] * 31 + [(300, 256)], 28, 4)[3] == 0 and way([(600, 1)] * 31 + [(30000, 256)], 28, 4)[1:3] == (0, 8)
    assert way([(40, 2)] * 256 + [(30000, 128)], 12, 2)[:3] == (3, 0, 0)  # more requests than are cut for
    assert way([(600, 1)] * 3 + [(300, 256)], 28, 4, padded_to=(300, 5))[0] == 3 and way([(300, 256)], 28, 4, padded_to=(300, 5))[0] == 3


# ---------------------------------------------------------------------------- streams, graphs


@pytest.mark.parametrize("dtype", DTYPES)
def test_another_stream(kernels, dtype):
    k = kernels[dtype]
    lengths, counts = [3000, 50], [1, 20]
    batch, cell, layout, qkv, found = packed_case(k, lengths, counts, 4, 2, 64, 16)
    want = k.paged_attention(qkv, layout, batch, cell, 0.125, None)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        wide = torch.randn((4096, 4096), device="cuda")
        later = torch.zeros_like(qkv)
        for _ in range(20):  # work before it on its stream, none on the others
            wide = wide @ wide * 1e-3
        later.copy_(qkv)
        got = k.paged_attention(later, layout, batch, cell, 0.125, None)
    stream.synchronize()
    assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("least", [(1, 1, 0), (0, 0, 0), (1, 1, 4), (0, 0, 4), (0, 0, 8)])
def test_captured_and_replayed(kernels, dtype, least, monkeypatch):
    """Two captured steps of different cells, replayed in turn with eager calls between them and with lengths, queries and pages changed under them: index arrays,
    store and attention in one graph."""
    k, page, kv_heads, heads, dim, tokens = kernels[dtype], 16, 2, 6, 64, 24
    force(monkeypatch, k, least)
    rng = torch.Generator().manual_seed(1)
    cases = []
    for index in range(2):
        lengths, counts = ([900, 40, 33], [20, 1, 3]) if index == 0 else ([50, 1200, 8], [1, 22, 1])
        batch, cell, layout, qkv, _ = packed_case(k, lengths, counts, heads, kv_heads, dim, page, seed=index)
        cases.append((lengths, counts, batch, cell, layout, qkv))

    def run(case, given):
        _, _, batch, cell, layout, qkv = case
        starts, new = given
        group = batch.groups[0]
        positions, _, query_start, contexts, mapping, compact = k.place_tokens(group.block_tables[None], case_slots, starts, new, page, tokens, group.width)
        step = dataclasses.replace(batch, query_start=query_start, context_lengths=contexts, groups=[dataclasses.replace(group, block_tables=compact[0], slot_mapping=mapping[0])],
                                   padded_to=(tokens, 3), scratch={})
        k.store_packed(qkv, layout, step, cell)
        return k.paged_attention(qkv, layout, step, cell, 0.125, None)

    case_slots = ints([0, 1, 2])
    given = [(ints([n - c for n, c in zip(case[0], case[1])]), ints(case[1])) for case in cases]
    graphs = []
    for case, lengths in zip(cases, given):
        run(case, lengths)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = run(case, lengths)
        graphs.append((graph, out))
    for turn in range(4):
        for case, lengths in zip(cases, given):
            case[5].copy_(torch.randn(case[5].shape, generator=rng))
            counts = [1, 1 + turn, 22 - turn] if turn % 2 else [20, 3 - turn // 2, 1 + turn // 2]
            lengths[1].copy_(ints(counts))
            lengths[0].copy_(ints([min(n - 24, 20 * turn) if n > 60 else 0 for n in case[0]]) if turn else lengths[0])
            lengths[1].copy_(ints([min(c, max(1, n - s)) for c, n, s in zip(counts, case[0], lengths[0].tolist())]))
        for graph, _ in graphs:
            graph.replay()
        for case, lengths, (_, out) in zip(cases, given, graphs):
            used = int(lengths[1].sum())
            assert torch.equal(out[:used], run(case, lengths)[:used])
    torch.cuda.synchronize()


# ---------------------------------------------------------------------------- together


@pytest.mark.parametrize("dtype", DTYPES)
def test_steps_of_growing_requests(kernels, dtype):
    """A prompt in portions, single tokens behind it and a second request beside them: index arrays from lengths, rotated rows stored, attention over all that was
    stored.  The oracle takes the queries and keys as the rotation left them."""
    k, page, heads, kv_heads, dim = kernels[dtype], 8, 6, 2, 96
    layout, need = HeadLayout(heads, kv_heads, dim), PackedKeyValue(kv_heads, dim)
    tables = ints([[[3, 9, 1, 14, 6, 11, -1, -1], [12, 0, 5, 8, -1, -1, -1, -1]]])
    cell = CacheCell(need, fields={"packed": torch.full((16, kv_heads, need.page_bytes(page)), 255, dtype=torch.uint8, device="cuda")}, group=0)
    frequencies = 1.0 / (1000.0 ** (torch.arange(0, dim, 2, device="cuda").float() / dim))
    seen, rng = [[torch.zeros((0, 2 * kv_heads, dim), dtype=torch.float64)] for _ in range(2)], torch.Generator().manual_seed(2)
    lengths = [0, 0]
    template = packed_case(k, [1], [1], heads, kv_heads, dim, page)[0]
    for counts in ([21, 0], [1, 9], [1, 1], [17, 1], [1, 12], [2, 2]):
        tokens = sum(counts)
        active = [index for index in range(2) if counts[index]]
        new = [counts[index] for index in active]
        positions, sequence, query_start, contexts, mapping, compact = k.place_tokens(tables, ints(active), ints([lengths[i] for i in active]), ints(new), page, tokens, 6)
        starts = [lengths[i] for i in active]
        from llmserve_amd.engine.batch import GroupBatch, SequenceChunk

        batch = dataclasses.replace(
            template, num_tokens=tokens, chunks=[SequenceChunk(str(i), i, s, c) for i, s, c in zip(active, starts, new)], positions=positions, token_sequence=sequence, query_start=query_start,
            context_lengths=contexts, groups=[GroupBatch(page, compact[0], mapping[0], 6)], max_query_length=max(new), max_context_length=max(s + c for s, c in zip(starts, new)), scratch={}, computed={},
        )
        qkv = torch.randn((tokens, layout.stride), generator=rng).to(dtype).cuda()
        unrotated = qkv.clone()
        got = k.rotate_store_attend(qkv, layout, batch, cell, frequencies, "half", dim ** -0.5, None)
        k.rotate_and_store(unrotated, layout, batch, None, frequencies, "half")
        rows, found, at = unrotated.double().cpu(), [], 0
        for index, count in zip(active, new):
            mine = rows[at:at + count]
            seen[index].append(kept(mine[:, heads * dim:].view(count, 2 * kv_heads, dim)))
            both = torch.cat(seen[index])
            found.append((mine[:, :heads * dim].view(count, heads, dim), both[:, :kv_heads], both[:, kv_heads:]))
            lengths[index] += count
            at += count
        ends = [lengths[i] for i in active]
        assert_near(got, expected_of(found, ends, new, dim ** -0.5, None), largest_of(found, new), dtype)
    for index in range(2):
        slots = [int(tables[0, index, p // page]) * page + p % page for p in range(lengths[index])]
        keys, values = k.packed_rows(cell, ints(slots), page)
        assert torch.equal(torch.cat((keys, values), 1).double().cpu(), torch.cat(seen[index]))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("pairing", ["adjacent", "half"])
@pytest.mark.parametrize("heads,kv_heads,dim,tokens,spare", [(4, 2, 64, 7, 0), (12, 2, 128, 33, 0), (5, 1, 96, 9, 0), (3, 3, 32, 5, 0), (6, 2, 192, 65, 0), (2, 1, 256, 3, 0), (4, 2, 64, 7, 3), (7, 1, 224, 2, 5)])
def test_rows_rotated_as_they_are_packed(kernels, dtype, pairing, heads, kv_heads, dim, tokens, spare):
    """The rows and the pages are those of rotating first and packing then, bit by bit."""
    k, page = kernels[dtype], 16
    batch = packed_case(k, [tokens], [tokens], heads, kv_heads, dim, page, seed=dim + tokens)[0]
    layout = HeadLayout(heads, kv_heads, dim, (heads + 2 * kv_heads) * dim + spare)
    need, generator = PackedKeyValue(kv_heads, dim), torch.Generator().manual_seed(dim)
    pages = -(-tokens // page) + 4
    slots = torch.randperm((pages - 1) * page, generator=generator)[:tokens]
    slots[tokens // 2] = -1 if dim % 128 else pages * page
    batch.groups[0].slot_mapping.copy_(slots.int())
    batch.positions.add_(11)
    frequencies = 1.0 / (1000.0 ** (torch.arange(0, dim, 2, device="cuda").float() / dim))
    rows = torch.randn((tokens, layout.stride), generator=generator).to(dtype).cuda()
    rows[1, heads * dim + 3] = float("inf")
    make = lambda: CacheCell(need, fields={"packed": torch.full((pages, kv_heads, need.page_bytes(page)), 255, dtype=torch.uint8, device="cuda")}, group=0)
    apart, cell, other = rows.clone(), make(), make()
    k.rotate_and_store(apart, layout, batch, None, frequencies, pairing)
    k.store_packed(apart, layout, batch, other)
    k.rotate_and_store(rows, layout, batch, cell, frequencies, pairing)
    torch.testing.assert_close(rows, apart, atol=0, rtol=0, equal_nan=True)
    assert torch.equal(cell.packed, other.packed)


# ---------------------------------------------------------------------------- whole models


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("name,graphs", [("window", True), ("window", False), ("long", True), ("long", False)])
def test_models_over_caches_in_4_bits(kernels, tmp_path, dtype, name, graphs, monkeypatch):
    """Portions, single tokens and both, replayed from graphs and launched: the logits are those of a plain model whose attention takes the keys and values that the
    cache holds, and what it holds is what the plain model's own keys and values round to (float32; but where a difference in the last bits decides)."""
    from llmserve_amd.weights import load_model_folder, write_model_folder

    config, page = (TINY_B, 8) if name == "window" else (dataclasses.replace(LONG, num_layers=2) if LONG.num_layers > 2 else LONG, 16)
    folder = write_model_folder(tmp_path / "model", config, 5, dtype=torch.float32 if dtype == torch.float32 else torch.bfloat16, **LOUD)
    k = kernels[dtype]
    runner = ModelRunner(load_model_folder(folder, dtype), k, CacheConfig(page, 160, 4, True), max_sequence_length=400, use_graphs=graphs)
    runs = [index for index, cell in enumerate(runner.cells) if cell is not None]
    prompts = {"a": random_tokens(110, config.vocab_size, 1), "b": random_tokens(61, config.vocab_size, 2)}
    at = {request: 0 for request in prompts}
    rows = {request: [] for request in prompts}
    held = {request: [[] for _ in runs] for request in prompts}
    steps = [{"a": 40}, {"a": 1, "b": 23}, {"a": 1, "b": 1}, {"a": 1, "b": 1}, {"a": 21, "b": 1}, {"a": 21, "b": 1}, {"a": 21, "b": 1}, {"b": 33}, {"a": 1}, {"a": 1}, {"a": 1}, {"a": 1}]
    with torch.inference_mode():
        for step in steps:
            entries = [StepEntry(request, prompts[request][at[request]:at[request] + count], list(range(count))) for request, count in step.items()]
            if all(len(entry.tokens) == 1 for entry in entries):
                entries = [StepEntry(entry.request_id, entry.tokens, (0,)) for entry in entries]
            logits, first = runner.step(entries, create_missing=True).cpu().double(), 0
            for request, count in step.items():
                rows[request].append(logits[first:first + count])
                first += count
                for layer, run in enumerate(runs):
                    begin, keys, values = runner.cache.gather(request, run)
                    assert begin <= at[request]
                    held[request][layer].append(torch.stack((keys, values))[:, at[request] - begin:].cpu().double())
                at[request] += count
    assert at == {"a": 110, "b": 61} and (not graphs or (runner.step_counts["replayed"] and runner._graphs))
    weights, plain_config = plain.read_weights(folder), plain.PlainConfig.from_folder(folder)
    attention, total, count = plain.causal_attention, 0.0, 0
    for request, tokens in prompts.items():
        both = [torch.cat(layer, 1) for layer in held[request]]
        calls = []

        def over_what_is_held(q, keys, values, scale, window=None):
            layer = len(calls)
            calls.append(layer)
            for own, cached in ((keys, both[layer][0]), (values, both[layer][1])):
                blocks = own.unflatten(-1, (-1, 32))
                spread = blocks.abs().amax(-1, keepdim=True)
                # a block's power is at most its largest element / 3.5, and an element moves by up to one (those between 6 and 7) ...
                nudge = (spread * (1e-4 if dtype == torch.float32 else 0.06)).expand_as(blocks).flatten(-2)
                assert bool(((cached - own).abs() <= (spread / 3.5).expand_as(blocks).flatten(-2) * 1.001 + 2 * nudge).all())
                if dtype == torch.float32:  # ... and is the nearest where the rows' own last bits do not decide
                    certain = (kept(own - nudge) == kept(own)) & (kept(own + nudge) == kept(own))
                    assert certain.double().mean() > 0.9 and torch.equal(cached[certain], kept(own)[certain])
            return attention(q, both[layer][0], both[layer][1], scale, window)

        monkeypatch.setattr(plain, "causal_attention", over_what_is_held)
        want = plain.forward(weights, plain_config, tokens)
        monkeypatch.setattr(plain, "causal_attention", attention)
        got, spread = torch.cat(rows[request]), float(want.std())
        bound = dict(atol=2e-5 * max(1.0, spread / 0.3), rtol=1e-4) if dtype == torch.float32 else dict(atol=BF16_LARGEST * spread, rtol=3e-2)
        torch.testing.assert_close(got, want, **bound)
        total, count = total + float((got - want).abs().mean()) / spread, count + 1
    if dtype == torch.bfloat16:
        assert total / count < BF16_MEAN
    runner.close()
