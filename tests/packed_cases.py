"""Keys and values in 4 bits, written from their definition in float64, and steps over pages of them."""

from __future__ import annotations

import math
import types

import torch


def kept(rows):
    """What pages in 4 bits keep of float64 [..., D], 32 neighbours a block."""
    x = rows.double().unflatten(-1, (-1, 32))
    largest = x.abs().amax(-1, keepdim=True)
    significand, exponent = torch.frexp(largest)
    exponent = torch.where(largest > 0, exponent - 1 + (significand >= 0.875).to(exponent.dtype), torch.tensor(-1000, dtype=exponent.dtype))
    unit = torch.pow(2.0, (exponent - 2).clamp(-125, 125).double())
    size = (x / unit).abs().clamp(max=6.0)
    step = torch.where(size < 2.0, 0.5, torch.where(size < 4.0, 1.0, 2.0))
    found = torch.copysign(torch.round(size / step) * step, x) * unit
    return torch.where(torch.isfinite(largest), found, math.nan).flatten(-2)


def reference(q, keys, values, scale, window, first_position):
    """softmax(q k^T scale) v in float64: q [n, heads, D] at positions from `first_position` on, keys and values [m, kv, D] of positions from 0 on.  A key that a
    query doesn't see has no part in its result, whatever it holds."""
    n, heads, _ = q.shape
    group = heads // keys.shape[1]
    out = torch.empty_like(q, dtype=torch.float64)
    for i in range(n):
        p = first_position + i
        first = max(0, p - window + 1) if window else 0
        for h in range(heads):
            scores = keys[first:p + 1, h // group].double() @ q[i, h].double() * scale
            out[i, h] = torch.softmax(scores, 0) @ values[first:p + 1, h // group].double()
    return out.flatten(1)


def packed_case(kernels, lengths, counts, heads, kv_heads, dim, page, seed=0, spare=3, window=None, row_stride=None, change=None, padded=0, group=0):
    """Requests with lengths[i] cached tokens of which the last counts[i] are this step's, on the GPU: every page byte is 0xff (no number) where no token lies, pages in any
    order.  -> (batch, cell, layout, qkv of the step, per request (q of its step, what is kept of its keys, of its values))."""
    from llmserve_amd.cache import CacheCell
    from llmserve_amd.engine.batch import GroupBatch, SequenceChunk, StepBatch
    from llmserve_amd.parts import HeadLayout, PackedKeyValue

    generator = torch.Generator().manual_seed(seed)
    layout = HeadLayout(heads, kv_heads, dim, row_stride)
    need = PackedKeyValue(kv_heads, dim, window)
    blocks = [max(1, math.ceil(n / page)) for n in lengths]
    pages = sum(blocks) + spare
    order = torch.randperm(pages, generator=generator).tolist()
    width = max(blocks) + padded
    tables = torch.full((len(lengths), width), -1, dtype=torch.int32)
    storage = torch.full((pages, kv_heads, need.page_bytes(page)), 255, dtype=torch.uint8, device="cuda")
    cell = CacheCell(need, fields={"packed": storage}, group=0)
    ints = lambda values: torch.tensor(values, dtype=torch.int32, device="cuda")
    rows, step, found = [], [], []
    for index, (length, count) in enumerate(zip(lengths, counts)):
        mine = [order.pop() for _ in range(blocks[index])]
        tables[index, :len(mine)] = torch.tensor(mine, dtype=torch.int32)
        full = torch.zeros((length, layout.stride))
        full[:, :layout.width] = torch.randn((length, layout.width), generator=generator)
        full[:, heads * dim:layout.width] *= torch.exp(torch.randn(2 * kv_heads * dim, generator=generator))
        if change is not None:
            change(index, full)
        full = full.to(kernels.dtype)
        slots = [mine[p // page] * page + p % page for p in range(length)]
        if length:
            earlier = types.SimpleNamespace(groups=[GroupBatch(page, tables, ints(slots), width)])
            kernels.store_packed(full.cuda(), layout, earlier, cell)
        mine_kv = kept(full[:, heads * dim:layout.width].double().view(length, 2 * kv_heads, dim)) if length else full.new_zeros((0, 2 * kv_heads, dim)).double()
        rows.append(full[length - count:])
        step += slots[length - count:]
        found.append((full[length - count:, :heads * dim].double().view(count, heads, dim), mine_kv[:, :kv_heads], mine_kv[:, kv_heads:]))
    starts = [sum(counts[:i]) for i in range(len(counts) + 1)]
    positions = [p for length, count in zip(lengths, counts) for p in range(length - count, length)]
    sequence = [i for i, count in enumerate(counts) for _ in range(count)]
    batch = StepBatch(
        num_tokens=sum(counts), chunks=[SequenceChunk(f"r{i}", i, n - c, c) for i, (n, c) in enumerate(zip(lengths, counts))], token_ids=ints([0] * sum(counts)),
        positions=ints(positions), token_sequence=ints(sequence), query_start=ints(starts), context_lengths=ints(lengths), state_slots=ints(list(range(len(lengths)))),
        groups=[GroupBatch(page, tables.cuda(), ints(step), width)], logit_rows=ints([]), num_logit_rows=0, max_query_length=max(counts), max_context_length=max(lengths),
    )
    return batch, cell, layout, torch.cat(rows).cuda(), found


def expected_of(found, lengths, counts, scale, window):
    return torch.cat([reference(q, k, v, scale, window, length - count) for (q, k, v), length, count in zip(found, lengths, counts)])


# A float32 result is exact but for sums in float32 (and products in three bfloat16 terms, 2^-24 of their largest).  In bfloat16 the weights are rounded once
# (half a step, 2^-9 of each at random, 2^-8 at most) and the result once more (2^-8 of itself at most).  An element is a sum of weights times values of no
# one sign, so what it may be off by goes by the largest value that its head keeps: half steps of 2^-8 of weights that add up to 1, twice.
def assert_near(got, want, values_largest, dtype):
    tolerance = 2.0 ** -8 * 2 if dtype == torch.bfloat16 else 64 * 2.0 ** -24
    off = (got.double().cpu() - want).abs()
    allowed = tolerance * torch.maximum(want.abs(), torch.as_tensor(values_largest).double())
    assert torch.equal(torch.isnan(got.cpu()), torch.isnan(want)), "rows that are no number"
    off, allowed = off[~torch.isnan(want)], allowed.expand_as(want)[~torch.isnan(want)]
    worst = (off / allowed).max().item() if off.numel() else 0.0
    assert worst <= 1.0, f"{worst:.3f} of what rounding allows"
