"""What operators over pages in 4 bits refuse, they refuse before anything is changed."""

from __future__ import annotations

import dataclasses

import pytest
import torch

from tests.packed_cases import packed_case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("tokens", [3, 2600])
def test_rows_are_not_rotated_where_their_pages_are_refused(dtype, tokens):
    """With few rows (rotated as they are packed) and with many (rotated first)."""
    from llmserve_amd.cache import CacheCell
    from llmserve_amd.kernels import HipKernels, KernelError
    from llmserve_amd.parts import PackedKeyValue

    k = HipKernels(dtype)
    heads, kv_heads, dim, page = 4, 4, 96, 16
    batch, cell, layout, qkv, _ = packed_case(k, [tokens], [tokens], heads, kv_heads, dim, page)
    group, frequencies = batch.groups[0], torch.ones(dim // 2, device="cuda")
    of_group = lambda **changes: dataclasses.replace(batch, groups=[dataclasses.replace(group, **changes)], scratch={}, computed={})
    before, held = qkv.clone(), cell.packed.clone()
    refused = [
        (of_group(slot_mapping=group.slot_mapping[:-1]), cell),
        (of_group(slot_mapping=group.slot_mapping.long()), cell),
        (of_group(page_size=8), cell),
        (batch, CacheCell(cell.need, fields={"packed": cell.packed[:, :1]}, group=0)),
        (batch, CacheCell(PackedKeyValue(kv_heads, 32), fields={"packed": cell.packed}, group=0)),
        (batch, CacheCell(cell.need, fields={"packed": torch.zeros(cell.packed.numel() + 8, dtype=torch.uint8, device="cuda")[8:].view_as(cell.packed)}, group=0)),  # not at a piece of 16 bytes
        (dataclasses.replace(batch, positions=batch.positions[:-1], scratch={}, computed={}), cell),
    ]
    for index, (step, of) in enumerate(refused):
        for pairing in ("adjacent", "half"):
            with pytest.raises(KernelError):
                k.rotate_and_store(qkv, layout, step, of, frequencies, pairing)
                pytest.fail(f"call {index} was taken")
            assert torch.equal(qkv, before), f"call {index} changed the rows"
    assert torch.equal(cell.packed, held)


def test_windows_wider_than_any_position():
    """They are no windows, also where 32 bits do not hold them."""
    from llmserve_amd.kernels import HipKernels

    k = HipKernels(torch.bfloat16)
    batch, cell, layout, qkv, _ = packed_case(k, [70, 40], [1, 30], 4, 2, 64, 16)
    want = k.paged_attention(qkv, layout, batch, cell, 0.125, None)
    for window in (70, (1 << 30) - 1, 1 << 30, (1 << 31) - 1, 1 << 31, (1 << 32) + 5):
        assert torch.equal(k.paged_attention(qkv, layout, batch, cell, 0.125, window), want), window
