"""What a runner's cache in 4 bits holds of a request, read back by the kernel library's `packed_rows`, is what the host reads page by page."""

from __future__ import annotations

import pytest
import torch

from llmserve_amd import CacheConfig, ModelRunner, StepEntry
from tests.tiny import TINY_B, random_tokens

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gathered_rows(dtype):
    from llmserve_amd.kernels import HipKernels
    from llmserve_amd.weights import random_model

    k, calls = HipKernels(dtype), []
    runner = ModelRunner(random_model(TINY_B, 0, dtype=dtype, device=k.device), k, CacheConfig(8, 80, 4, True), max_sequence_length=400)
    read = runner.cache.packed_rows
    runner.cache.packed_rows = lambda *given: calls.append(given) or read(*given)
    runs = [index for index, cell in enumerate(runner.cells) if cell is not None]
    runner.step([StepEntry("gone", random_tokens(50, TINY_B.vocab_size, 3), [49])], create_missing=True)
    runner.end_request("gone")  # (its pages are taken in another order)
    for count in (61, 1, 40):
        runner.step([StepEntry(name, random_tokens(count, TINY_B.vocab_size, count), [count - 1]) for name in ("a", "b")], create_missing=True)
    runner.cache.create("empty")
    firsts = set()
    for name in ("a", "b", "empty"):
        for run in runs:
            first, keys, values = runner.cache.gather(name, run)
            pages = list(runner.cache.iter_pages(name, run))
            assert first == (pages[0][0] if pages else 0) and len(calls) == 1
            calls.clear()
            firsts.add(first)
            for mine, theirs in ((keys, [k for _, k, _ in pages]), (values, [v for _, _, v in pages])):
                assert mine.dtype == torch.float32 and mine.shape[0] == runner.cache.sequences[name].length - first
                assert torch.equal(mine, torch.cat(theirs) if theirs else mine[:0])
    assert len(firsts) > 1  # (windows have given pages back)
    runner.close()
