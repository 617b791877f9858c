"""A launched step's index arrays: those made on the device from the requests' lengths are those packed on the host."""

from __future__ import annotations

import random

import pytest
import torch

from llmserve_amd import CacheConfig, StepEntry
from llmserve_amd.cache import CacheManager
from llmserve_amd.engine import build_step_batch
from llmserve_amd.registry import ARCHITECTURES
from tests.tiny import TINY_A, TINY_B

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def library():
    from llmserve_amd.kernels import HipKernels

    return HipKernels(torch.bfloat16, torch.device("cuda:0"))


def same_steps(made, packed) -> None:
    for name in ("num_tokens", "num_logit_rows", "max_query_length", "max_context_length", "every_row_wanted", "padded_to", "chunks"):
        assert getattr(made, name) == getattr(packed, name), name
    for name in ("token_ids", "positions", "token_sequence", "query_start", "context_lengths", "state_slots", "logit_rows"):
        mine, theirs = getattr(made, name), getattr(packed, name)
        assert mine.dtype == theirs.dtype and torch.equal(mine, theirs), name
    assert len(made.groups) == len(packed.groups)
    for mine, theirs in zip(made.groups, packed.groups):
        assert (mine.page_size, mine.width) == (theirs.page_size, theirs.width)
        assert torch.equal(mine.slot_mapping, theirs.slot_mapping) and torch.equal(mine.block_tables, theirs.block_tables)


@pytest.mark.parametrize("config,page", [(TINY_A, 4), (TINY_B, 8), (TINY_B, 3)])
@pytest.mark.parametrize("seed", [0, 1, 2])
def test_random_steps(library, config, page, seed):
    """Portions, single tokens, requests that end and whose pages others take, and windows (TINY_B) that pages fall behind."""
    rng = random.Random(seed)
    spec = ARCHITECTURES["Qwen2ForCausalLM"].build_spec(config)
    cache = CacheManager(spec, CacheConfig(block_size=page, num_blocks=160, max_sequences=6), max_sequence_length=200)
    live: list[str] = []
    for step in range(40):
        if len(live) < 6 and (not live or rng.random() < 0.4):
            live.append(f"r{step}")
            cache.create(live[-1])
        entries = []
        for name in rng.sample(live, rng.randint(1, len(live))):
            tokens = [rng.randrange(config.vocab_size) for _ in range(1 if rng.random() < 0.5 else rng.randint(2, 60))]
            if cache.sequences[name].length + len(tokens) <= 200 and cache.fits([(e.request_id, len(e.tokens)) for e in entries] + [(name, len(tokens))]):
                entries.append(StepEntry(name, tokens, rng.choice(([], [len(tokens) - 1], list(range(len(tokens)))))))
        if entries:
            reservations = [cache.reserve(entry.request_id, len(entry.tokens)) for entry in entries]
            same_steps(build_step_batch(reservations, entries, cache, library.device, library), build_step_batch(reservations, entries, cache, library.device))
        for name in list(live):
            if rng.random() < 0.1 or cache.sequences[name].length > 190:
                cache.free(name)
                live.remove(name)


def test_launched_steps_take_the_arrays_made_on_the_device(library):
    from llmserve_amd import ModelRunner
    from llmserve_amd.weights import random_model

    calls, kept = [], library.place_tokens
    runner = ModelRunner(random_model(TINY_B, 0, dtype=torch.bfloat16, device=library.device), library, CacheConfig(block_size=8, num_blocks=40, max_sequences=4))
    library.place_tokens = lambda *arguments: calls.append(arguments[5]) or kept(*arguments)
    try:
        logits = runner.step([StepEntry("a", list(range(30)), [29]), StepEntry("b", [7, 8], [0, 1])], create_missing=True)
    finally:
        del library.place_tokens
    assert calls == [32] and logits.shape == (3, TINY_B.vocab_size)
    runner.close()
