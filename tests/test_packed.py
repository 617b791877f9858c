"""Caches in 4 bits without a GPU: the pages' layout and what they stand for, which needs have the form, the cache's sizes and read path, the options that ask for it."""

from __future__ import annotations

import itertools

import pytest
import torch

from llmserve_amd import CacheConfig
from llmserve_amd.cache import CacheManager
from llmserve_amd.parts import PackedKeyValue, PagedKeyValue
from llmserve_amd.registry import ARCHITECTURES
from tests import dafutar_cases, dolezen_cases, dubesun_cases, katenex_cases, sozavik_cases, vagozen_cases
from tests.packed_cases import kept
from tests.tiny import TINY_A, TINY_B

NUMBERS = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def spec_of(config, architecture="Qwen2ForCausalLM"):
    return ARCHITECTURES[architecture].build_spec(config)


def page_bytes_of(keys: torch.Tensor, values: torch.Tensor) -> torch.Tensor:
    """[kv_heads, bytes] of a page with what `kept` leaves of keys and values [page, kv_heads, D] (every block of it with a largest element of 4 or 6 units), written
    byte by byte from the layout's description."""
    page, kv_heads, dim = keys.shape
    data = torch.zeros((kv_heads, page * (dim + dim // 16)), dtype=torch.uint8)
    value_codes, key_powers = page * dim // 2, page * dim
    value_powers = key_powers + page * dim // 32
    for which, rows in enumerate((keys, values)):
        for token, head, block in itertools.product(range(page), range(kv_heads), range(dim // 32)):
            elements = rows[token, head, block * 32 : block * 32 + 32].double()
            number = bool(torch.isfinite(elements).all())
            exponent = int(torch.frexp(elements.abs().max())[1]) - 3 if number and elements.abs().max() > 0 else -125
            power = exponent + 127 if number else 255
            at = key_powers + token * (dim // 32) + block if which == 0 else value_powers + (token // 8 * (dim // 32) + block) * 8 + token % 8
            data[head, at] = power
            for i, element in enumerate(elements.tolist()):
                code = (NUMBERS.index(abs(element) / 2.0 ** exponent) | (8 if str(element)[0] == "-" else 0)) if number else 0
                column = block * 32 + i
                byte = token * (dim // 2) + column // 2 if which == 0 else value_codes + ((token // 8 * (dim // 8) + column // 8) * 8 + token % 8) * 4 + column % 8 // 2
                data[head, byte] |= code << (column % 2 * 4)
    return data


@pytest.mark.parametrize("page,kv_heads,dim", [(8, 1, 32), (16, 2, 64), (24, 1, 96)])
def test_a_page_stands_for_what_is_kept(page, kv_heads, dim):
    generator = torch.Generator().manual_seed(dim)
    both = torch.randn((2, page, kv_heads, dim), generator=generator) * torch.exp(3 * torch.randn((2, page, kv_heads, 1), generator=generator))
    both[0, 3, 0, 5] = float("inf")
    both[1, 2, 0, :32] = 0.0
    both[1, 5, 0, :32] = torch.tensor([0.0, -0.0] * 16)
    want = kept(both)
    need = PackedKeyValue(kv_heads, dim)
    data = page_bytes_of(want[0], want[1])
    assert data.shape == (kv_heads, need.page_bytes(page)) == need.page_fields(page)["packed"]
    rows = need.token_rows({"packed": data}, page)
    for name, expected in (("keys", want[0]), ("values", want[1])):
        assert rows[name].dtype == torch.float32 and torch.equal(rows[name].isnan(), expected.isnan())
        assert torch.equal(rows[name].nan_to_num(0.0), expected.nan_to_num(0.0).float())


@pytest.mark.parametrize("dim", [0, 16, 48, 100, 288])
def test_heads_without_the_form(dim):
    with pytest.raises(ValueError, match="heads of 32 to 256"):
        PackedKeyValue(2, dim)


@pytest.mark.parametrize("page", [0, 1, 4, 12, -8])
def test_pages_without_the_form(page):
    with pytest.raises(ValueError, match="multiple of 8"):
        PackedKeyValue(2, 64).page_bytes(page)
    with pytest.raises(ValueError, match="multiple of 8"):
        PagedKeyValue(2, 64, packable=True).packed(page)


def test_needs_that_have_the_form():
    assert PagedKeyValue(2, 64, 100, packable=True).packed(16) == PackedKeyValue(2, 64, 100)
    for need in (PagedKeyValue(2, 64), PagedKeyValue(2, 64, keep_first=4, window=9, packable=True), PagedKeyValue(2, 64, chunk=32, packable=True)):
        with pytest.raises(ValueError, match="no form in 4 bits"):
            need.packed(16)
    # being able to is no difference between needs, and a cell that two share has to be for both
    assert PagedKeyValue(2, 64, packable=True) == PagedKeyValue(2, 64)
    for one, other in itertools.product((True, False), repeat=2):
        for window in (None, 7):
            assert PagedKeyValue(2, 64, packable=one).shared_with(PagedKeyValue(2, 64, window, packable=other)).packable is (one and other)


def test_packed_needs_shared():
    one = PackedKeyValue(2, 64, 9)
    assert one.shared_with(PackedKeyValue(2, 64, 30)) == PackedKeyValue(2, 64, 30)
    assert one.shared_with(PackedKeyValue(2, 64)) == PackedKeyValue(2, 64)
    for other in (PackedKeyValue(1, 64, 9), PackedKeyValue(2, 96, 9), PagedKeyValue(2, 64, 9)):
        assert one.shared_with(other) is None


def test_a_cache_in_4_bits():
    make = lambda packed, dtype: CacheManager(spec_of(TINY_B), CacheConfig(8, 12, 3, packed), max_sequence_length=64, dtype=dtype)
    plain, cache = make(False, torch.bfloat16), make(True, torch.bfloat16)
    assert len(cache.groups) == len(plain.groups) and not CacheConfig(8, 12, 3).packed
    size = lambda manager: sum(field.numel() * field.element_size() for group in manager.groups for field in group.storage.values())
    assert size(cache) * 64 == size(plain) * 17 and size(make(True, torch.float32)) == size(cache)
    for mine, theirs in zip(cache.groups, plain.groups):
        assert mine.need.window == theirs.need.window and mine.cells == theirs.cells
        assert set(mine.storage) == {"packed"} and mine.storage["packed"].dtype == torch.uint8
    cell = cache.cells()[0]
    cell = cell if not isinstance(cell, dict) else next(iter(cell.values()))
    assert cell.packed.shape == (12, TINY_B.num_key_value_heads, 8 * (32 + 2)) and cell.keys is None and cell.values is None


def test_reading_a_cache_in_4_bits():
    cache = CacheManager(spec_of(TINY_B), CacheConfig(8, 12, 3, True), max_sequence_length=64, dtype=torch.bfloat16)
    run = next(index for index, cell in enumerate(cache.cells()) if cell is not None)
    cache.create("empty")
    cache.create("a")
    first, keys, values = cache.gather("empty", run)
    assert (first, keys.shape, values.dtype) == (0, (0, 1, 32), torch.float32)
    cache.reserve("a", 11)
    group, _, index = cache._paged_cell(run)
    want = kept(torch.randn((2, 16, 1, 32), generator=torch.Generator().manual_seed(4)))
    for block, page in enumerate(cache.block_table("a")):
        group.storage["packed"][index, page] = page_bytes_of(want[0, block * 8 : block * 8 + 8], want[1, block * 8 : block * 8 + 8])
    first, keys, values = cache.gather("a", run)
    assert first == 0 and torch.equal(keys, want[0, :11].float()) and torch.equal(values, want[1, :11].float())


def test_models_without_the_form():
    with pytest.raises(ValueError, match="heads of 32 to 256"):
        CacheManager(spec_of(TINY_A), CacheConfig(16, 8, 2, True), max_sequence_length=64)  # heads of 16
    with pytest.raises(ValueError, match="multiple of 8"):
        CacheManager(spec_of(TINY_B), CacheConfig(4, 8, 2, True), max_sequence_length=64)
    for name, cases in (("Dafutar", dafutar_cases), ("Dolezen", dolezen_cases), ("Dubesun", dubesun_cases), ("Katenex", katenex_cases), ("Sozavik", sozavik_cases), ("Vagozen", vagozen_cases)):
        architecture = ARCHITECTURES[name]
        spec = architecture.build_spec(architecture.config_class.from_dict(cases.MIXED))
        with pytest.raises(ValueError, match="no form in 4 bits"):
            CacheManager(spec, CacheConfig(8, 8, 2, True), max_sequence_length=64)


def test_the_option(monkeypatch):
    """--packed-cache reaches the cache's configuration."""
    from llmserve_amd import cli, engine

    taken = {}
    monkeypatch.setattr(engine, "LLMEngine", lambda loaded, tokenizer, **options: taken.update(options))
    for command in ("generate", "benchmark"):
        for words, packed in (([], False), (["--packed-cache"], True)):
            cli._engine(cli.build_parser().parse_args([command, *words]), None, None, batch_size=2, mode="continuous")
            assert taken["cache_config"].packed is packed
