"""Sizes and refusals of a cache of 4 bits, without a GPU."""

import pytest
import torch

from tokensprint_amd.cache import CacheStorage, group_runs, packed_cache, page_bytes
from tokensprint_amd.cache.packed import packed_block_bytes
from tokensprint_amd.config import Config
from tokensprint_amd.parts.base import PagedKVNeed, PagedLatentNeed, SlotStateNeed

NEEDS = [PagedKVNeed(8, 128), PagedKVNeed(2, 48, 64), PagedLatentNeed(40), SlotStateNeed((3,)), PagedKVNeed(8, 128)]


def test_pages_of_4_bits_beside_other_caches():
    packed = CacheStorage(NEEDS, 32, 6, 2, torch.bfloat16, "cpu", kv_bits=4)
    wide = CacheStorage(NEEDS, 32, 6, 2, torch.bfloat16, "cpu")
    assert packed.views[0].k_pages.dtype == torch.uint8
    assert packed.views[0].k_pages.shape == (6, 8, 2, packed_block_bytes(128)) == packed.views[4].v_pages.shape
    assert packed.views[1].v_pages.shape == (6, 2, 2, packed_block_bytes(48))
    # latent vectors and states as ever
    assert packed.views[2].k_pages.shape == wide.views[2].k_pages.shape
    assert packed.views[2].k_pages.dtype == torch.bfloat16 and packed.views[2].v_pages is None
    assert packed.views[3].state.shape == wide.views[3].state.shape
    held = sum(t.numel() * t.element_size() for t in packed.k_tensors + packed.v_tensors if t is not None)
    groups, _ = group_runs(NEEDS)
    assert held == 6 * page_bytes(groups, 32, torch.bfloat16, 4)
    assert page_bytes(groups, 32, torch.bfloat16) == page_bytes(groups, 32, torch.bfloat16, None)


def test_bytes_of_a_block():
    # codes of 16 tokens, and four bytes a token and group of 64 elements
    assert packed_block_bytes(128) == 16 * (64 + 2 * 4)
    assert packed_block_bytes(64) == 16 * (32 + 4)
    assert packed_block_bytes(256) == 16 * (128 + 4 * 4)


@pytest.mark.parametrize("page,hd", [(8, 64), (24, 64), (1, 64), (16, 24), (16, 8), (16, 272)])
def test_sizes_that_are_not_built(page, hd):
    with pytest.raises(ValueError, match="4 bits"):
        packed_cache(4, 2, page, hd, "cpu")
    with pytest.raises(ValueError, match="4 bits"):
        CacheStorage([PagedKVNeed(2, hd)], page, 4, 1, torch.bfloat16, "cpu", kv_bits=4)


def test_refusals(tmp_path):
    with pytest.raises(ValueError):
        packed_cache(0, 2, 16, 64, "cpu")
    with pytest.raises(ValueError):
        CacheStorage(NEEDS, 32, 6, 2, torch.bfloat16, "cpu", kv_bits=8)
    with pytest.raises(ValueError, match="kv_bits"):
        Config(model=str(tmp_path), kv_bits=3)
    with pytest.raises(ValueError, match="power of two"):
        Config(model=str(tmp_path), kv_bits=4, kvcache_block_size=24)
    assert Config(model=str(tmp_path), kv_bits=4, kvcache_block_size=64).kv_bits == 4
