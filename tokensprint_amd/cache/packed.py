"""Keys and values held in 4 bits: sizes of their pages.

Up to 64 neighbouring elements of a head of one token are a group: a step in float16 (a
fifteenth of the way from the group's smallest element, or zero, to its largest, or zero), a
whole zero and a code of 4 bits an element, value = step * (code - zero); 4.5 bits an element
of a head of 128.  A page of P tokens keeps, per key/value head, P / 16 blocks of 16 tokens, keys
and values apart; inside, the bytes lie as the attention kernels read them (csrc/packed_kv.h).
What a cache holds is read back with the provider's `kv_values`.
"""

from __future__ import annotations

from functools import lru_cache

import torch

TOKENS = 16             # tokens of a block
GROUP = 64              # elements of a group


def packed_block_bytes(head_dim: int) -> int:
    """Bytes of 16 tokens' keys (or values) of one head."""
    groups = 1 if head_dim <= 64 else 2 if head_dim <= 128 else 4
    return 256 * (-(-head_dim // 32)) + 64 * groups


def check_packed(head_dim: int, page_size: int) -> None:
    """Raises ValueError where a cache of 4 bits is not built for these sizes."""
    if not 16 <= head_dim <= 256 or head_dim % 16:
        raise ValueError(f"keys and values in 4 bits: head size {head_dim} is no multiple of 16 "
                         "from 16 to 256")
    if page_size < TOKENS or page_size & (page_size - 1):
        raise ValueError(f"keys and values in 4 bits: page size {page_size} is no power of two "
                         f"from {TOKENS}")


@lru_cache(maxsize=1024)
def packed_pages_shape(num_pages: int, num_kv_heads: int, page_size: int,
                       head_dim: int) -> tuple[int, int, int, int]:
    """Shape of the uint8 tensor that holds keys, and of the one that holds values."""
    check_packed(head_dim, page_size)
    return num_pages, num_kv_heads, page_size // TOKENS, packed_block_bytes(head_dim)


def packed_cache(num_pages: int, num_kv_heads: int, page_size: int, head_dim: int, device):
    """An empty cache of 4 bits for one run, as a mixer sees it (a LayerCache of group 0)."""
    from tokensprint_amd.cache.storage import LayerCache
    if num_pages < 1 or num_kv_heads < 1:
        raise ValueError(f"a cache of {num_pages} pages and {num_kv_heads} key/value heads")
    shape = packed_pages_shape(num_pages, num_kv_heads, page_size, head_dim)
    return LayerCache(0, page_size, num_pages, torch.zeros(shape, dtype=torch.uint8, device=device),
                      torch.zeros(shape, dtype=torch.uint8, device=device))
