"""Layout of the paged 8-bit K/V cache (what the ``kv8_*`` ops read and write).

``num_pages`` pages of ``page_size`` tokens (a multiple of 16, at most 256), each
with ``kv_heads`` heads of ``head_dim`` values (a multiple of 32, at most 256), one
byte a value (``torch.float8_e4m3fn`` or ``torch.int8``):

* ``k_cache [num_pages, kv_heads, page_size, head_dim]``;
* ``v_cache [num_pages, kv_heads, page_size // 16, head_dim, 16]``: transposed in
  groups of 16 tokens, because the attention multiplies V from the left as V^T
  and so wants consecutive tokens of one dimension;
* ``k_scale``, ``v_scale`` fp32 ``[num_pages, kv_heads]``: a value is its byte
  times the scale of its page and head.

``block_table[b, j]`` (int32) is the page of sequence b's tokens
``[j * page_size, (j + 1) * page_size)``.  Scales are powers of two: dividing by
one is exact, so a stored byte is the one rounding of the value, and a page
whose scale grows when tokens are appended is moved to it by an exact shift
(e4m3 loses only what falls below its smallest values).  It costs int8 up to one
bit of its range, e4m3 nothing but that.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

TOKEN_GROUP = 16
MAX_PAGE_SIZE = 256
MAX_HEAD_DIM = 256
LEAST_SCALE = 2.0 ** -120
LARGEST = {torch.float8_e4m3fn: 448.0, torch.int8: 127.0}


class Kv8Cache(NamedTuple):
    """The four tensors of a cache, in the order the ops take them:
    ``native.kv8_decode_forward(q, *cache, block_table, lengths)``."""

    k_cache: torch.Tensor
    v_cache: torch.Tensor
    k_scale: torch.Tensor
    v_scale: torch.Tensor


def empty_cache(num_pages: int, kv_heads: int, page_size: int, head_dim: int, *,
                dtype: torch.dtype = torch.float8_e4m3fn, device="cuda") -> Kv8Cache:
    """A zero-filled cache, its scales those that the write gives a page of zeros."""
    if dtype not in LARGEST:
        raise ValueError("dtype must be float8_e4m3fn or int8")
    if not 0 < page_size <= MAX_PAGE_SIZE or page_size % TOKEN_GROUP:
        raise ValueError("page_size must be a multiple of 16, at most 256")
    if not 0 < head_dim <= MAX_HEAD_DIM or head_dim % 32:
        raise ValueError("head_dim must be a multiple of 32, at most 256")
    n = num_pages * kv_heads * page_size * head_dim
    k, v = (torch.zeros(n, dtype=torch.uint8, device=device).view(dtype) for _ in range(2))
    scale = torch.full((num_pages, kv_heads), LEAST_SCALE, dtype=torch.float32, device=device)
    return Kv8Cache(k.view(num_pages, kv_heads, page_size, head_dim),
                    v.view(num_pages, kv_heads, page_size // TOKEN_GROUP, head_dim, TOKEN_GROUP), scale, scale.clone())


def num_blocks(tokens: int, page_size: int) -> int:
    """Pages that ``tokens`` tokens of one sequence take."""
    return -(-tokens // page_size)
