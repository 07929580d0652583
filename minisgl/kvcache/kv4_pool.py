"""Paged K/V storage in 4 bits for multi-head (GQA) attention.

One byte tensor [2, layers, pages, local_kv_heads, block bytes]: a (page, head)
block holds its codes and then its scales (``minisgl.quant.kv4`` states the
format), so a page of one head is still one contiguous copy. 136 bytes per
token and head for 128-dim K and V heads, against 512 for the bf16 pool: 3.76
times the tokens in the same memory. The reference's pools are 16-bit only
(python/minisgl/kvcache/mha_pool.py:25-35).
"""

from __future__ import annotations

from typing import Sequence

import torch

from minisgl import ops
from minisgl.parallel import get_tp_info
from minisgl.quant.kv4 import kv4_block_bytes, kv4_check
from minisgl.utils import div_even

from .base import BaseKVCachePool


class MHAKV4Cache(BaseKVCachePool):
    """``dtype`` is the type of the rows that go in and come out (bf16 on a
    GPU, any float type on the CPU). The pool starts as zeros, which are
    finite values, so positions past the end of a sequence never are not."""

    def __init__(self, num_kv_heads: int, num_layers: int, head_dim: int, num_pages: int, page_size: int,
                 dtype: torch.dtype, device: torch.device) -> None:
        kv4_check(page_size, head_dim)
        local = div_even(num_kv_heads, get_tp_info().size, allow_replicate=True)
        self.local_kv_heads = local
        self.head_dim = head_dim
        self.page_size = page_size
        self.num_pages = num_pages
        self._num_layers = num_layers
        self._device = torch.device(device)
        self._dtype = dtype
        self.pool = torch.zeros((2, num_layers, num_pages, local, kv4_block_bytes(page_size, head_dim)),
                                dtype=torch.uint8, device=device)

    def k_cache(self, layer: int) -> torch.Tensor:
        return self.pool[0, layer]

    def v_cache(self, layer: int) -> torch.Tensor:
        return self.pool[1, layer]

    def store_kv(self, k: torch.Tensor, v: torch.Tensor, out_loc: torch.Tensor, layer: int) -> None:
        """Rows of k and v [T, heads * head_dim] or [T, heads, head_dim] as they are (no norm, no rotation)."""
        ops.store_kv4(k.flatten(1), v.flatten(1), self.pool, layer, out_loc, self.local_kv_heads,
                      self.head_dim, self.page_size)

    def load_kv(self, slots: torch.Tensor, layer: int):
        """The rows of ``slots`` as (k, v) [T, heads, head_dim]."""
        return ops.load_kv4(self.pool, layer, slots, self.local_kv_heads, self.head_dim, self.page_size,
                            dtype=self._dtype)

    def copy_pages(self, src: Sequence[int], dst: Sequence[int]) -> None:
        ops.copy_pages(self.pool, src, dst)

    @property
    def device(self) -> torch.device:
        return self._device

    @property
    def dtype(self) -> torch.dtype:
        return self._dtype

    @property
    def num_layers(self) -> int:
        return self._num_layers

    @staticmethod
    def bytes_per_page(num_kv_heads: int, num_layers: int, head_dim: int, page_size: int, dtype: torch.dtype) -> int:
        local = div_even(num_kv_heads, get_tp_info().size, allow_replicate=True)
        return 2 * num_layers * local * kv4_block_bytes(page_size, head_dim)
