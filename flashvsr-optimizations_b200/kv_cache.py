"""Paged FP8 store of attention keys and values.

:class:`FP8KVCache` keeps E4M3 codes with one fp32 scale per token and head, in pages that a
caller's page table strings into sequences: half the memory of a bf16 cache (0.52 of it at heads
of 128).  Rows are quantized as they are written and read back in bf16, for attention that takes
bf16 operands -- a streaming block that appends a chunk of tokens and attends over its window.
The reference's attention backends are outside this library; the store is what a W8A8 block adds
next to its quantized linears.
"""
from __future__ import annotations

import torch

from . import ops

__all__ = ["FP8KVCache"]


class FP8KVCache:
    """``num_pages`` pages of ``page_size`` slots; a slot holds one token's keys and values.

    k_codes, v_codes: float8_e4m3fn [num_pages, page_size, heads, head_dim]; k_scale, v_scale:
    fp32 [num_pages, page_size, heads].  head_dim a multiple of 8 up to 512.  The buffers are
    plain tensors (save, share or replace them); the object keeps nothing else.
    """

    def __init__(self, num_pages: int, page_size: int, heads: int, head_dim: int,
                 device: torch.device | str = "cuda"):
        if min(num_pages, page_size, heads, head_dim) <= 0 or head_dim % 8 or head_dim > 512:
            raise ValueError("FP8KVCache: sizes must be positive, head_dim a multiple of 8 up to 512")
        if torch.device(device).type != "cuda":
            raise RuntimeError("FP8KVCache: the store lives on a CUDA device (there is no CPU path)")
        shape = (num_pages, page_size, heads)
        self.k_codes = torch.zeros((*shape, head_dim), dtype=torch.float8_e4m3fn, device=device)
        self.v_codes = torch.zeros_like(self.k_codes)
        self.k_scale = torch.zeros(shape, dtype=torch.float32, device=device)
        self.v_scale = torch.zeros_like(self.k_scale)

    def write(self, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
        """Store bf16 k, v [tokens, heads, head_dim] at ``slots`` (int64 [tokens], negative: not
        stored); see ``ops.fp8_cache_write``."""
        ops.fp8_cache_write(k, v, slots, self.k_codes, self.k_scale, self.v_codes, self.v_scale)

    def read(self, page_table: torch.Tensor, lengths: torch.Tensor,
             max_len: int) -> tuple[torch.Tensor, torch.Tensor]:
        """(k, v) bf16 [batch, max_len, heads, head_dim], zero from each length on; see
        ``ops.fp8_cache_read``."""
        return ops.fp8_cache_read(self.k_codes, self.k_scale, self.v_codes, self.v_scale, page_table,
                                  lengths, max_len)

    def slots(self, page_table: torch.Tensor, positions: torch.Tensor) -> torch.Tensor:
        """The slots (int64, [batch * tokens]) of ``positions`` (integers [batch, tokens]; negative:
        padding, and so is its slot) of the sequences of ``page_table`` [batch, pages].  A position
        past the table, or on a page outside the store, gets a slot past the store, which ``write``
        reports."""
        pages, page = self.k_codes.shape[:2]
        if page_table.dim() != 2 or positions.dim() != 2 or positions.shape[0] != page_table.shape[0] or \
                any(t.dtype.is_floating_point or t.dtype == torch.bool for t in (page_table, positions)):
            raise ValueError("FP8KVCache.slots: expected integers, page_table [batch, pages] and positions "
                             f"[batch, tokens], got {tuple(page_table.shape)} and {tuple(positions.shape)}")
        at = positions.long()
        if page_table.shape[1] == 0:  # no entry to gather
            return torch.where(at < 0, -1, pages * page).reshape(-1)
        index = page_table.long().gather(1, (at.clamp_min(0) // page).clamp_max(page_table.shape[1] - 1))
        there = (at < page_table.shape[1] * page) & (index >= 0)
        slot = torch.where(there, index * page + at % page, pages * page)
        return torch.where(at < 0, -1, slot).reshape(-1)
