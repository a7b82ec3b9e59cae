"""A paged KV cache of one layer, held in 8 bits (no counterpart in the reference, which runs every
sequence from its first token).

``KV8Cache`` owns the tensors of the layout that ``include/mes_b200.h`` describes for ``mes_kv8_*``:
codes ``[pages, 2, Hkv, P, 128]`` (int8 or e4m3), one fp32 scale for each page, side (K or V) and kv
head, and, where eviction is wanted, the accumulated attention weight of every cached token.
``CacheStep`` names the tokens that one call adds or attends with: which pages each sequence has,
the offsets of its new tokens in the packed rows and how many tokens it has cached with them.
"""
from __future__ import annotations

import dataclasses

import torch

from .. import _C


@dataclasses.dataclass
class CacheStep:
    """New tokens of ``B`` sequences: ``block_table`` int32 ``[B, width]``, ``cu_new`` int32
    ``[B + 1]``, ``context_lens`` int32 ``[B]`` (the new tokens included), ``max_new`` an upper bound
    on the new tokens of one sequence."""
    block_table: torch.Tensor
    cu_new: torch.Tensor
    context_lens: torch.Tensor
    max_new: int


class KV8Cache:

    def __init__(self, num_pages: int, page_size: int, num_kv_heads: int,
                 dtype: torch.dtype = torch.int8, device: torch.device | str = "cuda",
                 track_weights: bool = False) -> None:
        if dtype not in _C.KV8_DTYPES:
            raise ValueError(f"a KV8Cache holds int8 or float8_e4m3fn, not {dtype}")
        if page_size not in _C.KV8_PAGE_SIZES:
            raise ValueError(f"the page size is one of {_C.KV8_PAGE_SIZES}, not {page_size}")
        shape = (num_pages, 2, num_kv_heads, page_size, 128)
        self.codes = torch.zeros(shape, dtype=torch.int8, device=device).view(dtype)
        self.scales = torch.zeros(shape[:3], dtype=torch.float32, device=device)
        self.sums = (torch.zeros(num_pages, num_kv_heads, page_size, dtype=torch.float32, device=device)
                     if track_weights else None)

    @property
    def page_size(self) -> int:
        return self.codes.shape[3]

    def append(self, k: torch.Tensor, v: torch.Tensor, step: CacheStep) -> None:
        """Quantise the new tokens' ``k`` / ``v`` (bf16 rows ``[T, Hkv * 128]``) into their pages."""
        _C.kv8_append(k, v, self.codes, self.scales, step.block_table, step.cu_new, step.context_lens,
                      step.max_new, self.sums)

    def attend(self, q: torch.Tensor, step: CacheStep, num_heads: int, scale: float,
               track: bool = True) -> torch.Tensor:
        """Causal attention of the new tokens' ``q`` (bf16 rows ``[T, num_heads * 128]``) over the
        cache, which holds their keys and values already; with ``track`` their weights are added
        to the cached tokens' sums (where the cache has them)."""
        return _C.kv8_attention(q, self.codes, self.scales, step.block_table, step.cu_new,
                                step.context_lens, num_heads, scale, step.max_new,
                                sums=self.sums if track else None)

    def evict(self, step: CacheStep, new_table: torch.Tensor, keep: int, recent: int):
        """Keep ``keep`` tokens of every sequence, the ``recent`` last ones among them, in the pages of
        ``new_table``; returns ``(kept, new_lens)`` (see ``_C.kv8_evict``)."""
        if self.sums is None:
            raise ValueError("eviction goes by the attention weights: make the cache with track_weights=True")
        return _C.kv8_evict(self.codes, self.scales, self.sums, step.block_table, step.context_lens,
                            new_table, keep, recent)

    def read(self, pages: torch.Tensor) -> torch.Tensor:
        """The values of ``pages`` (int32 ``[n]``), bf16 ``[n, 2, Hkv, P, 128]``."""
        return _C.kv8_read(self.codes, self.scales, pages)
