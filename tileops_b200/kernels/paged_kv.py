"""sm_100a kernel classes around a paged KV cache: the plan of a step (block tables and slot maps), the per-head norm and
rotation with the append, and the cache held in 4 bits with its append, read-back, decode and prefill (L1 of the operator
stack).

None of them has a counterpart in the reference, whose paged operators take finished block tables, rotate without the
norm and keep their caches in 16 or 8 bits (``src/tileops/ops/attention/gqa.py:765-1454``); the decode and prefill classes
stand beside :class:`GQADecodePagedFp8Sm100Kernel` and :class:`GQAPrefillPagedFp8CacheSm100Kernel`.
"""

from __future__ import annotations

from typing import Optional

import torch

from .. import functional as F
from .call_spec import ATTENTION_DTYPES
from .kernel_base import Kernel

__all__ = ["PagedKVPlanSm100Kernel", "PagedKVReleaseSm100Kernel", "QKNormRopeSm100Kernel", "Int4KVCacheAppendSm100Kernel",
           "Int4KVCacheGatherSm100Kernel", "GQADecodePagedInt4Sm100Kernel", "GQAPrefillPagedInt4CacheSm100Kernel"]

_INT4_DIMS = (64, 128)


def _check_int4(name: str, dim: int, page_size: int) -> None:
    if dim not in _INT4_DIMS:
        raise ValueError(f"{name} supports head dims {_INT4_DIMS}, got {dim}")
    if page_size <= 0 or page_size % 16 != 0:
        raise ValueError(f"{name} supports pages of a multiple of 16 tokens, got {page_size}")


class PagedKVPlanSm100Kernel(Kernel):
    supported_archs = [100]
    general = True

    def __init__(self, page_size, config: Optional[dict] = None, device_index=None) -> None:
        super().__init__(device_index=device_index)
        self.page_size = page_size
        self.init_config(config)

    def forward(self, seq_lens, new_lens, block_table, free_pages, free_count, total_tokens, inplace=False):
        return F.paged_kv_plan(seq_lens, new_lens, block_table, free_pages, free_count, total_tokens,
                               page_size=self.page_size, inplace=inplace)


class PagedKVReleaseSm100Kernel(PagedKVPlanSm100Kernel):
    def forward(self, finished, seq_lens, block_table, free_pages, free_count):
        F.paged_kv_release(finished, seq_lens, block_table, free_pages, free_count, page_size=self.page_size)


class QKNormRopeSm100Kernel(Kernel):
    """One launch: norm, rotation and, with a cache, the append."""

    supported_archs = [100]
    general = True

    def __init__(self, dim, eps, page_size=0, config: Optional[dict] = None, device_index=None) -> None:
        super().__init__(device_index=device_index)
        if dim <= 0 or dim % 8 != 0 or dim > 256:
            raise ValueError(f"{type(self).__name__} supports head dims that are multiples of 8 up to 256, got {dim}")
        self.dim, self.eps, self.page_size = dim, eps, page_size
        self.init_config(config)

    @property
    def default_config(self) -> dict:
        return {"threads": 128}

    def forward(self, q, k, positions, inv_turns, q_weight, k_weight, v=None, slot_mapping=None, k_pages=None,
                v_pages=None, kv_pages=None, return_k=True):
        return F.qk_norm_rope(q, k, positions, inv_turns, q_weight=q_weight, k_weight=k_weight, eps=self.eps, v=v,
                              slot_mapping=slot_mapping, k_pages=k_pages, v_pages=v_pages, kv_pages=kv_pages,
                              page_size=self.page_size, return_k=return_k)


class _Int4CacheBase(Kernel):
    supported_archs = [100]
    general = True

    def __init__(self, dim, page_size, dtype=None, config: Optional[dict] = None, device_index=None) -> None:
        super().__init__(device_index=device_index)
        _check_int4(type(self).__name__, dim, page_size)
        self.dim, self.page_size, self.dtype = dim, page_size, dtype
        self.init_config(config)

    @property
    def default_config(self) -> dict:
        return {"threads": 128}


class Int4KVCacheAppendSm100Kernel(_Int4CacheBase):
    def forward(self, k, v, slot_mapping, kv_pages):
        F.int4_cache_append(k, v, slot_mapping, kv_pages, page_size=self.page_size)


class Int4KVCacheGatherSm100Kernel(_Int4CacheBase):
    @property
    def default_config(self) -> dict:
        return {"threads": 288}

    def forward(self, kv_pages, block_table, cu_seqlens_kv, total_tokens):
        return F.int4_cache_gather(kv_pages, block_table, cu_seqlens_kv, total_tokens, dim=self.dim,
                                   page_size=self.page_size, dtype=self.dtype)


class GQADecodePagedInt4Sm100Kernel(Kernel):
    """Paged decode over a 4-bit cache: ``forward(Q[B,H,D], kv_pages, real_seqlen_kv[B] i32, block_table[B,W] i32)``.
    Constructor as :class:`GQADecodePagedFp8Sm100Kernel`.  ``config`` may set ``chunk_tiles`` (a fixed run length) and
    ``wait_log2`` (the limit of a device-side wait in clock ticks); ``threads`` describes the kernel."""

    supported_archs = [100]
    general = True

    @classmethod
    def applies(cls, call) -> bool:
        return call.dim in _INT4_DIMS and call.dtype in ATTENTION_DTYPES and call.page_size % 16 == 0

    def __init__(self, batch, heads, heads_kv, seqlen_kv, dim, page_size, dtype, sm_scale=None, softcap=0.0,
                 config: Optional[dict] = None, tune: bool = False, device_index=None) -> None:
        super().__init__(device_index=device_index)
        if heads % heads_kv != 0:
            raise ValueError("heads must be divisible by heads_kv")
        _check_int4(type(self).__name__, dim, page_size)
        if seqlen_kv % page_size != 0:
            raise ValueError(f"seqlen_kv={seqlen_kv} must be a multiple of page_size={page_size}")
        self.batch, self.heads, self.heads_kv = batch, heads, heads_kv
        self.seqlen_kv, self.dim, self.page_size, self.dtype = seqlen_kv, dim, page_size, dtype
        self.sm_scale = dim ** -0.5 if sm_scale is None else sm_scale
        self.softcap = 0.0 if softcap is None else softcap
        self.tune = tune
        self.init_config(config, tune)

    @property
    def default_config(self) -> dict:
        return {"threads": 160}

    def forward(self, Q, kv_pages, real_seqlen_kv, block_table, return_lse: bool = False, out_dtype=None):
        return F.gqa_decode_int4(Q, kv_pages, real_seqlen_kv, block_table, page_size=self.page_size,
                                 sm_scale=self.sm_scale, softcap=self.softcap, return_lse=return_lse, out_dtype=out_dtype,
                                 config=self.config)


class GQAPrefillPagedInt4CacheSm100Kernel(Kernel):
    """Paged prefill over a 4-bit cache: the cached tokens are read back into a packed 16-bit K/V
    (``tb200_int4_cache_gather``), the packed tcgen05 prefill runs on it, and the chunk is quantised into the pages
    (``tb200_int4_cache_append``), as :class:`GQAPrefillPagedFp8CacheSm100Kernel` does for an e4m3 cache."""

    supported_archs = [100]
    general = True

    @classmethod
    def applies(cls, call) -> bool:
        return call.dim in _INT4_DIMS and call.dtype in ATTENTION_DTYPES and call.page_size % 16 == 0

    def __init__(self, batch, heads, heads_kv, max_pages_per_req, page_size, dim, is_causal, dtype, sm_scale=None,
                 softcap=0.0, config: Optional[dict] = None, tune: bool = False, device_index=None) -> None:
        super().__init__(device_index=device_index)
        _check_int4(type(self).__name__, dim, page_size)
        self.batch, self.heads, self.heads_kv, self.dim = batch, heads, heads_kv, dim
        self.max_pages_per_req, self.page_size = max_pages_per_req, page_size
        self.is_causal, self.dtype = is_causal, dtype
        self.sm_scale = dim ** -0.5 if sm_scale is None else sm_scale
        self.softcap = 0.0 if softcap is None else softcap
        self.tune = tune
        self.init_config(config, tune)

    @property
    def default_config(self) -> dict:
        """Of the prefill kernel, as its siblings' (fixed)."""
        return {"block_M": 128, "block_N": 64, "threads": 192}

    def forward(self, q, k_new, v_new, kv_pages, cu_seqlens_q, cache_seqlens, block_table, max_seqlen_q):
        return F.gqa_prefill_paged_int4_cache(q, k_new, v_new, kv_pages, cu_seqlens_q, cache_seqlens, block_table,
                                              int(max_seqlen_q), page_size=self.page_size, is_causal=self.is_causal,
                                              sm_scale=self.sm_scale, softcap=self.softcap)
