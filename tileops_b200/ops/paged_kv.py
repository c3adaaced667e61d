"""Operators around a paged KV cache (L2): the plan of a serving step, the norm and rotation of q and k with the append,
and the 4-bit cache's append and read-back.  The attention over the 4-bit cache stands with its siblings in
:mod:`tileops_b200.ops.gqa`.

They are additions: the reference's paged operators (``src/tileops/ops/attention/gqa.py:765-1454``) take finished block
tables and rotated keys.  A decode step is

    plan = PagedKVCachePlanFwdOp(...)(seq_lens, new_lens, block_table, free_pages, free_count, total_tokens)
    q = QKNormRopeInt4KVCacheAppendFwdOp(...)(q, k, v, q_weight, k_weight, plan.positions, plan.slot_mapping, kv_pages)
    o = GroupedQueryAttentionDecodePagedInt4KVCacheFwdOp(...)(q, kv_pages, plan.seq_lens, block_table)

No call synchronises the host with the device, and each can be captured into a CUDA graph; an operator that rotates has to
have been called on the device once before, since its first call copies the frequencies there.
"""

from __future__ import annotations

import math
from typing import Dict, Optional

import torch

from .. import functional
from ..functional import PagedKVPlan, int4_page_bytes
from ..kernels import (
    Int4KVCacheAppendSm100Kernel,
    Int4KVCacheGatherSm100Kernel,
    PagedKVPlanSm100Kernel,
    PagedKVReleaseSm100Kernel,
    QKNormRopeSm100Kernel,
)
from .gqa import _validate_attention_dtype, _validate_positive
from .op_base import Op

__all__ = [
    "PagedKVCachePlanFwdOp",
    "PagedKVCacheReleaseFwdOp",
    "QKNormRopeFwdOp",
    "QKNormRopeKVCacheAppendFwdOp",
    "QKNormRopeInt4KVCacheAppendFwdOp",
    "Int4KVCacheAppendFwdOp",
    "Int4KVCacheGatherFwdOp",
]


class PagedKVCachePlanFwdOp(Op):
    """Block tables and slot maps of one step, built on the GPU from the requests' lengths.

    ``forward(seq_lens, new_lens, block_table, free_pages, free_count, total_tokens)``: request b holds ``seq_lens[b]``
    tokens and appends ``new_lens[b]`` (int32 ``[B]``).  Its new pages come off the top of the stack
    ``free_pages[0 .. free_count[0])`` in the order of the requests and are entered in ``block_table [B, W]`` in place.
    Returns a :class:`PagedKVPlan`: ``cu_seqlens_q [B + 1]``, ``slot_mapping`` and ``positions [total_tokens]``, and
    ``seq_lens [B]``, ``free_count [1]`` and ``granted [B]`` after the step.  A request is granted when its lengths fit the
    table and it needs no page or the stack holds enough for it and the requests in front of it; else its rows get slot
    -1 and it keeps its length.  A page id that is negative or too large for a 32-bit slot gives slot -1 as well; an append
    skips slots outside its pool.  ``total_tokens`` is the packed batch's row count; rows behind the last request get slot -1
    and position 0.  ``inplace=True`` updates ``seq_lens`` and ``free_count`` themselves, for a step that a CUDA graph
    replays.  ``free_pages`` and ``free_count`` ``None``: the table holds every page already (the host manages its pages)
    and only the maps are built.  At most 4096 requests.
    """

    def __init__(self, batch: int, max_pages_per_req: int, page_size: int,
                 kernel_map: Optional[Dict[str, type]] = None) -> None:
        _validate_positive(batch=batch, max_pages_per_req=max_pages_per_req, page_size=page_size)
        if batch > 4096:
            raise ValueError(f"at most 4096 requests, got {batch}")
        if max_pages_per_req * page_size > 1 << 30:
            raise ValueError("a request must hold at most 2^30 tokens")
        self.batch, self.max_pages_per_req, self.page_size = batch, max_pages_per_req, page_size
        self.dispatch_kernel(kernel_map)

    @property
    def default_kernel_map(self) -> Dict[str, type]:
        return {"paged_kv_plan_kernel": PagedKVPlanSm100Kernel}

    def _check(self, seq_lens, block_table) -> None:
        if seq_lens.shape != (self.batch,):
            raise ValueError(f"seq_lens must have shape ({self.batch},), got {tuple(seq_lens.shape)}")
        if block_table.shape != (self.batch, self.max_pages_per_req):
            raise ValueError(f"block_table shape must be ({self.batch}, {self.max_pages_per_req}), "
                             f"got {tuple(block_table.shape)}")

    def _kernel(self, slot, inputs):
        return self.get_or_build_kernel(slot, inputs, build=lambda: self.kernel_map[slot](self.page_size))

    def forward(self, seq_lens, new_lens, block_table, free_pages, free_count, total_tokens: int,
                inplace: bool = False) -> PagedKVPlan:
        self._check(seq_lens, block_table)
        self.total_tokens = int(total_tokens)
        return self._kernel("paged_kv_plan_kernel", (seq_lens, new_lens, block_table, free_pages, free_count))(
            seq_lens, new_lens, block_table, free_pages, free_count, total_tokens, inplace=inplace)


class PagedKVCacheReleaseFwdOp(PagedKVCachePlanFwdOp):
    """Gives the pages of finished requests back: ``forward(finished, seq_lens, block_table, free_pages, free_count)``
    pushes the pages of every request with ``finished[b]`` (bool ``[B]``) on the stack and sets its ``seq_lens`` to 0, all
    in place on the GPU.  The table keeps its entries."""

    @property
    def default_kernel_map(self) -> Dict[str, type]:
        return {"paged_kv_release_kernel": PagedKVReleaseSm100Kernel}

    def forward(self, finished, seq_lens, block_table, free_pages, free_count) -> None:
        self._check(seq_lens, block_table)
        self._kernel("paged_kv_release_kernel", (finished, seq_lens, block_table, free_pages, free_count))(
            finished, seq_lens, block_table, free_pages, free_count)


class QKNormRopeFwdOp(Op):
    """Per-head RMS norm of q and k and the GPT-NeoX rotation in the same pass.

    ``forward(q [T,H,D], k [T,Hkv,D], q_weight, k_weight, positions)`` returns the new q and k.  Per head
    ``y = x * rsqrt(mean(x^2) + eps) * weight`` (``weight`` ``[D]`` of q's dtype or fp32, or ``None``), then the first
    ``rotary_dim`` dims are rotated about their midpoint by ``positions[t] * inv_freq[j]`` (``positions`` int32 ``[T]``).
    Computed in fp32 with angles in fp64 and rounded once, so there is no cos / sin table and no largest position.
    ``inv_freq`` (``[rotary_dim / 2]``) replaces ``rope_base ** (-2 j / rotary_dim)``, for scaled rotations.  q, k and v may
    be parts of one projection's output (rows on 16-byte boundaries are read where they are).  ``dim`` is a multiple of 8
    up to 256, ``rotary_dim`` a multiple of 16 up to ``dim``, or 0.  The first call on a device copies the frequencies there and
    cannot be captured.
    """

    def __init__(self, heads: int, heads_kv: int, dim: int, rotary_dim: Optional[int] = None, rope_base: float = 10000.0,
                 eps: float = 1e-6, inv_freq: Optional[torch.Tensor] = None,
                 kernel_map: Optional[Dict[str, type]] = None) -> None:
        _validate_positive(heads=heads, heads_kv=heads_kv, dim=dim, rope_base=rope_base)
        if dim % 8 != 0 or dim > 256:
            raise ValueError(f"dim must be a multiple of 8 up to 256, got {dim}")
        rotary_dim = dim // 16 * 16 if rotary_dim is None and dim % 16 == 0 else rotary_dim
        if rotary_dim is None or rotary_dim < 0 or rotary_dim > dim or rotary_dim % 16 != 0:
            raise ValueError(f"rotary_dim must be a multiple of 16 in [0, {dim}], got {rotary_dim}")
        if not eps >= 0:
            raise ValueError("eps must be non-negative")
        self.heads, self.heads_kv, self.dim = heads, heads_kv, dim
        self.rotary_dim, self.rope_base, self.eps, self.inv_freq = rotary_dim, rope_base, eps, inv_freq
        half = rotary_dim // 2
        if inv_freq is None:
            turns = [rope_base ** (-j / half) / (2 * math.pi) for j in range(half)]
        else:
            if tuple(inv_freq.shape) != (half,):
                raise ValueError(f"inv_freq must have shape ({half},), got {tuple(inv_freq.shape)}")
            turns = [f / (2 * math.pi) for f in inv_freq.detach().double().cpu().tolist()]
        self._inv_turns = torch.tensor(turns, dtype=torch.float64)
        self._inv_turns_on: dict = {}
        self.dispatch_kernel(kernel_map)

    @property
    def default_kernel_map(self) -> Dict[str, type]:
        return {"qk_norm_rope_kernel": QKNormRopeSm100Kernel}

    _page_size = 0

    def _kernel(self, inputs):
        return self.get_or_build_kernel("qk_norm_rope_kernel", inputs, build=lambda: self.kernel_map["qk_norm_rope_kernel"](
            self.dim, self.eps, page_size=self._page_size))

    def _turns(self, device: torch.device) -> Optional[torch.Tensor]:
        """Frequencies in turns on ``device``, copied there by the first call."""
        if self.rotary_dim == 0:
            return None
        turns = self._inv_turns_on.get(device)
        if turns is None:
            if device.type == "cuda" and functional._capturing(device):
                raise RuntimeError(f"the first call of a {type(self).__name__} on a device copies its frequencies there, which a "
                                   "CUDA graph cannot hold: call it once before the capture")
            turns = self._inv_turns.to(device)
            self._inv_turns_on[device] = turns
        return turns

    def _check(self, q, k) -> None:
        shape = q.shape
        if shape[1:] != (self.heads, self.dim):
            raise ValueError(f"q must have shape [T, {self.heads}, {self.dim}], got {tuple(q.shape)}")
        if k.shape[1:] != (self.heads_kv, self.dim):
            raise ValueError(f"k must have shape [T, {self.heads_kv}, {self.dim}], got {tuple(k.shape)}")
        self.total_tokens = shape[0]       # for eval_roofline

    def forward(self, q, k, q_weight, k_weight, positions) -> tuple:
        self._check(q, k)
        return self._kernel((q, k, q_weight, k_weight, positions))(
            q, k, positions, self._turns(q.device), q_weight, k_weight)


class QKNormRopeKVCacheAppendFwdOp(QKNormRopeFwdOp):
    """:class:`QKNormRopeFwdOp` with the append to a paged cache of q's dtype in the same launch:
    ``forward(q, k, v, q_weight, k_weight, positions, slot_mapping, k_pages, v_pages)`` returns the new q; the new k and v
    go to the rows ``slot_mapping`` (int32 ``[T]``, as the plan gives it; rows outside the pool are skipped, rows of one
    call must be distinct) of ``k_pages`` / ``v_pages [pool_tokens,Hkv,D]``.  ``return_k=True`` returns (q, k), for a
    prefill that attends to its own chunk."""

    def forward(self, q, k, v, q_weight, k_weight, positions, slot_mapping, k_pages, v_pages, return_k: bool = False):
        self._check(q, k)
        return self._kernel((q, k, v, q_weight, k_weight, positions, slot_mapping, k_pages, v_pages))(
            q, k, positions, self._turns(q.device), q_weight, k_weight, v=v, slot_mapping=slot_mapping, k_pages=k_pages,
            v_pages=v_pages, return_k=return_k)


def _check_int4_sizes(dim: int, page_size: int) -> None:
    if dim not in (64, 128):
        raise ValueError(f"a 4-bit KV cache serves head dim 64 and 128, got {dim}")
    if page_size <= 0 or page_size % 16 != 0:
        raise ValueError(f"page_size must be a positive multiple of 16, got {page_size}")


class QKNormRopeInt4KVCacheAppendFwdOp(QKNormRopeFwdOp):
    """:class:`QKNormRopeKVCacheAppendFwdOp` with the 4-bit cache of :class:`Int4KVCacheAppendFwdOp`:
    ``forward(q, k, v, q_weight, k_weight, positions, slot_mapping, kv_pages)``.  The cache gets k as its 16-bit value
    quantises, bit for bit what the norm and an append of their own would leave."""

    def __init__(self, heads: int, heads_kv: int, dim: int, page_size: int, rotary_dim: Optional[int] = None,
                 rope_base: float = 10000.0, eps: float = 1e-6, inv_freq: Optional[torch.Tensor] = None,
                 kernel_map: Optional[Dict[str, type]] = None) -> None:
        _check_int4_sizes(dim, page_size)
        self.page_size = self._page_size = page_size
        super().__init__(heads, heads_kv, dim, rotary_dim, rope_base, eps, inv_freq, kernel_map)

    def forward(self, q, k, v, q_weight, k_weight, positions, slot_mapping, kv_pages, return_k: bool = False):
        self._check(q, k)
        return self._kernel((q, k, v, q_weight, k_weight, positions, slot_mapping, kv_pages))(
            q, k, positions, self._turns(q.device), q_weight, k_weight, v=v, slot_mapping=slot_mapping, kv_pages=kv_pages,
            return_k=return_k)


class Int4KVCacheAppendFwdOp(Op):
    """Quantises k and v ``[T,Hkv,D]`` into a paged cache of 4 bits: ``forward(k, v, slot_mapping, kv_pages)``.

    ``kv_pages`` is uint8 ``[pages, Hkv, page_size * (D + 8)]`` (:meth:`page_bytes`), modified in place; the library's header
    gives its layout and :func:`tileops_b200.functional.int4_cache_views` its parts.  Each row (one token of one KV head)
    has 15 equal steps between its smallest and largest value and a float16 scale and offset; value = scale * code +
    offset is off by at most half a step and 15 times the rounding of the scale (2^-11 of a step, or 2^-25 where the step is
    below 2^-14, float16's smallest normal number), and by the offset's rounding where it is no float16.  Values beyond +-65504
    saturate; a row with a NaN reads as NaN.  ``slot_mapping``: int32 ``[T]``, distinct, rows outside the pool are skipped."""

    def __init__(self, heads_kv: int, dim: int, page_size: int, kernel_map: Optional[Dict[str, type]] = None) -> None:
        _validate_positive(heads_kv=heads_kv)
        _check_int4_sizes(dim, page_size)
        self.heads_kv, self.dim, self.page_size = heads_kv, dim, page_size
        self.dispatch_kernel(kernel_map)

    @property
    def page_bytes(self) -> int:
        return int4_page_bytes(self.page_size, self.dim)

    @property
    def default_kernel_map(self) -> Dict[str, type]:
        return {"int4_kv_cache_append_kernel": Int4KVCacheAppendSm100Kernel}

    def forward(self, k, v, slot_mapping, kv_pages) -> None:
        if k.shape[1:] != (self.heads_kv, self.dim):
            raise ValueError(f"k must have shape [T, {self.heads_kv}, {self.dim}], got {tuple(k.shape)}")
        self.total_tokens = k.shape[0]
        slot = "int4_kv_cache_append_kernel"
        self.get_or_build_kernel(slot, (k, v, slot_mapping, kv_pages),
                                 build=lambda: self.kernel_map[slot](self.dim, self.page_size))(
            k, v, slot_mapping, kv_pages)


class Int4KVCacheGatherFwdOp(Op):
    """Reads a 4-bit cache back: ``forward(kv_pages, block_table, cu_seqlens_kv, total_tokens)`` returns K and V
    ``[total_tokens,Hkv,D]`` in ``dtype``; rows ``cu_seqlens_kv[b] .. cu_seqlens_kv[b + 1]`` are request b's tokens from 0 on.
    ``total_tokens`` may be an upper bound (rows behind the last request's are left uninitialised).  A page id outside the
    pool reads as NaN; float16 values saturate at +-65504."""

    def __init__(self, heads_kv: int, dim: int, page_size: int, dtype: torch.dtype = torch.bfloat16,
                 kernel_map: Optional[Dict[str, type]] = None) -> None:
        _validate_positive(heads_kv=heads_kv)
        _check_int4_sizes(dim, page_size)
        _validate_attention_dtype(dtype)
        self.heads_kv, self.dim, self.page_size, self.dtype = heads_kv, dim, page_size, dtype
        self.dispatch_kernel(kernel_map)

    @property
    def default_kernel_map(self) -> Dict[str, type]:
        return {"int4_kv_cache_gather_kernel": Int4KVCacheGatherSm100Kernel}

    def forward(self, kv_pages, block_table, cu_seqlens_kv, total_tokens: int) -> tuple:
        if kv_pages.ndim != 3 or kv_pages.shape[1] != self.heads_kv:
            raise ValueError(f"kv_pages must be [pages, {self.heads_kv}, {int4_page_bytes(self.page_size, self.dim)}], "
                             f"got {tuple(kv_pages.shape)}")
        self.total_tokens = int(total_tokens)
        slot = "int4_kv_cache_gather_kernel"
        return self.get_or_build_kernel(slot, (kv_pages, block_table, cu_seqlens_kv),
                                        build=lambda: self.kernel_map[slot](self.dim, self.page_size, self.dtype))(
            kv_pages, block_table, cu_seqlens_kv, total_tokens)
