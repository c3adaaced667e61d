"""Tensor-level wrappers over the C ABI: argument checks, workspace cache, launch.

These are what the kernel classes (``tileops_b200.kernels``) call.  They allocate the output
with torch, hand raw pointers and the current torch CUDA stream to the library, and never
synchronise with the device.
"""

from __future__ import annotations

import ctypes
from typing import NamedTuple, Optional, Tuple

import torch

from . import _native as N

# One workspace per (device, stream, problem shape).  The kernel leaves its counters zeroed, so
# the buffer is zero-filled only when it is created.  Keyed by stream because two launches that
# overlap on the GPU must not share scheduler counters, and by shape because the position of
# the counters inside the buffer depends on (batch, heads, heads_kv, dim): partial results of
# one shape would otherwise land on the counters of another.
_WORKSPACES: dict = {}


def _decode_workspace(device: torch.device, batch: int, heads: int, heads_kv: int, dim: int) -> torch.Tensor:
    need = N.lib().tb200_gqa_decode_workspace_bytes(batch, heads, heads_kv, dim)
    if need == 0:
        raise ValueError("invalid decode problem size")
    key = (device, torch.cuda.current_stream(device).cuda_stream, "decode", batch, heads, heads_kv, dim)
    ws = _WORKSPACES.get(key)
    if ws is None or ws.numel() < need:
        ws = torch.zeros(need, dtype=torch.uint8, device=device)
        _WORKSPACES[key] = ws
    return ws


def release_workspaces() -> None:
    """Drop every cached workspace (e.g. before measuring memory)."""
    _WORKSPACES.clear()


def _require_cuda(**tensors: Optional[torch.Tensor]) -> None:
    for name, t in tensors.items():
        if t is not None and not t.is_cuda:
            raise ValueError(f"{name} must be on a cuda device, got {t.device}")


def gqa_decode(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    *,
    real_seqlen_kv: "torch.Tensor | int",
    block_table: Optional[torch.Tensor] = None,
    page_size: int = 0,
    k_scale: Optional[torch.Tensor] = None,
    v_scale: Optional[torch.Tensor] = None,
    sm_scale: Optional[float] = None,
    softcap: float = 0.0,
    out_dtype: Optional[torch.dtype] = None,
    return_lse: bool = False,
    out: Optional[torch.Tensor] = None,
    lse_out: Optional[torch.Tensor] = None,
    config: Optional[dict] = None,
) -> "torch.Tensor | Tuple[torch.Tensor, torch.Tensor]":
    """Single-token GQA decode.

    q ``[B,H,D]``; paged cache (``block_table`` given): k/v ``[N,Hkv,D]``; contiguous cache:
    k/v ``[B,S,Hkv,D]``.  ``real_seqlen_kv`` is an int32 device tensor ``[B]`` or one int for
    all sequences.  An e4m3 cache needs ``k_scale``/``v_scale`` ``[N/page,Hkv]`` fp32.
    Returns o ``[B,H,D]`` (and the log2-domain LSE ``[B,H]`` fp32 when asked).  ``out`` /
    ``lse_out`` are optional preallocated contiguous destinations (e.g. slices of a
    communication buffer).  ``config`` selects a kernel variant (see ``_native.decode_flags``).
    """
    _require_cuda(q=q, k=k, v=v, block_table=block_table, k_scale=k_scale, v_scale=v_scale)
    if q.dim() != 3:
        raise ValueError(f"q must have shape [B, H, D], got {tuple(q.shape)}")
    B, H, D = q.shape
    paged = block_table is not None
    if paged:
        if k.dim() != 3 or v.shape != k.shape or k.shape[2] != D:
            raise ValueError(f"paged k/v must have shape [N, Hkv, {D}], got {tuple(k.shape)} / {tuple(v.shape)}")
        Hkv = k.shape[1]
        if block_table.dtype != torch.int32 or block_table.dim() != 2 or block_table.shape[0] != B:
            raise ValueError("block_table must be int32 with shape [B, num_pages]")
        if page_size <= 0:
            raise ValueError("page_size must be positive")
        block_table = block_table.contiguous()
    else:
        if k.dim() != 4 or v.shape != k.shape or k.shape[0] != B or k.shape[3] != D:
            raise ValueError(f"k/v must have shape [{B}, S, Hkv, {D}], got {tuple(k.shape)} / {tuple(v.shape)}")
        Hkv = k.shape[2]
    if H % Hkv != 0:
        raise ValueError("heads must be divisible by heads_kv")
    q = q.contiguous()
    k = k.contiguous()
    v = v.contiguous()
    fp8 = k.dtype == getattr(torch, "float8_e4m3fn", None)
    if fp8:
        if k_scale is None or v_scale is None:
            raise ValueError("an float8_e4m3fn cache needs k_scale and v_scale")
        if k_scale.dtype != torch.float32 or v_scale.dtype != torch.float32:
            raise ValueError("k_scale/v_scale must be torch.float32")
        k_scale, v_scale = k_scale.contiguous(), v_scale.contiguous()
    elif k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError(f"k/v dtype {k.dtype} must equal q dtype {q.dtype} (or be float8_e4m3fn)")

    lens_t = None
    uniform = 0
    if isinstance(real_seqlen_kv, torch.Tensor):
        _require_cuda(real_seqlen_kv=real_seqlen_kv)
        if real_seqlen_kv.dtype != torch.int32 or tuple(real_seqlen_kv.shape) != (B,):
            raise ValueError("real_seqlen_kv must be int32 with shape [B]")
        lens_t = real_seqlen_kv.contiguous()
    else:
        uniform = int(real_seqlen_kv)
        if not paged and uniform > k.shape[1]:
            raise ValueError(f"real_seqlen_kv {uniform} exceeds the cache length {k.shape[1]}")

    if out is not None:
        if tuple(out.shape) != (B, H, D) or not out.is_contiguous() or out.device != q.device:
            raise ValueError("out must be a contiguous [B, H, D] tensor on q's device")
        out_dtype = out.dtype
    out_dtype = q.dtype if out_dtype is None else out_dtype
    o = torch.empty((B, H, D), dtype=out_dtype, device=q.device) if out is None else out
    if lse_out is not None:
        if tuple(lse_out.shape) != (B, H) or lse_out.dtype != torch.float32 or not lse_out.is_contiguous():
            raise ValueError("lse_out must be a contiguous float32 [B, H] tensor")
        return_lse = True
    lse = lse_out if lse_out is not None else (
        torch.empty((B, H), dtype=torch.float32, device=q.device) if return_lse else None)
    ws = _decode_workspace(q.device, B, H, Hkv, D)
    scale = D ** -0.5 if sm_scale is None else float(sm_scale)
    if paged:
        tok_stride, head_stride, batch_stride = k.stride(0), k.stride(1), 0
    else:
        tok_stride, head_stride, batch_stride = k.stride(1), k.stride(2), k.stride(0)
    with torch.cuda.device(q.device):
        st = N.lib().tb200_gqa_decode(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), N.ptr(lse),
            N.ptr(lens_t), uniform, N.ptr(block_table), block_table.shape[1] if paged else 0,
            N.ptr(k_scale) if fp8 else None, N.ptr(v_scale) if fp8 else None,
            N.dtype_code(q.dtype), N.dtype_code(k.dtype), N.dtype_code(out_dtype),
            B, H, Hkv, D, int(page_size),
            tok_stride, head_stride, batch_stride,
            scale, float(softcap or 0.0), k.shape[0] if paged else 0, N.decode_flags(config),
            ws.data_ptr(), ws.numel(), N.current_stream(q.device))
    N.check(st, "tb200_gqa_decode")
    return (o, lse) if return_lse else o


def gqa_lse_merge(o_parts: torch.Tensor, lse_parts: torch.Tensor, out_dtype: torch.dtype,
                  return_lse: bool = False):
    """o_parts ``[R, ..., D]`` fp32 and lse_parts ``[R, ...]`` fp32 (log2 domain) -> merged o.

    Each part must be contiguous; the parts themselves may be strided along dim 0 (views into
    an all-gather buffer)."""
    _require_cuda(o_parts=o_parts, lse_parts=lse_parts)
    if o_parts.dtype != torch.float32 or lse_parts.dtype != torch.float32:
        raise ValueError("o_parts and lse_parts must be torch.float32")
    if tuple(o_parts.shape[:-1]) != tuple(lse_parts.shape):
        raise ValueError("o_parts must have shape lse_parts.shape + [D]")
    if not o_parts[0].is_contiguous():
        o_parts = o_parts.contiguous()
    if not lse_parts[0].is_contiguous():
        lse_parts = lse_parts.contiguous()
    R, D = o_parts.shape[0], o_parts.shape[-1]
    rows = lse_parts[0].numel()
    o_stride = o_parts.stride(0) if R > 1 else 0
    l_stride = lse_parts.stride(0) if R > 1 else 0
    o = torch.empty(o_parts.shape[1:], dtype=out_dtype, device=o_parts.device)
    lse = torch.empty(lse_parts.shape[1:], dtype=torch.float32, device=o_parts.device) if return_lse else None
    with torch.cuda.device(o_parts.device):
        st = N.lib().tb200_gqa_lse_merge(o_parts.data_ptr(), lse_parts.data_ptr(), o.data_ptr(), N.ptr(lse),
                                         R, rows, D, o_stride, l_stride, N.dtype_code(out_dtype),
                                         N.current_stream(o_parts.device))
    N.check(st, "tb200_gqa_lse_merge")
    return (o, lse) if return_lse else o


def _prefill_status(device: torch.device, need: int) -> torch.Tensor:
    """Zeroed status buffer of the prefill kernels, one per device (a kernel writes it only when a bounded
    device-side wait runs out).  A wait that ran out makes the launch - and, the word being sticky, every
    later launch on the device - return with its outputs unwritten.  So that this cannot pass unnoticed, the
    word has a mirror in pinned host memory: every prefill call first looks at the mirror (a plain host
    read, no synchronisation; it shows what launches that have completed by now left there), raises
    ``NativeLibraryError`` and clears the word if it is set, and after its launch queues a 4-byte copy of the
    word into the mirror on the same stream."""
    key = (device, "prefill_status")
    ws = _WORKSPACES.get(key)
    if ws is None or ws.numel() < need:
        ws = torch.zeros(max(need, 256), dtype=torch.uint8, device=device)
        _WORKSPACES[key] = ws
        _WORKSPACES[(device, "prefill_status_mirror")] = torch.zeros(1, dtype=torch.int32).pin_memory()
    mirror = _WORKSPACES[(device, "prefill_status_mirror")]
    code = int(mirror[0])
    if code:
        mirror.zero_()
        ws[:4].zero_()
        raise N.NativeLibraryError(
            f"an earlier prefill launch on {device} gave up on a device-side wait (code {code}); its outputs and "
            "those of the launches after it are not valid.  The status word has been cleared.")
    return ws


def _mirror_prefill_status(device: torch.device) -> None:
    ws = _WORKSPACES.get((device, "prefill_status"))
    mirror = _WORKSPACES.get((device, "prefill_status_mirror"))
    if ws is not None and mirror is not None:
        mirror.copy_(ws[:4].view(torch.int32), non_blocking=True)


def _device_of(device: "torch.device | str | int | None") -> torch.device:
    """A device with an explicit index (``"cuda"`` means the current device)."""
    d = torch.device("cuda" if device is None else device)
    if d.type == "cuda" and d.index is None:
        d = torch.device("cuda", torch.cuda.current_device())
    return d


def prefill_status(device: "torch.device | str | int | None" = None, reset: bool = False) -> int:
    """0 if no prefill launch on ``device`` (default: the current CUDA device) has timed out on a
    device-side wait, else the code of the wait that gave up (synchronises with the device).

    The word is sticky: once set, every later prefill launch on the device returns at once with its
    outputs unwritten, so after a suspected timeout poll this before using any output.  ``reset=True``
    clears the word after reading it."""
    ws = _WORKSPACES.get((_device_of(device), "prefill_status"))
    if ws is None:
        return 0
    code = int(ws[:4].view(torch.int32).item())
    if reset and code:
        ws[:4].zero_()
        _WORKSPACES[(_device_of(device), "prefill_status_mirror")].zero_()
    return code


def decode_status(device: "torch.device | str | int | None" = None) -> int:
    """Largest non-zero status word left by a decode launch in any cached workspace of ``device`` (601-603: a bounded wait
    of the TMA decode kernel or of the 4-bit decode ran out), or by a 4-bit decode in a replayed CUDA graph, else 0.
    Synchronises with the current stream; launches and replays on other streams have to be waited for first.  A workspace
    whose status is set is dropped from the cache (its counters are no longer trustworthy) and the next call allocates a
    fresh one; a graph clears its own counters on every replay."""
    dev, worst = _device_of(device), 0
    for key in [k for k in _WORKSPACES if len(k) > 2 and k[2] == "decode" and k[0] == dev]:
        code = int(_WORKSPACES[key][8:12].view(torch.int32).item())
        if code:
            worst = max(worst, code)
            del _WORKSPACES[key]
    if dev.type == "cuda" and torch.cuda.is_initialized():
        code = ctypes.c_int32(0)
        N.check(N.launch(dev, N.lib().tb200_gqa_decode_int4_status, ctypes.addressof(code), 1), "tb200_gqa_decode_int4_status")
        worst = max(worst, code.value)
    return worst


def decode_last_kernel() -> str:
    """Name of the kernel that served this thread's last decode call: ``"tma"`` (TMA producer warp + math
    warps), ``"cp_async"``, or ``""`` before the first call."""
    return {1: "tma", 2: "cp_async"}.get(int(N.lib().tb200_gqa_decode_last_kernel()), "")


def gqa_prefill(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, is_causal: bool = True,
                sm_scale: Optional[float] = None, softcap: float = 0.0, return_lse: bool = False,
                window_size_left: int = -1, window_size_right: int = -1, config: Optional[dict] = None):
    """Dense BSHD prefill: q ``[B,Sq,H,D]``, k/v ``[B,Skv,Hkv,D]`` -> o ``[B,Sq,H,D]`` (+ LSE
    ``[B,H,Sq]`` fp32, log2 domain)."""
    _require_cuda(q=q, k=k, v=v)
    if q.dim() != 4 or k.dim() != 4 or v.shape != k.shape:
        raise ValueError("q must be [B,Sq,H,D] and k/v [B,Skv,Hkv,D]")
    B, Sq, H, D = q.shape
    Skv, Hkv = k.shape[1], k.shape[2]
    if k.shape[0] != B or k.shape[3] != D:
        raise ValueError("k/v batch and head dim must match q")
    if H % Hkv != 0:
        raise ValueError("heads must be divisible by heads_kv")
    if k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError("q/k/v dtypes must match")
    q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    o = torch.empty_like(q)
    lse = torch.empty((B, H, Sq), dtype=torch.float32, device=q.device) if return_lse else None
    need = N.lib().tb200_gqa_prefill_workspace_bytes(B, H, Hkv, Sq, Skv, D)
    ws = _prefill_status(q.device, need)
    scale = D ** -0.5 if sm_scale is None else float(sm_scale)
    with torch.cuda.device(q.device):
        st = N.lib().tb200_gqa_prefill(q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), N.ptr(lse),
                                       N.dtype_code(q.dtype), B, Sq, Skv, H, Hkv, D, int(bool(is_causal)),
                                       scale, float(softcap or 0.0), int(window_size_left),
                                       int(window_size_right), N.prefill_flags(config), N.ptr(ws), need,
                                       N.current_stream(q.device))
    N.check(st, "tb200_gqa_prefill")
    _mirror_prefill_status(q.device)
    return (o, lse) if return_lse else o


def gqa_prefill_paged(q: torch.Tensor, k_new: torch.Tensor, v_new: torch.Tensor,
                      k_pages: Optional[torch.Tensor], v_pages: Optional[torch.Tensor],
                      cu_seqlens_q: torch.Tensor, cache_seqlens: Optional[torch.Tensor],
                      block_table: Optional[torch.Tensor], max_seqlen_q: int, *, page_size: int = 0,
                      is_causal: bool = True, sm_scale: Optional[float] = None, softcap: float = 0.0,
                      return_lse: bool = False, cu_seqlens_kv: Optional[torch.Tensor] = None,
                      window_size_left: int = -1, window_size_right: int = -1, config: Optional[dict] = None):
    """Packed prefill of one chunk per request over a paged cache, appending the chunk in place.

    q ``[total_q,H,D]``, k_new/v_new ``[total_q,Hkv,D]``, k_pages/v_pages ``[pool_tokens,Hkv,D]``
    (modified in place), cu_seqlens_q ``[B+1]``, cache_seqlens ``[B]``, block_table ``[B,W]`` (int32)
    -> o ``[total_q,H,D]`` (+ LSE ``[H,total_q]`` fp32, log2 domain).  With the three cache arguments
    ``None`` it is the packed varlen prefill without a cache; only then may ``cu_seqlens_kv``
    give k_new/v_new their own row ranges (bottom-right aligned causal mask per request).
    """
    _require_cuda(q=q, k_new=k_new, v_new=v_new, cu_seqlens_q=cu_seqlens_q)
    if q.dim() != 3 or k_new.dim() != 3 or v_new.shape != k_new.shape:
        raise ValueError("q must be [total_q,H,D] and k_new/v_new [total_kv,Hkv,D]")
    if cu_seqlens_kv is None and k_new.shape[0] != q.shape[0]:
        raise ValueError("k_new/v_new must have the rows of q unless cu_seqlens_kv is given")
    if cu_seqlens_kv is not None:
        if k_pages is not None:
            raise ValueError("cu_seqlens_kv cannot be combined with a cache")
        _require_cuda(cu_seqlens_kv=cu_seqlens_kv)
        if cu_seqlens_kv.dtype != torch.int32 or cu_seqlens_kv.shape != cu_seqlens_q.shape:
            raise ValueError("cu_seqlens_kv must be int32 with the shape of cu_seqlens_q")
        cu_seqlens_kv = cu_seqlens_kv.contiguous()
    total_q, H, D = q.shape
    Hkv = k_new.shape[1]
    if k_new.shape[2] != D or H % Hkv != 0:
        raise ValueError("head dim must match and heads must be divisible by heads_kv")
    if k_new.dtype != q.dtype or v_new.dtype != q.dtype:
        raise ValueError("q/k_new/v_new dtypes must match")
    if cu_seqlens_q.dtype != torch.int32 or cu_seqlens_q.dim() != 1:
        raise ValueError("cu_seqlens_q must be a 1-D int32 tensor")
    B = cu_seqlens_q.numel() - 1
    has_cache = k_pages is not None
    pool_tokens, bt_stride = 0, 0
    if has_cache:
        if v_pages is None or cache_seqlens is None or block_table is None:
            raise ValueError("k_pages, v_pages, cache_seqlens and block_table come together")
        _require_cuda(k_pages=k_pages, v_pages=v_pages, cache_seqlens=cache_seqlens, block_table=block_table)
        if k_pages.dtype != q.dtype or v_pages.dtype != q.dtype:
            raise ValueError("k_pages/v_pages must have the dtype of q")
        if not (k_pages.is_contiguous() and v_pages.is_contiguous()):
            raise ValueError("k_pages and v_pages must be contiguous (they are written in place)")
        if k_pages.dim() != 3 or tuple(k_pages.shape[1:]) != (Hkv, D) or v_pages.shape != k_pages.shape:
            raise ValueError("k_pages/v_pages must be [pool_tokens,Hkv,D]")
        if cache_seqlens.dtype != torch.int32 or block_table.dtype != torch.int32:
            raise ValueError("cache_seqlens and block_table must be int32")
        if cache_seqlens.shape != (B,) or block_table.dim() != 2 or block_table.shape[0] != B:
            raise ValueError("cache_seqlens must be [B] and block_table [B,W]")
        if block_table.stride(1) != 1:
            block_table = block_table.contiguous()
        pool_tokens, bt_stride = k_pages.shape[0], block_table.stride(0)
    q, k_new, v_new = q.contiguous(), k_new.contiguous(), v_new.contiguous()
    cu_seqlens_q = cu_seqlens_q.contiguous()
    o = torch.empty_like(q)
    lse = torch.empty((H, total_q), dtype=torch.float32, device=q.device) if return_lse else None
    if total_q == 0:
        return (o, lse) if return_lse else o
    need = N.lib().tb200_gqa_prefill_workspace_bytes(B, H, Hkv, int(max_seqlen_q), 0, D)
    ws = _prefill_status(q.device, need)
    scale = D ** -0.5 if sm_scale is None else float(sm_scale)
    with torch.cuda.device(q.device):
        st = N.lib().tb200_gqa_prefill_paged(
            q.data_ptr(), k_new.data_ptr(), v_new.data_ptr(), N.ptr(k_pages), N.ptr(v_pages), o.data_ptr(),
            N.ptr(lse), cu_seqlens_q.data_ptr(), N.ptr(cu_seqlens_kv), N.ptr(cache_seqlens) if has_cache else None,
            N.ptr(block_table) if has_cache else None, bt_stride, N.dtype_code(q.dtype), total_q,
            k_new.shape[0], B,
            int(max_seqlen_q), H, Hkv, D, int(page_size), pool_tokens, int(bool(is_causal)), scale,
            float(softcap or 0.0), int(window_size_left), int(window_size_right), N.prefill_flags(config),
            N.ptr(ws), need, N.current_stream(q.device))
    N.check(st, "tb200_gqa_prefill_paged")
    _mirror_prefill_status(q.device)
    return (o, lse) if return_lse else o


def rope_neox_packed(x: torch.Tensor, cos_table: torch.Tensor, sin_table: torch.Tensor,
                     cu_seqlens_q: torch.Tensor, cache_seqlens: Optional[torch.Tensor],
                     rotary_dim: Optional[int] = None) -> torch.Tensor:
    """GPT-NeoX rotary embedding of packed ``x [T,H,D]`` at positions ``cache_seqlens[b] + i`` for the
    i-th token of request b; tables ``[max_position, rotary_dim/2]`` in x's dtype.  Returns a new tensor."""
    _require_cuda(x=x, cos_table=cos_table, sin_table=sin_table, cu_seqlens_q=cu_seqlens_q)
    if x.dim() != 3:
        raise ValueError("x must be [tokens, heads, dim]")
    T, H, D = x.shape
    rotary_dim = D if rotary_dim is None else int(rotary_dim)
    if cos_table.dtype != x.dtype or sin_table.dtype != x.dtype:
        raise ValueError("cos/sin tables must have x's dtype")
    if cos_table.shape != sin_table.shape or cos_table.dim() != 2 or cos_table.shape[1] != rotary_dim // 2:
        raise ValueError(f"cos/sin tables must be [max_position, {rotary_dim // 2}]")
    if cu_seqlens_q.dtype != torch.int32 or (cache_seqlens is not None and cache_seqlens.dtype != torch.int32):
        raise ValueError("cu_seqlens_q and cache_seqlens must be int32")
    x = x.contiguous()
    y = torch.empty_like(x)
    # positions are range-checked by the caller (the operator does, on the host); no status word is passed
    with torch.cuda.device(x.device):
        st = N.lib().tb200_rope_neox_packed(
            x.data_ptr(), y.data_ptr(), cos_table.contiguous().data_ptr(), sin_table.contiguous().data_ptr(),
            cu_seqlens_q.contiguous().data_ptr(), N.ptr(cache_seqlens), N.dtype_code(x.dtype), T,
            cu_seqlens_q.numel() - 1, H, D, rotary_dim, cos_table.shape[0], None, N.current_stream(x.device))
    N.check(st, "tb200_rope_neox_packed")
    return y


def gqa_prefill_paged_fp8_cache(q: torch.Tensor, k_new: torch.Tensor, v_new: torch.Tensor, k_pages: torch.Tensor,
                                v_pages: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor,
                                cu_seqlens_q: torch.Tensor, cache_seqlens: torch.Tensor, block_table: torch.Tensor,
                                max_seqlen_q: int, *, page_size: int, is_causal: bool = True,
                                sm_scale: Optional[float] = None, softcap: float = 0.0,
                                fused: Optional[bool] = None) -> torch.Tensor:
    """Packed prefill of one chunk per request over an FP8-e4m3 paged cache with scalar scales
    (``k_scale`` / ``v_scale``: fp32 tensors of shape (1,)).

    Default (``fused=False``): three launches - the cached tokens are dequantised into a packed 16-bit K/V next
    to the chunk's own rows, the packed prefill runs on it, and the chunk is quantised into the pages (the
    packed buffer is sized by the capacity of the block table).  ``fused=True`` (head dim 128): ONE launch - the
    prefill kernel reads the e4m3 pages by TMA, four converter warps expand each tile in shared memory, the
    scalar scales are folded into the softmax, and the appending CTAs quantise the chunk into the pages.  It
    needs no packed copy of the cache but measured 20-30 % slower (every CTA that shares a KV head converts
    the same tiles again on schedulers the softmax already fills).  Nothing is read back from the
    device either way."""
    _require_cuda(q=q, k_new=k_new, v_new=v_new, k_pages=k_pages, v_pages=v_pages, k_scale=k_scale, v_scale=v_scale,
                  cu_seqlens_q=cu_seqlens_q, cache_seqlens=cache_seqlens, block_table=block_table)
    f8 = getattr(torch, "float8_e4m3fn")
    if k_pages.dtype != f8 or v_pages.dtype != f8:
        raise ValueError("k_pages and v_pages must be torch.float8_e4m3fn")
    if k_scale.dtype != torch.float32 or v_scale.dtype != torch.float32 or k_scale.numel() != 1 or v_scale.numel() != 1:
        raise ValueError("k_scale and v_scale must be fp32 tensors with one element")
    if not (k_pages.is_contiguous() and v_pages.is_contiguous()):
        raise ValueError("k_pages and v_pages must be contiguous (they are written in place)")
    total_q, H, D = q.shape
    Hkv = k_new.shape[1]
    B = cu_seqlens_q.numel() - 1
    q, k_new, v_new = q.contiguous(), k_new.contiguous(), v_new.contiguous()
    cu_seqlens_q, cache_seqlens = cu_seqlens_q.contiguous(), cache_seqlens.contiguous()
    if block_table.stride(1) != 1:
        block_table = block_table.contiguous()
    fused = bool(fused)
    if fused:
        if D != 128:
            raise ValueError("the fused e4m3-page prefill serves head dim 128")
        if k_pages.dim() != 3 or tuple(k_pages.shape[1:]) != (Hkv, D) or v_pages.shape != k_pages.shape:
            raise ValueError("k_pages/v_pages must be [pool_tokens,Hkv,D]")
        o = torch.empty_like(q)
        if total_q == 0:
            return o
        need = N.lib().tb200_gqa_prefill_workspace_bytes(B, H, Hkv, int(max_seqlen_q), 0, D)
        ws = _prefill_status(q.device, need)
        scale = D ** -0.5 if sm_scale is None else float(sm_scale)
        with torch.cuda.device(q.device):
            st = N.lib().tb200_gqa_prefill_paged_e4m3_cache(
                q.data_ptr(), k_new.data_ptr(), v_new.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(),
                k_scale.data_ptr(), v_scale.data_ptr(), o.data_ptr(), None, cu_seqlens_q.data_ptr(),
                cache_seqlens.data_ptr(), block_table.data_ptr(), block_table.stride(0), N.dtype_code(q.dtype),
                total_q, B, int(max_seqlen_q), H, Hkv, D, int(page_size), k_pages.shape[0], int(bool(is_causal)),
                scale, float(softcap or 0.0), N.ptr(ws), need, N.current_stream(q.device))
        N.check(st, "tb200_gqa_prefill_paged_e4m3_cache")
        _mirror_prefill_status(q.device)
        return o
    kv_lens = cache_seqlens + (cu_seqlens_q[1:] - cu_seqlens_q[:-1])
    cu_kv = torch.zeros(B + 1, dtype=torch.int32, device=q.device)
    cu_kv[1:] = torch.cumsum(kv_lens, 0)
    # The packed K/V is sized by what the block table can describe (its width x the page size per request)
    # plus the chunk: an upper bound known on the host, so that no length is read back from the device.  It is
    # the call's own: one kept for the shape would be shared by two host threads whose launches interleave.
    total_kv = B * block_table.shape[1] * int(page_size) + total_q
    bufs = tuple(torch.empty((total_kv, Hkv, D), dtype=q.dtype, device=q.device) for _ in range(2))
    k_all, v_all = bufs
    lib, stream = N.lib(), N.current_stream(q.device)
    with torch.cuda.device(q.device):
        st = lib.tb200_fp8_cache_gather(
            k_pages.data_ptr(), v_pages.data_ptr(), k_new.data_ptr(), v_new.data_ptr(), k_all.data_ptr(),
            v_all.data_ptr(), cu_seqlens_q.data_ptr(), cu_kv.data_ptr(), cache_seqlens.data_ptr(),
            block_table.data_ptr(), block_table.stride(0), k_scale.data_ptr(), v_scale.data_ptr(),
            N.dtype_code(q.dtype), total_kv, B, Hkv, D, int(page_size), stream)
        N.check(st, "tb200_fp8_cache_gather")
        o = gqa_prefill_paged(q, k_all, v_all, None, None, cu_seqlens_q, None, None, int(max_seqlen_q),
                              is_causal=is_causal, sm_scale=sm_scale, softcap=softcap, cu_seqlens_kv=cu_kv)
        st = lib.tb200_fp8_cache_append(
            k_new.data_ptr(), v_new.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), cu_seqlens_q.data_ptr(),
            cache_seqlens.data_ptr(), block_table.data_ptr(), block_table.stride(0), k_scale.data_ptr(),
            v_scale.data_ptr(), N.dtype_code(q.dtype), total_q, B, Hkv, D, int(page_size), stream)
        N.check(st, "tb200_fp8_cache_append")
    return o


def mma_issue_probe(n: int = 128, a_in_tmem: bool = False, repetitions: int = 200, device=None) -> "tuple[float, float]":
    """Clocks one ``tcgen05.mma`` (M = 128, K = 16, N = ``n``) takes to be accepted / to complete on the
    tensor pipe of ``device`` (``tb200_mma_issue_probe``; synchronises)."""
    dev = _device_of(device)
    out = torch.zeros(2, dtype=torch.int64, device=dev)
    with torch.cuda.device(dev):
        st = N.lib().tb200_mma_issue_probe(out.data_ptr(), int(n), int(bool(a_in_tmem)), int(repetitions),
                                           N.current_stream(dev))
    N.check(st, "tb200_mma_issue_probe")
    issued, done = (int(x) for x in out.cpu())
    if done < 0:
        raise N.NativeLibraryError("tb200_mma_issue_probe: the bounded wait for the last MMA ran out")
    return issued / (8.0 * repetitions), done / (8.0 * repetitions)


# ---- paged KV cache: plans, per-head norm + rotation + append, the cache in 4 bits -------------------------------------

class PagedKVPlan(NamedTuple):
    """What :func:`paged_kv_plan` returns; every field is an int32 tensor on the GPU."""
    cu_seqlens_q: torch.Tensor      # [B + 1]
    slot_mapping: torch.Tensor      # [total_tokens], -1: not to be stored
    positions: torch.Tensor         # [total_tokens]
    seq_lens: torch.Tensor          # [B], after the step
    free_count: Optional[torch.Tensor]   # [1], after the step
    granted: torch.Tensor           # [B], 1 or 0


def _fits(t: torch.Tensor, dtype: torch.dtype, shape: tuple, index: int) -> bool:
    """The short answer of the checks below for a contiguous tensor on GPU ``index``: these calls are short, and so is a decode
    step.  Where it is no, the check itself says what is wrong, if anything is."""
    return t.dtype is dtype and t.shape == shape and t.get_device() == index and t.is_contiguous()


def _check_vector(name: str, t: torch.Tensor, n: int, device: torch.device, dtype: torch.dtype = torch.int32) -> None:
    if _fits(t, dtype, (n,), device.index):
        return
    if t.dtype != dtype or t.dim() != 1 or t.shape[0] != n:
        raise ValueError(f"{name} must be {str(dtype)[6:]} with shape ({n},), got {t.dtype} {tuple(t.shape)}")
    if t.device != device:
        raise ValueError(f"{name} must be on {device}, got {t.device}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")


def _check_table(block_table: torch.Tensor, batch: int, device: torch.device) -> None:
    shape = block_table.shape
    if len(shape) == 2 and shape[1] > 0 and _fits(block_table, torch.int32, (batch, shape[1]), device.index):
        return
    if block_table.dtype != torch.int32 or block_table.dim() != 2 or block_table.shape[0] != batch:
        raise ValueError(f"block_table must be int32 with shape [{batch}, num_pages], got {block_table.dtype} "
                         f"{tuple(block_table.shape)}")
    if block_table.device != device:
        raise ValueError(f"block_table must be on {device}, got {block_table.device}")
    if block_table.shape[1] == 0:
        raise ValueError("block_table must have at least one column")
    if block_table.stride(1) != 1 and block_table.shape[1] > 1:
        raise ValueError("the rows of block_table must be contiguous")


def _check_rows_apart(block_table: torch.Tensor) -> None:
    """New pages are entered in the table: its rows must be places of their own (an expanded row is none)."""
    if block_table.shape[0] > 1 and block_table.stride(0) < block_table.shape[1]:
        raise ValueError("the rows of block_table must not overlap where pages are entered in it")


def paged_kv_plan(seq_lens: torch.Tensor, new_lens: torch.Tensor, block_table: torch.Tensor,
                  free_pages: Optional[torch.Tensor], free_count: Optional[torch.Tensor], total_tokens: int, *,
                  page_size: int, inplace: bool = False) -> PagedKVPlan:
    """Plan of a step that appends ``new_lens[b]`` tokens to request b, built on the GPU without a host
    synchronisation: pages come off the stack ``free_pages[0 .. free_count)`` into ``block_table`` (in place), and the
    packed batch gets its row ranges, positions and cache slots (:class:`PagedKVPlan`).

    ``total_tokens`` is the number of rows of the packed batch as the host knows it (at least ``sum(new_lens)``).  A
    request whose lengths do not fit the table, or for which the stack is short, is not granted: its rows get slot -1 and
    it keeps its length.  A page id that is negative or too large for a 32-bit slot gives slot -1 too.  ``inplace=True``
    updates ``seq_lens`` and ``free_count`` themselves (a step that a CUDA graph replays).  With ``free_pages`` and
    ``free_count`` ``None`` the table is taken to hold every page already."""
    _require_cuda(seq_lens=seq_lens)
    device, batch, total = seq_lens.device, seq_lens.shape[0], int(total_tokens)
    _check_vector("seq_lens", seq_lens, batch, device)
    _check_vector("new_lens", new_lens, batch, device)
    _check_table(block_table, batch, device)
    if (free_pages is None) != (free_count is None):
        raise ValueError("free_pages and free_count come together")
    if free_pages is not None:
        _check_vector("free_pages", free_pages, free_pages.numel(), device)
        _check_vector("free_count", free_count, 1, device)
        if not block_table.is_contiguous():
            _check_rows_apart(block_table)
    if total < 0:
        raise ValueError("total_tokens must not be negative")
    buf = seq_lens.new_empty(2 * total + 3 * batch + 2)     # one allocation; the slot map, written most, starts it
    slots, positions, cu, after, granted, count = buf.split_with_sizes([total, total, batch + 1, batch, batch, 1])
    if inplace:
        after, count = seq_lens, free_count
    if free_count is None:
        count = None
    st = N.launch(device, N.lib().tb200_paged_kv_plan, seq_lens.data_ptr(), new_lens.data_ptr(), block_table.data_ptr(),
                  block_table.stride(0), N.ptr(free_pages), 0 if free_pages is None else free_pages.shape[0],
                  N.ptr(free_count), cu.data_ptr(), slots.data_ptr(), positions.data_ptr(), after.data_ptr(),
                  N.ptr(count), granted.data_ptr(), batch, block_table.shape[1], int(page_size), total)
    N.check(st, "tb200_paged_kv_plan")
    return PagedKVPlan(cu, slots, positions, after, count, granted)


def paged_kv_release(finished: torch.Tensor, seq_lens: torch.Tensor, block_table: torch.Tensor, free_pages: torch.Tensor,
                     free_count: torch.Tensor, *, page_size: int) -> None:
    """Gives the pages of the requests with ``finished[b]`` (bool ``[B]``) back to the stack and sets their ``seq_lens`` to
    0; ``free_pages``, ``free_count`` and ``seq_lens`` are updated in place on the GPU."""
    _require_cuda(seq_lens=seq_lens)
    device, batch = seq_lens.device, seq_lens.shape[0]
    _check_vector("seq_lens", seq_lens, batch, device)
    _check_vector("finished", finished, batch, device, torch.bool)
    _check_table(block_table, batch, device)
    _check_vector("free_pages", free_pages, free_pages.numel(), device)
    _check_vector("free_count", free_count, 1, device)
    st = N.launch(device, N.lib().tb200_paged_kv_release, finished.data_ptr(), seq_lens.data_ptr(),
                  block_table.data_ptr(), block_table.stride(0), free_pages.data_ptr(), free_pages.shape[0],
                  free_count.data_ptr(), batch, block_table.shape[1], int(page_size))
    N.check(st, "tb200_paged_kv_release")


def _rows(t: torch.Tensor) -> "Tuple[torch.Tensor, int, int]":
    """``t [tokens, heads, dim]`` with its token and head strides, as it is when its rows start on 16-byte boundaries
    (parts of a fused projection's output do), else a contiguous copy."""
    tokens, heads, dim = t.shape
    tok, head, last = t.stride()
    if tokens <= 1:
        tok = heads * dim
    if heads <= 1:
        head = dim
    if ((last == 1 or dim == 1) and tok % 8 == 0 and head % 8 == 0 and t.data_ptr() % 16 == 0
            and tok < 1 << 31 and head < 1 << 31):
        return t, tok, head
    return t.clone(memory_format=torch.contiguous_format), heads * dim, dim


def int4_page_bytes(page_size: int, dim: int) -> int:
    """Bytes of one KV head's share of a page of the 4-bit cache: ``kv_pages`` is uint8
    ``[pages, heads_kv, int4_page_bytes(page_size, dim)]``."""
    return page_size * (dim + 8)


def int4_cache_views(kv_pages: torch.Tensor, page_size: int, dim: int) -> "Tuple[torch.Tensor, ...]":
    """Views of a 4-bit pool: K codes and V codes ``[pages, heads_kv, page_size / 16, 16, dim / 2]`` (uint8; dim 2j in
    the low half of byte j) and the parameters ``[pages, heads_kv, page_size / 16, 16, 4]`` (float16: K scale, K offset,
    V scale, V offset)."""
    records = kv_pages.view(kv_pages.shape[0], kv_pages.shape[1], page_size // 16, 16 * (dim + 8))
    k, v, params = records.split_with_sizes([8 * dim, 8 * dim, 128], -1)
    return k.unflatten(-1, (16, dim // 2)), v.unflatten(-1, (16, dim // 2)), params.view(torch.float16).unflatten(-1, (16, 4))


def _check_int4_pool(kv_pages: torch.Tensor, heads_kv: int, dim: int, page_size: int, device: torch.device) -> None:
    if (page_size > 0 and page_size % 16 == 0 and (dim == 128 or dim == 64) and kv_pages.data_ptr() % 16 == 0
            and _fits(kv_pages, torch.uint8, (kv_pages.shape[0], heads_kv, page_size * (dim + 8)), device.index)):
        return
    if page_size <= 0 or page_size % 16 != 0:
        raise ValueError(f"page_size must be a positive multiple of 16, got {page_size}")
    if dim not in (64, 128):
        raise ValueError(f"a 4-bit KV cache serves head dim 64 and 128, got {dim}")
    want = (heads_kv, int4_page_bytes(page_size, dim))
    if kv_pages.dtype != torch.uint8 or kv_pages.dim() != 3 or tuple(kv_pages.shape[1:]) != want:
        raise ValueError(f"kv_pages must be uint8 with shape [pages, {want[0]}, {want[1]}], got {kv_pages.dtype} "
                         f"{tuple(kv_pages.shape)}")
    if kv_pages.device != device:
        raise ValueError(f"kv_pages must be on {device}, got {kv_pages.device}")
    if not kv_pages.is_contiguous() or kv_pages.data_ptr() % 16:
        raise ValueError("kv_pages must be contiguous and start on a 16-byte boundary")


def _check_kv_rows(k: torch.Tensor, v: torch.Tensor) -> None:
    shape = k.shape
    if len(shape) == 3 and v.shape == shape and v.dtype is k.dtype and v.get_device() == k.get_device():
        return
    if k.dim() != 3 or v.shape != k.shape:
        raise ValueError(f"k and v must have the same shape [tokens, heads_kv, dim], got {tuple(k.shape)} and "
                         f"{tuple(v.shape)}")
    if v.dtype != k.dtype:
        raise ValueError(f"v must have the dtype of k, got {v.dtype} and {k.dtype}")
    if v.device != k.device:
        raise ValueError(f"v must be on {k.device}, got {v.device}")


def _check_weight(name: str, w: torch.Tensor, dtype: torch.dtype, dim: int, device: torch.device) -> torch.dtype:
    of = w.dtype
    if of is not dtype and of is not torch.float32:
        raise ValueError(f"{name} must have the dtype of q or be torch.float32, got {w.dtype}")
    _check_vector(name, w, dim, device, of)
    return of


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor, inv_turns: Optional[torch.Tensor], *,
                 q_weight: Optional[torch.Tensor] = None, k_weight: Optional[torch.Tensor] = None, eps: float = 1e-6,
                 v: Optional[torch.Tensor] = None, slot_mapping: Optional[torch.Tensor] = None,
                 k_pages: Optional[torch.Tensor] = None, v_pages: Optional[torch.Tensor] = None,
                 kv_pages: Optional[torch.Tensor] = None, page_size: int = 0, return_k: bool = True):
    """Per-head RMS norm of q ``[T,H,D]`` and k ``[T,Hkv,D]``, then the GPT-NeoX rotation of their first ``2 *
    len(inv_turns)`` dims by ``positions[t]`` (int32 ``[T]``), in one pass; ``inv_turns`` is float64, frequencies over
    2 pi (``None``: no rotation).  Computed in fp32, rounded once.  Returns q (and k when ``return_k``) as new contiguous
    tensors.

    With ``k_pages`` / ``v_pages`` (``[pool_tokens,Hkv,D]``, the dtype of q) or ``kv_pages`` (the 4-bit pool) the same
    launch also stores k and v ``[T,Hkv,D]`` at the rows ``slot_mapping`` (int32 ``[T]``; rows outside the pool are
    skipped, rows of one call must be distinct)."""
    _require_cuda(q=q)
    q_shape, k_shape = q.shape, k.shape
    if len(q_shape) != 3 or len(k_shape) != 3 or k_shape[0] != q_shape[0] or k_shape[2] != q_shape[2]:
        raise ValueError(f"q must be [tokens, heads, dim] and k [tokens, heads_kv, dim], got {tuple(q.shape)} and "
                         f"{tuple(k.shape)}")
    device, dtype = q.device, q.dtype
    index = device.index
    if dtype is not torch.bfloat16 and dtype is not torch.float16:
        raise ValueError(f"Expected dtype torch.float16 or torch.bfloat16, got {dtype}")
    if k.dtype is not dtype or k.get_device() != index:
        raise ValueError(f"k must have the dtype and device of q, got {k.dtype} on {k.device}")
    T, H, D = q_shape
    Hkv = k_shape[1]
    _check_vector("positions", positions, T, device)
    half, turns = 0, None
    if inv_turns is not None:
        half, turns = inv_turns.numel(), inv_turns.data_ptr()
        _check_vector("inv_turns", inv_turns, half, device, torch.float64)
    weight_dtype, q_w, k_w = dtype, None, None
    if q_weight is not None:
        weight_dtype, q_w = _check_weight("q_weight", q_weight, dtype, D, device), q_weight.data_ptr()
    if k_weight is not None:
        k_dtype, k_w = _check_weight("k_weight", k_weight, dtype, D, device), k_weight.data_ptr()
        if q_weight is not None and k_dtype is not weight_dtype:
            raise ValueError("q_weight and k_weight must have the same dtype")
        weight_dtype = k_dtype
    kind, pool_tokens, k_cache, v_cache, slots, v_at, v_tok, v_head = N.CACHE_NONE, 0, None, None, None, None, 0, 0
    if kv_pages is not None or k_pages is not None:
        if v is None or slot_mapping is None:
            raise ValueError("v and slot_mapping come with a cache")
        _check_kv_rows(k, v)
        _check_vector("slot_mapping", slot_mapping, T, device)
        slots = slot_mapping.data_ptr()
        if kv_pages is not None:
            if k_pages is not None or v_pages is not None:
                raise ValueError("kv_pages cannot be combined with k_pages / v_pages")
            _check_int4_pool(kv_pages, Hkv, D, page_size, device)
            kind, k_cache, pool_tokens = N.CACHE_INT4, kv_pages.data_ptr(), kv_pages.shape[0] * page_size
        else:
            if v_pages is None:
                raise ValueError("k_pages and v_pages come together")
            kind, k_cache, v_cache = N.CACHE_16BIT, k_pages.data_ptr(), v_pages.data_ptr()
            pool = k_pages.shape
            want = (pool[0], Hkv, D) if len(pool) == 3 else None
            if not (_fits(k_pages, dtype, want, index) and _fits(v_pages, dtype, want, index)
                    and (k_cache | v_cache) % 16 == 0):
                for name, t in (("k_pages", k_pages), ("v_pages", v_pages)):
                    if want is None or tuple(t.shape) != want or t.dtype != dtype:
                        raise ValueError(f"{name} must be [pool_tokens, {Hkv}, {D}] with dtype {dtype}, got "
                                         f"{tuple(t.shape)} {t.dtype}")
                    if t.device != device or not t.is_contiguous() or t.data_ptr() % 16:
                        raise ValueError(f"{name} must be contiguous, on {device}, and start on a 16-byte boundary")
            pool_tokens = pool[0]
        v, v_tok, v_head = _rows(v)
        v_at = v.data_ptr()
    q_out = torch.empty_like(q, memory_format=torch.contiguous_format)
    k_out = torch.empty_like(k, memory_format=torch.contiguous_format) if return_k else None
    q, q_tok, q_head = _rows(q)
    k, k_tok, k_head = _rows(k)
    st = N.launch(device, N.lib().tb200_qk_norm_rope, q.data_ptr(), k.data_ptr(), v_at, q_out.data_ptr(), N.ptr(k_out), q_w, k_w,
                  N.dtype_code(weight_dtype), turns, positions.data_ptr(), slots, k_cache, v_cache, N.dtype_code(dtype), kind,
                  T, H, Hkv, D, 2 * half, q_tok, q_head, k_tok, k_head, v_tok, v_head, page_size, pool_tokens, eps)
    N.check(st, "tb200_qk_norm_rope")
    return (q_out, k_out) if return_k else q_out


def int4_cache_append(k: torch.Tensor, v: torch.Tensor, slot_mapping: torch.Tensor, kv_pages: torch.Tensor, *,
                      page_size: int) -> None:
    """Quantises k and v ``[T,Hkv,D]`` into the rows ``slot_mapping`` (int32 ``[T]``) of the 4-bit pool, in place: 15
    steps between a row's smallest and largest value, one float16 scale and offset per token and KV head (error at most
    half a step, 15 times the rounding of the scale - 2^-11 of a step, or 2^-25 below float16's normal numbers - and the
    rounding of the offset).  Rows outside the pool are skipped; rows of one call must be distinct."""
    _require_cuda(k=k)
    _check_kv_rows(k, v)
    device, dtype = k.device, k.dtype
    if dtype is not torch.bfloat16 and dtype is not torch.float16:
        raise ValueError(f"Expected dtype torch.float16 or torch.bfloat16, got {dtype}")
    T, Hkv, D = k.shape
    _check_vector("slot_mapping", slot_mapping, T, device)
    _check_int4_pool(kv_pages, Hkv, D, page_size, device)
    k, k_tok, k_head = _rows(k)
    v, v_tok, v_head = _rows(v)
    st = N.launch(device, N.lib().tb200_int4_cache_append, k.data_ptr(), v.data_ptr(), slot_mapping.data_ptr(),
                  kv_pages.data_ptr(), N.dtype_code(dtype), T, Hkv, D, page_size, kv_pages.shape[0] * page_size,
                  k_tok, k_head, v_tok, v_head)
    N.check(st, "tb200_int4_cache_append")


def int4_cache_gather(kv_pages: torch.Tensor, block_table: torch.Tensor, cu_seqlens_kv: torch.Tensor, total_tokens: int, *,
                      dim: int, page_size: int, dtype: torch.dtype, cache_seqlens: Optional[torch.Tensor] = None,
                      cu_seqlens_new: Optional[torch.Tensor] = None, k_new: Optional[torch.Tensor] = None,
                      v_new: Optional[torch.Tensor] = None,
                      out: "Optional[Tuple[torch.Tensor, torch.Tensor]]" = None) -> "Tuple[torch.Tensor, torch.Tensor]":
    """Reads the 4-bit pool back: rows ``cu_seqlens_kv[b] .. cu_seqlens_kv[b + 1]`` of the returned K and V
    ``[total_tokens,Hkv,dim]`` are request b's tokens 0, 1, ... in ``dtype``.  ``total_tokens`` may be an upper bound; rows
    behind ``cu_seqlens_kv[-1]`` are left as they were (uninitialised in a new tensor).

    With ``cache_seqlens``, ``cu_seqlens_new``, ``k_new`` and ``v_new`` only the first ``cache_seqlens[b]`` rows of a request
    come from the cache and the rest from rows ``cu_seqlens_new[b] ..`` of ``k_new`` / ``v_new``, which have
    ``cu_seqlens_new[-1]`` rows; a negative ``cache_seqlens[b]`` makes the request NaN."""
    _require_cuda(kv_pages=kv_pages)
    if kv_pages.dim() != 3:
        raise ValueError(f"kv_pages must be [pages, heads_kv, page bytes], got {tuple(kv_pages.shape)}")
    if dtype not in (torch.float16, torch.bfloat16):
        raise ValueError(f"Expected dtype torch.float16 or torch.bfloat16, got {dtype}")
    device, Hkv, total = kv_pages.device, kv_pages.shape[1], int(total_tokens)
    _check_int4_pool(kv_pages, Hkv, dim, page_size, device)
    batch = block_table.shape[0]
    _check_table(block_table, batch, device)
    _check_vector("cu_seqlens_kv", cu_seqlens_kv, batch + 1, device)
    if total < 0:
        raise ValueError("total_tokens must not be negative")
    if cache_seqlens is not None:
        if cu_seqlens_new is None or k_new is None or v_new is None:
            raise ValueError("cache_seqlens, cu_seqlens_new, k_new and v_new come together")
        _check_vector("cache_seqlens", cache_seqlens, batch, device)
        _check_vector("cu_seqlens_new", cu_seqlens_new, batch + 1, device)
        _check_kv_rows(k_new, v_new)
        if tuple(k_new.shape[1:]) != (Hkv, dim) or k_new.dtype != dtype or k_new.device != device:
            raise ValueError(f"k_new and v_new must be [tokens, {Hkv}, {dim}] with dtype {dtype} on {device}")
        k_new, v_new = (t if t.is_contiguous() and t.data_ptr() % 16 == 0
                        else t.clone(memory_format=torch.contiguous_format) for t in (k_new, v_new))
    given, shape = out, (total, Hkv, dim)
    if out is None:
        k_out = kv_pages.new_empty(shape, dtype=dtype)
        out = k_out, torch.empty_like(k_out)
    for t in given or ():
        if tuple(t.shape) != (total, Hkv, dim) or t.dtype != dtype or t.device != device or not t.is_contiguous():
            raise ValueError(f"out must be two contiguous [{total}, {Hkv}, {dim}] tensors with dtype {dtype} on {device}")
    st = N.launch(device, N.lib().tb200_int4_cache_gather, kv_pages.data_ptr(), block_table.data_ptr(),
                  block_table.stride(0), block_table.shape[1], cu_seqlens_kv.data_ptr(), N.ptr(cache_seqlens),
                  N.ptr(cu_seqlens_new), N.ptr(k_new), N.ptr(v_new), out[0].data_ptr(), out[1].data_ptr(),
                  N.dtype_code(dtype), total, batch, Hkv, dim, page_size, kv_pages.shape[0])
    N.check(st, "tb200_int4_cache_gather")
    return out


def _capturing(device: torch.device) -> bool:
    """Is the current stream of ``device`` (which need not be the current one) under capture?"""
    if device.index == torch.cuda.current_device():
        return torch.cuda.is_current_stream_capturing()
    with torch.cuda.device(device):
        return torch.cuda.is_current_stream_capturing()


def _decode_int4_workspace(device: torch.device, batch: int, heads: int, heads_kv: int, dim: int) -> torch.Tensor:
    """Scratch of the 4-bit decode.  Eager calls keep one buffer per (device, stream, shape), as the other decode calls do.
    A call under capture gets one of its own from the graph's pool, cleared by a node of the graph: two graphs, or a
    graph and an eager call, that run at the same time then never share counters.  A wait that runs out in such a launch is
    recorded outside the buffer as well (:func:`decode_status`)."""
    capturing = _capturing(device)
    key = (device, torch._C._cuda_getCurrentRawStream(device.index), "decode", batch, heads, heads_kv, dim, "int4")
    ws = None if capturing else _WORKSPACES.get(key)
    if ws is None:
        need = N.lib().tb200_gqa_decode_int4_workspace_bytes(batch, heads, heads_kv, dim)
        if need == 0:
            raise ValueError("invalid decode problem size")
        ws = torch.empty(need, dtype=torch.uint8, device=device)
        ws[:(batch * heads + 8) * 4].zero_()            # TB200_DECODE_INT4_ZERO_BYTES
        if not capturing:
            _WORKSPACES[key] = ws
    return ws


def gqa_decode_int4(q: torch.Tensor, kv_pages: torch.Tensor, real_seqlen_kv: torch.Tensor, block_table: torch.Tensor, *,
                    page_size: int, sm_scale: Optional[float] = None, softcap: float = 0.0,
                    out_dtype: Optional[torch.dtype] = None, return_lse: bool = False, config: Optional[dict] = None):
    """Single-token GQA decode over the 4-bit paged cache: q ``[B,H,D]``, ``kv_pages`` uint8
    ``[pages,Hkv,page_size*(D+8)]``, ``real_seqlen_kv [B]`` and ``block_table [B,W]`` int32 -> o ``[B,H,D]`` (and the
    log2-domain LSE ``[B,H]`` fp32).  An empty sequence gives zeros (LSE -inf); a page id outside the pool or a length
    beyond the table makes that sequence NaN."""
    _require_cuda(q=q)
    if q.dim() != 3:
        raise ValueError(f"q must have shape [B, H, D], got {tuple(q.shape)}")
    if q.dtype not in (torch.float16, torch.bfloat16):
        raise ValueError(f"Expected dtype torch.float16 or torch.bfloat16, got {q.dtype}")
    if kv_pages.dim() != 3:
        raise ValueError(f"kv_pages must be [pages, heads_kv, page bytes], got {tuple(kv_pages.shape)}")
    B, H, D = q.shape
    device, Hkv = q.device, kv_pages.shape[1]
    if Hkv == 0 or H % Hkv != 0:
        raise ValueError("heads must be divisible by heads_kv")
    _check_int4_pool(kv_pages, Hkv, D, page_size, device)
    _check_vector("real_seqlen_kv", real_seqlen_kv, B, device)
    _check_table(block_table, B, device)
    if not q.is_contiguous() or q.data_ptr() % 16:
        q = q.clone(memory_format=torch.contiguous_format)
    out_dtype = q.dtype if out_dtype is None else out_dtype
    o = torch.empty_like(q, dtype=out_dtype)
    lse = torch.empty((B, H), dtype=torch.float32, device=device) if return_lse else None
    if B == 0:
        return (o, lse) if return_lse else o
    ws = _decode_int4_workspace(device, B, H, Hkv, D)
    st = N.launch(device, N.lib().tb200_gqa_decode_int4, q.data_ptr(), kv_pages.data_ptr(), o.data_ptr(), N.ptr(lse),
                  real_seqlen_kv.data_ptr(), block_table.data_ptr(), block_table.stride(0), block_table.shape[1],
                  N.dtype_code(q.dtype), N.dtype_code(out_dtype), B, H, Hkv, D, page_size, kv_pages.shape[0],
                  D ** -0.5 if sm_scale is None else float(sm_scale), float(softcap or 0.0), N.decode_flags(config),
                  ws.data_ptr(), ws.numel())
    N.check(st, "tb200_gqa_decode_int4")
    return (o, lse) if return_lse else o


def gqa_prefill_paged_int4_cache(q: torch.Tensor, k_new: torch.Tensor, v_new: torch.Tensor, kv_pages: torch.Tensor,
                                 cu_seqlens_q: torch.Tensor, cache_seqlens: torch.Tensor, block_table: torch.Tensor,
                                 max_seqlen_q: int, *, page_size: int, is_causal: bool = True,
                                 sm_scale: Optional[float] = None, softcap: float = 0.0) -> torch.Tensor:
    """Packed prefill of one chunk per request over the 4-bit paged cache, appending the chunk: the cached tokens are read
    back as packed 16-bit K/V next to the chunk's own rows, the packed prefill runs on it, and the chunk is quantised into
    the pages.  The packed buffer is sized by the capacity of the block table (K and V of B W page_size + T tokens) and
    given back to the allocator after the call; nothing is read back from the device.  ``cache_seqlens[b]`` outside what
    the table holds makes request b NaN; a chunk that the table has no room for is attended to but not stored."""
    _require_cuda(q=q, k_new=k_new, v_new=v_new, kv_pages=kv_pages)
    total_q, H, D = q.shape
    Hkv, B, device = k_new.shape[1], cu_seqlens_q.numel() - 1, q.device
    if total_q == 0:
        return torch.empty_like(q)
    new_lens = cu_seqlens_q[1:] - cu_seqlens_q[:-1]
    slots = paged_kv_plan(cache_seqlens, new_lens, block_table, None, None, total_q, page_size=page_size).slot_mapping
    # A request that claims more tokens than its table has (or fewer than none) gets rows of its own that read as NaN: none
    # of the others' move out of the buffer.
    capacity = block_table.shape[1] * int(page_size)
    cu_kv = torch.zeros(B + 1, dtype=torch.int32, device=device)
    cu_kv[1:] = torch.cumsum(cache_seqlens.clamp(0, capacity) + new_lens, 0)
    total_kv = B * capacity + total_q
    # The call's own: a buffer kept for the shape would be shared by two host threads whose launches interleave.
    bufs = tuple(torch.empty((total_kv, Hkv, D), dtype=q.dtype, device=device) for _ in range(2))
    k_all, v_all = int4_cache_gather(kv_pages, block_table, cu_kv, total_kv, dim=D, page_size=page_size, dtype=q.dtype,
                                     cache_seqlens=cache_seqlens, cu_seqlens_new=cu_seqlens_q, k_new=k_new, v_new=v_new,
                                     out=bufs)
    o = gqa_prefill_paged(q, k_all, v_all, None, None, cu_seqlens_q, None, None, int(max_seqlen_q), is_causal=is_causal,
                          sm_scale=sm_scale, softcap=softcap, cu_seqlens_kv=cu_kv)
    int4_cache_append(k_new, v_new, slots, kv_pages, page_size=page_size)
    return o
