"""Bounding a paged KV cache: attention weights per cached token, and the eviction of the tokens with the least of them.

A serving loop that keeps a cache at a budget calls, beside ``flash_decode``, ``accumulate_attention_weights`` (with the
query and the lse of the decode) and, when a sequence has outgrown its budget, ``evict_kvcache``.  After an eviction a token's
place in the cache is no longer its position: the append then takes ``positions``.

The kernels are in ``libfdk.so`` (include/fdk.h: fdk_accumulate_weights, fdk_kv_evict); there is no fallback path.
"""
from __future__ import annotations

import ctypes as C
from typing import Optional, Tuple

import torch

from . import _lib
from ._lib import FdkAttnWeightsArgs, FdkKvEvictArgs
from .flash_decode import (_LIB, _MXFP4_CODES, _check_block_scales, _fdk_dtype, _launch_on, _on_stream, _row_values,
                           _stream_handle)


def _meta(t: Optional[torch.Tensor]):
    return None if t is None else (t.shape, t.stride(), t.dtype, t.device)


def _check_cache(cache, block_table, kv_lens):
    if block_table.dim() != 2 or block_table.dtype != torch.int32 or block_table.stride(-1) != 1:
        raise ValueError("block_table must be int32 [batch, max_pages] with contiguous rows")
    batch = block_table.shape[0]
    if kv_lens.dtype != torch.int32 or tuple(kv_lens.shape) != (batch,) or (batch > 1 and kv_lens.stride(0) != 1):
        raise ValueError(f"kv_lens must be contiguous int32 [{batch}]")
    if cache.dim() != 4 or cache.stride(-1) != 1:
        raise ValueError("caches must be [num_pages, page_size, kv_heads, head_dim] with a contiguous last axis")
    return batch


def _check_devices(first, **tensors):
    for name, t in tensors.items():
        if t is None:
            continue
        if not t.is_cuda:
            raise ValueError(f"{name} must live on the GPU (got {t.device}); there is no CPU path")
        if t.device != first.device:
            raise ValueError(f"{name} is on {t.device}, the cache on {first.device}")


def _check_weights(name, w, batch, kv_heads, length=None):
    if w.dtype != torch.float32 or w.dim() != 3 or tuple(w.shape[:2]) != (batch, kv_heads) or w.stride(-1) != 1 or \
            (length is not None and w.shape[2] != length):
        raise ValueError(f"{name} must be fp32 [{batch}, {kv_heads}, {'tokens' if length is None else length}] with a contiguous last axis")


_WEIGHTS_TEMPLATES = {}      # layout key -> validated argument block without pointers


def accumulate_attention_weights(q: torch.Tensor, k_cache: torch.Tensor, block_table: torch.Tensor, kv_lens: torch.Tensor,
                                 lse: torch.Tensor, sm_scale: float, weights: torch.Tensor, *, soft_cap: float = 0.0,
                                 k_scale: Optional[torch.Tensor] = None, stream=None) -> torch.Tensor:
    """Add what one query token per sequence attends to: ``weights[b, kvh, n] += sum_h exp(logit(b, h, n) - lse[b, h])``
    over the q heads ``h`` of kv head ``kvh``, for the ``kv_lens[b]`` cached tokens.

    q, k_cache, block_table, kv_lens, sm_scale, soft_cap, k_scale   as in ``flash_decode`` (16-bit, fp8 and MXFP4 caches)
    lse        [B, Hq] fp32, what ``flash_decode`` returned for this query; where the tokens are spread over several ranks, the
               merged one (``inter_rank_combine(..., all_ranks_lse=, lse_out=)``): the lse of a packed result is in 16 bits
    weights    [B, Hkv, S] fp32, updated in place; S must cover every length (tokens past S are left out)
    Returns ``weights``.  Every weight is summed in a fixed order: the same bits on every run."""
    key = (_meta(q), _meta(k_cache), _meta(block_table), _meta(kv_lens), _meta(lse), _meta(weights), _meta(k_scale), sm_scale, soft_cap)
    hit = _WEIGHTS_TEMPLATES.get(key)
    if hit is not None:
        a = FdkAttnWeightsArgs.from_buffer_copy(hit)
    else:
        batch = _check_cache(k_cache, block_table, kv_lens)
        _, page_size, kv_heads, _ = k_cache.shape
        d = _row_values(k_cache)
        if q.dim() != 3 or q.shape[0] != batch or q.shape[2] != d or q.stride(-1) != 1:
            raise ValueError(f"q must be [{batch}, q_heads, {d}] with a contiguous last axis, got {tuple(q.shape)}")
        if q.shape[1] % kv_heads:
            raise ValueError(f"{q.shape[1]} q heads are no multiple of {kv_heads} kv heads")
        if lse.dtype != torch.float32 or tuple(lse.shape) != (batch, q.shape[1]) or lse.stride(-1) != 1:
            raise ValueError(f"lse must be fp32 [{batch}, {q.shape[1]}] with contiguous heads")
        _check_weights("weights", weights, batch, kv_heads)
        _check_devices(k_cache, q=q, k_cache=k_cache, block_table=block_table, kv_lens=kv_lens, lse=lse, weights=weights, k_scale=k_scale)
        a = FdkAttnWeightsArgs()
        a.struct_size = C.sizeof(FdkAttnWeightsArgs)
        a.q_dtype, a.kv_dtype = _fdk_dtype(q.dtype, "q"), _fdk_dtype(k_cache.dtype, "k_cache")
        if a.kv_dtype == _lib.FDK_MXFP4:
            _check_block_scales("k_scale", k_scale, k_cache)
            a.kbs_stride_page, a.kbs_stride_tok, a.kbs_stride_head = k_scale.stride()[:3]
        elif k_scale is not None:
            if a.kv_dtype != _lib.FDK_FP8_E4M3:
                raise ValueError("k_scale is only meaningful for an fp8 or MXFP4 KV cache")
            if k_scale.dtype != torch.float32 or k_scale.numel() != kv_heads or not k_scale.is_contiguous():
                raise ValueError(f"k_scale must be a contiguous fp32 tensor of {kv_heads} per-kv-head scales")
        a.q_stride_b, a.q_stride_h = q.stride(0), q.stride(1)
        a.k_stride_page, a.k_stride_tok, a.k_stride_head = k_cache.stride()[:3]
        a.table_stride_b = block_table.stride(0) if batch > 1 else max(block_table.stride(0), block_table.shape[1])
        a.lse_stride_b = lse.stride(0) if batch > 1 else max(lse.stride(0), q.shape[1])
        a.weights_stride_b, a.weights_stride_h = weights.stride(0), weights.stride(1)
        a.batch, a.num_q_heads, a.num_kv_heads, a.head_dim = batch, q.shape[1], kv_heads, d
        a.page_size, a.max_pages, a.weights_len = page_size, block_table.shape[1], weights.shape[2]
        a.sm_scale, a.soft_cap = float(sm_scale), float(soft_cap) if soft_cap else 0.0
    a.q, a.k_cache, a.block_table, a.kv_lens = q.data_ptr(), k_cache.data_ptr(), block_table.data_ptr(), kv_lens.data_ptr()
    a.lse, a.weights = lse.data_ptr(), weights.data_ptr()
    if k_scale is not None:
        if a.kv_dtype == _lib.FDK_MXFP4:
            a.k_block_scale = k_scale.data_ptr()
        else:
            a.k_scale = k_scale.data_ptr()
    _launch_on(q.device, stream, _LIB.fdk_accumulate_weights, a)
    if hit is None:
        if len(_WEIGHTS_TEMPLATES) >= 256:
            _WEIGHTS_TEMPLATES.clear()
        _WEIGHTS_TEMPLATES[key] = bytes(a)
    return weights


_EVICT_TEMPLATES = {}


def _evict_buffers(weights, kv_lens, keep, weights_out, kv_lens_out, kept, workspace_bytes):
    batch, kv_heads = weights.shape[:2]
    if weights_out is None:
        weights_out = torch.empty(weights.shape, dtype=torch.float32, device=weights.device)
    if kv_lens_out is None:
        kv_lens_out = torch.empty(kv_lens.shape, dtype=torch.int32, device=weights.device)
    if kept is None:
        kept = torch.empty((batch, kv_heads, keep), dtype=torch.int32, device=weights.device)
    buf = torch.empty(workspace_bytes, dtype=torch.uint8, device=weights.device)
    return weights_out, kv_lens_out, kept, buf


def evict_kvcache(key_cache: torch.Tensor, value_cache: torch.Tensor, block_table: torch.Tensor, kv_lens: torch.Tensor,
                  weights: torch.Tensor, keep: int, recent: int, *, k_scale: Optional[torch.Tensor] = None,
                  v_scale: Optional[torch.Tensor] = None, weights_out: Optional[torch.Tensor] = None,
                  kv_lens_out: Optional[torch.Tensor] = None, kept: Optional[torch.Tensor] = None,
                  stream=None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Bring every sequence back to at most ``keep`` tokens: its last ``recent`` ones and, of the others, those with the
    largest weights (ties: the lowest slots; a NaN counts as the largest).  Every kv head chooses for itself; the survivors
    move to slots 0, 1, ... in their order, in place.

    key_cache, value_cache  [num_pages, P, Hkv, D] (any row length that is a multiple of 32 values; 16-bit, fp8), or MXFP4
                 codes with their block scales k_scale / v_scale, which move along; the scales of an fp8 cache do not depend on
                 the tokens and are not asked for.  value_cache may be a view of key_cache's rows (latent attention)
    block_table  [B, max_pages] int32, kv_lens [B] int32, weights [B, Hkv, S] fp32 with S covering every length
    keep, recent 1 <= keep <= S, 0 <= recent <= keep; a sequence of at most ``keep`` tokens stays as it is

    Rows move within a sequence's own pages: no other sequence may share them.  (A row that would come from or go to a page number
    outside the pool is left out.)

    Returns ``(kv_lens_out [B] int32 = min(kv_lens, keep), kept [B, Hkv, keep] int32, weights_out [B, Hkv, S])``: ``kept`` is
    the slot that the token in each slot had before (-1 behind the new length), ``weights_out`` the survivors' weights and 0
    behind them.  ``weights_out`` may be ``weights`` and ``kv_lens_out`` may be ``kv_lens``.  Rows behind the new length keep
    their contents and pages their owners: a page that holds no token any more is the caller's to reuse."""
    keep, recent = int(keep), int(recent)
    key = (_meta(key_cache), _meta(value_cache), _meta(block_table), _meta(kv_lens), _meta(weights), keep, recent, _meta(k_scale),
           _meta(v_scale), _meta(weights_out), _meta(kv_lens_out), _meta(kept))
    hit = _EVICT_TEMPLATES.get(key)
    if hit is not None:
        a = FdkKvEvictArgs.from_buffer_copy(hit)
    else:
        batch = _check_cache(key_cache, block_table, kv_lens)
        _check_cache(value_cache, block_table, kv_lens)
        if value_cache.shape[:3] != key_cache.shape[:3] or value_cache.dtype != key_cache.dtype:
            raise ValueError("caches must share their pages, heads and dtype")
        kv_heads = key_cache.shape[2]
        _check_weights("weights", weights, batch, kv_heads)
        length = weights.shape[2]
        if not 1 <= keep <= length:
            raise ValueError(f"keep = {keep} outside [1, {length}]")
        if not 0 <= recent <= keep:
            raise ValueError(f"recent = {recent} outside [0, keep = {keep}]")
        _check_devices(key_cache, key_cache=key_cache, value_cache=value_cache, block_table=block_table, kv_lens=kv_lens, weights=weights,
                       k_scale=k_scale, v_scale=v_scale, weights_out=weights_out, kv_lens_out=kv_lens_out, kept=kept)
        a = FdkKvEvictArgs()
        a.struct_size = C.sizeof(FdkKvEvictArgs)
        a.kv_dtype = _fdk_dtype(key_cache.dtype, "key_cache")
        if key_cache.dtype in _MXFP4_CODES:
            _check_block_scales("k_scale", k_scale, key_cache)
            _check_block_scales("v_scale", v_scale, value_cache)
            a.kbs_stride_page, a.kbs_stride_tok, a.kbs_stride_head = k_scale.stride()[:3]
            a.vbs_stride_page, a.vbs_stride_tok, a.vbs_stride_head = v_scale.stride()[:3]
        elif k_scale is not None or v_scale is not None:
            raise ValueError("k_scale / v_scale: only the block scales of an MXFP4 cache move with its rows")
        if weights_out is not None:
            _check_weights("weights_out", weights_out, batch, kv_heads, length)
        if kv_lens_out is not None and (kv_lens_out.dtype != torch.int32 or tuple(kv_lens_out.shape) != (batch,) or
                                        not kv_lens_out.is_contiguous()):
            raise ValueError(f"kv_lens_out must be contiguous int32 [{batch}]")
        if kept is not None and (kept.dtype != torch.int32 or tuple(kept.shape) != (batch, kv_heads, keep) or not kept.is_contiguous()):
            raise ValueError(f"kept must be contiguous int32 {[batch, kv_heads, keep]}")
        a.k_stride_page, a.k_stride_tok, a.k_stride_head = key_cache.stride()[:3]
        a.v_stride_page, a.v_stride_tok, a.v_stride_head = value_cache.stride()[:3]
        a.table_stride_b = block_table.stride(0) if batch > 1 else max(block_table.stride(0), block_table.shape[1])
        a.weights_stride_b, a.weights_stride_h = weights.stride(0), weights.stride(1)
        a.batch, a.num_kv_heads, a.head_dim, a.v_head_dim = batch, kv_heads, _row_values(key_cache), _row_values(value_cache)
        a.page_size, a.max_pages, a.weights_len = key_cache.shape[1], block_table.shape[1], length
        a.keep, a.recent, a.num_pages = keep, recent, key_cache.shape[0]
        a.workspace_bytes = _LIB.fdk_kv_evict_workspace_bytes(C.byref(a))
    if stream is None:
        weights_out, kv_lens_out, kept, buf = _evict_buffers(weights, kv_lens, keep, weights_out, kv_lens_out, kept, a.workspace_bytes)
    else:
        # (the kernels run on that stream: the workspace must go back to its pool, not to the current stream's)
        with _on_stream(weights.device, _stream_handle(stream)):
            weights_out, kv_lens_out, kept, buf = _evict_buffers(weights, kv_lens, keep, weights_out, kv_lens_out, kept, a.workspace_bytes)
    a.weights_out_stride_b, a.weights_out_stride_h = weights_out.stride(0), weights_out.stride(1)
    a.k_cache, a.v_cache = key_cache.data_ptr(), value_cache.data_ptr()
    if k_scale is not None:
        a.k_block_scale, a.v_block_scale = k_scale.data_ptr(), v_scale.data_ptr()
    a.block_table, a.kv_lens, a.weights = block_table.data_ptr(), kv_lens.data_ptr(), weights.data_ptr()
    a.weights_out, a.kept, a.kv_lens_out, a.workspace = weights_out.data_ptr(), kept.data_ptr(), kv_lens_out.data_ptr(), buf.data_ptr()
    _launch_on(weights.device, stream, _LIB.fdk_kv_evict, a)
    if hit is None:
        if len(_EVICT_TEMPLATES) >= 256:
            _EVICT_TEMPLATES.clear()
        _EVICT_TEMPLATES[key] = bytes(a)
    return kv_lens_out, kept, weights_out
