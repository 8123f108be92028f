"""Paged KV cache of a decoder stack: the producer of the tensors the decode and append operators take.

Host-side mirror of the reference's ``PagedKVCache`` (mega_triton_kernel/models/paged_kv_cache.py:28-58): one K
pool and one V pool ``[num_blocks, PAGE_SIZE, Hkv, D]`` shared by all layers, ``block_tables
[num_layers, B, max_blocks_per_seq]`` int32 cut from ONE permutation of the pool (no page belongs to two
sequences or two layers), one ``kv_lens [B]`` int32 for all layers, ``inc_offset`` and ``get_layer_kv_cache``
with the reference's meaning.

Differences, all additions:
  * the two pools share one allocation, the V pool 256 bytes (modulo 512) off the K pool (``alloc_kv_pools``);
  * the pools start zeroed (the reference fills them with random numbers), ``fill="randn"`` restores that;
  * ``dtype=torch.float8_e4m3fn`` keeps 1-byte pools plus per-layer, per-kv-head fp32 scales
    (``k_scale, v_scale [num_layers, Hkv]``, given by the caller);
  * ``dtype=torch.float4_e2m1fn_x2`` keeps MXFP4 pools: packed codes ``[num_blocks, PAGE_SIZE, Hkv, D/2]`` and, in
    ``k_block_scale`` / ``v_block_scale``, a scale byte per 32 values, written by ``append``;
  * the lengths are tracked on the host as well (``max_kv_len``), so the decode can be planned for the real
    length without reading ``kv_lens`` back from the GPU (both bounds: the sequences advance together, so
    the decode may use per-sequence chunks) - a hint that is wrong never changes results;
  * ``append`` / ``decode`` run the two operators of this package on one layer's view;
  * ``accumulate`` / ``evict`` keep the cache at a budget: attention weights per cached token, and the eviction of the
    tokens with the least of them from all layers.  From then on ``append`` takes the tokens' positions from a count of
    the tokens seen (``next_positions``), not from their places in the cache; the cos / sin tables then need a row for every
    token that a sequence will ever see, not for ``max_length`` of them.

The class itself allocates with torch and launches nothing; it works on any torch device (the operators do not).
"""
from __future__ import annotations

import contextlib
from typing import Optional, Tuple

import torch


_MXFP4 = getattr(torch, "float4_e2m1fn_x2", None)


def alloc_kv_pools(shape, dtype, device, zero: bool = True, v_shape=None) -> Tuple[torch.Tensor, torch.Tensor]:
    """A K pool and a V pool of ``shape`` (the V pool of ``v_shape``, if its rows have a length of their own) in ONE
    allocation, the V pool placed 256 bytes (modulo 512) off the K pool.

    Why the placement: MI355X's memory system tells two halves apart by address bit 8.  The rows of one kv head
    (``head_dim`` x element size bytes every ``Hkv`` rows) have that bit in common when the pools start on the usual
    large boundaries, and the K row and the V row of a token then meet in the same half; a workgroup that reads one
    kv head (the plan for batches that fill the GPU by themselves) keeps half of the memory system idle.  With the V
    pool shifted by 256 bytes its two streams go to different halves: measured, batch 32 x 8 kv heads x 4096 tokens,
    82.5 -> 80.3 us with a 16-bit cache and 48.9 -> 45.1 us with an fp8 cache; plans whose workgroups read two or more
    heads do not care (within 0.6 %).  Shapes, strides and dtypes are those of two separate tensors."""
    def bytes_of(sh):
        n = torch.empty((), dtype=dtype).element_size()
        for x in sh:
            n *= int(x)
        return n
    v_shape = tuple(shape) if v_shape is None else tuple(v_shape)
    nbytes, v_nbytes = bytes_of(shape), bytes_of(v_shape)
    span = (nbytes + 511) // 512 * 512
    make = torch.zeros if zero else torch.empty
    buf = make(span + v_nbytes + 1024, dtype=torch.uint8, device=device)
    base = (-buf.data_ptr()) % 512 if buf.is_cuda else 0
    k = buf[base: base + nbytes].view(dtype).view(shape)
    v = buf[base + span + 256: base + span + 256 + v_nbytes].view(dtype).view(v_shape)
    return k, v


class PagedKVCache:

    def __init__(self, PAGE_SIZE: int = 1, num_layers: int = 32, batch_size: int = 1, max_length: int = 1024,
                 num_kv_heads: int = 8, head_dim: int = 128, dtype=torch.bfloat16, *, device=None,
                 fill: str = "zeros", generator: Optional[torch.Generator] = None,
                 k_scale: Optional[torch.Tensor] = None, v_scale: Optional[torch.Tensor] = None) -> None:
        if PAGE_SIZE <= 0 or num_layers <= 0 or batch_size <= 0 or max_length <= 0:
            raise ValueError("PAGE_SIZE, num_layers, batch_size and max_length must be positive")
        if fill not in ("zeros", "randn"):
            raise ValueError("fill must be 'zeros' or 'randn'")
        if device is None:
            device = torch.device("cuda", torch.cuda.current_device())
        self.device = torch.device(device)
        self.page_size = PAGE_SIZE
        self.max_num_blocks_per_seq = (max_length + PAGE_SIZE - 1) // PAGE_SIZE
        self.num_layers = num_layers
        self.batch_size = batch_size
        self.max_length = max_length
        self.num_kv_heads = num_kv_heads
        self.head_dim = head_dim
        self.dtype = dtype
        num_blocks = self.max_num_blocks_per_seq * batch_size * num_layers
        if num_blocks >= 2 ** 31:
            raise ValueError("block ids are int32")
        shape = (num_blocks, PAGE_SIZE, num_kv_heads, head_dim)
        fp8 = dtype == torch.float8_e4m3fn
        self.mxfp4 = dtype == _MXFP4
        if self.mxfp4 and (fill != "zeros" or head_dim % 32):
            raise ValueError("an MXFP4 cache starts zeroed and has rows of a multiple of 32 values")
        if fp8:
            if k_scale is None or v_scale is None:
                raise ValueError("an fp8 cache needs k_scale and v_scale [num_layers, Hkv]")
            for s in (k_scale, v_scale):
                if tuple(s.shape) != (num_layers, num_kv_heads) or s.dtype != torch.float32:
                    raise ValueError("k_scale / v_scale must be fp32 [num_layers, Hkv]")
            self.k_scale = k_scale.to(self.device).contiguous()
            self.v_scale = v_scale.to(self.device).contiguous()
        else:
            self.k_scale = self.v_scale = None
        # (one allocation for both pools, the V pool 256 bytes off the K pool modulo 512: see alloc_kv_pools)
        self.k_block_scale = self.v_block_scale = None
        if self.mxfp4:
            # In memory [num_blocks, Hkv, PAGE_SIZE, ...]: a row is half a 128-byte line or less, and a decode workgroup, which
            # reads one kv head, then finds its rows side by side instead of sharing every line with the neighbouring head's
            # (4 sequences x 8 kv heads x 131072 tokens: 97 us against 106 us).
            by_head = (num_blocks, num_kv_heads, PAGE_SIZE)
            k, v = alloc_kv_pools(by_head + (head_dim // 2,), torch.uint8, self.device, zero=True)
            self.key_cache, self.value_cache = k.view(dtype).transpose(1, 2), v.view(dtype).transpose(1, 2)
            self.k_block_scale, self.v_block_scale = (
                torch.zeros(by_head + (head_dim // 32,), dtype=torch.uint8, device=self.device).transpose(1, 2) for _ in range(2))
        else:
            self.key_cache, self.value_cache = alloc_kv_pools(shape, dtype, self.device, zero=True)
        if fill == "randn":
            # drawn on the host so that a seed gives the same cache on every device
            draw = torch.bfloat16 if fp8 else dtype
            self.key_cache.copy_(torch.randn(shape, generator=generator, dtype=draw).to(dtype))
            self.value_cache.copy_(torch.randn(shape, generator=generator, dtype=draw).to(dtype))
        perm = torch.randperm(num_blocks, generator=generator).to(torch.int32)
        self.block_tables = perm.reshape(num_layers, batch_size, self.max_num_blocks_per_seq).to(self.device)
        self.kv_lens = torch.zeros(batch_size, dtype=torch.int32, device=self.device)
        self._host_len = 0
        self._seen = None               # [B] int32: tokens each sequence has seen, once some of them were evicted
        self._host_seen = 0             # the same count on the host

    # ---- the reference's interface -----------------------------------------------------------------------------
    def inc_offset(self, seq_len: int) -> None:
        """Every sequence grows by ``seq_len`` tokens (paged_kv_cache.py:52-54).  Call BEFORE appending them: the
        append operator expects lengths that already count the new tokens."""
        if seq_len < 0 or self._host_len + seq_len > self.max_length:
            raise ValueError(f"{self._host_len} + {seq_len} tokens exceed max_length = {self.max_length}")
        self.kv_lens += seq_len
        if self._seen is not None:
            self._seen += seq_len
        self._host_len += seq_len
        self._host_seen += seq_len

    def get_layer_kv_cache(self, layer_idx: int) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
        """``(key_cache, value_cache, block_table [B, max_blocks_per_seq], kv_lens [B])`` of one layer
        (paged_kv_cache.py:56-57); views, nothing is copied."""
        return self.key_cache, self.value_cache, self.block_tables[layer_idx], self.kv_lens

    # ---- additions ---------------------------------------------------------------------------------------------
    @property
    def max_kv_len(self) -> int:
        """Length of every sequence as the host knows it (all sequences advance together)."""
        return self._host_len

    @property
    def nbytes(self) -> int:
        scales = 0 if self.k_block_scale is None else self.k_block_scale.numel()
        return 2 * (self.key_cache.numel() * self.key_cache.element_size() + scales)

    def reset(self) -> None:
        """Forget all tokens; the pages keep their contents and their owners."""
        self.kv_lens.zero_()
        self._host_len = self._host_seen = 0
        self._seen = None

    def layer_scales(self, layer_idx: int):
        if self.mxfp4:
            return self.k_block_scale, self.v_block_scale          # a byte per row and block: pools like the rows'
        if self.k_scale is None:
            return None, None
        return self.k_scale[layer_idx], self.v_scale[layer_idx]

    def append(self, layer_idx: int, qkv: torch.Tensor, q_rms_weight: torch.Tensor, k_rms_weight: torch.Tensor,
               cos_cache: torch.Tensor, sin_cache: torch.Tensor, q_rms_eps: float = 1e-6, k_rms_eps: float = 1e-6,
               q_norm_rope: Optional[torch.Tensor] = None, stream=None, **kwargs) -> torch.Tensor:
        """Norm + rotary + append of ``qkv [B, T, Hq + 2 Hkv, D]`` into one layer, after ``inc_offset(T)``.
        ``positions`` / ``rope_sections`` / ``rope_interleaved`` as in ``qk_norm_rope_update_kvcache``; after an eviction
        ``positions`` defaults to ``next_positions(T)``, which the tables must have rows for.  Returns the normalised, rotated
        query ``[B, T, Hq, D]``."""
        from . import qk_norm_rope_update_kvcache
        if qkv.shape[1] > self._host_len:
            raise ValueError("call inc_offset(T) before append: kv_lens must count the new tokens")
        k, v, table, lens = self.get_layer_kv_cache(layer_idx)
        ks, vs = self.layer_scales(layer_idx)
        if self._seen is not None and kwargs.get("positions") is None:
            # (the operator turns a position behind the tables' end by their last row)
            if self._host_seen > min(cos_cache.shape[-2], sin_cache.shape[-2]):
                raise ValueError(f"the cos / sin tables have {cos_cache.shape[-2]} positions, the sequences have seen {self._host_seen} "
                                 "tokens: longer tables, or positions")
            with self._on(stream):
                kwargs["positions"] = self.next_positions(qkv.shape[1])
        return qk_norm_rope_update_kvcache(qkv, k, v, table, lens, q_rms_weight, k_rms_weight, cos_cache, sin_cache,
                                           q_norm_rope, q_rms_eps, k_rms_eps, k_scale=ks, v_scale=vs, stream=stream, **kwargs)

    def _on(self, stream):
        """torch's work in line with the kernels on ``stream``: it reads and holds what they read and write."""
        if stream is None:
            return contextlib.nullcontext()
        from .flash_decode import _on_stream, _stream_handle
        return _on_stream(self.device, _stream_handle(stream))

    def next_positions(self, new_tokens: int) -> torch.Tensor:
        """Positions ``[B, T]`` int32 of the T tokens that ``inc_offset(T)`` has just counted: how many tokens their
        sequence had seen before them, evicted ones among them."""
        seen = self.kv_lens if self._seen is None else self._seen
        return seen[:, None] - new_tokens + torch.arange(new_tokens, dtype=torch.int32, device=self.device)

    def accumulate(self, layer_idx: int, q: torch.Tensor, lse: torch.Tensor, sm_scale: float, weights: torch.Tensor, **kwargs):
        """``accumulate_attention_weights`` of a decode's query and lse over one layer; weights ``[B, Hkv, S]``."""
        from . import accumulate_attention_weights
        k, _, table, lens = self.get_layer_kv_cache(layer_idx)
        ks, _ = self.layer_scales(layer_idx)
        if ks is not None:
            kwargs.setdefault("k_scale", ks)
        return accumulate_attention_weights(q, k, table, lens, lse, sm_scale, weights, **kwargs)

    def evict(self, weights: torch.Tensor, keep: int, recent: int, stream=None) -> Optional[torch.Tensor]:
        """Bring every layer back to at most ``keep`` tokens by its weights ``[num_layers, B, Hkv, S]``, which move along
        (see ``evict_kvcache``).  Returns ``kept [num_layers, B, Hkv, keep]``, or None if nothing had to go.  Not to be captured
        into a graph: it changes the host's count of tokens, which a replay does not."""
        from . import evict_kvcache
        if weights.dim() != 4 or weights.shape[0] != self.num_layers or weights.shape[3] < self._host_len:
            raise ValueError(f"weights must be [{self.num_layers}, B, Hkv, S] with S >= {self._host_len} tokens")
        if self._host_len <= keep:
            return None
        with self._on(stream):
            from .flash_decode import _capturing
            if _capturing():
                raise ValueError("an eviction changes the host's count of tokens: not under graph capture (evict_kvcache can be captured)")
            kept = torch.empty((self.num_layers, self.batch_size, self.num_kv_heads, keep), dtype=torch.int32, device=self.device)
            seen = self.kv_lens.clone() if self._seen is None else self._seen
        scales = {} if not self.mxfp4 else dict(k_scale=self.k_block_scale, v_scale=self.v_block_scale)
        for layer in range(self.num_layers):
            # (the layers share kv_lens: the last one changes it)
            lens_out = self.kv_lens if layer == self.num_layers - 1 else None
            evict_kvcache(self.key_cache, self.value_cache, self.block_tables[layer], self.kv_lens, weights[layer], keep, recent,
                          weights_out=weights[layer], kept=kept[layer], kv_lens_out=lens_out, stream=stream, **scales)
        self._seen = seen
        self._host_len = keep
        return kept

    def decode(self, layer_idx: int, q: torch.Tensor, sm_scale: float, **kwargs):
        """``flash_decode`` of ``q [B, Hq, D]`` over one layer, planned for the host-known length.
        Returns ``(out [B, Hq, D], lse [B, Hq] fp32)``."""
        from . import flash_decode
        k, v, table, lens = self.get_layer_kv_cache(layer_idx)
        ks, vs = self.layer_scales(layer_idx)
        if ks is not None:
            kwargs.setdefault("k_scale", ks)
            kwargs.setdefault("v_scale", vs)
        kwargs.setdefault("max_kv_len", max(self._host_len, 1))
        kwargs.setdefault("min_kv_len", self._host_len)          # all sequences advance together
        return flash_decode(q, k, v, table, lens, sm_scale, **kwargs)
