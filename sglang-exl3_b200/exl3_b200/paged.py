"""Paged key-value cache over the C ABI: tokens appended with the position rotation
applied on the way (``rope_append``), and the attention of each sequence's newest tokens
over its pages (``attention``).

A layer's cache is a pair of tensors ``[pages, page_size, kv_heads, head_dim]`` (any stride
order whose last dimension is contiguous, e.g. a permuted ``[pages, kv_heads, page_size,
head_dim]`` pool), fp16, bf16 or ``float8_e4m3fn`` with one fp32 scale per kv head.  A slot
is ``page * page_size + offset``.  Sequences have lengths of their own, read on the device:
both calls are CUDA-graph capturable and keep working as the lengths grow.

The fused sub-layers of ``exl3_b200.decode`` read a dense cache with one position for the
whole batch; these operators serve batches whose sequences differ, around the EXL3 linears
(``ops.matmul_multi`` for q/k/v, ``ops.matmul`` for o).
"""

from __future__ import annotations

import functools
from typing import Optional, Tuple, Union

import torch

from . import _lib

_IN = {torch.float16: _lib.DTYPE_F16, torch.bfloat16: _lib.DTYPE_BF16, torch.float32: _lib.DTYPE_F32}
_CACHE = {torch.float16: _lib.DTYPE_F16, torch.bfloat16: _lib.DTYPE_BF16, torch.float8_e4m3fn: _lib.DTYPE_E4M3}


_E4M3 = torch.float8_e4m3fn


def _cache(k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: Optional[torch.Tensor],
           v_scale: Optional[torch.Tensor]) -> tuple:
    """The fields of ``exl3b200_paged_cache``."""
    if not k_cache.is_cuda:
        raise RuntimeError("EXL3 B200 ops require CUDA tensors (there is no CPU path)")
    dtype, shape, strides = k_cache.dtype, k_cache.shape, k_cache.stride()
    if dtype not in _CACHE or len(shape) != 4 or shape[3] not in (64, 128):
        raise RuntimeError("caches must be fp16, bf16 or float8_e4m3fn [pages, page_size, kv_heads, 64 or 128]")
    if v_cache.dtype != dtype or v_cache.shape != shape or v_cache.stride() != strides:
        raise RuntimeError("k and v caches must have the same type, shape and strides")
    pages, page_size, kv_heads, dim = shape
    s0, s1, s2, s3 = strides
    if s3 != 1:
        raise RuntimeError("caches must have unit stride in their last dimension")
    if not (pages and page_size and kv_heads):
        raise RuntimeError("caches must not be empty")
    if pages == 1:
        s0 = 0
    if page_size == 1:
        s1 = 0
    if kv_heads == 1:
        s2 = 0
    if (pages > 1 and not s0) or (page_size > 1 and not s1) or (kv_heads > 1 and not s2):
        raise RuntimeError("caches must not be expanded views")
    ks = vs = 0
    if k_scale is not None:
        ks = _scale(k_scale, dtype, kv_heads)
    if v_scale is not None:
        vs = _scale(v_scale, dtype, kv_heads)
    return (k_cache.data_ptr(), v_cache.data_ptr(), _CACHE[dtype], pages, page_size, kv_heads, dim, s0, s1, s2, ks, vs)


def _scale(s: torch.Tensor, dtype: torch.dtype, kv_heads: int) -> int:
    if dtype != _E4M3:
        raise RuntimeError("k_scale and v_scale belong to float8_e4m3fn caches")
    if s.dtype != torch.float32 or s.numel() != kv_heads or not s.is_contiguous():
        raise RuntimeError("k_scale and v_scale must be contiguous fp32 [kv_heads]")
    return s.data_ptr()


def _device(index: int, *tensors: Optional[torch.Tensor]) -> None:
    for t in tensors:
        if t is not None and t.get_device() != index:
            raise RuntimeError("paged tensors must share a CUDA device")


@functools.lru_cache(maxsize=4096)
def _scratch_size(rows_per_seq: int, heads: int, kv_heads: int, dim: int) -> int:
    return _lib.lib().exl3b200_paged_attention_scratch_size(rows_per_seq, heads, kv_heads, dim)


def _rows(t: torch.Tensor, copy: bool = True):
    """An input [rows, heads, head_dim] whose heads begin on 16-byte boundaries (itself, or a
    copy), its address and its row and head strides; None where it is not and may not be copied."""
    s0, s1, s2 = t.stride()
    p = t.data_ptr()
    vec = 4 if t.dtype == torch.float32 else 8
    if s2 != 1 or (s0 | s1) % vec or p % 16:
        # (the stride of a dimension of one does not count)
        s0, s1 = s0 if t.size(0) > 1 else 0, s1 if t.size(1) > 1 else 0
        if s2 != 1 or (s0 | s1) % vec or p % 16:
            return _rows(t.clone(memory_format=torch.contiguous_format), False) if copy else None
    return t, p, s0, s1


def rope_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                positions: torch.Tensor, slots: torch.Tensor, inv_freq: torch.Tensor,
                q_out: Optional[torch.Tensor] = None, interleaved: bool = False,
                k_scale: Optional[torch.Tensor] = None, v_scale: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Rotate ``q`` and ``k`` by their tokens' ``positions`` and write ``k`` and ``v`` into
    the caches' ``slots`` (``exl3b200_rope_append``); returns the rotated q.

    ``q [tokens, q_heads, head_dim]``, ``k``/``v [tokens, kv_heads, head_dim]``: fp16, bf16
    or fp32, e.g. column slices of one fused q/k/v output.  ``inv_freq`` fp32: the first
    ``2 * len(inv_freq)`` dims of a head turn (a multiple of 16), in pairs (i, i + r/2), or
    (2i, 2i + 1) with ``interleaved``.  ``positions`` and ``slots``: int64 ``[tokens]``; a
    negative slot writes nothing (padding rows), one past the pool neither, and is recorded
    in ``ops.device_status``.  The slots of one call must differ.  ``q_out`` (default: new,
    in the cache's type, bf16 for an e4m3 cache) may be ``q``; an expanded view is refused."""
    c = _cache(k_cache, v_cache, k_scale, v_scale)
    index = k_cache.get_device()
    if not (q.get_device() == k.get_device() == v.get_device() == positions.get_device() == slots.get_device()
            == inv_freq.get_device() == index):
        raise RuntimeError("paged tensors must share a CUDA device")
    _device(index, v_cache, q_out, k_scale, v_scale)
    src, cache = q.dtype, k_cache.dtype
    if src not in _IN or k.dtype != src or v.dtype != src:
        raise RuntimeError("q, k and v must be of one type: fp16, bf16 or fp32")
    shape = q.shape
    if len(shape) != 3 or shape[2] != c[6]:
        raise RuntimeError("q must be [tokens, q_heads, head_dim]")
    tokens, heads, dim = shape
    if k.shape != (tokens, c[5], dim) or v.shape != k.shape:
        raise RuntimeError("k and v must be [tokens, kv_heads, head_dim]")
    if (positions.dtype != torch.int64 or slots.dtype != torch.int64 or positions.shape != (tokens,)
            or slots.shape != (tokens,)):
        raise RuntimeError("positions and slots must be int64 [tokens]")
    rotary = 2 * inv_freq.numel()
    if inv_freq.dtype != torch.float32 or rotary > dim or rotary % 16:
        raise RuntimeError("inv_freq must be fp32 with half of the rotated dims, a multiple of 8 up to head_dim / 2")
    if q_out is None:
        q_out = torch.empty_like(q, dtype=torch.bfloat16 if cache == _E4M3 else cache,
                                 memory_format=torch.contiguous_format)
    elif q_out.shape != shape or q_out.dtype not in (torch.float16, torch.bfloat16):
        raise RuntimeError("q_out must be fp16 or bf16, shaped like q")
    elif cache != _E4M3 and q_out.dtype != cache:
        raise RuntimeError("q_out must have the cache's type")
    if tokens == 0 or heads == 0:
        return q_out
    out = _rows(q_out, copy=False)
    if out is None:
        raise RuntimeError("q_out's heads must begin on 16-byte boundaries with unit stride")
    q, qp, q0, q1 = _rows(q)
    k, kp, k0, k1 = _rows(k)
    v, vp, v0, v1 = _rows(v)
    positions, slots, inv_freq = positions.contiguous(), slots.contiguous(), inv_freq.contiguous()
    args = _lib.pack_rope_append(*c, qp, kp, vp, out[1], positions.data_ptr(), slots.data_ptr(), inv_freq.data_ptr(),
                                 q0, q1, k0, k1, v0, v1, out[2], out[3], tokens, heads, rotary, bool(interleaved),
                                 _IN[src], _IN[q_out.dtype])
    _lib.launch("exl3b200_rope_append", index, args)
    return q_out


def attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor,
              seq_lens: torch.Tensor, rows_per_seq: int = 1, scale: Optional[float] = None, softcap: float = 0.0,
              window: int = 0, k_scale: Optional[torch.Tensor] = None, v_scale: Optional[torch.Tensor] = None,
              out: Optional[torch.Tensor] = None,
              return_lse: bool = False) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """Attention of each sequence's newest ``rows_per_seq`` tokens over its pages
    (``exl3b200_paged_attention``).

    ``q [sequences * rows_per_seq, q_heads, head_dim]`` fp16 or bf16 (the caches' type
    unless that is e4m3), rotated; rows ``R s + j`` are sequence ``s``'s tokens at positions
    ``seq_lens[s] - R + j``, whose keys and values the caches hold already.  A row sees the
    positions up to its own, of those the last ``window`` when that is positive.
    ``block_table`` int32 ``[sequences, max_pages]`` (entries past a sequence's pages, or
    before its window, are not read), ``seq_lens`` int32 ``[sequences]``.  ``scale`` defaults
    to ``head_dim ** -0.5``; ``softcap`` > 0 caps scores at ``softcap * tanh(s / softcap)``.
    Rows that see nothing (an empty sequence) are zeros, their ``lse`` is -inf.  Returns
    ``out`` (q's type; a given one must not be an expanded view), with ``return_lse`` also
    fp32 ``lse [rows, q_heads]``."""
    c = _cache(k_cache, v_cache, k_scale, v_scale)
    index = k_cache.get_device()
    if not q.get_device() == block_table.get_device() == seq_lens.get_device() == index:
        raise RuntimeError("paged tensors must share a CUDA device")
    _device(index, v_cache, k_scale, v_scale, out)
    dtype, shape = q.dtype, q.shape
    if dtype not in (torch.float16, torch.bfloat16) or len(shape) != 3 or shape[2] != c[6]:
        raise RuntimeError("q must be fp16 or bf16 [rows, q_heads, head_dim]")
    if k_cache.dtype not in (dtype, _E4M3):
        raise RuntimeError("q must have the caches' type (or the caches be float8_e4m3fn)")
    rows, heads, dim = shape
    kv_heads, R, window, softcap = c[5], int(rows_per_seq), int(window), float(softcap)
    if block_table.dtype != torch.int32 or block_table.dim() != 2 or block_table.stride(1) != 1:
        raise RuntimeError("block_table must be int32 [sequences, max_pages] with unit column stride")
    seqs, max_pages = block_table.shape
    if seq_lens.dtype != torch.int32 or seq_lens.shape != (seqs,) or not seq_lens.is_contiguous():
        raise RuntimeError("seq_lens must be contiguous int32 [sequences]")
    if R < 1 or rows != seqs * R or max_pages < 1:
        raise RuntimeError("q must have rows_per_seq rows for each sequence, block_table a column")
    if heads < 1 or heads % kv_heads or R * (heads // kv_heads) > _lib.PAGED_MAX_ROWS:
        raise RuntimeError(f"q_heads must be a multiple of kv_heads, rows_per_seq * group at most {_lib.PAGED_MAX_ROWS}")
    if window < 0 or not (softcap == 0.0 or 1e-6 <= softcap < float("inf")):
        raise RuntimeError("window must not be negative, softcap 0 or at least 1e-6")
    scale = dim ** -0.5 if scale is None else float(scale)
    if not 0.0 < scale < float("inf"):
        raise RuntimeError("scale must be positive")
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
        op, o0, o1 = out.data_ptr(), heads * dim, dim
    else:
        got = _rows(out, copy=False) if out.shape == shape and out.dtype == dtype else None
        if got is None:
            raise RuntimeError("out must be shaped like q, of its type, heads on 16-byte boundaries with unit stride")
        _, op, o0, o1 = got
    lse = q.new_empty((rows, heads), dtype=torch.float32) if return_lse else None
    if rows:
        q, qp, q0, q1 = _rows(q)
        n = _scratch_size(R, heads, kv_heads, dim)
        # the scratch is the call's own (a captured graph keeps its own, too)
        scratch = q.new_empty(n, dtype=torch.uint8)
        args = _lib.pack_paged_attention(*c, qp, op, lse.data_ptr() if return_lse else 0, block_table.data_ptr(),
                                         seq_lens.data_ptr(), q0, q1, o0, o1,
                                         block_table.stride(0) if seqs > 1 else max_pages, seqs, R, heads, max_pages,
                                         min(window, 2 ** 31 - 1), _IN[dtype], scale, softcap)
        _lib.launch("exl3b200_paged_attention", index, args, scratch.data_ptr(), n)
    return (out, lse) if return_lse else out
