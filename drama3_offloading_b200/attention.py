"""What Drama-3's full-attention layers do around the cache, served by libd3b200.so.

* ``qk_norm_rope`` -- the RMS norm of every query and key head and the rotation
  by position, one pass; ``qk_norm_rope_write`` also puts K and V into a
  ``kvcache.PagedKV``.
* ``paged_attention`` -- causal attention of new tokens over the cache: single
  decode tokens, a few drafted ones, prefill chunks, or a ragged mix of them.

No call syncs; each allocates only its outputs and workspace from torch's
allocator, so any of them can be captured in a CUDA graph, and calls on
different streams share nothing.  A bounded wait that ran out inside a kernel
is reported by ``moe.check_errors()``.
"""
from __future__ import annotations

import torch

from . import _lib
from .kvcache import (DTYPES, PagedKV, _raw_stream, elsewhere, fresh, in_place, index, output, place,
                      rows)


def rope_frequencies(rotary_dim: int, theta: float = 10000.0, device="cuda") -> torch.Tensor:
    """``theta ** (-2 i / rotary_dim)`` for the pairs i: float64 [rotary_dim / 2]."""
    i = torch.arange(0, rotary_dim, 2, dtype=torch.float64, device=device)
    return theta ** (-i / rotary_dim)


def _norm_rope(q, k, v, q_weight, k_weight, positions, inv_freq, cache, slots, eps, weight_offset,
               interleaved, out, stream):
    dtype, dev = q.dtype, q.get_device()
    if dtype is not torch.bfloat16 and dtype is not torch.float16:
        raise TypeError(f"q must be bfloat16 or float16, got {dtype}")
    if q.dim() != 3 or k.dim() != 3:
        raise ValueError("q and k must be [tokens, heads, head_dim]")
    tokens, heads, dim = q.shape
    kv_heads = k.shape[1]
    rows(k, "k", kv_heads, dim, dtype, dev)
    if k.shape[0] != tokens:
        raise ValueError("q and k must have the same tokens")
    for w in (q_weight, k_weight):
        if w.dtype is not dtype or w.numel() != dim:
            raise TypeError(f"q_weight and k_weight must be {dtype} [{dim}]")
        if w.get_device() != dev:
            raise ValueError(f"a weight is on {w.device}, not on device {dev}")
    if inv_freq.dtype is not torch.float64 or inv_freq.dim() != 1:
        raise TypeError("inv_freq must be float64 [rotary_dim / 2]")
    if inv_freq.get_device() != dev:
        raise ValueError(f"inv_freq is on {inv_freq.device}, not on device {dev}")
    index(positions, "positions", tokens, dev)
    if cache is not None:
        cache.rows_dtype(dtype)
        rows(v, "v", kv_heads, dim, dtype, dev)
        if v.shape[0] != tokens or cache.kv_heads != kv_heads or cache.head_dim != dim:
            raise ValueError("v and the cache must have k's tokens and heads")
        if cache.device_index != dev:
            raise ValueError(f"the cache is on {cache.device}, not on device {dev}")
        index(slots, "slots", tokens, dev)
    if elsewhere(dev, stream):
        with place(dev, stream):
            return _norm_rope(q, k, v, q_weight, k_weight, positions, inv_freq, cache, slots, eps,
                              weight_offset, interleaved, out, None)
    q, q_at, q0, q1 = in_place(q)
    k, k_at, k0, k1 = in_place(k)
    q_weight, k_weight = q_weight.contiguous(), k_weight.contiguous()
    qw, kw = q_weight.data_ptr(), k_weight.data_ptr()
    if (qw | kw) & 15:
        q_weight, k_weight = q_weight.clone(), k_weight.clone()
        qw, kw = q_weight.data_ptr(), k_weight.data_ptr()
    positions, inv_freq = positions.contiguous(), inv_freq.contiguous()
    qo, ko = out if isinstance(out, tuple) else (out, None)
    qo, qo_at, qo0, qo1 = fresh(q, heads, dim) if qo is None else output(qo, q.shape, dtype, dev)
    if cache is None:
        ko, ko_at, ko0, ko1 = fresh(k, kv_heads, dim) if ko is None else output(ko, k.shape, dtype, dev)
        v_at, v0, v1, slots_at, slot_bytes, ref = 0, 0, 0, 0, 4, None
    else:
        v, v_at, v0, v1 = in_place(v)
        slots = slots.contiguous()
        ko_at, ko0, ko1 = 0, 0, 0
        slots_at, slot_bytes, ref = slots.data_ptr(), slots.element_size(), cache.ref
    rc = _lib.packed("d3_qk_norm_rope")(_lib.NORM_ROPE.pack(
        q_at, k_at, v_at, q0, q1, k0, k1, v0, v1, qo_at, ko_at, qo0, qo1, ko0, ko1, qw, kw,
        positions.data_ptr(), inv_freq.data_ptr(), slots_at, positions.element_size(), slot_bytes,
        tokens, heads, kv_heads, dim, 2 * inv_freq.shape[0], 1 if interleaved else 0, DTYPES[dtype],
        eps, weight_offset), ref, _raw_stream(dev))
    if rc:
        _lib.raise_status(rc, "d3_qk_norm_rope")
    return qo, ko


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, q_weight: torch.Tensor,
                 k_weight: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor, *,
                 eps: float = 1e-6, weight_offset: float = 0.0, interleaved: bool = False,
                 out: tuple | None = None, stream=None):
    """Norm and rotation of q ``[tokens, heads, head_dim]`` and k ``[tokens,
    kv_heads, head_dim]`` (bf16 or fp16; views of a wider projection are read
    in place): ``x / sqrt(mean(x^2) + eps) * (weight + weight_offset)`` for each
    head, then the first ``2 * len(inv_freq)`` dims turned by
    ``positions * inv_freq`` in pairs of halves (or, ``interleaved``, of
    neighbours).  ``weight_offset=1`` for zero-centred weights.  ``out=(q_out,
    k_out)`` may be ``(q, k)``.  The mean is float32, the angle float64;
    len(inv_freq) is a multiple of 8.  Returns (q, k)."""
    return _norm_rope(q, k, None, q_weight, k_weight, positions, inv_freq, None, None, eps,
                      weight_offset, interleaved, out, stream)


def qk_norm_rope_write(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, q_weight: torch.Tensor,
                       k_weight: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor,
                       cache: PagedKV, slots: torch.Tensor, *, eps: float = 1e-6,
                       weight_offset: float = 0.0, interleaved: bool = False,
                       out: torch.Tensor | None = None, stream=None) -> torch.Tensor:
    """``qk_norm_rope`` whose K, and V as it is, go straight into ``cache`` at
    ``slots`` (as ``kvcache.write`` would put them; K is rounded once, from
    fp32).  ``out`` may be ``q``.  Returns q."""
    return _norm_rope(q, k, v, q_weight, k_weight, positions, inv_freq, cache, slots, eps,
                      weight_offset, interleaved, out, stream)[0]


def paged_attention(q: torch.Tensor, cache: PagedKV, page_table: torch.Tensor,
                    kv_lens: torch.Tensor, cu_q: torch.Tensor | None = None, *, max_q: int = 1,
                    max_kv: int | None = None, scale: float | None = None,
                    out: torch.Tensor | None = None, stream=None) -> torch.Tensor:
    """softmax(scale * q k^T) v of new tokens over their sequences' cached keys.

    q ``[tokens, heads, head_dim]``; sequence b has the rows ``cu_q[b] ..
    cu_q[b + 1]`` (int32 ``[batch + 1]``; None: one row a sequence), the last of
    its ``kv_lens[b]`` (int32) cached tokens, so row i of n sees the keys
    ``[0, kv_lens[b] - n + i]``; a row that sees none gives zeros.  Key j lies
    in page ``page_table[b, j // page_size]`` (int32 ``[batch, pages]``); ids
    outside the cache read as zeros.  Lengths behind the table's width count as
    the width.  ``max_q`` and ``max_kv`` bound the new tokens and the length of
    a sequence (default: one token, the table's width); they choose the launch:
    a sequence that exceeds them is answered too, more slowly.  ``scale``
    defaults to head_dim ** -0.5.  ``out`` may be ``q``; rows of it behind the
    last sequence are left as they were.

    A row whose visible scores hold NaN or +inf, or -inf alone, gives NaN, as the
    formula does; a score of -inf among others takes its key away.  Keys that a
    row's mask hides may hold anything.  Values are multiplied by
    zero there: an infinity or NaN in V reaches rows of the same sequence and
    call that do not see its key; over codes, with float16 queries and more than
    16 rows of a KV head, that holds for values which float16 cannot hold, too.

    Scores and sums are float32.  Probabilities are rounded to q's type before
    they meet V (over codes and up to 16 rows of a KV head to float16, the values'
    scales in them): about 1.4 times the error of rounding the result alone."""
    if q.dim() != 3:
        raise ValueError("q must be [tokens, heads, head_dim]")
    tokens, heads, dim = q.shape
    dev, dtype = q.get_device(), q.dtype
    code = cache.rows_dtype(dtype)
    kv_heads = cache.kv_heads
    if dim != cache.head_dim:
        raise ValueError(f"q's head_dim {dim}, the cache's {cache.head_dim}")
    if heads % kv_heads or heads // kv_heads > 128:
        raise ValueError(f"{heads} heads over {kv_heads} KV heads")
    if page_table.dtype is not torch.int32 or page_table.dim() != 2:
        raise TypeError("page_table must be int32 [batch, pages]")
    batch, pages = page_table.shape
    index(kv_lens, "kv_lens", batch, dev)
    if cu_q is not None:
        index(cu_q, "cu_q", batch + 1, dev)
    elif tokens < batch:
        raise ValueError(f"{tokens} rows for {batch} sequences of one row each")
    if kv_lens.dtype is not torch.int32 or (cu_q is not None and cu_q.dtype is not torch.int32):
        raise TypeError("kv_lens and cu_q must be int32")
    if cache.device_index != dev or page_table.get_device() != dev:
        raise ValueError(f"the cache or page_table is not on q's device {q.device}")
    if max_q < 1:
        raise ValueError("max_q must be at least 1")
    if scale is None:
        scale = dim ** -0.5
    elif not 0.0 < scale < float("inf"):
        raise ValueError(f"scale {scale}: must be positive")
    top = pages * cache.page_size
    max_kv = top if max_kv is None else max(0, min(max_kv, top))
    if out is not None:
        out, o_at, o0, o1 = output(out, q.shape, dtype, dev)
    if elsewhere(dev, stream):
        with place(dev, stream):
            return paged_attention(q, cache, page_table, kv_lens, cu_q, max_q=max_q, max_kv=max_kv,
                                   scale=scale, out=out)
    q, q_at, q0, q1 = in_place(q)
    kv_lens = kv_lens.contiguous()
    cu_at = 0
    if cu_q is not None:
        cu_q = cu_q.contiguous()
        cu_at = cu_q.data_ptr()
    t0, t1 = page_table.stride()
    if t1 != 1:
        page_table = page_table.contiguous()
        t0 = page_table.stride(0)
    if out is None:
        out, o_at, o0, o1 = fresh(q, heads, dim)
    if max_q > tokens:
        max_q = tokens or 1
    a = _lib.ATTENTION.pack(q_at, q0, q1, o_at, o0, o1, page_table.data_ptr(), t0, kv_lens.data_ptr(),
                            cu_at, pages, batch, tokens, heads, max_q, max_kv, code, scale)
    # the workspace depends on the kernels that max_q asks for alone
    key = max_q * (heads // kv_heads) > 16
    need = cache.workspace.get(key)
    if need is None:
        need = _lib.load().d3_paged_attention_workspace_size(
            _lib.Attention.from_buffer_copy(a), _lib.KVCache.from_address(cache.ref))
        if need:
            cache.workspace[key] = need
    ws = q.new_empty(need // 2 or 8)
    rc = _lib.packed("d3_paged_attention")(a, cache.ref, cache.error_word.data_ptr(), ws.data_ptr(),
                                           need, _raw_stream(dev))
    if rc:
        _lib.raise_status(rc, "d3_paged_attention")
    return out
