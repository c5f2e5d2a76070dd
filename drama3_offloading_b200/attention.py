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

from . import _lib, moe
from .kvcache import DTYPES, PagedKV, aligned, index, on_device, rows


def rope_frequencies(rotary_dim: int, theta: float = 10000.0, device="cuda") -> torch.Tensor:
    """``theta ** (-2 i / rotary_dim)`` for the pairs i: float64 [rotary_dim / 2]."""
    i = torch.arange(0, rotary_dim, 2, dtype=torch.float64, device=device)
    return theta ** (-i / rotary_dim)


def _norm_rope(q, k, v, q_weight, k_weight, positions, inv_freq, cache, slots, eps, weight_offset,
               interleaved, out, stream):
    if q.dtype not in (torch.bfloat16, torch.float16):
        raise TypeError(f"q must be bfloat16 or float16, got {q.dtype}")
    if q.dim() != 3 or k.dim() != 3:
        raise ValueError("q and k must be [tokens, heads, head_dim]")
    tokens, heads, dim = q.shape
    kv_heads, dev = k.shape[1], q.device
    q, k = rows(q, "q", heads, dim, q.dtype), rows(k, "k", kv_heads, dim, q.dtype)
    if k.shape[0] != tokens:
        raise ValueError("q and k must have the same tokens")
    for w, name in ((q_weight, "q_weight"), (k_weight, "k_weight")):
        if w.dtype != q.dtype or w.numel() != dim:
            raise TypeError(f"{name} must be {q.dtype} [{dim}]")
    q_weight, k_weight = q_weight.contiguous(), k_weight.contiguous()
    if inv_freq.dtype != torch.float64 or inv_freq.dim() != 1:
        raise TypeError("inv_freq must be float64 [rotary_dim / 2]")
    inv_freq = inv_freq.contiguous()
    positions = index(positions, "positions", tokens, dev)
    for t in (k, q_weight, k_weight, inv_freq):
        if t.device != dev:
            raise ValueError(f"a tensor is on {t.device}, q on {dev}")
    if cache is not None:
        cache.rows_dtype(q.dtype)
        v = rows(v, "v", kv_heads, dim, q.dtype)
        if v.shape[0] != tokens or cache.kv_heads != kv_heads or cache.head_dim != dim:
            raise ValueError("v and the cache must have k's tokens and heads")
        if v.device != dev or cache.device != dev:
            raise ValueError(f"v or the cache is not on {dev}")
        slots = index(slots, "slots", tokens, dev)

    def take(t, like, name):
        if t is None:
            return torch.empty(like.shape, dtype=like.dtype, device=dev)
        if t.shape != like.shape or t.dtype != like.dtype or t.device != dev or not aligned(t):
            raise ValueError(f"{name} must be {like.dtype} {tuple(like.shape)} on {dev}, its rows "
                             "contiguous on 16-byte boundaries")
        return t

    def go(st):
        qo, ko = (out if isinstance(out, tuple) else (out, None)) if out is not None else (None, None)
        qo = take(qo, q, "out")
        ko = take(ko, k, "out") if cache is None else None
        a = _lib.NormRope(
            q.data_ptr(), k.data_ptr(), v.data_ptr() if cache is not None else None,
            q.stride(0), q.stride(1), k.stride(0), k.stride(1),
            v.stride(0) if cache is not None else 0, v.stride(1) if cache is not None else 0,
            qo.data_ptr(), ko.data_ptr() if ko is not None else None, qo.stride(0), qo.stride(1),
            ko.stride(0) if ko is not None else 0, ko.stride(1) if ko is not None else 0,
            q_weight.data_ptr(), k_weight.data_ptr(), positions.data_ptr(), inv_freq.data_ptr(),
            slots.data_ptr() if cache is not None else None, positions.element_size(),
            slots.element_size() if cache is not None else 4, tokens, heads, kv_heads, dim,
            2 * inv_freq.shape[0], 1 if interleaved else 0, DTYPES[q.dtype], eps, weight_offset)
        _lib.call("d3_qk_norm_rope", a, cache.ref if cache is not None else None, st)
        return qo, ko
    return on_device(dev, go, stream=stream)


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
    k_out)`` may be ``(q, k)``.  Returns (q, k)."""
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
    outside the cache read as zeros.  ``max_q`` and ``max_kv`` bound the new
    tokens and the length of a sequence (they choose the launch; default: one
    token, the table's width).  ``scale`` defaults to head_dim ** -0.5.  Rows
    of ``out`` behind the last sequence are left as they were."""
    if q.dim() != 3:
        raise ValueError("q must be [tokens, heads, head_dim]")
    tokens, heads, dim = q.shape
    dev = q.device
    code = cache.rows_dtype(q.dtype)
    q = rows(q, "q", heads, cache.head_dim, q.dtype)
    if heads % cache.kv_heads or heads // cache.kv_heads > 128:
        raise ValueError(f"{heads} heads over {cache.kv_heads} KV heads")
    if page_table.dtype != torch.int32 or page_table.dim() != 2:
        raise TypeError("page_table must be int32 [batch, pages]")
    if page_table.stride(1) != 1:
        page_table = page_table.contiguous()
    batch, pages = page_table.shape
    kv_lens = index(kv_lens, "kv_lens", batch, dev)
    if cu_q is not None:
        cu_q = index(cu_q, "cu_q", batch + 1, dev)
    elif tokens < batch:
        raise ValueError(f"{tokens} rows for {batch} sequences of one row each")
    if kv_lens.dtype != torch.int32 or (cu_q is not None and cu_q.dtype != torch.int32):
        raise TypeError("kv_lens and cu_q must be int32")
    if cache.device != dev or page_table.device != dev:
        raise ValueError(f"the cache or page_table is not on {dev}")
    if max_q < 1:
        raise ValueError("max_q must be at least 1")
    scale = dim ** -0.5 if scale is None else float(scale)
    if not 0.0 < scale < float("inf"):
        raise ValueError(f"scale {scale}: must be positive")
    top = pages * cache.page_size
    max_kv = top if max_kv is None else min(max_kv, top)
    if out is not None and (out.shape != q.shape or out.dtype != q.dtype or out.device != dev
                            or not aligned(out)):
        raise ValueError(f"out must be {q.dtype} {tuple(q.shape)} on {dev}, its rows contiguous on "
                         "16-byte boundaries")

    def go(st):
        o = out if out is not None else torch.empty(tokens, heads, dim, dtype=q.dtype, device=dev)
        a = _lib.Attention(
            q.data_ptr(), q.stride(0), q.stride(1), o.data_ptr(), o.stride(0), o.stride(1),
            page_table.data_ptr(), page_table.stride(0), kv_lens.data_ptr(),
            cu_q.data_ptr() if cu_q is not None else None, pages, batch, tokens, heads,
            min(max_q, max(tokens, 1)), max(max_kv, 0), code,
            scale)
        need = _lib.load().d3_paged_attention_workspace_size(a, cache.ref)
        ws = torch.empty(max(need, 16), dtype=torch.uint8, device=dev)
        _lib.call("d3_paged_attention", a, cache.ref, moe.error_word(dev).data_ptr(),
                  ws.data_ptr(), need, st)
        return o
    return on_device(dev, go, stream=stream)
