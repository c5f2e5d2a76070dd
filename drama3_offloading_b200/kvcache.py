"""Paged K/V cache of one attention layer, 16-bit or e4m3, served by libd3b200.so.

* ``PagedKV`` holds the buffers: pages of ``page_size`` tokens, every KV head's
  rows of a page together (``[pages, kv_heads, page_size, head_dim]``).  A
  token's *slot* is ``page * page_size + offset``.
* ``write(cache, k, v, slots)`` puts new rows in, quantising them where the
  cache is e4m3: one fp32 scale ``max|row| / 448`` per (token, head), the row
  as codes ``e4m3(row / scale)``.
* ``read(cache, slots)`` gives rows back as 16-bit values.

``attention.qk_norm_rope_write`` fills the cache in the same pass as the norm
and rotation, ``attention.paged_attention`` reads it.  All of it is free of
host syncs and allocates only outputs, so a decode step that uses it can be
captured in a CUDA graph.

The reference keeps attention state in upstream fish-speech's dense buffers
(bin/prefix_kv.py:184-339 snapshots them); paging and quantising are this
framework's own.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib, moe

DTYPES = {torch.bfloat16: _lib.D3_BF16, torch.float16: _lib.D3_F16,
          torch.float8_e4m3fn: _lib.D3_E4M3}


_device = torch._C._cuda_getDevice if hasattr(torch._C, "_cuda_getDevice") else torch.cuda.current_device
if hasattr(torch._C, "_cuda_getCurrentRawStream"):
    _raw_stream = torch._C._cuda_getCurrentRawStream
else:
    def _raw_stream(index):
        return torch.cuda.current_stream(index).cuda_stream


def elsewhere(device: torch.device, stream) -> bool:
    """Whether a call on ``device`` and ``stream`` (None: the current one) needs
    ``place`` around it -- and around the copies it may make of its arguments."""
    if device.type != "cuda":
        raise ValueError(f"tensors on {device}: a CUDA device is needed")
    return stream is not None or _device() != device.index


def place(device: torch.device, stream):
    """Context in which ``device`` is the current device and ``stream`` (or the
    device's current one) its current stream: outputs and workspaces made in it
    belong to that stream."""
    return torch.cuda.stream(stream if stream is not None else torch.cuda.current_stream(device))


def rows(t: torch.Tensor, name: str, heads: int, dim: int, dtype) -> None:
    """Checks ``t`` as [tokens, heads, dim] rows of ``dtype``."""
    if t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    shape = t.shape
    if len(shape) != 3 or shape[1] != heads or shape[2] != dim:
        raise ValueError(f"{name} must be [tokens, {heads}, {dim}], got {tuple(shape)}")


def in_place(t: torch.Tensor) -> torch.Tensor:
    """``t``, or a copy if its rows do not lie as the kernels read them:
    contiguous dims, rows on 16-byte boundaries."""
    if not aligned(t):
        t = t.contiguous()
        if t.data_ptr() % 16:
            t = t.clone()
    return t


def aligned(t: torch.Tensor) -> bool:
    s = t.stride()
    return (s[2] == 1 and s[0] % 8 == 0 and s[1] % 8 == 0 and s[0] > 0 and s[1] > 0
            and t.data_ptr() % 16 == 0)


def index(t: torch.Tensor, name: str, tokens: int, device) -> None:
    """Checks ``t`` as int32 or int64 [tokens] on ``device``."""
    if t.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"{name} must be int32 or int64, got {t.dtype}")
    if t.dim() != 1 or t.shape[0] != tokens:
        raise ValueError(f"{name} must be [{tokens}], got {tuple(t.shape)}")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, not on {device}")


class PagedKV:
    """One layer's cache.  ``k``, ``v``: ``[pages, kv_heads, page_size,
    head_dim]`` of ``dtype`` (bf16, fp16 or float8_e4m3fn); ``k_scale``,
    ``v_scale``: float32 ``[pages, kv_heads, page_size]`` of an e4m3 cache,
    else None.  head_dim 128 or 256; page_size 16, 32, 64 or 128."""

    def __init__(self, pages: int, page_size: int, kv_heads: int, head_dim: int,
                 dtype=torch.bfloat16, device="cuda"):
        if dtype not in DTYPES:
            raise TypeError(f"cache dtype {dtype}: bfloat16, float16 or float8_e4m3fn")
        shape = (pages, kv_heads, page_size, head_dim)
        k = torch.zeros(shape, dtype=dtype, device=device)
        v = torch.zeros_like(k)
        ks = vs = None
        if dtype == torch.float8_e4m3fn:
            ks = torch.ones(shape[:3], dtype=torch.float32, device=device)
            vs = torch.ones_like(ks)
        self._take(k, v, ks, vs)

    @classmethod
    def from_tensors(cls, k, v, k_scale=None, v_scale=None) -> "PagedKV":
        """A cache over buffers the caller has."""
        self = cls.__new__(cls)
        self._take(k, v, k_scale, v_scale)
        return self

    def _take(self, k, v, ks, vs):
        if k.dtype not in DTYPES:
            raise TypeError(f"cache dtype {k.dtype}: bfloat16, float16 or float8_e4m3fn")
        if k.dim() != 4 or v.shape != k.shape or v.dtype != k.dtype:
            raise ValueError("k and v must be [pages, kv_heads, page_size, head_dim] of one type")
        e4m3 = k.dtype == torch.float8_e4m3fn
        if e4m3 != (ks is not None) or e4m3 != (vs is not None):
            raise ValueError("an e4m3 cache has k_scale and v_scale, a 16-bit one has neither")
        for t in (k, v, ks, vs):
            if t is not None and (not t.is_contiguous() or t.device != k.device):
                raise ValueError("cache buffers must be contiguous and on one device")
        for t in (ks, vs):
            if t is not None and (t.dtype != torch.float32 or t.shape != k.shape[:3]):
                raise ValueError("scales must be float32 [pages, kv_heads, page_size]")
        if k.shape[3] not in (128, 256) or k.shape[2] not in (16, 32, 64, 128):
            raise ValueError(f"head_dim {k.shape[3]} (128 or 256), page_size {k.shape[2]} "
                             "(16, 32, 64 or 128)")
        if min(k.shape) < 1 or k.shape[0] * k.shape[1] * k.shape[2] >= 1 << 31:
            raise ValueError("pages * kv_heads * page_size must be in 1 .. 2^31 - 1")
        self.k, self.v, self.k_scale, self.v_scale = k, v, ks, vs
        self.pages, self.kv_heads, self.page_size, self.head_dim = k.shape
        self.dtype, self.device = k.dtype, k.device
        self.desc = _lib.KVCache(k.data_ptr(), v.data_ptr(), ks.data_ptr() if e4m3 else None,
                                 vs.data_ptr() if e4m3 else None, *k.shape, DTYPES[k.dtype])
        self.ref = ctypes.addressof(self.desc)
        self.e4m3 = e4m3
        self.workspace: dict = {}         # bytes an attention call needs, by its kernels
        # made here, not inside a capture
        self.error_word = moe.error_word(k.device) if k.device.type == "cuda" else None

    def rows_dtype(self, dtype) -> int:
        """The ABI's code of 16-bit rows this cache takes and gives."""
        code = DTYPES.get(dtype)
        if code is None or code == _lib.D3_E4M3:
            raise TypeError(f"rows must be bfloat16 or float16, got {dtype}")
        if not self.e4m3 and dtype != self.dtype:
            raise TypeError(f"a {self.dtype} cache takes and gives {self.dtype} rows, not {dtype}")
        return code


def write(cache: PagedKV, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor,
          stream=None) -> None:
    """Rows k, v ``[tokens, kv_heads, head_dim]`` (bf16 or fp16; views of a wider
    tensor are read in place) into ``slots`` (int32 or int64 ``[tokens]``).
    Slots outside the cache -- -1, say, for padding -- are skipped.  The slots
    of one call are distinct: a slot named twice keeps parts of either row."""
    dev = cache.device
    dtype = k.dtype
    code = cache.rows_dtype(dtype)
    rows(k, "k", cache.kv_heads, cache.head_dim, dtype)
    rows(v, "v", cache.kv_heads, cache.head_dim, dtype)
    tokens = k.shape[0]
    if v.shape[0] != tokens or k.device != dev or v.device != dev:
        raise ValueError("k and v must have the same tokens and the cache's device")
    index(slots, "slots", tokens, dev)
    if elsewhere(dev, stream):
        with place(dev, stream):
            return write(cache, k, v, slots)
    k, v, slots = in_place(k), in_place(v), slots.contiguous()
    ks, vs = k.stride(), v.stride()
    rc = _lib.packed("d3_kv_write")(cache.ref, k.data_ptr(), ks[0], ks[1], v.data_ptr(), vs[0], vs[1],
                                    code, tokens, slots.data_ptr(), slots.element_size(),
                                    _raw_stream(dev.index))
    if rc:
        _lib.raise_status(rc, "d3_kv_write")


def read(cache: PagedKV, slots: torch.Tensor, dtype=None, stream=None):
    """(k, v) rows ``[tokens, kv_heads, head_dim]`` at ``slots`` as ``dtype``
    (the cache's own type, or bfloat16 for an e4m3 cache).  A slot outside the
    cache reads as zeros."""
    dev = cache.device
    if dtype is None:
        dtype = torch.bfloat16 if cache.e4m3 else cache.dtype
    code = cache.rows_dtype(dtype)
    index(slots, "slots", slots.shape[0] if slots.dim() else 0, dev)
    if elsewhere(dev, stream):
        with place(dev, stream):
            return read(cache, slots, dtype)
    slots = slots.contiguous()
    tokens = slots.shape[0]
    k, v = torch.empty((2, tokens, cache.kv_heads, cache.head_dim), dtype=dtype, device=dev).unbind(0)
    rc = _lib.packed("d3_kv_read")(cache.ref, slots.data_ptr(), slots.element_size(), tokens, code,
                                   k.data_ptr(), v.data_ptr(), _raw_stream(dev.index))
    if rc:
        _lib.raise_status(rc, "d3_kv_read")
    return k, v
