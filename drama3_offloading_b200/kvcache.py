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


def elsewhere(device: int, stream) -> bool:
    """Whether a call on CUDA device ``device`` and ``stream`` (None: the current
    one) needs ``place`` around it -- and around the copies it may make of its
    arguments."""
    if device < 0:
        raise ValueError("tensors on the CPU: a CUDA device is needed")
    if stream is not None and stream.device_index != device:
        raise ValueError(f"stream is of device {stream.device_index}, the tensors are on {device}")
    return stream is not None or _device() != device


def place(device: int, stream):
    """Context in which ``device`` is the current device and ``stream`` (or the
    device's current one) its current stream: outputs and workspaces made in it
    belong to that stream."""
    return torch.cuda.stream(stream if stream is not None else torch.cuda.current_stream(device))


def rows(t: torch.Tensor, name: str, heads: int, dim: int, dtype, device: int) -> None:
    """Checks ``t`` as [tokens, heads, dim] rows of ``dtype`` on ``device``."""
    if t.dtype is not dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    shape = t.shape
    if len(shape) != 3 or shape[1] != heads or shape[2] != dim:
        raise ValueError(f"{name} must be [tokens, {heads}, {dim}], got {tuple(shape)}")
    if t.get_device() != device:
        raise ValueError(f"{name} is on {t.device}, not on device {device}")


def index(t: torch.Tensor, name: str, tokens: int, device: int) -> None:
    """Checks ``t`` as int32 or int64 [tokens] on ``device``."""
    if t.dtype is not torch.int32 and t.dtype is not torch.int64:
        raise TypeError(f"{name} must be int32 or int64, got {t.dtype}")
    shape = t.shape
    if len(shape) != 1 or shape[0] != tokens:
        raise ValueError(f"{name} must be [{tokens}], got {tuple(shape)}")
    if t.get_device() != device:
        raise ValueError(f"{name} is on {t.device}, not on device {device}")


def _free(t: torch.Tensor):
    """(token stride, head stride) of ``t``'s rows, the stride of a dimension of
    size 1 -- any number, of one token of an odd pitch, say -- replaced by a
    contiguous tensor's."""
    heads, dim = t.shape[1:]
    s0, s1, _ = t.stride()
    return heads * dim if t.shape[0] == 1 else s0, dim if heads == 1 else s1


def in_place(t: torch.Tensor):
    """(``t``, address, token stride, head stride), or those of a copy if the
    rows do not lie as the kernels read them: contiguous dims, rows on 16-byte
    boundaries."""
    s0, s1, s2 = t.stride()
    at = t.data_ptr()
    if s2 == 1 and not at & 15:
        if s0 > 0 and s1 > 0 and not (s0 | s1) & 7:
            return t, at, s0, s1
        s0, s1 = _free(t)
        if s0 > 0 and s1 > 0 and not (s0 | s1) & 7:
            return t, at, s0, s1
    t = t.contiguous()
    if t.data_ptr() & 15:
        t = t.clone()
    # (what is contiguous for torch may keep such a stride)
    heads, dim = t.shape[1:]
    return t, t.data_ptr(), heads * dim, dim


def output(t: torch.Tensor, shape, dtype, device: int):
    """(``t``, address, token stride, head stride) of an output the caller gives."""
    if t.shape == shape and t.dtype is dtype and t.get_device() == device:
        s0, s1, s2 = t.stride()
        at = t.data_ptr()
        if s2 == 1 and not at & 15:
            if s0 <= 0 or s1 <= 0 or (s0 | s1) & 7:
                s0, s1 = _free(t)
            if s0 > 0 and s1 > 0 and not (s0 | s1) & 7:
                return t, at, s0, s1
    raise ValueError(f"out must be {dtype} {tuple(shape)} on device {device}, its rows contiguous on "
                     "16-byte boundaries")


def fresh(like: torch.Tensor, heads: int, dim: int):
    """(new rows, address, token stride, head stride) of ``like``'s tokens."""
    t = like.new_empty((like.shape[0], heads, dim))
    return t, t.data_ptr(), heads * dim, dim


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
        self.dtype, self.device, self.device_index = k.dtype, k.device, k.get_device()
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
    dev, dtype = cache.device_index, k.dtype
    code = cache.rows_dtype(dtype)
    rows(k, "k", cache.kv_heads, cache.head_dim, dtype, dev)
    rows(v, "v", cache.kv_heads, cache.head_dim, dtype, dev)
    tokens = k.shape[0]
    if v.shape[0] != tokens:
        raise ValueError("k and v must have the same tokens")
    index(slots, "slots", tokens, dev)
    if elsewhere(dev, stream):
        with place(dev, stream):
            return write(cache, k, v, slots)
    k, k_at, k0, k1 = in_place(k)
    v, v_at, v0, v1 = in_place(v)
    slots = slots.contiguous()
    rc = _lib.packed("d3_kv_write")(cache.ref, k_at, k0, k1, v_at, v0, v1, code, tokens,
                                    slots.data_ptr(), slots.element_size(), _raw_stream(dev))
    if rc:
        _lib.raise_status(rc, "d3_kv_write")


def read(cache: PagedKV, slots: torch.Tensor, dtype=None, stream=None):
    """(k, v) rows ``[tokens, kv_heads, head_dim]`` at ``slots`` as ``dtype``
    (the cache's own type, or bfloat16 for an e4m3 cache).  A slot outside the
    cache reads as zeros."""
    dev = cache.device_index
    if dtype is None:
        dtype = torch.bfloat16 if cache.e4m3 else cache.dtype
    code = cache.rows_dtype(dtype)
    index(slots, "slots", slots.shape[0] if slots.dim() else 0, dev)
    if elsewhere(dev, stream):
        with place(dev, stream):
            return read(cache, slots, dtype)
    slots = slots.contiguous()
    tokens = slots.shape[0]
    k, v = torch.empty((2, tokens, cache.kv_heads, cache.head_dim), dtype=dtype,
                       device=cache.device).unbind(0)
    rc = _lib.packed("d3_kv_read")(cache.ref, slots.data_ptr(), slots.element_size(), tokens, code,
                                   k.data_ptr(), v.data_ptr(), _raw_stream(dev))
    if rc:
        _lib.raise_status(rc, "d3_kv_read")
    return k, v
