"""Refusals of the K/V cache and attention calls, without a GPU: wrong types,
shapes and sizes raise before anything is launched; the C ABI returns its
status codes."""
import ctypes

import pytest
import torch

from drama3_offloading_b200 import _lib, attention, kvcache

BF, FP, E4 = torch.bfloat16, torch.float16, torch.float8_e4m3fn


def cache(kind=BF, pages=2, page=16, heads=2, dim=128):
    return kvcache.PagedKV(pages, page, heads, dim, kind, "cpu")


def test_cache_shapes():
    c = cache(E4)
    assert c.k.shape == (2, 2, 16, 128) and c.k_scale.shape == (2, 2, 16)
    assert cache().k_scale is None
    for kw in ({"page": 48}, {"page": 8}, {"dim": 64}, {"dim": 192}, {"pages": 0}, {"heads": 0}):
        with pytest.raises(ValueError):
            cache(**kw)
    with pytest.raises(TypeError):
        cache(torch.float32)
    k = torch.zeros(2, 2, 16, 128, dtype=BF)
    with pytest.raises(ValueError):
        kvcache.PagedKV.from_tensors(k, k[:1])
    with pytest.raises(ValueError):
        kvcache.PagedKV.from_tensors(k, k.transpose(0, 1).contiguous().transpose(0, 1)[:, :, ::1].mT.contiguous().mT)
    with pytest.raises(ValueError):
        kvcache.PagedKV.from_tensors(k, k, torch.ones(2, 2, 16), torch.ones(2, 2, 16))
    with pytest.raises(ValueError):
        kvcache.PagedKV.from_tensors(k.to(E4), k.to(E4))
    with pytest.raises(ValueError):
        kvcache.PagedKV.from_tensors(k.to(E4), k.to(E4), torch.ones(2, 2, 8), torch.ones(2, 2, 16))


def test_write_and_read_refusals():
    k = torch.zeros(3, 2, 128, dtype=BF)
    slots = torch.arange(3)
    with pytest.raises(TypeError):
        kvcache.write(cache(), k.half(), k.half(), slots)        # fp16 rows, bf16 cache
    with pytest.raises(TypeError):
        kvcache.write(cache(E4), k.float(), k.float(), slots)
    with pytest.raises(TypeError):
        kvcache.write(cache(), k, k.half(), slots)
    with pytest.raises(ValueError):
        kvcache.write(cache(), k[:, :1], k, slots)
    with pytest.raises(ValueError):
        kvcache.write(cache(), k, k[:2], slots)
    with pytest.raises(ValueError):
        kvcache.write(cache(), k, k, slots[:2])
    with pytest.raises(TypeError):
        kvcache.write(cache(), k, k, slots.float())
    with pytest.raises(TypeError):
        kvcache.read(cache(), slots, dtype=FP)
    with pytest.raises(ValueError):
        kvcache.read(cache(), slots[:, None])


def test_norm_rope_refusals():
    q, k = torch.zeros(3, 4, 128, dtype=BF), torch.zeros(3, 2, 128, dtype=BF)
    w, pos = torch.zeros(128, dtype=BF), torch.arange(3)
    f = attention.rope_frequencies(64, device="cpu")
    assert f.dtype == torch.float64 and f.shape == (32,) and float(f[0]) == 1.0
    bad = [(q.float(), k, w, w, pos, f), (q, k.half(), w, w, pos, f), (q, k, w.float(), w, pos, f),
           (q, k, w, w[:64], pos, f), (q, k, w, w, pos.float(), f), (q, k, w, w, pos, f.float())]
    for a in bad:
        with pytest.raises(TypeError):
            attention.qk_norm_rope(*a)
    for a in [(q[0], k, w, w, pos, f), (q, k[:2], w, w, pos, f), (q, k, w, w, pos[:2], f)]:
        with pytest.raises(ValueError):
            attention.qk_norm_rope(*a)
    v = torch.zeros(3, 2, 128, dtype=BF)
    with pytest.raises(ValueError):
        attention.qk_norm_rope_write(q, k, v, w, w, pos, f, cache(heads=3), pos)
    with pytest.raises(ValueError):
        attention.qk_norm_rope_write(q, k, v[:, :1], w, w, pos, f, cache(), pos)
    with pytest.raises(TypeError):
        attention.qk_norm_rope_write(q, k, v, w, w, pos, f, cache(FP), pos)
    with pytest.raises(ValueError):
        attention.qk_norm_rope_write(q, k, v, w, w, pos, f, cache(), pos[:1])


def test_attention_refusals():
    q = torch.zeros(2, 4, 128, dtype=BF)
    table, lens = torch.zeros(2, 2, dtype=torch.int32), torch.ones(2, dtype=torch.int32)
    cu = torch.arange(3, dtype=torch.int32)
    c = cache()
    call = attention.paged_attention
    for a, kw in [((q.half(), c, table, lens), {}), ((q.float(), cache(E4), table, lens), {}),
                  ((q, c, table.long(), lens), {}), ((q, c, table, lens.long()), {}),
                  ((q, c, table, lens, cu.long()), {}), ((q, c, table, lens.float()), {})]:
        with pytest.raises(TypeError):
            call(*a, **kw)
    for a, kw in [((q[0], c, table, lens), {}), ((q[:, :3], c, table, lens), {}), ((q[:1], c, table, lens), {}),
                  ((q, c, table, lens[:1]), {}), ((q, c, table, lens, cu[:2]), {}),
                  ((q, c, table, lens), {"max_q": 0}), ((q, c, table, lens), {"out": q[:1]}),
                  ((q, c, table, lens), {"out": torch.zeros(2, 4, 256, dtype=BF)[..., ::2]}),
                  ((torch.zeros(2, 4, 256, dtype=BF), c, table, lens), {}),
                  ((torch.zeros(2, 2 * 129, 128, dtype=BF), c, table, lens), {})]:
        with pytest.raises(ValueError):
            call(*a, **kw)


def test_abi_statuses():
    lib = _lib.load()
    P = ctypes.c_void_p
    c = _lib.KVCache(16, 16, None, None, 4, 2, 64, 128, _lib.D3_BF16)
    r = ctypes.byref(c)
    z = P(16)
    write = lambda dt=0, tok=128, sb=4, k=16: lib.d3_kv_write(r, P(k), tok, 128, z, 128, 128, dt, 3, z, sb, P(0))
    assert write(dt=1) == -1 and write(dt=2) == -1 and write(sb=2) == -1
    assert write(tok=130) == -3 and write(k=8) == -3
    assert lib.d3_kv_write(None, z, 128, 128, z, 128, 128, 0, 3, z, 4, P(0)) == -1
    assert lib.d3_kv_write(r, z, 128, 128, z, 128, 128, 0, 0, z, 4, P(0)) == 0
    assert lib.d3_kv_read(r, z, 4, 3, 1, z, z, P(0)) == -1
    assert lib.d3_kv_read(r, z, 4, 3, 0, P(8), z, P(0)) == -3
    c.dtype = _lib.D3_E4M3
    assert write() == -1 and b"scales" in lib.d3_last_error()
    c.dtype = _lib.D3_BF16
    c.page_size = 48
    assert write() == -5
    c.page_size, c.head_dim = 64, 64
    assert write() == -5
    c.head_dim, c.pages = 128, 1 << 25
    assert write() == -6
    c.pages = 4
    n = _lib.NormRope(q=16, k=16, v=16, q_out=16, q_weight=16, k_weight=16, positions=16, inv_freq=16, slots=16,
                      pos_bytes=4, slot_bytes=4, tokens=2, heads=4, kv_heads=2, head_dim=128, rotary_dim=64)
    assert lib.d3_qk_norm_rope(n, None, P(0)) == -1          # no k_out, no cache
    n.rotary_dim = 24
    assert lib.d3_qk_norm_rope(n, r, P(0)) == -5
    n.rotary_dim = 144
    assert lib.d3_qk_norm_rope(n, r, P(0)) == -5
    n.rotary_dim, n.kv_heads = 64, 1
    assert lib.d3_qk_norm_rope(n, r, P(0)) == -1
    n.kv_heads, n.q_token = 2, 4
    assert lib.d3_qk_norm_rope(n, r, P(0)) == -3
    a = _lib.Attention(q=16, q_token=512, q_head=128, out=16, out_token=512, out_head=128, page_table=16,
                       table_stride=4, kv_lens=16, table_pages=4, batch=2, tokens=2, heads=4, max_q=1, max_kv=256,
                       scale=0.1)
    need = lib.d3_paged_attention_workspace_size(a, r)
    assert need > 0
    run = lambda ws=16, size=need, err=16: lib.d3_paged_attention(a, r, P(err), P(ws), ctypes.c_size_t(size), P(0))
    assert run(size=need - 1) == -7 and run(ws=0) == -7 and run(ws=24) == -3 and run(err=0) == -1
    a.heads = 5
    assert run() == -1 and lib.d3_paged_attention_workspace_size(a, r) == 0
    a.heads, a.tokens = 4, 1
    assert run() == -1                                        # fewer rows than sequences
    a.tokens, a.q_head = 2, 4
    assert run() == -3
    a.q_head, a.heads = 128, 2 * 129
    assert run() == -5
    a.heads, a.max_q = 4, 0
    assert run() == -1
    a.max_q, a.batch = 1, 0
    assert run() == 0                                         # nothing to do
