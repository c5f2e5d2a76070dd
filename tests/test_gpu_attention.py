"""GPU parity of the paged K/V cache, the norm and rotation, and the attention
over the cache, through the public Python calls, against 64-bit plain forms
(tests/attention_reference.py, which derives the tolerances)."""
import pytest
import torch

import attention_reference as ref
from conftest import cuda_available

pytestmark = [pytest.mark.gpu,
              pytest.mark.skipif(not cuda_available(), reason="needs a CUDA GPU")]

from drama3_offloading_b200 import attention, kvcache, moe  # noqa: E402

DEV = torch.device("cuda:0")
BF, FP, E4 = torch.bfloat16, torch.float16, torch.float8_e4m3fn


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def randn(g, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=g, device=DEV) * scale).to(dtype)


def poison(cache):
    """NaN wherever nothing has been written."""
    for x in (cache.k, cache.v):
        if x.dtype == E4:
            x.view(torch.uint8).fill_(0x7F)
        else:
            x.fill_(float("nan"))
    for s in (cache.k_scale, cache.v_scale):
        if s is not None:
            s.fill_(float("nan"))
    return cache


def at(cache, x, slots):
    """Rows of a cache buffer [pages, heads, page(, D)] at slots: [T, heads(, D)]."""
    return x.view(torch.uint8)[slots // cache.page_size, :, slots % cache.page_size].view(x.dtype) \
        if x.dtype == E4 else x[slots // cache.page_size, :, slots % cache.page_size]


# ---------------------------------------------------------------- cache

@pytest.mark.parametrize("dim", [128, 256])
@pytest.mark.parametrize("dtype,kind", [(BF, BF), (FP, FP), (BF, E4), (FP, E4)])
@pytest.mark.parametrize("tokens,page", [(1, 16), (77, 32), (1300, 64), (2500, 128)])
def test_write_and_read(dim, dtype, kind, tokens, page):
    g = gen(tokens)
    heads = 3
    cache = poison(kvcache.PagedKV(-(-tokens // page) + 2, page, heads, dim, kind, DEV))
    before = cache.k.clone()
    wide = randn(g, tokens, 2 * heads + 1, dim, dtype=dtype, scale=3.0)
    wide[0, 0] = 0                                     # a row of zeros: scale 1
    k, v = wide[:, :heads], wide[:, heads:2 * heads]   # strided views
    slots = torch.randperm(cache.pages * page, generator=g, device=DEV)[:tokens]
    if tokens % 2 == 0:
        slots = slots.to(torch.int32)
    kvcache.write(cache, k, v, slots)
    s = slots.long()
    for x, buf, sc in ((k, cache.k, cache.k_scale), (v, cache.v, cache.v_scale)):
        if kind == E4:
            code, scale = (t.to(DEV) for t in ref.quantise(x.cpu()))
            assert torch.equal(at(cache, sc, s), scale)
            assert torch.equal(at(cache, buf, s).view(torch.uint8), code.view(torch.uint8))
        else:
            assert torch.equal(at(cache, buf, s), x)
    # nothing else was touched
    rest = torch.ones(cache.pages * page, dtype=torch.bool, device=DEV)
    rest[s] = False
    other = rest.nonzero()[:, 0]
    assert torch.equal(at(cache, cache.k, other).contiguous().view(torch.uint8),
                       at(cache, before, other).contiguous().view(torch.uint8))
    got = kvcache.read(cache, slots, dtype=dtype)
    for x, buf, sc, y in ((k, cache.k, cache.k_scale, got[0]), (v, cache.v, cache.v_scale, got[1])):
        want = (at(cache, buf, s).float() * at(cache, sc, s)[..., None]).to(dtype) if kind == E4 else x
        assert torch.equal(y, want)


def test_slots_outside_are_skipped_and_read_as_zeros():
    g = gen(1)
    cache = kvcache.PagedKV(2, 16, 2, 128, E4, DEV)
    k, v = randn(g, 5, 2, 128, dtype=BF), randn(g, 5, 2, 128, dtype=BF)
    slots = torch.tensor([3, -1, 32, 31, -2 ** 40], device=DEV)
    kvcache.write(cache, k, v, slots)
    assert int((cache.k_scale != 1).sum()) == 4       # two rows of two heads
    rk, rv = kvcache.read(cache, slots)
    assert torch.equal(rk[[1, 2, 4]], torch.zeros_like(rk[:3]))
    assert torch.equal(rv[[1, 2, 4]], torch.zeros_like(rv[:3]))
    assert float((rv[0].float() - v[0].float()).abs().max()) < 0.3
    kvcache.write(cache, k[:0], v[:0], slots[:0])     # no tokens
    assert kvcache.read(cache, slots[:0])[0].shape == (0, 2, 128)


def test_infinities_and_nan_stay_in_their_row():
    cache = kvcache.PagedKV(1, 16, 1, 128, E4, DEV)
    k = torch.ones(3, 1, 128, dtype=BF, device=DEV)
    k[1, 0, 5] = float("nan")
    k[2, 0, 7] = float("inf")
    kvcache.write(cache, k, k, torch.arange(3, device=DEV))
    r = kvcache.read(cache, torch.arange(3, device=DEV))[0]
    assert torch.equal(r[0], k[0])
    assert r[1].isnan().sum() == 1 and bool(r[1, 0, 5].isnan())
    # an infinite scale: nothing of the row is finite
    assert not r[2].isfinite().any()


# ---------------------------------------------------------------- norm, rotation

@pytest.mark.parametrize("dim,rotary", [(128, 128), (128, 32), (256, 64), (256, 256), (256, 16), (128, 48)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("tokens,heads,kv_heads", [(1, 8, 2), (37, 5, 5), (1303, 6, 1)])
def test_norm_rope(dim, rotary, interleaved, dtype, tokens, heads, kv_heads):
    g = gen(tokens + rotary)
    wide = randn(g, tokens, heads + kv_heads, dim, dtype=dtype, scale=2.0)
    wide[0, 0] = 0                                     # a row of zeros stays one
    q, k = wide[:, :heads], wide[:, heads:]
    qw, kw = randn(g, dim, dtype=dtype, scale=0.3), randn(g, dim, dtype=dtype, scale=0.3)
    pos = torch.randint(0, 2 ** 20, (tokens,), generator=g, device=DEV)
    pos[-1] = 0
    if tokens == 37:
        pos = pos.to(torch.int32)
    f = attention.rope_frequencies(rotary, 10000000.0, DEV)
    qo, ko = attention.qk_norm_rope(q, k, qw, kw, pos, f, eps=1e-6, weight_offset=1.0,
                                    interleaved=interleaved)
    for x, w, y in ((q, qw, qo), (k, kw, ko)):
        want = ref.norm_rope(x, w, pos, f, 1e-6, 1.0, interleaved)
        assert y.dtype == dtype and y.is_contiguous()
        assert bool(((y.double() - want).abs() <= ref.norm_rope_bound(want, dtype)).all())
    # in place, over the same views
    attention.qk_norm_rope(q, k, qw, kw, pos, f, eps=1e-6, weight_offset=1.0,
                           interleaved=interleaved, out=(q, k))
    assert torch.equal(q, qo) and torch.equal(k, ko)


@pytest.mark.parametrize("dim,kind,dtype", [(256, E4, BF), (256, BF, BF), (128, E4, FP), (128, FP, FP)])
@pytest.mark.parametrize("tokens", [1, 130, 1500])
def test_norm_rope_write(dim, kind, dtype, tokens):
    g = gen(tokens)
    heads, hk, page = 6, 2, 32
    wide = randn(g, tokens, heads + 2 * hk, dim, dtype=dtype, scale=2.0)
    q, k, v = wide[:, :heads], wide[:, heads:heads + hk], wide[:, heads + hk:]
    qw, kw = randn(g, dim, dtype=dtype, scale=0.3) + 1, randn(g, dim, dtype=dtype, scale=0.3) + 1
    pos = torch.arange(5000, 5000 + tokens, device=DEV)
    f = attention.rope_frequencies(64, 10000.0, DEV)
    cache = poison(kvcache.PagedKV(-(-tokens // page) + 1, page, hk, dim, kind, DEV))
    slots = torch.randperm(cache.pages * page, generator=g, device=DEV)[:tokens]
    slots[tokens // 2] = -1 if tokens > 1 else slots[0]
    qo = attention.qk_norm_rope_write(q, k, v, qw, kw, pos, f, cache, slots)
    plain_q, _ = attention.qk_norm_rope(q, k, qw, kw, pos, f)
    assert torch.equal(qo, plain_q)
    keep = (slots >= 0).nonzero()[:, 0]
    s = slots[keep]
    want = ref.norm_rope(k, kw, pos, f, 1e-6, 0.0, False)[keep]
    slack = 64 * 2.0 ** -24 * want.abs().amax(-1, keepdim=True)
    if kind == E4:
        sc = at(cache, cache.k_scale, s).double()
        assert bool(((sc * 448 / want.abs().amax(-1) - 1).abs() < 2.0 ** -17).all())
        got = at(cache, cache.k, s).float().double() * sc[..., None]
        # half a step of a code: 2^-4 of the value, or of the least normal one
        assert bool(((got - want).abs() <= 2.0 ** -4 * want.abs() + 2.0 ** -10 * sc[..., None] + slack).all())
        code, scale = (t.to(DEV) for t in ref.quantise(v[keep].cpu()))
        assert torch.equal(at(cache, cache.v, s).view(torch.uint8), code.view(torch.uint8))
        assert torch.equal(at(cache, cache.v_scale, s), scale)
    else:
        got = at(cache, cache.k, s).double()
        assert bool(((got - want).abs() <= ref.norm_rope_bound(want, dtype)).all())
        assert torch.equal(at(cache, cache.v, s), v[keep])


# ---------------------------------------------------------------- attention

def make_batch(g, lens, heads, hk, dim, page, dtype, kind, q_scale=2.0, extra=0, spare=3):
    """lens: (new tokens, cached tokens) of each sequence.  Pages in random
    order; everything that no sequence holds is NaN."""
    need = [-(-kv // page) for _, kv in lens]
    cache = poison(kvcache.PagedKV(sum(need) + spare, page, hk, dim, kind, DEV))
    order = torch.randperm(cache.pages, generator=g, device=DEV).to(torch.int32)
    table = torch.full((len(lens), max(need + [1]) + 1), -7, dtype=torch.int32, device=DEV)
    first = 0
    for b, (n, kv) in enumerate(lens):
        table[b, :need[b]] = order[first:first + need[b]]
        first += need[b]
        if kv:
            i = torch.arange(kv, device=DEV)
            slots = table[b].long()[i // page] * page + i % page
            kvcache.write(cache, randn(g, kv, hk, dim, dtype=dtype), randn(g, kv, hk, dim, dtype=dtype), slots)
    total = sum(n for n, _ in lens)
    q = randn(g, total + extra, heads, dim, dtype=dtype, scale=q_scale)
    cu = torch.tensor([sum(n for n, _ in lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32, device=DEV)
    kv = torch.tensor([kv for _, kv in lens], dtype=torch.int32, device=DEV)
    return cache, table, q, cu, kv


def check(out, want, bound, rows=None):
    live = ~want[:, 0, 0].isnan()
    err = (out.double() - want)[live].abs()
    worst = (err / bound[live].clamp_min(1e-300)).max() if err.numel() else 0.0
    assert bool((err <= bound[live]).all()), f"worst error {float(worst):.3g} of its bound"


DECODE = [(1, 1), (1, 0), (1, 15), (1, 16), (1, 17), (1, 63), (1, 64), (1, 65), (1, 127), (1, 128), (1, 129), (1, 700)]
FEW = [(3, 3), (2, 1), (5, 64), (4, 0), (1, 33), (5, 129), (3, 500), (0, 70), (4, 1000)]
CHUNK = [(130, 130), (17, 17), (64, 700), (0, 5), (33, 20), (1, 900), (257, 300), (3, 40)]


@pytest.mark.parametrize("lens", [DECODE, FEW, CHUNK], ids=["decode", "few", "chunk"])
@pytest.mark.parametrize("dim,heads,hk,page", [(256, 8, 2, 64), (256, 16, 2, 32), (128, 8, 8, 16), (128, 12, 2, 128),
                                               (256, 3, 1, 16), (128, 20, 1, 64)])
@pytest.mark.parametrize("dtype,kind", [(BF, BF), (FP, FP), (BF, E4), (FP, E4)], ids=["bf", "fp", "bf8", "fp8"])
def test_attention(lens, dim, heads, hk, page, dtype, kind):
    cache, table, q, cu, kv = make_batch(gen(heads + page), lens, heads, hk, dim, page, dtype, kind, extra=2)
    out = torch.full_like(q, 7.0)
    max_q = max(n for n, _ in lens)
    got = attention.paged_attention(q, cache, table, kv, cu, max_q=max_q, out=out)
    moe.check_errors(DEV)
    assert got is out
    want, bound = ref.attention(q, cache, table, kv, cu)
    check(out, want, bound)
    assert bool((out[-2:] == 7.0).all())              # rows behind the last sequence
    for b, (n, length) in enumerate(lens):            # rows that see nothing
        gone = max(0, min(n, n - length))
        assert bool((out[int(cu[b]):int(cu[b]) + gone] == 0).all())
    # the same call again gives the same bits
    again = attention.paged_attention(q, cache, table, kv, cu, max_q=max_q)
    assert torch.equal(again[:-2], out[:-2])


@pytest.mark.parametrize("dim,heads,hk,page,dtype,kind", [(256, 8, 2, 64, BF, BF), (128, 8, 2, 16, FP, E4)])
@pytest.mark.parametrize("n", [1, 40])
def test_attention_split_over_one_long_sequence(dim, heads, hk, page, dtype, kind, n):
    """A sequence long enough that every SM takes a part of it."""
    cache, table, q, cu, kv = make_batch(gen(9), [(n, 30011), (n, 5)], heads, hk, dim, page, dtype, kind)
    out = attention.paged_attention(q, cache, table, kv, cu, max_q=n)
    moe.check_errors(DEV)
    check(out, *ref.attention(q, cache, table, kv, cu))


def test_attention_without_cu_q_and_with_strided_q():
    cache, table, q, cu, kv = make_batch(gen(4), DECODE, 8, 2, 256, 64, BF, BF)
    wide = torch.randn(q.shape[0], 11, 256, device=DEV).to(BF)
    wide[:, 2:10] = q
    out = attention.paged_attention(wide[:, 2:10], cache, table, kv, scale=0.1)
    check(out, *ref.attention(q, cache, table, kv, scale=0.1))
    # int-like limits that are too low still give whole answers
    low = attention.paged_attention(q, cache, table, kv, max_kv=1, scale=0.1)
    check(low, *ref.attention(q, cache, table, kv, scale=0.1))


@pytest.mark.parametrize("kind", [BF, E4])
@pytest.mark.parametrize("n", [1, 30])
def test_attention_bad_pages_read_as_zeros(kind, n):
    cache, table, q, cu, kv = make_batch(gen(5), [(n, 200), (n, 100)], 8, 2, 128, 16, BF, kind)
    table[0, 3], table[0, 5], table[1, 0], table[1, 2] = -1, cache.pages, 2 ** 31 - 1, -2 ** 31
    out = attention.paged_attention(q, cache, table, kv, cu, max_q=n)
    moe.check_errors(DEV)
    check(out, *ref.attention(q, cache, table, kv, cu))


@pytest.mark.parametrize("n", [1, 33])
def test_attention_peaked_scores_and_large_values(n):
    """Scores of hundreds, where all but one key vanish, and queries and values
    far from 1."""
    for dtype, kind in ((BF, BF), (BF, E4)):
        cache, table, q, cu, kv = make_batch(gen(6), [(n, 333), (n, 90)], 8, 2, 256, 64, dtype, kind, q_scale=60.0)
        out = attention.paged_attention(q, cache, table, kv, cu, max_q=n)
        check(out, *ref.attention(q, cache, table, kv, cu))
        out = attention.paged_attention(q * 2.0 ** 20, cache, table, kv, cu, max_q=n, scale=2.0 ** -26)
        check(out, *ref.attention(q * 2.0 ** 20, cache, table, kv, cu, scale=2.0 ** -26))


@pytest.mark.parametrize("n", [1, 20])
@pytest.mark.parametrize("kind", [BF, E4])
def test_attention_far_pages(n, kind):
    """Pages whose elements lie behind 2^32."""
    page, hk, dim = 128, 2, 256
    pages = (1 << 32) // (page * hk * dim) + 40
    k = torch.empty(pages, hk, page, dim, dtype=kind, device=DEV)
    v = torch.empty_like(k)
    sc = [torch.ones(k.shape[:3], device=DEV) for _ in range(2)] if kind == E4 else [None, None]
    cache = kvcache.PagedKV.from_tensors(k, v, *sc)
    g = gen(8)
    table = torch.tensor([[pages - 1, 0, pages - 7]], dtype=torch.int32, device=DEV)
    i = torch.arange(300, device=DEV)
    slots = table[0].long()[i // page] * page + i % page
    kvcache.write(cache, randn(g, 300, hk, dim, dtype=BF), randn(g, 300, hk, dim, dtype=BF), slots)
    near = torch.tensor([0, 1, 2], device=DEV)
    small = kvcache.PagedKV.from_tensors(*(x[table[0].long()].contiguous() if x is not None else None
                                           for x in (k, v, *sc)))
    rk, rv = kvcache.read(cache, slots, dtype=BF)
    sk, sv = kvcache.read(small, i, dtype=BF)
    assert torch.equal(rk, sk) and torch.equal(rv, sv)
    q = randn(g, n, 8, dim, dtype=BF)
    kv = torch.tensor([300], dtype=torch.int32, device=DEV)
    cu = torch.tensor([0, n], dtype=torch.int32, device=DEV)
    out = attention.paged_attention(q, cache, table, kv, cu, max_q=n)
    assert torch.equal(out, attention.paged_attention(q, small, near[None].int(), kv, cu, max_q=n))
    check(out, *ref.attention(q, small, near[None].int(), kv, cu))


# ---------------------------------------------------------------- together

def step_inputs(g, tokens, heads, hk, dim, dtype):
    wide = randn(g, tokens, heads + 2 * hk, dim, dtype=dtype)
    return wide[:, :heads], wide[:, heads:heads + hk], wide[:, heads + hk:]


@pytest.mark.parametrize("kind", [BF, E4])
def test_prefill_then_decode_in_a_captured_graph(kind):
    """A prompt in two chunks, then decode steps replayed from one graph: the
    same rows as one chunk over all tokens, for the plain form."""
    g = gen(11)
    heads, hk, dim, page, total, prompt = 8, 2, 256, 64, 150, 130
    cache = poison(kvcache.PagedKV(8, page, hk, dim, kind, DEV))
    table = torch.tensor([[5, 2, 7]], dtype=torch.int32, device=DEV)
    q, k, v = step_inputs(g, total, heads, hk, dim, BF)
    qw, kw = randn(g, dim, dtype=BF, scale=0.2) + 1, randn(g, dim, dtype=BF, scale=0.2) + 1
    f = attention.rope_frequencies(64, 10000000.0, DEV)
    pos = torch.arange(total, device=DEV)
    slots = table[0].long()[pos // page] * page + pos % page
    out, qs = torch.empty(total, heads, dim, dtype=BF, device=DEV), []
    for lo, hi in ((0, 100), (100, prompt)):
        qr = attention.qk_norm_rope_write(q[lo:hi], k[lo:hi], v[lo:hi], qw, kw, pos[lo:hi], f, cache, slots[lo:hi])
        qs.append(qr)
        attention.paged_attention(qr, cache, table, torch.tensor([hi], dtype=torch.int32, device=DEV),
                                  torch.tensor([0, hi - lo], dtype=torch.int32, device=DEV), max_q=hi - lo,
                                  out=out[lo:hi])
    qb, kb, vb = (x[:1].clone() for x in (q, k, v))
    pb, sb, lb = pos[:1].clone(), slots[:1].clone(), torch.ones(1, dtype=torch.int32, device=DEV)
    qo, ob = torch.empty_like(qb), torch.empty_like(qb)

    def step():
        attention.qk_norm_rope_write(qb, kb, vb, qw, kw, pb, f, cache, sb, out=qo)
        attention.paged_attention(qo, cache, table, lb, out=ob)
    sb.fill_(-1)
    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for t in range(prompt, total):
        for dst, src in ((qb, q), (kb, k), (vb, v), (pb, pos), (sb, slots)):
            dst.copy_(src[t:t + 1])
        lb.fill_(t + 1)
        graph.replay()
        out[t] = ob[0]
        qs.append(qo.clone())
    moe.check_errors(DEV)
    kv = torch.tensor([total], dtype=torch.int32, device=DEV)
    cu = torch.tensor([0, total], dtype=torch.int32, device=DEV)
    check(out, *ref.attention(torch.cat(qs), cache, table, kv, cu))


def test_streams_and_graphs_share_nothing():
    """Two captured graphs and eager calls on a third stream, all at once."""
    big = make_batch(gen(21), [(1, 4000)] * 4, 8, 2, 256, 64, BF, BF)
    few = make_batch(gen(22), [(2, 3000), (2, 100)], 8, 2, 256, 64, BF, BF)
    call = lambda x: attention.paged_attention(x[2], x[0], x[1], x[4], x[3], max_q=2)
    want = [call(x) for x in (big, few)]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for x in (big, few):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(call(x))
        graphs.append(gr)
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    got = []
    for _ in range(20):
        for gr, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                gr.replay()
        got.append(attention.paged_attention(few[2], few[0], few[1], few[4], few[3], max_q=2, stream=streams[2]))
    torch.cuda.synchronize()
    moe.check_errors(DEV)
    for o, w in zip(outs, want):
        assert torch.equal(o, w)
    for o in got:
        assert torch.equal(o, want[1])


@pytest.mark.parametrize("dtype,kind,heads,hk,dim", [(FP, E4, 16, 4, 128), (BF, BF, 8, 2, 256)])
def test_many_calls_in_a_row_give_the_same_bits(dtype, kind, heads, hk, dim):
    """Chunks and single tokens mixed, hundreds of launches back to back (each
    early behind the one before): no wait runs out, no bit changes."""
    g = gen(31)
    lens = [(1, 2100), (140, 900), (1, 5), (65, 3500), (301, 301), (1, 800), (90, 2000)]
    cache, table, q, cu, kv = make_batch(g, lens, heads, hk, dim, 16, dtype, kind)
    call = lambda: attention.paged_attention(q, cache, table, kv, cu, max_q=301)
    want = call()
    check(want, *ref.attention(q, cache, table, kv, cu))
    same = torch.ones((), dtype=torch.bool, device=DEV)
    for _ in range(10):
        for o in [call() for _ in range(40)]:
            same &= (o == want).all()
    assert bool(same)
    moe.check_errors(DEV)
