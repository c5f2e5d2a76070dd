"""Calls of the paged attention and the cache operators where an answer depends
on more than their formulas: values next to a sequence's end, rows that are not
finite, scales far apart, broken offsets, odd strides.  Against 64-bit forms or
against the same call in another form."""
import pytest
import torch

import attention_reference as ref
from conftest import cuda_available

pytestmark = [pytest.mark.gpu,
              pytest.mark.skipif(not cuda_available(), reason="needs a CUDA GPU")]

from drama3_offloading_b200 import attention, kvcache, moe  # noqa: E402

DEV = torch.device("cuda:0")
BF, FP, E4 = torch.bfloat16, torch.float16, torch.float8_e4m3fn


def batch(seed, lens, heads, hk, dim, page, dtype, kind):
    """(cache, table, q, cu_q, kv_lens) of sequences of (new tokens, keys), their
    pages one behind the other; rows behind a sequence's end are NaN."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=g, device=DEV).to(dtype)
    need = [-(-kv // page) for _, kv in lens]
    cache = kvcache.PagedKV(max(1, sum(need)), page, hk, dim, kind, DEV)
    for x in (cache.k, cache.v):
        x.view(torch.uint8).fill_(0x7F) if kind == E4 else x.fill_(float("nan"))
    table = torch.zeros(len(lens), max(need + [1]), dtype=torch.int32, device=DEV)
    first = 0
    for b, (_, kv) in enumerate(lens):
        table[b, :need[b]] = torch.arange(first, first + need[b], device=DEV)
        if kv:
            kvcache.write(cache, rnd(kv, hk, dim), rnd(kv, hk, dim), first * page + torch.arange(kv, device=DEV))
        first += need[b]
    cu = torch.tensor([0] + [n for n, _ in lens]).cumsum(0).to(torch.int32).to(DEV)
    kv = torch.tensor([kv for _, kv in lens], dtype=torch.int32, device=DEV)
    return cache, table, rnd(int(cu[-1]), heads, dim), cu, kv


def call(c, q=None, **kw):
    cache, table, q0, cu, kv = c
    n = int((cu[1:] - cu[:-1]).max())
    return attention.paged_attention(q0 if q is None else q, cache, table, kv, cu, max_q=n, **kw)


def check(out, want, bound):
    live = ~want[:, 0, 0].isnan()
    assert bool(((out.double() - want)[live].abs() <= bound[live]).all())
    moe.check_errors(DEV)


# ---------------------------------------------------------------- behind the end

@pytest.mark.parametrize("dim,page,dtype,kind", [(256, 16, BF, BF), (128, 64, FP, FP), (256, 64, BF, E4), (128, 16, FP, E4)])
def test_many_ends_inside_a_tile(dim, page, dtype, kind):
    """Hundreds of sequences whose last rows are cleared in a slot that is loaded
    again at once: the same bits from every call, and the formula's."""
    lens = [(1, 1 + (13 * i) % 79) for i in range(600)]
    c = batch(1, lens, 4, 2, dim, page, dtype, kind)
    out = call(c)
    check(out, *ref.attention(c[2], c[0], c[1], c[4], c[3]))
    same = torch.ones((), dtype=torch.bool, device=DEV)
    for _ in range(20):
        same &= (call(c) == out).all()
    assert bool(same)


# ---------------------------------------------------------------- broken offsets

@pytest.mark.parametrize("max_q", [1, 1000])
def test_offsets_that_go_back_and_forth_are_refused(max_q):
    """Every second sequence has all rows: 500 x 1000 rows over 243 million keys
    each are more key tiles than 31 bits count.  Nothing is read or written for
    them, the error word says why, and the next call is right."""
    cache = kvcache.PagedKV(4, 16, 1, 128, BF, DEV)
    q = torch.randn(1000, 1, 128, device=DEV).to(BF)
    pages = 15_200_000
    table = torch.zeros(1, pages, dtype=torch.int32, device=DEV).expand(1000, -1)
    cu = torch.zeros(1001, dtype=torch.int32, device=DEV)
    cu[1::2] = 1000
    kv = torch.full((1000,), pages * 16, dtype=torch.int32, device=DEV)
    out = torch.full_like(q, 5.0)
    moe.check_errors(DEV)
    try:
        attention.paged_attention(q, cache, table, kv, cu, max_q=max_q, out=out)
        with pytest.raises(RuntimeError, match="code 58: .*cu_q"):
            moe.check_errors(DEV)
    finally:
        moe.error_word(DEV).zero_()
    assert bool((out == 5.0).all())
    lens = torch.full((1000,), 50, dtype=torch.int32, device=DEV)
    got = attention.paged_attention(q, cache, table[:, :4], lens, max_q=max_q)
    check(got, *ref.attention(q, cache, table[:, :4], lens))


# ---------------------------------------------------------------- not finite

def plain(q, cache, table, kv_lens, cu):
    """(out, bound) in 64 bits where scores may be infinite or NaN; rows that see
    no key are zeros.  The bound is tests/attention_reference.py's with the
    largest |v| in the place of the weighted mean of |v|, over finite scores."""
    T, H, D = q.shape
    k, v = ref.values(cache)
    G, out = H // cache.kv_heads, torch.zeros(T, H, D, dtype=torch.float64, device=DEV)
    bound = torch.zeros_like(out)
    step = ref.half_step(q.dtype) * (2 if cache.e4m3 else 1)
    for b, L in enumerate(kv_lens.tolist()):
        q0, q1 = int(cu[b]), int(cu[b + 1])
        n = q1 - q0
        if L == 0:
            continue
        at = table[b].long()
        kk, vv = (x[at].transpose(0, 1).reshape(cache.kv_heads, -1, D)[:, :L] for x in (k, v))
        see = torch.arange(L, device=DEV)[None] <= torch.arange(L - n, L, device=DEV)[:, None]
        for h in range(H):
            x = q[q0:q1, h].double()
            s = (x @ kk[h // G].T * D ** -0.5).masked_fill(~see, -torch.inf)
            p = torch.where(see.any(-1, keepdim=True), torch.softmax(s, -1), 0.0)
            out[q0:q1, h] = p @ vv[h // G]
            qk = (x.abs() @ kk[h // G].abs().T).nan_to_num(0, 0, 0).amax(-1, keepdim=True) * D ** -0.5
            score = qk * (D + 8) * 2.0 ** -24 + 2.0 ** -21
            bound[q0:q1, h] = vv[h // G].abs().amax() * (step + 2 * score + L * 2.0 ** -23 + 2.0 ** -24)
    fin = torch.finfo(q.dtype)
    return out, bound + ref.half_step(q.dtype) * out.nan_to_num().abs() + fin.smallest_normal * ref.half_step(q.dtype)


def same_kind(out, want, bound):
    """NaN where the formula has NaN, zeros and values where it has them."""
    assert torch.equal(out.isnan(), want.isnan())
    ok = ~want.isnan()
    assert bool(((out.double() - want)[ok].abs() <= bound[ok]).all())
    moe.check_errors(DEV)


# one piece a sequence, and sequences that several SMs share
WHOLE, SPLIT = [(0, 40), (2, 1), (0, 0)], [(0, 5000), (2, 1)]
SHAPES = [(256, 8, 2, 64, BF, BF), (128, 8, 2, 16, FP, FP), (256, 8, 2, 64, BF, E4), (128, 12, 2, 32, FP, E4)]


def some(lens, n, seed, shape):
    """A batch whose first sequences have n new tokens (0 stands for n)."""
    return batch(seed, [(a or n, kv) for a, kv in lens], shape[1], shape[2], shape[0], *shape[3:])


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("lens", [WHOLE, SPLIT], ids=["whole", "split"])
@pytest.mark.parametrize("n", [1, 3, 40])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_a_query_that_is_not_finite_gives_nan_to_its_row_alone(shape, lens, n, bad):
    c = some(lens, n, 3, shape)
    q = c[2].clone()
    q[n - 1, 1] = bad                                  # the last row, one head of it
    q[-1, 0, 5] = bad                                  # sequence of two rows and one key, or of n and none
    want, bound = plain(q, c[0], c[1], c[4], c[3])
    assert bool(want[n - 1, 1].isnan().all()) and int(want.isnan().any(-1).sum()) == (2 if lens is SPLIT else 1)
    same_kind(call(c, q), want, bound)


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("lens", [WHOLE, SPLIT], ids=["whole", "split"])
@pytest.mark.parametrize("n", [1, 3, 40])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_a_visible_key_that_is_not_finite(shape, lens, n, bad):
    """NaN, or an infinite score above all others, gives NaN; a score of -inf
    takes its key away.  Rows that do not see the key are as they were."""
    c = some(lens, n, 4, shape)
    q, kv, page = c[2].clone(), lens[0][1], c[0].page_size
    q[:, ::2, 9], q[:, 1::2, 9] = 1.0, -1.0
    for j in (kv - 2, 7):                              # the last row but one sees the former
        k = c[0].k.clone()
        where = (int(c[1][0, j // page]), 1, j % page)
        if c[0].e4m3:                                  # as a row with one such element is written
            c[0].k[where].view(torch.uint8)[9] = 0x7F
        else:
            c[0].k[where][9] = bad
        want, bound = plain(q, c[0], c[1], c[4], c[3])
        gone = want[n - 1].isnan().all(-1).sum()
        assert int(gone) == shape[1] // shape[2] // (1 if c[0].e4m3 or bad != bad else 2)
        same_kind(call(c, q), want, bound)
        c[0].k.copy_(k)


@pytest.mark.parametrize("shape", SHAPES[:2])
@pytest.mark.parametrize("lens", [WHOLE, SPLIT], ids=["whole", "split"])
@pytest.mark.parametrize("n", [1, 3, 40])
def test_scores_of_minus_infinity_alone(shape, lens, n):
    """As the quotient 0 / 0, and unlike a row that sees no key."""
    c = some(lens, n, 5, shape)
    c[0].k[..., 0] = float("-inf")
    q = c[2].clone()
    q[..., 0] = 1.0
    want, bound = plain(q, c[0], c[1], c[4], c[3])
    assert bool(want[:n].isnan().all())
    same_kind(call(c, q), want, bound)


# ---------------------------------------------------------------- codes

@pytest.mark.parametrize("dim,heads,hk,page,dtype", [(256, 8, 2, 64, BF), (128, 8, 2, 16, FP), (256, 16, 2, 32, FP), (128, 12, 2, 128, BF)])
@pytest.mark.parametrize("n", [1, 2, 40])
@pytest.mark.parametrize("length", [50, 300, 4000])
def test_values_far_above_those_that_count(dim, heads, hk, page, dtype, n, length):
    """Every 20th key has values 2^22 times the others' and a score that takes
    it out: what is left is theirs, with all of its bits."""
    c = batch(7, [(n, length), (n, max(1, length // 3))], heads, hk, dim, page, dtype, E4)
    cache, table, q, cu, kv = c
    q[..., 0] = 20.0
    g = torch.Generator(device=DEV).manual_seed(2)
    for b, L in enumerate(kv.tolist()):
        k, v = (torch.randn(L, hk, dim, generator=g, device=DEV) for _ in range(2))
        k[..., 0] = 0.0
        v *= 2.0 ** -7
        loud = torch.arange(L, device=DEV) % 20 == 3
        k[loud, :, 0] = -40.0
        v[loud] *= 2.0 ** 22
        i = torch.arange(L, device=DEV)
        kvcache.write(cache, k.to(dtype), v.to(dtype).clamp(-3e4, 3e4), table[b].long()[i // page] * page + i % page)
    want, _ = ref.attention(q, cache, table, kv, cu)
    # as in the reference's bound, but instead of 2^-24 of the largest value a half
    # step 2^-25 of fp16 over the unit 2^15, which is at most twice a scale, for
    # each key: 2^-39 of the largest value
    K, V = ref.values(cache)
    bound = torch.zeros_like(want)
    step = 2 * ref.half_step(dtype)
    for b, L in enumerate(kv.tolist()):
        r = slice(int(cu[b]), int(cu[b + 1]))
        at = table[b].long()
        kk, vv = (x[at].transpose(0, 1).reshape(hk, -1, dim)[:, :L] for x in (K, V))
        see = torch.arange(L, device=DEV)[None] <= torch.arange(L - n, L, device=DEV)[:, None]
        for h in range(heads):
            x, kh, vh = q[r, h].double(), kk[h // (heads // hk)], vv[h // (heads // hk)]
            p = torch.softmax((x @ kh.T * dim ** -0.5).masked_fill(~see, -torch.inf), -1).nan_to_num()
            qk = (x.abs() @ kh.abs().T).amax(-1, keepdim=True) * dim ** -0.5
            err = step + 2 * (qk * (dim + 8) * 2.0 ** -24 + 2.0 ** -21) + L * 2.0 ** -23
            bound[r, h] = p @ vh.abs() * err + L * 2.0 ** -39 * vh.abs().amax()
    fin = torch.finfo(dtype)
    bound += ref.half_step(dtype) * want.abs() + fin.smallest_normal * ref.half_step(dtype)
    check(call((cache, table, q, cu, kv)), want, bound)


@pytest.mark.parametrize("dim,heads,hk,page", [(256, 8, 2, 64), (128, 8, 2, 16), (256, 16, 2, 32), (128, 12, 2, 128)])
@pytest.mark.parametrize("n", [1, 2, 40])
@pytest.mark.parametrize("top", [2.0 ** 18, 2.0 ** 24, -2.0 ** 120])
def test_a_query_element_far_above_the_others(dim, heads, hk, page, n, top):
    """One element of a row is huge and meets zeros in every key: the scores are
    the other elements'.  The bound counts |q| |k|, so nothing of it is the huge
    one's; queries that become fp16 may lose a step 2^-25 over 2^14, of the
    largest element, of each element."""
    c = batch(8, [(n, 300), (n, 70)], heads, hk, dim, page, BF, E4)
    cache, table, q, cu, kv = c
    cache.k[..., 5] = 0
    big = q.clone()
    big[..., 5] = top
    want, bound = ref.attention(big, cache, table, kv, cu)
    K, V = ref.values(cache)
    fin = lambda x: x.nan_to_num()
    lost = 2.0 ** -39 * abs(top) * fin(K).abs().sum(-1).amax() * dim ** -0.5
    if top < 2.0 ** 30:
        bound = bound + 2 * lost * fin(V).abs().amax()
        got = call((cache, table, big, cu, kv))
        check(got, want, bound)
    else:       # too far above: what is left of the others is under fp16's least step or not, but finite
        got = call((cache, table, big, cu, kv))
        moe.check_errors(DEV)
        assert bool(got.isfinite().all())


# ---------------------------------------------------------------- views

@pytest.mark.parametrize("kind", [BF, E4])
@pytest.mark.parametrize("t", [slice(0, 1), slice(2, 3), slice(1, 2), slice(0, 5)])
def test_tokens_cut_from_a_buffer_of_an_odd_pitch(kind, t):
    """Rows 2568 bytes apart: one of them (its pitch means nothing) as several."""
    pitch = torch.randn(5, 1284, device=DEV).to(BF)
    x = pitch[:, :1024].view(5, 8, 128)[t]
    q, k, v = x[:, :4], x[:, 4:6], x[:, 6:]
    n = x.shape[0]
    w, f = torch.ones(128, dtype=BF, device=DEV), attention.rope_frequencies(64, device=DEV)
    pos, slots = torch.arange(n, device=DEV), torch.arange(n, device=DEV) + 3
    table = torch.zeros(1, 1, dtype=torch.int32, device=DEV)
    lens, cu = torch.tensor([n + 3], dtype=torch.int32, device=DEV), torch.tensor([0, n], dtype=torch.int32, device=DEV)

    def run(q, k, v):
        cache = kvcache.PagedKV(1, 16, 2, 128, kind, DEV)
        kvcache.write(cache, k, v, slots)
        first = kvcache.read(cache, slots, dtype=BF)
        turned = attention.qk_norm_rope(q, k, w, w, pos, f)
        qw = attention.qk_norm_rope_write(q, k, v, w, w, pos, f, cache, slots)
        a = attention.paged_attention(q, cache, table, lens, cu, max_q=n)
        return (*first, *turned, qw, a, *kvcache.read(cache, slots, dtype=BF))
    for a, b in zip(run(q, k, v), run(q.clone(), k.clone(), v.clone())):
        assert torch.equal(a, b)
    if n == 1 and q.data_ptr() % 16 == 0:              # ... and as outputs
        want = run(q, k, v)
        cache = kvcache.PagedKV(1, 16, 2, 128, kind, DEV)
        kvcache.write(cache, k, v, slots)
        attention.qk_norm_rope_write(q.clone(), k, v, w, w, pos, f, cache, slots)
        before = pitch.clone()
        assert attention.paged_attention(q, cache, table, lens, out=q) is q
        assert torch.equal(q, want[5])
        back = before[:, :1024].view(5, 8, 128)[t]
        attention.qk_norm_rope(back[:, :4], back[:, 4:6], w, w, pos, f, out=(q, k))
        assert torch.equal(q, want[2]) and torch.equal(k, want[3])
    moe.check_errors(DEV)


# ---------------------------------------------------------------- zeros

@pytest.mark.parametrize("dim", [128, 256])
@pytest.mark.parametrize("dtype", [BF, FP])
def test_a_negative_zero_keeps_its_sign(dim, dtype):
    """Codes are those of the formula bit for bit, 0x80 for -0 among them, and
    read back as -0; in rows of zeros as in others."""
    g = torch.Generator(device=DEV).manual_seed(1)
    x = torch.randn(70, 2, dim, generator=g, device=DEV).to(dtype)
    x[torch.rand(x.shape, generator=g, device=DEV) < 0.2] = -0.0
    x[3], x[4], x[5, :, 1:] = -0.0, 0.0, -0.0
    w, f = torch.ones(dim, dtype=dtype, device=DEV), attention.rope_frequencies(64, device=DEV)
    slots = torch.arange(70, device=DEV)
    code, scale = (t.to(DEV) for t in ref.quantise(x.cpu()))
    assert int((code.view(torch.uint8) == 0x80).sum()) > 1000
    for call in (lambda c: kvcache.write(c, x, x, slots),
                 lambda c: attention.qk_norm_rope_write(x, x, x, w, w, slots, f, c, slots)):
        cache = kvcache.PagedKV(5, 16, 2, dim, E4, DEV)
        call(cache)
        put = lambda t: t.transpose(1, 2).reshape(80, 2, *t.shape[3:])[:70]
        assert torch.equal(put(cache.v.view(torch.uint8)), code.view(torch.uint8))
        assert torch.equal(put(cache.v_scale), scale)
        back = kvcache.read(cache, slots, dtype=dtype)[1]
        want = (code.float() * scale[..., None]).to(dtype)
        assert torch.equal(back.view(torch.int16), want.view(torch.int16))


@pytest.mark.parametrize("dim,heads,hk,page,dtype", [(256, 8, 2, 64, BF), (128, 8, 2, 16, FP)])
@pytest.mark.parametrize("n", [1, 2, 40])
@pytest.mark.parametrize("share", [0.5, 1.0])
def test_negative_scales(dim, heads, hk, page, dtype, n, share):
    """A caller's own cache (value = code * scale) may have them, here and there
    or everywhere."""
    c = batch(11, [(n, 300), (n, 70)], heads, hk, dim, page, dtype, E4)
    g = torch.Generator(device=DEV).manual_seed(4)
    for s in (c[0].k_scale, c[0].v_scale):
        turn = torch.rand(s.shape, generator=g, device=DEV) < share
        s.mul_(torch.where(turn, -1.0, 1.0)).mul_(2.0 ** torch.randint(-3, 4, s.shape, generator=g, device=DEV))
    check(call(c), *ref.attention(c[2], c[0], c[1], c[4], c[3]))
