"""Calls of the paged attention and the cache operators at the edges of what
their documentation allows, against the 64-bit plain forms."""
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
    """(cache, table, q, cu_q, kv_lens): lens of (new tokens, keys); what no
    sequence has written is NaN, table entries behind a sequence are garbage."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    width = max(-(-kv // page) for _, kv in lens) + 1
    used = sum(-(-kv // page) for _, kv in lens)
    cache = kvcache.PagedKV(used + 2, page, hk, dim, kind, DEV)
    for x in (cache.k, cache.v):
        x.view(torch.uint8).fill_(0x7F) if kind == E4 else x.fill_(float("nan"))
    for s in (cache.k_scale, cache.v_scale):
        if s is not None:
            s.fill_(float("nan"))
    ids = torch.randperm(used + 2, generator=g, device=DEV).to(torch.int32)
    table = torch.full((len(lens), width), 2 ** 31 - 1, dtype=torch.int32, device=DEV)
    slots, at = [], 0
    for b, (_, kv) in enumerate(lens):
        n = -(-kv // page)
        table[b, :n] = ids[at:at + n]
        i = torch.arange(kv, device=DEV)
        slots.append(ids[at:at + n].long()[i // page] * page + i % page)
        at += n
    slots = torch.cat(slots)
    rnd = lambda *s: torch.randn(*s, generator=g, device=DEV).to(dtype)
    kvcache.write(cache, rnd(slots.numel(), hk, dim), rnd(slots.numel(), hk, dim), slots)
    ns = torch.tensor([0] + [n for n, _ in lens])
    cu = ns.cumsum(0).to(torch.int32).to(DEV)
    kv = torch.tensor([kv for _, kv in lens], dtype=torch.int32, device=DEV)
    return cache, table, rnd(int(cu[-1]), heads, dim), cu, kv


def check(out, want, bound):
    live = ~want[:, 0, 0].isnan()
    assert bool(((out.double() - want)[live].abs() <= bound[live]).all())
    moe.check_errors(DEV)


@pytest.mark.parametrize("heads,hk", [(128, 1), (100, 1), (65, 1), (40, 1), (34, 2)])
@pytest.mark.parametrize("dim,kind", [(128, BF), (256, E4), (128, E4)])
def test_many_query_heads_on_a_kv_head(heads, hk, dim, kind):
    c = batch(heads, [(1, 300), (3, 130), (2, 2), (9, 700)], heads, hk, dim, 32, BF, kind)
    check(attention.paged_attention(c[2], c[0], c[1], c[4], c[3], max_q=9),
          *ref.attention(c[2], c[0], c[1], c[4], c[3]))
    one = batch(heads + 1, [(1, 300), (1, 1), (1, 0)], heads, hk, dim, 32, BF, kind)
    check(attention.paged_attention(one[2], one[0], one[1], one[4]), *ref.attention(one[2], one[0], one[1], one[4]))


@pytest.mark.parametrize("heads,n", [(9, 1), (12, 1), (16, 1), (5, 3), (3, 5), (2, 8), (1, 16), (1, 13)])
@pytest.mark.parametrize("dim,page,dtype,kind", [(256, 64, BF, BF), (256, 16, BF, E4), (128, 128, FP, E4), (128, 32, FP, FP)])
def test_nine_to_sixteen_rows(heads, n, dim, page, dtype, kind):
    lens = [(n, 700), (n, n), (1, 129), (n, 0), (n, 128), (0, 50), (n, 257)]
    c = batch(heads * n, lens, heads, 1, dim, page, dtype, kind)
    check(attention.paged_attention(c[2], c[0], c[1], c[4], c[3], max_q=n),
          *ref.attention(c[2], c[0], c[1], c[4], c[3]))


@pytest.mark.parametrize("kind", [BF, E4])
@pytest.mark.parametrize("said", [1, 2, 3, 39, 41, 10 ** 6])
def test_max_q_that_is_not_the_longest(said, kind):
    """max_q chooses the launch, not the answer."""
    c = batch(7, [(40, 200), (1, 77), (2, 300), (5, 5)], 8, 2, 128, 16, BF, kind)
    check(attention.paged_attention(c[2], c[0], c[1], c[4], c[3], max_q=said, max_kv=said),
          *ref.attention(c[2], c[0], c[1], c[4], c[3]))


@pytest.mark.parametrize("kind", [BF, E4])
def test_a_thousand_sequences(kind):
    lens = [(1, (37 * i) % 150) for i in range(1000)]
    c = batch(1, lens, 4, 2, 128, 16, BF, kind)
    want = ref.attention(c[2], c[0], c[1], c[4])
    check(attention.paged_attention(c[2], c[0], c[1], c[4]), *want)
    # said to be a padded batch of chunks
    check(attention.paged_attention(c[2], c[0], c[1], c[4], c[3], max_q=64), *want)
    mixed = [((31 * i) % 40 if i % 7 == 0 else 1, (37 * i) % 150) for i in range(700)]
    c = batch(2, mixed, 4, 2, 128, 16, BF, kind)
    check(attention.paged_attention(c[2], c[0], c[1], c[4], c[3], max_q=40),
          *ref.attention(c[2], c[0], c[1], c[4], c[3]))


@pytest.mark.parametrize("n", [1, 40])
def test_lengths_behind_the_table_and_empty_calls(n):
    c = batch(3, [(n, 200), (n, 64)], 8, 2, 256, 64, BF, BF)
    table = c[1][:, :3].contiguous()                   # 192 tokens wide
    check(attention.paged_attention(c[2], c[0], table, c[4], c[3], max_q=n),
          *ref.attention(c[2], c[0], table, c[4], c[3]))
    out = attention.paged_attention(c[2], c[0], c[1][:, :0], c[4], c[3], max_q=n)
    assert bool((out == 0).all())                      # a table of no pages: rows see nothing
    none = attention.paged_attention(c[2][:0], c[0], c[1], c[4], torch.zeros_like(c[3]), max_q=n)
    assert none.shape == (0, 8, 256)
    kept = torch.full_like(c[2], 3.0)
    attention.paged_attention(c[2], c[0], c[1][:0], c[4][:0], c[3][:1], max_q=n, out=kept)
    assert bool((kept == 3.0).all())                   # no sequences: no row is anyone's
    moe.check_errors(DEV)


@pytest.mark.parametrize("kind", [BF, E4])
@pytest.mark.parametrize("n", [1, 3, 40])
def test_broadcast_and_misaligned_queries_and_outputs_in_place(n, kind):
    c = batch(5, [(n, 333), (n, 90)], 8, 2, 128, 32, BF, kind)
    q = c[2][:, :1].expand(-1, 8, -1)                  # head stride 0
    got = attention.paged_attention(q, c[0], c[1], c[4], c[3], max_q=n)
    check(got, *ref.attention(q, c[0], c[1], c[4], c[3]))
    odd = torch.empty(c[2].numel() + 1, dtype=BF, device=DEV)[1:].view_as(c[2]).copy_(c[2])
    out = attention.paged_attention(c[2], c[0], c[1], c[4], c[3], max_q=n)
    assert torch.equal(attention.paged_attention(odd, c[0], c[1], c[4], c[3], max_q=n), out)
    back = c[2].transpose(0, 1).contiguous().transpose(0, 1)      # heads outermost
    assert torch.equal(attention.paged_attention(back, c[0], c[1], c[4], c[3], max_q=n), out)
    tall = c[1].t().contiguous().t()                   # a table whose columns are contiguous
    assert torch.equal(attention.paged_attention(c[2], c[0], tall, c[4], c[3], max_q=n), out)
    mine = c[2].clone()
    assert attention.paged_attention(mine, c[0], c[1], c[4], c[3], max_q=n, out=mine) is mine
    assert torch.equal(mine, out)
    moe.check_errors(DEV)


@pytest.mark.parametrize("n", [1, 40])
def test_sequences_that_share_pages(n):
    c = batch(6, [(n, 150), (n, 150), (n, 40)], 8, 2, 256, 64, BF, E4)
    table = c[1].clone()
    table[1, :2], table[2, 0] = table[0, :2], table[0, 0]
    check(attention.paged_attention(c[2], c[0], table, c[4], c[3], max_q=n),
          *ref.attention(c[2], c[0], table, c[4], c[3]))


@pytest.mark.parametrize("kind", [BF, E4])
def test_a_stream_given_to_every_call(kind):
    """Each call on the stream it is told, in order there, whatever the current
    one is."""
    c = batch(8, [(3, 200), (40, 90)], 8, 2, 128, 32, BF, kind)
    w = torch.ones(128, dtype=BF, device=DEV)
    f = attention.rope_frequencies(64, device=DEV)
    pos = torch.arange(43, device=DEV)
    k = torch.randn(43, 2, 128, device=DEV).to(BF)
    free = (set(range(c[0].pages)) - set(c[1].flatten().tolist()))
    slots = torch.full((43,), -1, dtype=torch.int32, device=DEV)
    slots[:32] = min(free) * 32 + torch.arange(32, device=DEV)
    other = kvcache.PagedKV.from_tensors(*(x.clone() if x is not None else None
                                           for x in (c[0].k, c[0].v, c[0].k_scale, c[0].v_scale)))

    def run(cache, **kw):
        q = attention.qk_norm_rope_write(c[2], k, k, w, w, pos, f, cache, slots, **kw)
        a = attention.paged_attention(q, cache, c[1], c[4], c[3], max_q=40, **kw)
        kvcache.write(cache, k[:1], k[1:2], slots[:1], **kw)
        return (q, a, *kvcache.read(cache, slots[:32], dtype=BF, **kw),
                *attention.qk_norm_rope(c[2], k, w, w, pos, f, **kw))
    want = run(c[0])
    torch.cuda.synchronize()
    side = torch.cuda.Stream(device=DEV)
    side.wait_stream(torch.cuda.current_stream())
    got = run(other, stream=side)
    side.synchronize()
    with torch.cuda.stream(side):
        again = run(other)
    side.synchronize()
    for a, b, d in zip(want, got, again):
        assert torch.equal(a, b) and torch.equal(a, d)
    moe.check_errors(DEV)


@pytest.mark.parametrize("kind", [BF, E4])
def test_a_slot_named_twice_harms_no_other(kind):
    cache = kvcache.PagedKV(4, 16, 2, 128, kind, DEV)
    k = torch.randn(40, 2, 128, device=DEV).to(BF)
    slots = torch.arange(40, device=DEV) + 10
    kvcache.write(cache, k, k, slots)
    before = [x.clone() for x in kvcache.read(cache, torch.arange(64, device=DEV), dtype=BF)]
    slots[7] = slots[3]
    kvcache.write(cache, 2 * k, 2 * k, slots)
    after = kvcache.read(cache, torch.arange(64, device=DEV), dtype=BF)
    twice = torch.zeros(64, dtype=torch.bool, device=DEV)
    twice[slots] = True
    for b, a in zip(before, after):
        assert torch.equal(a[~twice], b[~twice])
        twice[13] = False                              # the slot named twice: parts of either
        assert torch.equal(a[twice], 2 * b[twice])
        twice[13] = True


def test_keys_hidden_by_the_mask_may_hold_anything():
    """K rows that a row's mask hides, infinite or NaN, change nothing for it."""
    for n, dtype in ((5, BF), (40, BF), (40, FP)):
        c = batch(9, [(n, 100)], 8, 2, 128, 32, dtype, dtype)
        want, bound = ref.attention(c[2], c[0], c[1], c[4], c[3])
        page, at = int(c[1][0, 3]), 99 % 32            # the last key: the last row alone sees it
        for bad in (float("inf"), float("nan"), float("-inf")):
            c[0].k[page, :, at] = bad
            out = attention.paged_attention(c[2], c[0], c[1], c[4], c[3], max_q=n)
            check(out[:n - 1], want[:n - 1], bound[:n - 1])
