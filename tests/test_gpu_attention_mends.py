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
