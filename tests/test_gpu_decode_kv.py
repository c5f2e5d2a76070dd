"""DecodeStack over the paged K/V cache: the norm and rotation, the cache write
and the attention as a decode token's full-attention layer calls them, eager
and in the captured step."""
import pytest
import torch

import attention_reference as ref
from conftest import cuda_available

pytestmark = [pytest.mark.gpu,
              pytest.mark.skipif(not cuda_available(), reason="needs a CUDA GPU")]

from drama3_offloading_b200 import attention, decode, moe  # noqa: E402

DEV = torch.device("cuda:0")
CTX = 200                                              # not a multiple of the page


def stack(kind, **kw):
    return decode.DecodeStack(layers=8, experts=16, hidden=512, inter=512, topk=4, capacity=8,
                              dense_gib=0.06, kv_context=CTX, device=DEV, l2_warm_mib=1.0,
                              kv_cache=kind, **kw)


def test_dense_is_the_default_and_unknown_kinds_are_refused():
    s = stack("dense")
    assert sorted(s.kv) == [3, 7] and not s.paged and s.launches_per_step() == 32
    assert s.kv_bytes == 2 * 2 * CTX * 2 * 256 * 2
    with pytest.raises(ValueError, match="kv_cache"):
        stack("fp8")


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
def test_layer_attention_against_the_plain_form(kind):
    """One layer's attention, step by step round the ring's end, against the
    64-bit form over the cache the step left; the operators between (the
    projection, the addition) are torch's, the same on both sides."""
    s = stack(kind)
    g = torch.Generator(device=DEV).manual_seed(3)
    cache = s.paged[3]
    for pos in (CTX, CTX + 1, 3 * CTX - 1, 3 * CTX):
        s.kv_pos.fill_(pos)
        h0 = torch.randn(1, 512, generator=g, device=DEV).to(torch.bfloat16)
        s.h.copy_(h0)
        before = [t.clone() for t in s._paged_state()]
        _, slot = s._next()
        s._paged_attention(3, slot)
        kv = (h0 @ s.kv_proj[3].t()).view(1, 4, 256)
        at = (slot // 64, slice(None), slot % 64)
        # the ring's slot holds the token's K, turned to its position, and V
        want = ref.norm_rope(kv[:, :2], s.qk_norm, s.kv_pos, s.inv_freq, 1e-6, 0.0, False)
        K, V = ref.values(cache)
        # (codes: half a step of the row's type and of 2^-3 of a code; amax / 448 is a
        # code's scale, so one of its smallest steps, 2^-9, is amax / 448 * 2^-9)
        tol = ref.norm_rope_bound(want, torch.bfloat16)
        small = lambda x: x.abs().amax(-1, keepdim=True) / 448 * 2.0 ** -9
        if kind == "e4m3":
            tol = want.abs() * 2.0 ** -4 * 1.001 + small(want) + tol
        assert ((K[at] - want).abs() <= tol).all()
        v = kv[:, 2:].double()
        vtol = v.abs() * 2.0 ** -4 * 1.001 + small(v) if kind == "e4m3" else 0
        assert ((V[at] - v).abs() <= vtol).all()
        # ... and no other slot has changed
        for old, new in zip(before[1:], s._paged_state()[1:]):
            old, new = old.view(torch.uint8), new.view(torch.uint8)
            if new.data_ptr() in (cache.k.data_ptr(), cache.v.data_ptr()):
                old[slot // 64, :, slot % 64] = new[slot // 64, :, slot % 64]
                assert torch.equal(old, new)
        q = attention.qk_norm_rope(h0.view(1, 2, 256), kv[:, :2], s.qk_norm, s.qk_norm, s.kv_pos,
                                   s.inv_freq)[0]
        out, bound = ref.attention(q, cache, s.kv_table, s.kv_lens)
        # the sum's own rounding, a half step, and the addend's
        got, plain = s.h.double().view(1, 2, 256), h0.double().view(1, 2, 256) + 0.25 * out
        assert ((got - plain).abs() <= 0.25 * bound + (plain.abs() + 0.25 * bound) * 2.0 ** -8).all()
    moe.check_errors()


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
def test_steps_eager_captured_and_restored(kind):
    """The captured step walks the ring as the eager one does, bit for bit, from
    a reset and from a snapshot."""
    s = stack(kind)
    assert s.launches_per_step() == 32 + 6
    s.reset()
    s.h.fill_(0.5)
    eager = []
    for _ in range(5):
        s.step()
        eager.append(s.h.clone())
    assert int(s.kv_pos) == CTX + 5 and torch.isfinite(eager[-1].float()).all()
    state = [t.clone() for t in s._paged_state()]
    g = s.capture()                                    # resets
    assert int(s.kv_pos) == CTX
    s.h.fill_(0.5)
    snap = None
    for i in range(5):
        if i == 2:
            snap = s.snapshot()
        g.replay()
        assert torch.equal(s.h, eager[i]), i
    for a, b in zip(state, s._paged_state()):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    s.restore(snap)
    for i in range(2, 5):
        g.replay()
        assert torch.equal(s.h, eager[i]), i
    s.reset()
    assert int(s.kv_pos) == CTX
    s.sample_fetch_timing(2)
    assert int(s.kv_pos) == CTX + 2
    moe.check_errors()
