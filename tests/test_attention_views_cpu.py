"""How the rows of the cache and attention calls are read and written in place,
without a GPU: strides of dimensions of size 1 carry no meaning.  And where a
call runs: never on a stream of another device."""
from types import SimpleNamespace

import pytest
import torch

from drama3_offloading_b200 import kvcache

BF = torch.bfloat16


def addresses(at, s0, s1, shape):
    return [[at + 2 * (t * s0 + h * s1) for h in range(shape[1])] for t in range(shape[0])]


def of_views():
    """Views [tokens, heads, 128] of all sorts: odd pitches, heads outermost,
    single tokens and heads, broadcast ones, odd addresses, no rows at all."""
    pitch = torch.randn(5, 1284).to(BF)
    odd = pitch[:, :1024].view(5, 8, 128)
    wide = torch.randn(5, 11, 128).to(BF)
    tall = torch.randn(8, 5, 128).to(BF).transpose(0, 1)
    flat = torch.randn(1 + 5 * 8 * 128).to(BF)[1:].view(5, 8, 128)
    cols = torch.randn(5, 130).to(BF)
    views = [odd, odd[:1], odd[2:3], odd[:, :1], odd[1:2, :1], odd[:0], wide[:, 2:10], wide[:1, 3:4], tall, tall[:1],
             tall[:, :1], flat, flat[:1], cols[:, None, :128], cols[3:4, None, :128], cols[:1, None, 1:129],
             wide[:1].expand(5, -1, -1), wide[:1, :1].expand(1, 8, -1), wide[:1, :1].expand(1, 1, 128),
             torch.empty(0).to(BF).as_strided((0, 8, 128), (3, 5, 1)),
             torch.randn(400).to(BF).as_strided((1, 1, 128), (7, 3, 1)),
             torch.randn(400).to(BF).as_strided((1, 1, 128), (0, 0, 1)),
             torch.randn(7, 256).to(BF)[:1, None, ::2]]
    return views


@pytest.mark.parametrize("i", range(len(of_views())))
def test_rows_are_read_where_they_lie(i):
    x = of_views()[i]
    t, at, s0, s1 = kvcache.in_place(x)
    assert s0 > 0 and s1 > 0 and s0 % 8 == 0 and s1 % 8 == 0 and at % 16 == 0
    assert torch.equal(t, x)
    if x.numel():
        want = [[t[a, h].data_ptr() for h in range(x.shape[1])] for a in range(x.shape[0])]
        assert addresses(at, s0, s1, x.shape) == want and t.stride(-1) == 1


def test_aligned_rows_of_one_token_or_head_are_not_copied():
    pitch = torch.randn(8, 1284).to(BF)[:, :1024].view(8, 8, 128)     # rows 2568 bytes apart
    for x in (pitch[:1], pitch[2:3], pitch[:1, :1], pitch[:1, 3:4]):
        assert kvcache.in_place(x)[0] is x
    assert kvcache.in_place(pitch[:2])[0] is not pitch


def test_outputs_of_one_token_or_head():
    pitch = torch.randn(5, 1284).to(BF)[:, :1024].view(5, 8, 128)
    for x in (pitch[:1], pitch[2:3], pitch[:1, :1]):
        t, at, s0, s1 = kvcache.output(x, x.shape, BF, -1)
        assert t is x and at == x.data_ptr() and s0 % 8 == 0 and s1 % 8 == 0 and s0 > 0 and s1 > 0
    for x in (pitch[:2], pitch[1:2], pitch[:1].expand(5, -1, -1), pitch[:1, :1].expand(1, 8, -1)):
        with pytest.raises(ValueError):
            kvcache.output(x, x.shape, BF, -1)


def test_a_stream_of_another_device_is_refused():
    """(such a call would else leave the stream for its device's current one)"""
    for device, of in ((0, 1), (1, 0)):
        with pytest.raises(ValueError, match="stream"):
            kvcache.elsewhere(device, SimpleNamespace(device_index=of))
    assert kvcache.elsewhere(1, SimpleNamespace(device_index=1))
