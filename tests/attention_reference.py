"""Plain 64-bit forms of the K/V cache and attention operators, for tests, and
the error each operator's roundings allow."""
import math

import torch

E4 = torch.float8_e4m3fn


def half_step(dtype) -> float:
    """Largest relative error of one rounding to ``dtype``."""
    return torch.finfo(dtype).eps / 2


def quantise(x: torch.Tensor):
    """(codes e4m3, scale fp32) of rows x [..., D] by the cache's formula; fp32
    divisions, as the formula says."""
    x = x.float()
    amax = x.abs().amax(-1)
    scale = torch.where(amax > 0, amax / torch.full_like(amax, 448.0), torch.ones_like(amax))
    return (x / scale[..., None]).to(E4), scale


def norm_rope(x, weight, positions, inv_freq, eps, offset, interleaved):
    """x [T, heads, D] -> float64."""
    y = x.double()
    y = y / (y.square().mean(-1, keepdim=True) + eps).sqrt() * (weight.double() + offset)
    half = inv_freq.numel()
    a = positions.double()[:, None, None] * inv_freq.double()
    c, s = a.cos(), a.sin()
    i = torch.arange(half, device=x.device)
    p, q = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    u, v = y[..., p], y[..., q]
    y = y.clone()
    y[..., p], y[..., q] = u * c - v * s, v * c + u * s
    return y


def norm_rope_bound(ref, dtype):
    """Rounding to dtype, the fp32 steps before it (a sum of squares, a root, a
    quotient, two products and the rotation's three operations with its sine and
    cosine: under 32 steps of 2^-24 of the larger of the pair) and the subnormal
    step of fp16."""
    big = ref.abs().amax(-1, keepdim=True)
    return half_step(dtype) * ref.abs() + 32 * 2.0 ** -24 * 2 * big + torch.finfo(dtype).smallest_normal * half_step(dtype)


def values(cache):
    """(k, v) of a PagedKV as float64 [pages, heads, page, D]."""
    out = []
    for x, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
        y = x.double() if x.dtype != E4 else x.float().double()
        out.append(y if s is None else y * s.double()[..., None])
    return out


def attention(q, cache, table, kv_lens, cu_q=None, scale=None):
    """(out, bound) float64 [T, heads, D]; rows of no sequence are NaN in out."""
    T, H, D = q.shape
    scale = D ** -0.5 if scale is None else scale
    k, v = values(cache)
    ps, G = cache.page_size, H // cache.kv_heads
    out = torch.full((T, H, D), math.nan, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    lens = kv_lens.tolist()
    cu = cu_q.tolist() if cu_q is not None else list(range(len(lens) + 1))
    e4 = cache.dtype == E4
    # the probabilities are rounded to 16 bits (and, over codes, so are scaled
    # values); the products of D terms and the sums of L terms are fp32
    step = half_step(q.dtype) * (2 if e4 else 1)
    for b, L in enumerate(lens):
        n, q0 = cu[b + 1] - cu[b], cu[b]
        L = min(L, table.shape[1] * ps)
        kk, vv = (torch.zeros(cache.kv_heads, L, D, dtype=torch.float64, device=q.device) for _ in range(2))
        for j in range(0, L, ps):
            page = int(table[b, j // ps])
            if 0 <= page < cache.pages:
                m = min(ps, L - j)
                kk[:, j:j + m], vv[:, j:j + m] = k[page, :, :m], v[page, :, :m]
        for h in range(H):
            x = q[q0:q0 + n, h].double()
            s = x @ kk[h // G].T * scale
            see = torch.arange(L, device=q.device)[None] <= torch.arange(L - n, L, device=q.device)[:, None]
            s = s.masked_fill(~see, -math.inf)
            any_ = see.any(-1, keepdim=True)
            p = torch.where(any_, torch.softmax(s, -1), torch.zeros_like(s)) if L else s
            out[q0:q0 + n, h] = p @ vv[h // G]
            if L:
                mass = p @ vv[h // G].abs()
                qk = (x.abs() @ kk[h // G].abs().T).amax(-1, keepdim=True) * abs(scale)
                score = qk * (D + 8) * 2.0 ** -24 + 2.0 ** -21
                bound[q0:q0 + n, h] = mass * (step + 2 * score + L * 2.0 ** -23)
                bound[q0:q0 + n, h] += 2.0 ** -24 * vv[h // G].abs().amax() if e4 or q.dtype == torch.float16 else 0
    fin = torch.finfo(q.dtype)
    bound += half_step(q.dtype) * out.nan_to_num().abs() + fin.smallest_normal * half_step(q.dtype)
    return out, bound
