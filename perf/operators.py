"""The attention side of a decode step or a prefill chunk, for measuring: the
norm and rotation of queries and keys, the paged K/V cache that takes keys and
values (16-bit, or e4m3 with a scale per token and head), and the attention
that reads it.

With ``own`` false, ``run`` computes each operator with elementary torch
operations in 32 bits (angles in 64); with ``own`` true it makes the calls of
``drama3_offloading_b200.kvcache`` and ``drama3_offloading_b200.attention``.
"""
import math
import random

import torch

own = False

E4M3_MAX = 448.0
EPS = 1e-6
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "e4m3": torch.float8_e4m3fn}


# ---------------------------------------------------------------- cases

def listed():
    return [
        # one decode token of the 8-query, 2-KV-head, 256-wide attention layers: latency
        {"name": "rope_step", "op": "rope_write", "tokens": 1, "heads": 8, "kv_heads": 2, "dim": 256,
         "rotary": 64, "interleaved": False, "page": 64, "dtype": "bf16", "cache": "bf16", "far": 2048},
        # an odd decode batch far into long documents, norm and rotation alone
        {"name": "rope_batch", "op": "rope", "tokens": 257, "heads": 32, "kv_heads": 8, "dim": 128,
         "rotary": 128, "interleaved": True, "page": 0, "dtype": "fp16", "cache": "", "far": 1000000},
        # a large prefill step: K and V quantised into the cache in the same pass
        {"name": "rope_chunk", "op": "rope_write", "tokens": 8192, "heads": 16, "kv_heads": 2, "dim": 256,
         "rotary": 64, "interleaved": False, "page": 64, "dtype": "bf16", "cache": "e4m3", "far": 32768},
        # a decode batch's keys and values quantised and read back
        {"name": "cache_batch", "op": "write_read", "tokens": 61, "kv_heads": 2, "dim": 256, "page": 16,
         "dtype": "bf16", "cache": "e4m3"},
        # many prompts' keys and values moved through the cache (a prefix stored and restored)
        {"name": "cache_bulk", "op": "write_read", "tokens": 50001, "kv_heads": 8, "dim": 128, "page": 32,
         "dtype": "fp16", "cache": "e4m3"},
        # one decode token over the 2048-token context of the decode benchmark
        {"name": "attend_step", "op": "attend", "batch": 1, "singles": 1, "q_lo": 1, "q_hi": 1, "ctx_lo": 2047,
         "ctx_hi": 2047, "heads": 8, "kv_heads": 2, "dim": 256, "page": 64, "dtype": "bf16", "cache": "bf16"},
        # a ragged decode batch on a quantised cache
        {"name": "attend_batch", "op": "attend", "batch": 64, "singles": 64, "q_lo": 1, "q_hi": 1, "ctx_lo": 17,
         "ctx_hi": 8001, "heads": 16, "kv_heads": 2, "dim": 256, "page": 32, "dtype": "bf16", "cache": "e4m3"},
        # few very long sequences, one token each
        {"name": "attend_long", "op": "attend", "batch": 4, "singles": 4, "q_lo": 1, "q_hi": 1, "ctx_lo": 100000,
         "ctx_hi": 131071, "heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "dtype": "fp16", "cache": "fp16"},
        # a few drafted tokens a sequence, checked together
        {"name": "attend_verify", "op": "attend", "batch": 24, "singles": 0, "q_lo": 3, "q_hi": 7, "ctx_lo": 333,
         "ctx_hi": 6000, "heads": 16, "kv_heads": 2, "dim": 256, "page": 64, "dtype": "bf16", "cache": "bf16"},
        # a 2048-token prefill chunk at the start of a prompt
        {"name": "attend_chunk0", "op": "attend", "batch": 1, "singles": 0, "q_lo": 2048, "q_hi": 2048, "ctx_lo": 0,
         "ctx_hi": 0, "heads": 8, "kv_heads": 2, "dim": 256, "page": 64, "dtype": "bf16", "cache": "bf16"},
        # the same chunk far into a document, more query heads
        {"name": "attend_chunk30k", "op": "attend", "batch": 1, "singles": 0, "q_lo": 2048, "q_hi": 2048,
         "ctx_lo": 30720, "ctx_hi": 30720, "heads": 16, "kv_heads": 2, "dim": 256, "page": 64, "dtype": "bf16",
         "cache": "bf16"},
        # a serving step that mixes chunks with single tokens, quantised cache
        {"name": "attend_mixed", "op": "attend", "batch": 12, "singles": 8, "q_lo": 100, "q_hi": 301, "ctx_lo": 0,
         "ctx_hi": 6001, "heads": 32, "kv_heads": 8, "dim": 128, "page": 16, "dtype": "fp16", "cache": "e4m3"},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rope", "rope_write", "write_read", "attend", "attend", "attend"])
    dim = rng.choice([128, 256])
    kv_heads = rng.choice([1, 2, 4, 8])
    heads = kv_heads * rng.choice([1, 2, 3, 4, 6, 8])
    dtype = rng.choice(["bf16", "fp16"])
    page = rng.choice([16, 32, 64, 128])
    cache = rng.choice([dtype, "e4m3"])
    if op == "rope":
        return {"op": op, "tokens": _log(rng, 1, 8192), "heads": heads, "kv_heads": kv_heads, "dim": dim,
                "rotary": rng.choice([32, 64, dim]), "interleaved": rng.random() < 0.5, "page": 0, "dtype": dtype,
                "cache": "", "far": _log(rng, 16, 1000000)}
    if op == "rope_write":
        return {"op": op, "tokens": _log(rng, 1, 8192), "heads": heads, "kv_heads": kv_heads, "dim": dim,
                "rotary": rng.choice([32, 64, dim]), "interleaved": rng.random() < 0.5, "page": page, "dtype": dtype,
                "cache": cache, "far": _log(rng, 16, 1000000)}
    if op == "write_read":
        return {"op": op, "tokens": _log(rng, 1, 50000), "kv_heads": kv_heads, "dim": dim, "page": page,
                "dtype": dtype, "cache": cache}
    kind = rng.choice(["single", "single", "few", "chunk", "mixed"])
    if kind == "single":
        batch = _log(rng, 1, 128)
        singles, q_lo, q_hi = batch, 1, 1
    elif kind == "few":
        batch, singles = _log(rng, 1, 32), 0
        q_lo, q_hi = rng.randint(1, 4), rng.randint(4, 8)
    elif kind == "chunk":
        batch, singles = rng.randint(1, 3), 0
        q_hi = _log(rng, 16, 2048)
        q_hi = max(16, min(q_hi, 2 ** 17 // (batch * heads)))
        q_lo = max(1, q_hi - rng.randint(0, 40))
    else:
        batch = rng.randint(3, 12)
        singles, q_lo, q_hi = rng.randint(1, batch - 1), rng.randint(9, 60), rng.randint(60, 300)
    # contexts up to 131072 tokens, as far as 1 GB of cached elements and the
    # plain form's scores (9e8 of them) go
    most = min(131071, 2 ** 30 // (batch * kv_heads * dim * 2), int(9e8 // (batch * heads * q_hi)))
    ctx_hi = _log(rng, 16, max(16, most))
    ctx_lo = rng.randint(0, ctx_hi)
    return {"op": "attend", "batch": batch, "singles": singles, "q_lo": q_lo, "q_hi": q_hi, "ctx_lo": ctx_lo,
            "ctx_hi": ctx_hi, "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page, "dtype": dtype,
            "cache": cache}


def _spread(lo, hi, n):
    """n lengths evenly spread over [lo, hi]; hi alone when n is 1."""
    return [hi - (hi - lo) * i // max(1, n - 1) for i in range(n)]


def _lengths(case):
    """(new tokens, tokens before them) of each sequence, before the shuffle."""
    n, one = case["batch"], case["singles"]
    return [1] * one + _spread(case["q_lo"], case["q_hi"], n - one), _spread(case["ctx_lo"], case["ctx_hi"], n)


def work(case):
    d, hk = case["dim"], case["kv_heads"]
    row = d + 4 if case["cache"] == "e4m3" else 2 * d        # one cached row of one head
    if case["op"] == "attend":
        q, ctx = _lengths(case)
        total_q, total_ctx = sum(q), sum(ctx)
        # every new token sees the context before it (mean over the shuffled pairing) and itself
        seen = total_q * total_ctx / len(ctx) + sum(n * (n + 1) / 2 for n in q)
        return {"bytes": 2 * total_q * case["heads"] * d * 2 + (total_q + total_ctx) * hk * 2 * row,
                "flops": 4 * case["heads"] * d * seen}
    t = case["tokens"]
    if case["op"] == "write_read":
        return {"bytes": 2 * t * 2 * hk * (2 * d + row), "flops": t * 2 * hk * d * 4}
    heads = case["heads"]
    if case["op"] == "rope":
        return {"bytes": 2 * t * (heads + hk) * d * 2, "flops": t * (heads + hk) * d * 8}
    back = 2 * hk * (row + 2 * d) if case["cache"] == "e4m3" else 0
    return {"bytes": t * ((2 * heads + 2 * hk) * d * 2 + 2 * hk * row + back), "flops": t * (heads + hk) * d * 8}


# ---------------------------------------------------------------- inputs

def _randn(g, *shape, dtype, scale=1.0):
    return (torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32) * scale).to(dtype)


def _empty_cache(case, pages):
    shape = (pages, case["kv_heads"], case["page"], case["dim"])
    dt = DTYPES[case["cache"]]
    c = {"k": torch.zeros(shape, dtype=dt, device="cuda"), "v": torch.zeros(shape, dtype=dt, device="cuda"),
         "k_scale": None, "v_scale": None}
    if dt == torch.float8_e4m3fn:
        c["k_scale"] = torch.ones(shape[:3], dtype=torch.float32, device="cuda")
        c["v_scale"] = torch.ones(shape[:3], dtype=torch.float32, device="cuda")
    return c


def _handle(c):
    from drama3_offloading_b200 import kvcache
    return kvcache.PagedKV.from_tensors(c["k"], c["v"], c["k_scale"], c["v_scale"])


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rng = random.Random(seed)
    dt, d, hk = DTYPES[case["dtype"]], case["dim"], case["kv_heads"]
    s = {"case": case, "dtype": dt}
    if case["op"] == "attend":
        q_lens, ctx = _lengths(case)
        rng.shuffle(q_lens)
        rng.shuffle(ctx)
        kv = [a + b for a, b in zip(q_lens, ctx)]
        page = case["page"]
        need = [-(-n // page) for n in kv]
        pages = sum(need) + 2
        order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
        table = torch.zeros(len(kv), max(need), dtype=torch.int32, device="cuda")
        at = 0
        for b, n in enumerate(need):
            table[b, :n] = order[at:at + n]
            at += n
        c = _empty_cache(case, pages)
        # values as the cache holds them: normalised keys, plain values
        for name in ("k", "v"):
            x = c[name]
            if x.dtype == torch.float8_e4m3fn:
                x.copy_(torch.randn(x.shape, generator=g, device="cuda").mul_(100.0).clamp_(-E4M3_MAX, E4M3_MAX))
                c[name + "_scale"].uniform_(0.004, 0.016, generator=g)
            else:
                x.copy_(torch.randn(x.shape, generator=g, device="cuda"))
        s.update(cache=c, table=table, max_q=max(q_lens), max_kv=max(kv),
                 kv_lens=torch.tensor(kv, dtype=torch.int32, device="cuda"),
                 cu_q=torch.tensor([sum(q_lens[:i]) for i in range(len(kv) + 1)], dtype=torch.int32, device="cuda"),
                 # scores of a few units, so that some keys stand out as they do in use
                 q=_randn(g, sum(q_lens), case["heads"], d, dtype=dt, scale=2.0))
        if own:
            s["handle"] = _handle(c)
        return s
    t = case["tokens"]
    if case["cache"]:
        pages = -(-t // case["page"]) + 1
        c = _empty_cache(case, pages)
        order = torch.randperm(pages, generator=g, device="cuda")
        slots = (order[:, None] * case["page"] + torch.arange(case["page"], device="cuda")).reshape(-1)[:t]
        s.update(cache=c, slots=slots.contiguous())
        if own:
            s["handle"] = _handle(c)
    if case["op"] == "write_read":
        s.update(k=_randn(g, t, hk, d, dtype=dt), v=_randn(g, t, hk, d, dtype=dt))
        return s
    heads = case["heads"]
    # one projection's output, seen as queries, keys and values (strided rows)
    wide = _randn(g, t, heads + 2 * hk, d, dtype=dt)
    start = rng.randrange(max(1, case["far"] - t))
    half = case["rotary"] // 2
    s.update(q=wide[:, :heads], k=wide[:, heads:heads + hk], v=wide[:, heads + hk:],
             q_weight=_randn(g, d, dtype=dt, scale=0.2), k_weight=_randn(g, d, dtype=dt, scale=0.2),
             positions=torch.arange(start, start + t, dtype=torch.int64, device="cuda"),
             inv_freq=10000000.0 ** (-torch.arange(half, dtype=torch.float64, device="cuda") / half))
    return s


# ---------------------------------------------------------------- plain forms

def _norm_rope(x, w, s):
    """The norm of each head with weights 1 + w, then the rotation, in 32 bits."""
    case = s["case"]
    y = x.float()
    y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + EPS) * (1.0 + w.float())
    r = case["rotary"]
    angle = s["positions"].double()[:, None] * s["inv_freq"]
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    if case["interleaved"]:
        a, b = y[..., 0:r:2], y[..., 1:r:2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = y[..., :r // 2], y[..., r // 2:r]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((turned, y[..., r:]), -1)


def _put(c, name, x, slots):
    """Rows x [T, heads, D] (32 bits) into the cache's slots."""
    cache = c[name]
    page, off = slots // cache.shape[2], slots % cache.shape[2]
    if cache.dtype == torch.float8_e4m3fn:
        amax = x.abs().amax(-1)
        # a tensor divides: a number would be turned into its rounded reciprocal
        scale = torch.where(amax > 0, amax / torch.full_like(amax, E4M3_MAX), torch.ones_like(amax))
        c[name + "_scale"][page, :, off] = scale
        cache.view(torch.uint8)[page, :, off] = (x / scale[..., None]).to(torch.float8_e4m3fn).view(torch.uint8)
    else:
        cache[page, :, off] = x.to(cache.dtype)


def _get(c, name, slots, dtype):
    cache = c[name]
    page, off = slots // cache.shape[2], slots % cache.shape[2]
    if cache.dtype == torch.float8_e4m3fn:
        x = cache.view(torch.uint8)[page, :, off].view(torch.float8_e4m3fn).float()
        return (x * c[name + "_scale"][page, :, off][..., None]).to(dtype)
    return cache[page, :, off].to(dtype)


def _pages(c, name, table):
    """All pages of each sequence in order: [B, heads, L, D] in 32 bits."""
    x = c[name][table.long()] if c[name].dtype != torch.float8_e4m3fn else \
        c[name].view(torch.uint8)[table.long()].view(torch.float8_e4m3fn)
    x = x.float()
    if c[name + "_scale"] is not None:
        x = x * c[name + "_scale"][table.long()][..., None]
    return x.transpose(1, 2).flatten(2, 3)


def _attend(s):
    q, cu, kv_lens = s["q"], s["cu_q"].long(), s["kv_lens"].long()
    t, heads, d = q.shape
    k, v = (_pages(s["cache"], n, s["table"]) for n in ("k", "v"))
    b, hk, length, _ = k.shape
    n = cu[1:] - cu[:-1]
    i = torch.arange(s["max_q"], device=q.device)
    at = (cu[:-1, None] + i).clamp_(max=t - 1)                              # [B, Q] rows of q
    qp = q.float()[at].reshape(b, len(i), hk, heads // hk, d).permute(0, 2, 1, 3, 4)
    score = (qp.reshape(b, hk, -1, d) @ k.transpose(2, 3)).mul_(d ** -0.5)
    last = kv_lens[:, None] - n[:, None] + i                                # last visible key of each row
    hidden = torch.arange(length, device=q.device) > last[..., None]
    score = score.reshape(b, hk, len(i), heads // hk, length).masked_fill_(hidden[:, None, :, None], -math.inf)
    score = score.sub_(score.amax(-1, keepdim=True)).exp_()
    total = score.sum(-1, keepdim=True)
    out = (score.reshape(b, hk, -1, length) @ v).reshape(b, hk, len(i), heads // hk, d) / total
    out = out.permute(0, 2, 1, 3, 4).reshape(b, len(i), heads, d)
    row = torch.arange(t, device=q.device)
    seq = torch.searchsorted(cu[1:], row, right=True)
    return out[seq, row - cu[seq]].to(q.dtype)


def run(s):
    case = s["case"]
    if own:
        from drama3_offloading_b200 import attention, kvcache
        if case["op"] == "attend":
            return attention.paged_attention(s["q"], s["handle"], s["table"], s["kv_lens"], s["cu_q"],
                                             max_q=s["max_q"], max_kv=s["max_kv"])
        if case["op"] == "write_read":
            kvcache.write(s["handle"], s["k"], s["v"], s["slots"])
            return kvcache.read(s["handle"], s["slots"], dtype=s["dtype"])
        if case["op"] == "rope":
            return attention.qk_norm_rope(s["q"], s["k"], s["q_weight"], s["k_weight"], s["positions"],
                                          s["inv_freq"], eps=EPS, weight_offset=1.0,
                                          interleaved=case["interleaved"])
        q = attention.qk_norm_rope_write(s["q"], s["k"], s["v"], s["q_weight"], s["k_weight"], s["positions"],
                                         s["inv_freq"], s["handle"], s["slots"], eps=EPS, weight_offset=1.0,
                                         interleaved=case["interleaved"])
        if case["cache"] == "e4m3":
            return (q, *kvcache.read(s["handle"], s["slots"], dtype=s["dtype"]))
        return q, s["cache"]["k"], s["cache"]["v"]
    if case["op"] == "attend":
        return _attend(s)
    dt, c = s["dtype"], s.get("cache")
    if case["op"] == "write_read":
        _put(c, "k", s["k"].float(), s["slots"])
        _put(c, "v", s["v"].float(), s["slots"])
        return _get(c, "k", s["slots"], dt), _get(c, "v", s["slots"], dt)
    q, k = _norm_rope(s["q"], s["q_weight"], s), _norm_rope(s["k"], s["k_weight"], s)
    if case["op"] == "rope":
        return q.to(dt), k.to(dt)
    _put(c, "k", k, s["slots"])
    _put(c, "v", s["v"].float(), s["slots"])
    if case["cache"] == "e4m3":
        return q.to(dt), _get(c, "k", s["slots"], dt), _get(c, "v", s["slots"], dt)
    return q.to(dt), c["k"], c["v"]


# ---------------------------------------------------------------- 64 bits

def _e4m3_64(x):
    """Nearest e4m3 value (ties to even) of 64-bit values within +-448."""
    _, e = torch.frexp(x)
    step = torch.ldexp(torch.ones_like(x), (e - 1).clamp(min=-6) - 3)
    return torch.round(x / step) * step


def _held_64(x, kind):
    """What a cache of that kind holds of the rows x, as 64-bit values.  The
    scale is a 32-bit number, and so is the quotient that becomes a code: with
    16-bit rows the quotient often is the middle of two codes."""
    if kind != "e4m3":
        return x
    amax = x.abs().amax(-1, keepdim=True)
    scale = torch.where(amax > 0, amax / E4M3_MAX, torch.ones_like(amax)).float().double()
    return _e4m3_64((x / scale).float().double().clamp(-E4M3_MAX, E4M3_MAX)) * scale


def _turn_64(x, w, s):
    case = s["case"]
    y = x.double()
    y = y / torch.sqrt((y ** 2).sum(-1, keepdim=True) / y.shape[-1] + EPS) * (w.double() + 1.0)
    half = case["rotary"] // 2
    z = torch.polar(torch.ones((), dtype=torch.float64, device=y.device),
                    s["positions"].double()[:, None, None] * s["inv_freq"])
    i = torch.arange(half, device=y.device)
    first, second = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + half)
    z = torch.complex(y[..., first], y[..., second]) * z
    y[..., first], y[..., second] = z.real, z.imag
    return y


def _attend_64(s):
    q, c = s["q"].double(), s["cache"]
    t, heads, d = q.shape
    out = torch.zeros(t, heads, d, dtype=torch.float64, device=q.device)
    cu, kv = s["cu_q"].tolist(), s["kv_lens"].tolist()
    group = heads // c["k"].shape[1]
    for b, length in enumerate(kv):
        pages = s["table"][b, :-(-length // c["k"].shape[2])].tolist()
        n = cu[b + 1] - cu[b]
        see = torch.arange(length, device=q.device)[None] <= torch.arange(length - n, length, device=q.device)[:, None]
        for h in range(c["k"].shape[1]):
            rows = []
            for name in ("k", "v"):
                x = torch.stack([c[name].view(torch.uint8)[p, h] for p in pages]).view(c[name].dtype).double()
                if c[name + "_scale"] is not None:
                    x = x * torch.stack([c[name + "_scale"][p, h] for p in pages]).double()[..., None]
                rows.append(x.flatten(0, 1)[:length])
            for j in range(h * group, (h + 1) * group):
                p = torch.softmax(torch.where(see, q[cu[b]:cu[b + 1], j] @ rows[0].T / math.sqrt(d), -math.inf), -1)
                out[cu[b]:cu[b + 1], j] = p @ rows[1]
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "attend":
        return _attend_64(s)
    kind = case["cache"]
    if case["op"] == "write_read":
        return _held_64(s["k"].double(), kind), _held_64(s["v"].double(), kind)
    q, k = _turn_64(s["q"], s["q_weight"], s), _turn_64(s["k"], s["k_weight"], s)
    if case["op"] == "rope":
        return q, k
    k, v = _held_64(k, kind), _held_64(s["v"].double(), kind)
    if kind == "e4m3":
        return q, k, v
    whole = []
    for x in (k, v):
        full = torch.zeros(s["cache"]["k"].shape, dtype=torch.float64, device="cuda")
        for h in range(case["kv_heads"]):
            full[s["slots"] // case["page"], h, s["slots"] % case["page"]] = x[:, h]
        whole.append(full)
    return q, whole[0], whole[1]
