"""The operators of a serving step over a key-value cache in pages, as cases
that can be timed: block tables and slot maps from request lengths, rotary
positions with the rows' way into the cache (16-bit rows, or the fused 8- and
4-bit rows of the quantizers), and the attention of one new token per request
over its pages.

``listed()`` holds the cases, ``draw(rng)`` gives further ones over the same
ranges.  ``prepare`` makes caches, tables and activations from a seed; ``run``
is one pass, in elementary torch operations in 32 bits, or (``own``) through the
public entry points of ``fbgemm_b200.paged``; ``exact`` is the same from the
definitions in 64 bits.

Cached rows are N(0,1) values, quantized where the cache is; queries are wide
enough for the softmax to favour some rows.  Pages are scattered over the cache
and the lengths of a batch are spread evenly, or evenly over their logarithm,
between two bounds, in an order of the seed's.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

TORCH = {"float16": torch.float16, "bfloat16": torch.bfloat16}


# ---- the cases ---------------------------------------------------------------

def listed():
    return [
        # One decode step of a full batch: every request gets one more token, some of them a new page.
        dict(name="slots_decode_b256", op="slots", batch=256, lo=16, hi=8_192, new_lo=1, new_hi=1, page=16, spare=0),
        # Prompts of many requests enter the cache at once, the maps padded to a captured graph's capacity.
        dict(name="slots_prefill_b64", op="slots", batch=64, lo=1, hi=512, new_lo=64, new_hi=2_048, page=32, spare=4_097),
        # One decode step: a token per request rotated and stored, 16-bit rows.
        dict(name="append_bf16_decode_t64", op="append", tokens=64, heads=32, kv_heads=8, dim=128, rot=128, axes="",
             interleaved=False, type="bfloat16", bits=16, page=16, order="heads", max_pos=32_768),
        # Prompts with images in them (time, height, width positions) into an 8-bit cache.
        dict(name="append_int8_prefill_3_axes", op="append", tokens=8_192, heads=32, kv_heads=8, dim=128, rot=128,
             axes="16,24,24", interleaved=False, type="bfloat16", bits=8, page=64, order="heads", max_pos=32_768),
        # Odd count of tokens, half of each head rotated in adjacent pairs, 4-bit rows in order of tokens.
        dict(name="append_int4_t1001_d96", op="append", tokens=1_001, heads=12, kv_heads=4, dim=96, rot=48, axes="",
             interleaved=True, type="float16", bits=4, page=16, order="tokens", max_pos=8_192),
        # The smallest: one request, a short answer so far.
        dict(name="decode_bf16_b1_129", op="decode", batch=1, lo=129, hi=129, spread="even", heads=32, kv_heads=8, dim=128,
             type="bfloat16", bits=16, page=16, order="heads", window=0, empty=0),
        # One request over a long document: the length has to be split over the chip.
        dict(name="decode_bf16_b1_128k", op="decode", batch=1, lo=131_072, hi=131_072, spread="even", heads=32, kv_heads=8,
             dim=128, type="bfloat16", bits=16, page=16, order="heads", window=0, empty=0),
        # A serving batch with requests of all lengths.
        dict(name="decode_bf16_b64_ragged", op="decode", batch=64, lo=128, hi=8_192, spread="log", heads=32, kv_heads=8,
             dim=128, type="bfloat16", bits=16, page=16, order="heads", window=0, empty=0),
        # 8-bit rows, long requests, eight query heads for each cached one.
        dict(name="decode_int8_b32_16k", op="decode", batch=32, lo=2_048, hi=16_384, spread="even", heads=64, kv_heads=8,
             dim=128, type="bfloat16", bits=8, page=64, order="heads", window=0, empty=0),
        # 4-bit rows, many requests, rows in order of tokens.
        dict(name="decode_int4_b128", op="decode", batch=128, lo=64, hi=4_096, spread="log", heads=32, kv_heads=8, dim=128,
             type="float16", bits=4, page=32, order="tokens", window=0, empty=0),
        # Odd batch, heads and width, a sliding window that starts inside a page, requests without a token and with one.
        dict(name="decode_fp16_b7_d80_window", op="decode", batch=7, lo=1, hi=5_003, spread="even", heads=15, kv_heads=3,
             dim=80, type="float16", bits=16, page=32, order="tokens", window=1_000, empty=1),
        # All query heads on one wide cached head.
        dict(name="decode_fp16_b48_one_kv_head_d256", op="decode", batch=48, lo=512, hi=6_000, spread="even", heads=16,
             kv_heads=1, dim=256, type="float16", bits=16, page=64, order="heads", window=0, empty=0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of an operator that listed() holds."""
    op = rng.choice(["slots", "append", "append", "decode", "decode", "decode"])
    order = rng.choice(["heads", "tokens"])
    kind = rng.choice(["float16", "bfloat16"])
    bits = rng.choice([16, 16, 8, 4])
    page = rng.choice([8, 16, 32, 64, 128])
    if op == "slots":
        prompts = rng.random() < 0.5
        lo = _log(rng, 1, 512)
        return dict(op=op, batch=_log(rng, 1, 64 if prompts else 1_024), lo=lo, hi=lo + _log(rng, 1, 8_000),
                    new_lo=rng.randint(0, 64) if prompts else 1, new_hi=_log(rng, 65, 2_048) if prompts else rng.randint(1, 4),
                    page=page, spare=rng.choice([0, rng.randint(1, 5_000)]))
    dim = rng.choice([64, 80, 96, 112, 128, 128, 192, 256] if bits != 4 else [64, 96, 128, 128, 160, 256])
    kv_heads = rng.choice([1, 2, 3, 4, 8, 8, 10])
    heads = kv_heads * rng.choice([1, 2, 4, 4, 5, 8, 16] if kv_heads <= 4 else [1, 2, 4, 4, 5, 8])
    if op == "append":
        rot = rng.choice([dim, dim, dim // 32 * 16])
        axes = rng.choice(["", "", "%d,%d,%d" % (rot // 2 - 2 * (rot // 6), rot // 6, rot // 6)])
        room = 8_192 * 48 * 128 // ((heads + 2 * kv_heads) * dim)
        return dict(op=op, tokens=_log(rng, 1, min(room, 8_192)), heads=heads, kv_heads=kv_heads, dim=dim, rot=rot, axes=axes,
                    interleaved=rng.random() < 0.5, type=kind, bits=bits, page=page, order=order,
                    max_pos=_log(rng, 1_024, 65_536))
    batch = _log(rng, 1, 160)
    room = 64 * 8_192 * 8 * 128 // (batch * kv_heads * dim)     # rows of the longest request, as in the largest listed case
    hi = _log(rng, 16, max(17, min(131_072, room)))
    return dict(op=op, batch=batch, lo=_log(rng, 1, hi), hi=hi, spread=rng.choice(["even", "log"]), heads=heads,
                kv_heads=kv_heads, dim=dim, type=kind, bits=bits, page=page, order=order,
                window=rng.choice([0, 0, 0, rng.randint(1, 2 * hi)]), empty=rng.choice([0, 0, batch // 4]))


# ---- inputs ------------------------------------------------------------------

def _spread(n, lo, hi, how="even"):
    """n whole numbers from lo to hi, evenly or evenly over their logarithm."""
    at = (np.arange(n) + 0.5) / n
    v = lo + (hi - lo) * at if how == "even" else lo * (hi / lo) ** at
    return np.clip(np.rint(v), lo, hi).astype(np.int64)


def _row_bytes(bits, dim):
    return 2 * dim if bits == 16 else dim + 8 if bits == 8 else dim // 2 + 4


def _device():
    return torch.device("cuda", torch.cuda.current_device())


def _generator(seed):
    return torch.Generator(_device()).manual_seed(int(seed) & 0x7FFFFFFFFFFF)


def _shuffled(v, g):
    """The numbers of an array in an order of the generator's, int32 on the device."""
    t = torch.from_numpy(np.asarray(v, dtype=np.int32)).to(_device())
    return t[torch.randperm(t.numel(), generator=g, device=t.device)].contiguous()


def _cache(case, pages, g):
    """K and V rows [pages, page, kv_heads, row] of N(0,1) values; quantized rows lie 16 bytes apart or a multiple of it."""
    bits, dim, row = case["bits"], case["dim"], _row_bytes(case["bits"], case["dim"])
    pitch = (row + 15) // 16 * 16
    shape = (pages, case["kv_heads"], case["page"]) if case["order"] == "heads" else (pages, case["page"], case["kv_heads"])
    out = []
    for _ in range(2):
        if bits == 16:
            c = torch.randn(shape + (dim,), generator=g, device=_device(), dtype=TORCH[case["type"]])
        else:
            c = torch.zeros(shape + (pitch,), device=_device(), dtype=torch.uint8)
            flat = c.view(-1, pitch)
            for a in range(0, flat.shape[0], 1 << 19):
                some = flat[a:a + (1 << 19)]
                some[:, :row] = _quantized(torch.randn((some.shape[0], dim), generator=g, device=_device()), bits)
            c = c[..., :row]
        out.append(c.permute(0, 2, 1, 3) if case["order"] == "heads" else c)
    return out


def _slots_inputs(case, seed):
    g = _generator(seed)
    B, page = case["batch"], case["page"]
    lengths = _shuffled(_spread(B, case["lo"], case["hi"], "log"), g)
    new = _shuffled(_spread(B, case["new_lo"], case["new_hi"]), g)
    total = int(_spread(B, case["new_lo"], case["new_hi"]).sum())
    have = (lengths + page - 1) // page
    need = int(((lengths + new + page - 1) // page - have).sum())
    width = (case["hi"] + case["new_hi"] + page - 1) // page
    used = int(have.sum())
    ids = torch.randperm(used + need + 64, generator=g, device=_device()).to(torch.int32)
    tables = torch.full((B, width), -1, dtype=torch.int32, device=_device())
    mask = torch.arange(width, device=_device())[None] < have[:, None]
    tables[mask] = ids[:used]
    free = ids[used:].contiguous()
    return dict(lengths=lengths, new=new, tables=tables, free=free,
                num_free=torch.tensor([free.numel()], dtype=torch.int32, device=_device()),
                page=page, capacity=total + case["spare"])


def _append_inputs(case, seed):
    g = _generator(seed)
    T, H, K, D, R = case["tokens"], case["heads"], case["kv_heads"], case["dim"], case["rot"]
    pages = (2 * T + case["page"] - 1) // case["page"] + 1
    k_cache, v_cache = _cache(case, pages, g)
    qkv = torch.randn((T, (H + 2 * K) * D), generator=g, device=_device()).to(TORCH[case["type"]])
    q, k, v = (x.view(T, -1, D) for x in qkv.split([H * D, K * D, K * D], 1))      # as a projection leaves them
    sections = [int(x) for x in case["axes"].split(",")] if case["axes"] else None
    shape = (len(sections), T) if sections else (T,)
    positions = torch.randint(0, case["max_pos"], shape, generator=g, device=_device(), dtype=torch.int32)
    slots = torch.randperm(pages * case["page"], generator=g, device=_device())[:T].contiguous()
    angles = torch.arange(case["max_pos"], device=_device(), dtype=torch.float64)[:, None] * 10_000.0 ** (
        -torch.arange(0, R, 2, device=_device(), dtype=torch.float64) / R)
    cos_sin = torch.cat([angles.cos(), angles.sin()], 1).float()
    axis = torch.repeat_interleave(torch.arange(len(sections) if sections else 1, device=_device()),
                                   torch.tensor(sections or [R // 2], device=_device()))
    return dict(q=q, k=k, v=v, slots=slots, positions=positions, cos_sin=cos_sin, sections=sections, axis=axis,
                k_cache=k_cache, v_cache=v_cache)


def _lengths(case):
    v = _spread(case["batch"], case["lo"], case["hi"], case["spread"])
    v[:case["empty"]] = 0
    return v


def _decode_inputs(case, seed):
    g = _generator(seed)
    page = case["page"]
    lengths = _shuffled(_lengths(case), g)
    counts = (lengths + page - 1) // page
    total = int(((_lengths(case) + page - 1) // page).sum())
    pages = total + 5
    k_cache, v_cache = _cache(case, pages, g)
    width = (case["hi"] + page - 1) // page
    tables = torch.zeros((case["batch"], width), dtype=torch.int32, device=_device())
    mask = torch.arange(width, device=_device())[None] < counts[:, None]
    tables[mask] = torch.randperm(pages, generator=g, device=_device())[:total].to(torch.int32)
    q = torch.randn((case["batch"], case["heads"], case["dim"]), generator=g, device=_device()) * 2.0
    return dict(q=q.to(TORCH[case["type"]]), tables=tables, lengths=lengths, k_cache=k_cache, v_cache=v_cache,
                scale=case["dim"] ** -0.5)


_INPUTS = {"slots": _slots_inputs, "append": _append_inputs, "decode": _decode_inputs}


def prepare(case, seed):
    return {"case": dict(case), **_INPUTS[case["op"]](case, seed)}


# ---- the plain forms ---------------------------------------------------------

def _slots_plain(s):
    page, capacity, tables = s["page"], s["capacity"], s["tables"]
    lengths, new = s["lengths"], s["new"]
    have = (lengths + page - 1) // page
    want = (lengths + new + page - 1) // page
    need = want - have
    before = torch.cumsum(need, 0) - need
    j = torch.arange(tables.shape[1], device=tables.device)[None]
    take = s["num_free"] - 1 - (before[:, None] + j - have[:, None])
    fresh = s["free"][take.clamp(0, s["free"].numel() - 1)]
    tables.copy_(torch.where((j >= have[:, None]) & (j < want[:, None]), fresh, tables))
    ends = torch.cumsum(new, 0)
    t = torch.arange(capacity, device=tables.device)
    request = torch.searchsorted(ends, t, right=True)
    there = t < ends[-1]
    r = request.clamp(max=lengths.numel() - 1)
    position = lengths[r] + t - (ends - new)[r]
    slot = tables[r, (position // page).clamp(max=tables.shape[1] - 1)].long() * page + position % page
    return {"slots": torch.where(there, slot, -1), "positions": torch.where(there, position, 0).int(),
            "requests": torch.where(there, request, -1).int(),
            "offsets": torch.cat([torch.zeros_like(ends[:1]), ends]).int(), "lengths": lengths + new,
            "num_free": s["num_free"] - need.sum(dtype=torch.int32), "tables": tables}


def _quantized(x, bits):
    """Fused rows of fp32 values: codes and fp32 scale, bias (8 bits), or codes and fp16 scale, bias (4 bits)."""
    low, high = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    if bits == 8:
        span = high - low
        most = torch.full_like(span, 255.0)
        codes = torch.round((x - low) * (most / (span + 1e-8))).to(torch.uint8)
        scale_bias = torch.cat([span / most, low], -1)
    else:
        low = low.half().float()
        span = high - low
        scale = torch.where(span == 0, 1.0, span / torch.full_like(span, 15.0)).half().float()
        scale = torch.where((scale == 0) | torch.isinf(1.0 / scale), 1.0, scale)
        codes = torch.round((x - low) * (torch.ones_like(scale) / scale)).clamp(0, 15).to(torch.uint8)
        codes = codes[..., ::2] | (codes[..., 1::2] << 4)
        scale_bias = torch.cat([scale, low], -1).half()
    return torch.cat([codes, scale_bias.view(torch.uint8)], -1)


def _rotated(x, cos, sin, rot, interleaved):
    x = x.float()
    turn, rest = x[..., :rot], x[..., rot:]
    a, b = (turn[..., ::2], turn[..., 1::2]) if interleaved else (turn[..., :rot // 2], turn[..., rot // 2:])
    a, b = a * cos - b * sin, b * cos + a * sin
    turn = torch.stack([a, b], -1).flatten(-2) if interleaved else torch.cat([a, b], -1)
    return torch.cat([turn, rest], -1)


def _append_plain(s):
    case = s["case"]
    rot, page = case["rot"], case["page"]
    of_axis = s["cos_sin"][s["positions"].view(-1, case["tokens"]).long()]           # [axes, tokens, rot]
    pair = torch.arange(rot // 2, device=of_axis.device)
    cos, sin = of_axis[s["axis"], :, pair].T[:, None], of_axis[s["axis"], :, pair + rot // 2].T[:, None]
    q = _rotated(s["q"], cos, sin, rot, case["interleaved"])
    k = _rotated(s["k"], cos, sin, rot, case["interleaved"])
    p, at = s["slots"] // page, s["slots"] % page
    for cache, x in ((s["k_cache"], k), (s["v_cache"], s["v"].float())):
        cache[p, at] = x.to(cache.dtype) if case["bits"] == 16 else _quantized(x, case["bits"])
    # (Quantized rows are compared as they lie in the cache, code, scale and bias bytes: the row format is fixed to the
    # bit, and equal bytes are equal values.)
    return {"q": q.to(s["q"].dtype), "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _values(rows, bits, dim, dtype=torch.float32):
    """What cached rows stand for."""
    if bits == 16:
        return rows.to(dtype)
    at = dim * bits // 8
    scale, bias = rows[..., at:].contiguous().view(torch.float32 if bits == 8 else torch.float16).to(dtype).split(1, -1)
    codes = rows[..., :at]
    if bits == 4:
        codes = torch.stack([codes & 15, codes >> 4], -1).flatten(-2)
    return codes.to(dtype) * scale + bias


def _decode_plain(s):
    case, q, lengths = s["case"], s["q"], s["lengths"]
    B, H, D = q.shape
    K, bits = case["kv_heads"], case["bits"]
    k, v = (_values(c[s["tables"].long()], bits, D).flatten(1, 2) for c in (s["k_cache"], s["v_cache"]))
    qs = q.float().view(B, K, H // K, D)
    scores = torch.matmul(qs, k.permute(0, 2, 3, 1)) * s["scale"]                     # [B, K, H/K, tokens]
    t = torch.arange(k.shape[1], device=q.device)[None]
    first = (lengths - case["window"]).clamp(min=0) if case["window"] else torch.zeros_like(lengths)
    seen = ((t < lengths[:, None]) & (t >= first[:, None]))[:, None, None]
    scores = torch.where(seen, scores, -math.inf)
    most = scores.amax(-1, keepdim=True)
    weights = torch.where(seen, torch.exp(scores - most), 0.0)
    total = weights.sum(-1, keepdim=True)
    out = torch.matmul(weights / total, v.permute(0, 2, 1, 3))
    empty = (lengths == 0)[:, None, None]
    lse = torch.where(empty, -math.inf, (most + total.log()).squeeze(-1))
    out = torch.where(empty[..., None], 0.0, out)
    return {"out": out.view(B, H, D).to(q.dtype), "lse": lse.view(B, H)}


_PLAIN = {"slots": _slots_plain, "append": _append_plain, "decode": _decode_plain}


# ---- the framework's calls ---------------------------------------------------

def _handle(s):
    """The cache as a serving program holds it: made once for its tensors."""
    if "handle" not in s:
        from fbgemm_b200 import paged

        bits = s["case"]["bits"]
        s["handle"] = paged.PagedKVCache(s["k_cache"], s["v_cache"], bit_rate=None if bits == 16 else bits)
    return s["handle"]


def _slots_own(s):
    from fbgemm_b200 import paged

    r = paged.paged_slots(s["lengths"], s["new"], s["tables"], s["free"], s["num_free"], s["page"], s["capacity"])
    return {"slots": r.slots, "positions": r.positions, "requests": r.requests, "offsets": r.offsets,
            "lengths": r.lengths, "num_free": r.num_free, "tables": s["tables"]}


def _append_own(s):
    from fbgemm_b200 import paged

    q = paged.rotary_append(_handle(s), s["q"], s["k"], s["v"], s["slots"], s["positions"], s["cos_sin"],
                            sections=s["sections"], interleaved=s["case"]["interleaved"])
    return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _decode_own(s):
    from fbgemm_b200 import paged

    out, lse = paged.paged_attention(_handle(s), s["q"], s["tables"], s["lengths"], scale=s["scale"],
                                     window=s["case"]["window"], return_lse=True)
    return {"out": out, "lse": lse}


_OWN = {"slots": _slots_own, "append": _append_own, "decode": _decode_own}


def run(state):
    return (_OWN if own else _PLAIN)[state["case"]["op"]](state)


# ---- what a pass cannot do without -------------------------------------------

def work(case):
    if case["op"] == "slots":
        B, page = case["batch"], case["page"]
        lengths = _spread(B, case["lo"], case["hi"], "log")
        new = _spread(B, case["new_lo"], case["new_hi"])
        rows = int(new.sum()) + case["spare"]
        pages = int(((lengths + new + page - 1) // page - (lengths + page - 1) // page).sum())   # about: the orders differ
        return {"bytes": 16 * B + 8 * pages + 16 * rows + 12, "flops": 0}
    if case["op"] == "append":
        T, H, K, D, R = case["tokens"], case["heads"], case["kv_heads"], case["dim"], case["rot"]
        axes = len(case["axes"].split(",")) if case["axes"] else 1
        moved = 2 * T * (H + 2 * K) * D + 2 * T * H * D + 2 * T * K * _row_bytes(case["bits"], D)
        table = min(T, case["max_pos"]) * R * 4                                    # each position's angles, once
        return {"bytes": moved + table + T * (8 + 4 * axes), "flops": 3 * T * (H + K) * R}
    B, H, D = case["batch"], case["heads"], case["dim"]
    lengths = _lengths(case)
    rows = int((np.minimum(lengths, case["window"]) if case["window"] else lengths).sum())
    pages = int(((lengths + case["page"] - 1) // case["page"]).sum())
    return {"bytes": 2 * rows * case["kv_heads"] * _row_bytes(case["bits"], D) + 4 * (pages + B) + B * H * (4 * D + 4),
            "flops": 4 * rows * H * D}


# ---- the definitions in 64 bits ----------------------------------------------

def _exact_append(case, s):
    T, D, R = case["tokens"], case["dim"], case["rot"]
    half = R // 2
    first = torch.arange(half, device=_device()) * (2 if case["interleaved"] else 1)
    second = first + (1 if case["interleaved"] else half)
    position = s["positions"].reshape(-1, T)[s["axis"]].long().T                    # [T, R/2]
    pair = torch.arange(half, device=_device())
    c = s["cos_sin"][position, pair].double()[:, None]
    n = s["cos_sin"][position, pair + half].double()[:, None]

    def turned(x):
        x = x.double()
        y = x.clone()
        y[..., first] = x[..., first] * c - x[..., second] * n
        y[..., second] = x[..., second] * c + x[..., first] * n
        return y

    if case["bits"] != 16:
        return {"q": turned(s["q"]), "k_cache": None, "v_cache": None}
    got = {"q": turned(s["q"])}
    for name, rows in (("k", turned(s["k"])), ("v", s["v"].double())):
        cache = s[name + "_cache"].double()
        cache[s["slots"] // case["page"], s["slots"] % case["page"]] = rows
        got[name + "_cache"] = cache
    return got


def _exact_decode(case, s):
    B, H, D = s["q"].shape
    K, page = case["kv_heads"], case["page"]
    out = torch.zeros((B, H, D), dtype=torch.float64, device=_device())
    lse = torch.full((B, H), -math.inf, dtype=torch.float64, device=_device())
    for b, n in enumerate(s["lengths"].tolist()):
        first = max(0, n - case["window"]) if case["window"] else 0
        if n == 0:
            continue
        t = torch.arange(first, n, device=_device())
        where = s["tables"][b, t // page].long()
        k, v = (_values(s[x][where, t % page], case["bits"], D, torch.float64) for x in ("k_cache", "v_cache"))
        q = s["q"][b].double().view(K, H // K, D)
        score = torch.einsum("kgd,tkd->kgt", q, k) * s["scale"]
        lse[b] = torch.logsumexp(score, -1).view(H)
        out[b] = torch.einsum("kgt,tkd->kgd", torch.softmax(score, -1), v).reshape(H, D)
    return {"out": out, "lse": lse}


def exact(case, seed):
    if case["op"] == "slots":
        return None
    s = _INPUTS[case["op"]](case, seed)
    return (_exact_append if case["op"] == "append" else _exact_decode)(case, s)
