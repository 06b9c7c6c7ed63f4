"""The paged key-value cache on the GPU, against plain implementations in 64
bits (and, for what is stored, bit for bit against the oracle's quantizers)."""
import math
from concurrent.futures import ThreadPoolExecutor

import numpy as np
import pytest
import torch

import fbgemm_b200 as F
from fbgemm_b200 import _capi, paged

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
HALF_STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}     # the largest relative error of one rounding


# ---- slots -------------------------------------------------------------------

def slots_plain(lengths, new, tables, free, num_free, page, capacity):
    """The definition, request after request and row after row."""
    B, W = tables.shape
    tables = tables.copy()
    slots, positions, requests = (np.full(capacity, v, dtype=t) for v, t in ((-1, np.int64), (0, np.int32), (-1, np.int32)))
    offsets = np.zeros(B + 1, np.int32)
    top, row, bad = int(num_free), 0, None
    if not 0 <= top <= len(free):
        bad = 0
    for b in range(B):
        L, n = max(int(lengths[b]), 0), max(int(new[b]), 0)
        have, want = -(-L // page), -(-(L + n) // page)
        if bad is None and (want - have > top or want > W or row + n > capacity):
            bad = b
        if bad is not None:
            break
        for j in range(have, want):
            top -= 1
            tables[b, j] = free[top]
        for t in range(L, L + n):
            p = int(tables[b, t // page])
            slots[row], positions[row], requests[row] = (p * page + t % page if p >= 0 else -1), t, b
            row += 1
        offsets[b + 1] = row
    if bad is not None:
        n = max(int(lengths[bad]), 0) + max(int(new[bad]), 0)
        return dict(slots=np.full(capacity, -1), positions=np.zeros(capacity), requests=np.full(capacity, -1),
                    offsets=np.zeros(B + 1), lengths=lengths, num_free=[num_free], tables=None), [
                        _capi.STATUS_NO_PAGES, bad, min(n, 2 ** 31 - 1), int(num_free)]
    return dict(slots=slots, positions=positions, requests=requests, offsets=offsets,
                lengths=np.maximum(lengths, 0) + np.maximum(new, 0), num_free=[top], tables=tables), None


def check_slots(lengths, new, tables, free, num_free, page, capacity, pad=0):
    lengths, new, free = (np.asarray(x, dtype=np.int32) for x in (lengths, new, free))
    tables = np.asarray(tables, dtype=np.int32)
    want, record = slots_plain(lengths, new, tables, free, num_free, page, capacity)
    wide = torch.full((tables.shape[0], tables.shape[1] + pad), -7, dtype=torch.int32, device=DEV)
    t = wide[:, :tables.shape[1]]
    t.copy_(torch.from_numpy(tables))
    dev = [torch.from_numpy(x).to(DEV) for x in (lengths, new, free)]
    got = paged.paged_slots(dev[0], dev[1], t, dev[2], torch.tensor([num_free], dtype=torch.int32, device=DEV), page, capacity)
    ok, info = F.status_read(0)
    assert ok == (record is None) and (ok or info == record), (info, record)
    for name in ("slots", "positions", "requests", "offsets", "lengths", "num_free"):
        np.testing.assert_array_equal(getattr(got, name).cpu().numpy(), want[name], err_msg=name)
    np.testing.assert_array_equal(t.cpu().numpy(), tables if want["tables"] is None else want["tables"])
    assert pad == 0 or (wide[:, tables.shape[1]:] == -7).all()
    for x, before in zip(dev, (lengths, new, free)):
        np.testing.assert_array_equal(x.cpu().numpy(), before)


def slots_case(rng, B, page, most, fresh, width=None):
    lengths, new = rng.integers(0, most + 1, B), rng.integers(0, fresh + 1, B)
    need = -(-(lengths + new) // page)
    width = width or max(1, int(need.max()))
    ids = rng.permutation(int(need.sum()) + 50)
    tables = rng.integers(-5, 5, (B, width))
    at = 0
    for b in range(B):
        k = -(-int(lengths[b]) // page)
        tables[b, :k] = ids[at:at + k]
        at += k
    return lengths, new, tables, ids[at:]


@pytest.mark.parametrize("B,page,most,fresh,spare,pad", [
    (1, 16, 0, 1, 0, 0), (1, 1, 5, 3, 2, 0), (3, 16, 100, 1, 5, 3), (7, 8, 40, 33, 0, 0), (64, 32, 700, 90, 100, 1),
    (511, 16, 300, 1, 1, 0), (513, 4, 60, 2, 0, 0), (1500, 128, 2000, 3, 0, 5), (5000, 16, 50, 1, 7, 0), (2, 65536, 70000, 9000, 3, 0),
])
def test_slots(B, page, most, fresh, spare, pad):
    rng = np.random.default_rng(B)
    lengths, new, tables, free = slots_case(rng, B, page, most, fresh)
    check_slots(lengths, new, tables, free, len(free), page, int(new.sum()) + spare, pad)


def test_slots_largest_batch_and_requests_that_get_nothing():
    rng = np.random.default_rng(1)
    lengths, new, tables, free = slots_case(rng, _capi.PAGED_MAX_BATCH, 16, 40, 1)
    check_slots(lengths, new, tables, free, len(free), 16, int(new.sum()) + 1)
    check_slots([3, 0, 9], [0, 0, 0], [[1, -1, -1], [-1, -1, -1], [4, 6, 2]], [5], 1, 4, 0)
    check_slots([3, 0, 9], [0, 2, 0], [[1, -1, -1], [-1, -1, -1], [4, 6, 2]], [5], 1, 4, 2)
    check_slots([-3, -1], [2, -5], [[7], [7]], [5, 8], 2, 4, 3)                 # negative counts are 0
    check_slots([2], [1], [[-1]], [5], 1, 4, 1)                                 # an entry that was never set: no slot


def test_slots_only_part_of_the_stack_is_free():
    check_slots([4, 4], [1, 5], [[0, -1, -1], [1, -1, -1]], [9, 8, 7, 6, 5], 3, 4, 6)
    check_slots([4, 4], [1, 5], [[0, -1, -1], [1, -1, -1]], [9, 8, 7, 6, 5], 5, 4, 6)


@pytest.mark.parametrize("lengths,new,width,num_free,capacity", [
    ([4, 4, 4], [1, 5, 1], 3, 2, 7),            # pages run out at the second request
    ([4, 4, 4], [1, 1, 9], 3, 5, 11),           # the table is too narrow for the last
    ([4, 4, 4], [1, 1, 1], 3, 5, 2),            # the maps are too short
    ([4, 4, 4], [1, 1, 1], 3, -1, 3), ([4, 4, 4], [1, 1, 1], 3, 6, 3),   # not the height of this stack
    ([4, 2147483647, 4], [1, 2147483647, 1], 3, 5, 7), ([4, 4, 4], [2147483647, 2147483647, 2147483647], 3, 5, 7),
])
def test_slots_all_or_nothing(lengths, new, width, num_free, capacity):
    tables = np.arange(3 * width).reshape(3, width)
    check_slots(lengths, new, tables, [20, 21, 22, 23, 24], num_free, 4, capacity)


# ---- rotary append -----------------------------------------------------------

def make_cache(pages, page, heads, dim, bits, dtype, order="heads", pitch=None, seed=0):
    """A cache of random bytes (NaN among them), and row alignment as asked."""
    n = paged.row_bytes(dim, None if bits == 16 else bits)
    pitch = pitch or ((n + 15) // 16 * 16)
    shape = {"heads": (pages, heads, page), "tokens": (pages, page, heads), "pages last": (heads, page, pages)}[order]
    to = {"heads": (0, 2, 1, 3), "tokens": (0, 1, 2, 3), "pages last": (2, 1, 0, 3)}[order]
    g = torch.Generator(DEV).manual_seed(seed)
    rows = [torch.randint(0, 256, shape + (pitch,), generator=g, device=DEV, dtype=torch.uint8) for _ in range(2)]
    if bits == 16:
        rows = [x.view(dtype)[..., :dim].permute(to) for x in rows]
    else:
        rows = [x[..., :n].permute(to) for x in rows]
    return paged.PagedKVCache(*rows, bit_rate=None if bits == 16 else bits)


def angles(max_pos, rot):
    a = np.arange(max_pos)[:, None] * 10000.0 ** (-np.arange(0, rot, 2) / rot)
    return torch.from_numpy(np.concatenate([np.cos(a), np.sin(a)], 1).astype(np.float32)).to(DEV)


def turned(x, cos, sin, rot, interleaved):
    """x [tokens, heads, dim] with cos, sin [tokens, rot / 2], in the arrays' own precision."""
    y = x.copy()
    a = np.arange(rot // 2) * (2 if interleaved else 1)
    b = a + (1 if interleaved else rot // 2)
    c, s = cos[:, None], sin[:, None]
    y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., b] * c + x[..., a] * s
    return y


def to_type(x, dtype):
    return torch.from_numpy(np.ascontiguousarray(x)).to(dtype)


APPENDS = [
    # tokens, heads, kv_heads, dim, rot, sections, interleaved, bits, type, page, order, pitch
    (1, 4, 2, 64, 64, None, False, 16, "bf16", 16, "heads", None),
    (5, 3, 1, 16, 16, None, False, 16, "f16", 1, "tokens", None),
    (37, 10, 5, 80, 80, None, True, 16, "bf16", 4, "tokens", 176),
    (70, 8, 8, 256, 64, (10, 11, 11), False, 16, "f16", 32, "pages last", None),
    (33, 6, 3, 112, 48, (0, 20, 4), True, 16, "bf16", 8, "heads", None),
    (64, 8, 2, 128, 128, (16, 24, 24), False, 8, "bf16", 16, "heads", None),
    (9, 4, 4, 16, 16, None, True, 8, "f16", 2, "tokens", 24),
    (130, 5, 1, 208, 96, None, False, 8, "f16", 64, "tokens", 220),
    (65, 8, 4, 96, 96, (5, 6, 7, 30), False, 4, "f16", 16, "heads", None),
    (31, 2, 2, 32, 32, None, True, 4, "bf16", 8, "tokens", 20),
    (1100, 32, 3, 256, 128, None, False, 4, "bf16", 16, "pages last", 132),
    (1025, 7, 7, 64, 0, None, False, 8, "bf16", 16, "heads", None),        # nothing is turned
    (40, 0, 2, 128, 128, None, False, 8, "f16", 16, "heads", None),        # no queries
]


@pytest.mark.parametrize("tokens,heads,kv,dim,rot,sections,interleaved,bits,kind,page,order,pitch", APPENDS)
def test_append(oracle, tokens, heads, kv, dim, rot, sections, interleaved, bits, kind, page, order, pitch):
    dtype, rng = TYPES[kind], np.random.default_rng(tokens + dim)
    pages, max_pos = 2 * tokens // page + 3, 501
    cache = make_cache(pages, page, kv, dim, bits, dtype, order, pitch)
    before = [cache.k.clone(), cache.v.clone()]
    qkv = torch.from_numpy(rng.standard_normal((tokens, (heads + 2 * kv) * dim + 8)).astype(np.float32)).to(dtype).to(DEV)
    q, k, v = (x.view(tokens, n, dim) for x, n in zip(qkv[:, :-8].split([heads * dim, kv * dim, kv * dim], 1), (heads, kv, kv)))
    slots = rng.permutation(pages * page)[:tokens]
    slots[rng.random(tokens) < 0.2] = -1
    axes = len(sections) if sections else 1
    pos = rng.integers(0, max_pos, (axes, tokens)).astype(np.int32)
    table = angles(max_pos, rot) if rot else None
    dpos = torch.from_numpy(pos).to(DEV)
    got = paged.rotary_append(cache, q if heads else None, k, v, torch.from_numpy(slots).to(DEV),
                              None if not rot else dpos if sections else dpos[0], table, sections=sections, interleaved=interleaved)
    assert F.status_read(0)[0]
    xs = [x.float().cpu().numpy() for x in (q, k, v)]
    if rot:
        axis = np.repeat(np.arange(axes), sections or [rot // 2])
        t32 = table.cpu().numpy()
        pair = np.arange(rot // 2)
        cos, sin = t32[pos[axis].T, pair], t32[pos[axis].T, pair + rot // 2]
        exact = turned(xs[0].astype(np.float64), cos.astype(np.float64), sin.astype(np.float64), rot, interleaved)
        xs[0], xs[1] = turned(xs[0], cos, sin, rot, interleaved), turned(xs[1], cos, sin, rot, interleaved)
    if heads:
        assert torch.equal(got.cpu(), to_type(xs[0], dtype))      # the same roundings in the same order: the same bits
        if rot:
            # three roundings of products and sums of two values each, then one to the type
            wide = np.abs(q.double().cpu().numpy()).max() * 2 * 3 * 2.0 ** -24
            assert (np.abs(got.double().cpu().numpy() - exact) <= HALF_STEP[dtype] * np.abs(exact) + wide + 2.0 ** -25).all()
    for rows, x, was in ((cache.k, xs[1], before[0]), (cache.v, xs[2], before[1])):
        want = was.clone()
        flat = x.reshape(tokens * kv, dim)
        if bits == 16:
            new = to_type(x, dtype)
        else:
            new = torch.from_numpy(oracle.quantize_8bit(flat) if bits == 8 else oracle.quantize_nbit(4, flat)).view(tokens, kv, -1)
        for t, s in enumerate(slots):
            if s >= 0:
                want[s // page, s % page] = new[t].to(DEV)
        assert torch.equal(rows.contiguous().view(torch.uint8), want.contiguous().view(torch.uint8))   # other rows as they were


@pytest.mark.parametrize("bits", [16, 8, 4])
def test_append_special_rows(oracle, bits):
    """Constant rows, zeros, infinities and NaN, the type's largest and smallest values: the quantizers' bytes."""
    rows = torch.zeros(12, 64, dtype=torch.bfloat16)
    rows[1], rows[2], rows[3] = 3.5, -3.5, 1e-38
    rows[4, 5], rows[5, 6], rows[6, 7], rows[7] = math.inf, -math.inf, math.nan, math.nan
    rows[8] = torch.finfo(torch.bfloat16).max
    rows[9, ::2], rows[9, 1::2] = 60000.0, -60000.0
    rows[10] = torch.arange(64) * 2.0 ** -133
    rows[11] = torch.arange(64)
    cache = make_cache(1, 16, 1, 64, bits, torch.bfloat16)
    x = rows.view(12, 1, 64).to(DEV)
    paged.rotary_append(cache, None, x, x, torch.arange(12, device=DEV))
    assert F.status_read(0)[0]
    if bits != 16:   # what this library's own quantizers give
        f = rows.float().to(DEV)
        want = (F.FloatToFused8BitRowwiseQuantizedSBFloat(f) if bits == 8 else F.FloatToFusedNBitRowwiseQuantizedSBHalf(4, f)).cpu()
    for got in (cache.k, cache.v):
        got = got[0, :12, 0].contiguous().cpu()
        if bits == 16:      # a NaN is a NaN, of whatever bits
            assert torch.equal(got.isnan(), rows.isnan())
            got, want = got.nan_to_num(0.0).view(torch.uint8), rows.nan_to_num(0.0).view(torch.uint8)
        assert torch.equal(got.view(torch.uint8), want.view(12, -1))


def test_append_reports_what_is_outside():
    cache = make_cache(4, 4, 2, 64, 8, torch.float16)
    k = torch.randn(3, 2, 64, device=DEV).half()
    before = cache.k.clone(), cache.v.clone()
    table = angles(10, 64)

    def call(slots, positions):
        q = paged.rotary_append(cache, k, k, k, torch.tensor(slots, device=DEV),
                                torch.tensor(positions, dtype=torch.int32, device=DEV), table)
        return q, F.status_read(0)

    for value in (10, -1, 2 ** 31 - 1):
        q, (ok, info) = call([-1, 3, -1], [0, value, 0])
        assert not ok and info == [_capi.STATUS_BAD_INDEX, 1, 0, value]
        assert torch.equal(q[1], k[1])                                   # unturned
    for value in (16, -2, 2 ** 62):
        _, (ok, info) = call([-1, -1, value], [0, 0, 0])
        assert not ok and info[:2] == [_capi.STATUS_BAD_PAGE, 2]
    assert torch.equal(cache.k, before[0]) and torch.equal(cache.v, before[1])
    assert F.status_read(0)[0]                                          # reading cleared it


def test_rows_that_append_stores_are_rows_that_the_lookups_read():
    """A page's rows as a table of the 8-bit lookup: the dequantized rows, bit for bit those of the quantizer's table."""
    cache = paged.PagedKVCache.allocate(3, 16, 1, 64, bit_rate=8, device=DEV, row_alignment=1)
    x = torch.randn(48, 1, 64, device=DEV).to(torch.bfloat16)
    paged.rotary_append(cache, None, x, x, torch.arange(48, device=DEV))
    table = cache.k.reshape(48, 72)
    k = F.GenerateEmbeddingSpMDMWithStrides(64, False, False, no_bag=True, index_dtype=np.int64, offset_dtype=np.int64)
    out = [torch.empty(48 * 64, device=DEV) for _ in range(2)]
    order = torch.randperm(48, device=DEV)
    for o, t in zip(out, (table, F.FloatToFused8BitRowwiseQuantizedSBFloat(x[:, 0].float()))):
        assert k(48, 48, 48, t, order, None, None, o)
    assert torch.equal(out[0], out[1])


# ---- attention ---------------------------------------------------------------

def values(rows, bits, dim):
    """Cached rows [.., row bytes or values] in 64 bits; (scale, codes about the middle of their range, bias about it)."""
    if bits == 16:
        return rows.double(), None
    at = dim * bits // 8
    scale, bias = rows[..., at:].contiguous().view(torch.float32 if bits == 8 else torch.float16).double().split(1, -1)
    codes = rows[..., :at]
    if bits == 4:
        codes = torch.stack([codes & 15, codes >> 4], -1).flatten(-2)
    middle = 128 if bits == 8 else 8
    c = codes.double()
    return c * scale + bias, (scale, c - middle, bias + middle * scale)


def check_attention(cache, q, tables, lengths, scale=None, window=0, requests=None):
    """Against the formula in 64 bits, within what the roundings add up to."""
    B, H, D = q.shape
    bits = cache.bit_rate or 16
    K, page, G = cache.kv_heads, cache.page_size, H // cache.kv_heads
    out, lse = paged.paged_attention(cache, q, tables, lengths, scale=scale, window=window, return_lse=True)
    ok, info = F.status_read(0)
    assert ok, info
    again = paged.paged_attention(cache, q, tables, lengths, scale=scale, window=window)
    assert torch.equal(out.view(torch.int16), again.view(torch.int16))      # a fixed order of sums
    scale = D ** -0.5 if scale is None else scale
    # A weight is rounded to fp16, beside bf16 rows to bf16.
    weight = HALF_STEP[torch.bfloat16 if cache.dtype == torch.bfloat16 else torch.float16]
    for b, n in enumerate(lengths.tolist()):
        if requests is not None and b not in requests:
            continue
        got, got_lse = out[b].double().view(K, G, D), lse[b].double().view(K, G)
        if n == 0:
            assert (got == 0).all() and (got_lse == -math.inf).all()
            continue
        t = torch.arange(max(0, n - window) if window else 0, n, device=DEV)
        where = tables[b, t // page].long()
        kd, kq = values(cache.k[where, t % page], bits, D)     # [rows, K, D]
        vd, vq = values(cache.v[where, t % page], bits, D)
        x = q[b].double().view(K, G, D)
        s = scale * torch.einsum("kgd,tkd->kgt", x, kd)
        top = s.amax(-1, keepdim=True)
        e = (s - top).exp()
        p = e / e.sum(-1, keepdim=True)
        o, full_lse = torch.einsum("kgt,tkd->kgd", p, vd), (top + e.sum(-1, keepdim=True).log()).squeeze(-1)
        # Scores: D products summed in fp32 (the tensor cores may drop bits below 2^-22 of a step's largest term, D / 16
        # steps), five more operations; codes and centred biases beside quantized rows.
        size = torch.einsum("kgd,tkd->kgt", x.abs(), kd.abs()) if kq is None else (
            torch.einsum("kgd,tkd->kgt", x.abs(), kq[0].abs() * kq[1].abs())
            + kq[2].abs()[..., 0].T[:, None] * x.abs().sum(-1, keepdim=True))
        off = abs(scale) * size.amax(-1) * (D / 16 + 8) * 2.0 ** -22 + (s.abs().amax(-1) + 16) * 2.0 ** -22
        # Sums over rows: a step of 16 drops as much, and joining splits and warps a few more; ex2 is off by 2^-22.
        steps = (len(t) / 16 + 64) * 2.0 ** -22
        mass = torch.einsum("kgt,tkd->kgd", p, vd.abs())
        heavy = mass if vq is None else torch.einsum("kgt,tkd->kgd", p, vq[0].abs() * vq[1].abs())
        both = mass if vq is None else heavy + torch.einsum("kgt,tkd->kgd", p, vq[2].abs().expand(-1, -1, D))
        # fp16 numbers below 2^-14 are 2^-24 apart, so a small weight is off by 2^-25; weights are 2^10 times their size
        # relative to a row's that is not above the largest (and beside quantized rows to the largest scale): 2^-35 each.
        small = len(t) * 2.0 ** -35 * (vd.abs().max() if vq is None else vq[0].abs().max() * 128)
        # Beside quantized rows the sums are of whole codes, sum w c and middle * sum w, and only their difference is of centred
        # ones: where that is 0 (codes 8 and 8, w s = 0.29: 2.3 - 2.3, off by 1.2e-7) their own roundings stay.  Each is at most
        # held = sum p s 2^bits.  A step of 16 rows rounds its sum, by 2^-22 held, and drops what lies 2^-22 below its largest
        # term, a subnormal code being aligned as 64 (4-bit) or 1024 (8-bit) would be, 4 * 2^bits: over all steps 4 * 2^-22
        # held; the products with the middle and the unit, the difference and its sum with the biases: 4 * 2^-24 held each side.
        held = 0 if vq is None else torch.einsum("kgt,tkd->kgd", p, vq[0].abs()) * 2.0 ** bits * (len(t) / 16 + 6) * 2.0 ** -22
        most = HALF_STEP[q.dtype] * o.abs() + weight * heavy + (2 * off[..., None] + steps) * both + held + small + 2.0 ** -25
        bad = (got - o).abs() - most
        assert (bad <= 0).all(), (b, n, (got - o).abs().max(), bad.max())
        assert ((got_lse - full_lse).abs() <= 2 * off + steps + full_lse.abs() * 2.0 ** -22).all(), (b, n)
    return out, lse


def fill(cache, seed=0):
    """N(0,1) rows everywhere, through the cache's own way in."""
    n = cache.num_pages * cache.page_size
    g = torch.Generator(DEV).manual_seed(seed)
    dtype = cache.dtype or torch.float16
    for a in range(0, n, 4096):
        m = min(4096, n - a)
        k, v = (torch.randn(m, cache.kv_heads, cache.head_dim, generator=g, device=DEV).to(dtype) for _ in range(2))
        paged.rotary_append(cache, None, k, v, torch.arange(a, a + m, device=DEV))
    assert F.status_read(0)[0]


def spoil(cache, slots):
    """Rows that nobody may look at: NaN, or NaN scales."""
    p, t = torch.div(slots, cache.page_size, rounding_mode="floor"), slots % cache.page_size
    for rows in (cache.k, cache.v):
        if cache.bit_rate is None:
            rows[p, t] = math.nan
        else:
            rows[p, t] = 0xFF


def place(lengths, page, rng, pages_free=2):
    """Scattered pages for each request; entries behind them are no pages at all."""
    need = [-(-n // page) for n in lengths]
    ids = rng.permutation(sum(need) + pages_free)
    tables = np.full((len(lengths), max(1, max(need)) + 1), 0x7FFFFFF0, dtype=np.int32)
    at = 0
    for b, n in enumerate(need):
        tables[b, :n] = ids[at:at + n]
        at += n
    return tables, sum(need) + pages_free


ATTENTIONS = [
    # lengths, heads, kv_heads, dim, bits, type, page, order, pitch, window
    ([1], 1, 1, 16, 16, "f16", 16, "heads", None, 0),
    ([0], 2, 1, 64, 16, "bf16", 8, "heads", None, 0),
    ([0, 1, 2, 15, 16, 17], 8, 2, 64, 16, "bf16", 16, "tokens", None, 0),
    ([63, 64, 65, 127, 128, 129, 300], 32, 4, 128, 16, "bf16", 16, "heads", None, 0),
    ([700, 0, 33], 5, 1, 128, 16, "f16", 1, "tokens", 272, 0),
    ([5000, 3, 1024], 9, 1, 128, 16, "f16", 64, "heads", None, 0),
    ([777, 40], 32, 2, 128, 16, "bf16", 32, "tokens", None, 0),
    ([333, 90], 48, 2, 64, 16, "f16", 16, "heads", None, 0),
    ([400, 7, 1000], 15, 3, 80, 16, "f16", 32, "tokens", None, 0),
    ([100, 1300], 12, 1, 256, 16, "bf16", 16, "heads", None, 0),
    ([250, 31], 6, 3, 208, 16, "f16", 128, "pages last", None, 0),
    ([20000], 4, 1, 128, 16, "bf16", 16, "heads", None, 0),
    ([1, 2, 3, 500, 129, 1000], 8, 2, 64, 16, "bf16", 16, "heads", None, 1),
    ([1, 70, 300, 500, 129, 1000], 8, 2, 128, 16, "f16", 16, "heads", None, 77),
    ([300, 999, 0], 8, 1, 256, 16, "f16", 8, "tokens", None, 500),
    ([0, 1, 31, 32, 33, 64, 65, 128, 257], 8, 1, 128, 8, "bf16", 16, "heads", None, 0),
    ([999, 1500], 64, 4, 128, 8, "f16", 64, "tokens", None, 0),
    ([999, 15], 3, 1, 112, 8, "f16", 16, "tokens", 120, 0),
    ([257, 600], 4, 2, 64, 8, "bf16", 4, "heads", 72, 0),
    ([260, 77], 34, 2, 48, 8, "bf16", 16, "heads", None, 0),
    ([500, 3000], 5, 1, 256, 8, "f16", 32, "heads", None, 0),
    ([129, 1], 8, 1, 256, 8, "bf16", 32, "pages last", 268, 100),
    ([0, 1, 63, 64, 65, 256, 257, 1000], 8, 2, 128, 4, "bf16", 16, "heads", None, 0),
    ([900, 450], 32, 2, 128, 4, "f16", 16, "tokens", 68, 0),
    ([321, 5], 3, 3, 32, 4, "f16", 2, "heads", 20, 0),
    ([321, 1234], 20, 2, 64, 4, "bf16", 16, "tokens", None, 200),
    ([1025, 60], 7, 1, 96, 4, "bf16", 16, "heads", None, 0),
    ([513, 60], 11, 1, 160, 4, "f16", 256, "heads", None, 0),
    ([513, 60], 4, 2, 256, 4, "f16", 16, "pages last", 132, 0),
    ([30000, 5], 2, 1, 64, 4, "f16", 16, "heads", None, 0),
    # windows that begin in either half of a page, pages of 32 rows and more for two steps of 16
    ([1000, 47, 0, 33, 2077], 8, 2, 64, 16, "bf16", 32, "heads", None, 45),
    ([1000, 47, 0, 33, 2077], 8, 2, 128, 8, "f16", 64, "heads", None, 531),
    ([1000, 47, 0, 33, 2077], 8, 2, 128, 4, "bf16", 32, "tokens", None, 16),
    ([15, 16, 17, 31, 32, 33], 4, 1, 64, 8, "bf16", 128, "heads", None, 9),
]


@pytest.mark.parametrize("lengths,heads,kv,dim,bits,kind,page,order,pitch,window", ATTENTIONS)
def test_attention(lengths, heads, kv, dim, bits, kind, page, order, pitch, window):
    rng = np.random.default_rng(sum(lengths) + dim)
    tables, pages = place(lengths, page, rng)
    cache = make_cache(pages, page, kv, dim, bits, TYPES[kind], order, pitch)
    fill(cache)
    used = np.zeros(pages * page, bool)
    for b, n in enumerate(lengths):
        t = np.arange(max(0, n - window) if window else 0, n)
        used[tables[b, t // page].astype(np.int64) * page + t % page] = True
    spoil(cache, torch.from_numpy(np.flatnonzero(~used)).to(DEV))
    wide = torch.randn(len(lengths), heads * dim + 16, device=DEV).to(TYPES[kind]) * 3
    q = wide[:, 8:8 + heads * dim].view(len(lengths), heads, dim)          # rows of a wider activation
    padded = torch.full((tables.shape[0], tables.shape[1] + 3), -1, dtype=torch.int32, device=DEV)
    view = padded[:, :tables.shape[1]]
    view.copy_(torch.from_numpy(tables))
    check_attention(cache, q, view, torch.tensor(lengths, dtype=torch.int32, device=DEV), window=window)


@pytest.mark.parametrize("bits,kind", [(16, "bf16"), (16, "f16"), (8, "bf16"), (4, "f16")])
def test_attention_of_many_requests_of_all_lengths(bits, kind):
    """Requests that share pages, short ones alone and among longer ones (more items than workers)."""
    rng = np.random.default_rng(bits)
    pages, page = 60, 16
    cache = make_cache(pages, page, 4, 64, bits, TYPES[kind])
    fill(cache)
    for B, longest in ((150, 400), (500, 1500)):
        lengths = [int(x) for x in np.exp(rng.uniform(-1, math.log(longest), B))]
        tables = torch.from_numpy(rng.integers(0, pages, (B, longest // page + 1)).astype(np.int32)).to(DEV)
        q = torch.randn(B, 8, 64, device=DEV).to(TYPES[kind])
        check_attention(cache, q, tables, torch.tensor(lengths, dtype=torch.int32, device=DEV), scale=0.3)


@pytest.mark.parametrize("bits,kind,page", [(16, "bf16", 16), (8, "f16", 64), (4, "f16", 8)])
def test_attention_with_workers_of_either_size(bits, kind, page):
    """So long that a second set of workers takes the last quarter; the requests go over the same pages again and again."""
    rng = np.random.default_rng(bits)
    pages = 3000 // page
    cache = make_cache(pages, page, 8, 64, bits, TYPES[kind])
    fill(cache)
    lengths = [300_001, 5, 250_000, 0, 40_000]
    tables = torch.from_numpy(rng.integers(0, pages, (5, 300_001 // page + 1)).astype(np.int32)).to(DEV)
    q = torch.randn(5, 8, 64, device=DEV).to(TYPES[kind])
    check_attention(cache, q, tables, torch.tensor(lengths, dtype=torch.int32, device=DEV))


@pytest.mark.parametrize("bits", [16, 8, 4])
def test_attention_over_one_page_of_one_head(bits):
    """Dimensions of one have no stride."""
    for page in (1, 16, 64):
        cache = make_cache(1, page, 1, 64, bits, torch.float16)
        fill(cache)
        q = torch.randn(3, 2, 64, device=DEV).half()
        tables = torch.zeros(3, 1, dtype=torch.int32, device=DEV)
        check_attention(cache, q, tables, torch.tensor([page, 0, (page + 1) // 2], dtype=torch.int32, device=DEV))


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("bits", [16, 8, 4])
def test_attention_weights_far_apart(bits, kind):
    """One row outweighs tens of thousands that matter together: weights of 2^-20 keep their bits."""
    dtype, n = TYPES[kind], 20000
    cache = paged.PagedKVCache.allocate(n // 16, 16, 1, 64, dtype=dtype, bit_rate=None if bits == 16 else bits, device=DEV)
    k = torch.zeros(n, 1, 64, device=DEV, dtype=dtype)
    k[:, 0, 1] = 1.0
    k[7, 0, 0] = 14.0      # score 14 against 0: weight e^-14 = 2^-20 for the others
    v = torch.randn(n, 1, 64, device=DEV).to(dtype) * 0.01 + 1.0
    v[7] = 0.5
    paged.rotary_append(cache, None, k, v, torch.arange(n, device=DEV))
    q = torch.zeros(1, 2, 64, device=DEV, dtype=dtype)
    q[0, :, 0] = 1.0
    tables = torch.arange(n // 16, dtype=torch.int32, device=DEV)[None]
    check_attention(cache, q, tables, torch.tensor([n], dtype=torch.int32, device=DEV), scale=1.0)


def test_attention_scales_far_apart():
    """8-bit rows whose scales differ by 2^40, small ones first, last and alone; queries beyond fp16's range."""
    n = 600
    for back in (False, True):
        cache = paged.PagedKVCache.allocate(40, 16, 1, 64, bit_rate=8, device=DEV)
        k = torch.randn(n, 1, 64, device=DEV).bfloat16() * 1e-3
        v = (torch.randn(n, 1, 64, device=DEV) * 2.0 ** torch.linspace(-30, 10, n, device=DEV)[:, None, None]).bfloat16()
        v = v.flip(0) if back else v
        paged.rotary_append(cache, None, k, v, torch.arange(n, device=DEV))
        q = torch.randn(2, 4, 64, device=DEV).bfloat16()
        q[1] *= 1e5
        q[1, 1] *= 2.0 ** -100
        tables = torch.arange(40, dtype=torch.int32, device=DEV)[None].expand(2, 40).contiguous()
        check_attention(cache, q, tables, torch.tensor([n, n], dtype=torch.int32, device=DEV), scale=0.01)
        check_attention(cache, q, tables, torch.tensor([3, 1], dtype=torch.int32, device=DEV), scale=0.01)


@pytest.mark.parametrize("bits", [16, 8])
def test_attention_infinities_and_nan(bits):
    """What a row that is seen holds goes the formula's way, and stays with its head and request."""
    dtype = torch.bfloat16
    cache = paged.PagedKVCache.allocate(16, 16, 2, 64, dtype=dtype, bit_rate=None if bits == 16 else bits, device=DEV)
    fill(cache)
    q = torch.randn(3, 4, 64, device=DEV).to(dtype)
    tables = torch.arange(15, dtype=torch.int32, device=DEV).view(3, 5)
    lengths = torch.tensor([80, 50, 80], dtype=torch.int32, device=DEV)
    clean = paged.paged_attention(cache, q, tables, lengths)
    if bits == 16:
        cache.v[1, 3, 0, 9] = math.nan
        cache.k[12, 0, 1] = math.nan
    else:
        cache.v[1, 3, 0, 64:68] = 0xFF      # the scale: a NaN
        cache.k[12, 0, 1, 64:68] = 0xFF
    got, lse = paged.paged_attention(cache, q, tables, lengths, return_lse=True)
    assert F.status_read(0)[0]
    hit = torch.zeros_like(got, dtype=torch.bool)
    if bits == 16:
        hit[0, :2, 9] = True
    else:
        hit[0, :2] = True
    hit[2, 2:] = True
    assert torch.equal(got.isnan(), hit) and torch.equal(got[~hit], clean[~hit])
    assert lse[2, 2:].isnan().all() and not lse[:2].isnan().any()
    if bits == 16:
        cache.k[12, 0, 1] = 0
        cache.v[1, 3, 0, 9] = 0
        cache.k[5:10] = 0
        cache.k[5:10, :, :, 0] = -math.inf     # every score of request 1 is -inf: 0 / 0
        q[1, :, 0] = 1.0
        got, lse = paged.paged_attention(cache, q, tables, lengths, return_lse=True)
        assert got[1].isnan().all() and (lse[1] == -math.inf).all()
        cache.k[6, 4, :, 0] = 1.0              # one finite score among them takes all the weight
        got, lse = paged.paged_attention(cache, q, tables, lengths, return_lse=True)
        assert torch.equal(got[1].view(2, 2, 64), cache.v[6, 4][:, None].expand(2, 2, 64))
        assert torch.allclose(lse[1], torch.full((4,), 0.125, device=DEV), rtol=2.0 ** -20)
        cache.k[6, 4, :, 0] = math.inf         # inf - inf
        assert paged.paged_attention(cache, q, tables, lengths)[1].isnan().all()


def test_attention_splits_join():
    """Results over two halves of the rows, joined by their logarithms, are the result over all."""
    cache = paged.PagedKVCache.allocate(300, 16, 2, 128, device=DEV)
    fill(cache)
    q = torch.randn(2, 8, 128, device=DEV).bfloat16()
    tables = torch.randperm(300, device=DEV).to(torch.int32)[:280].view(2, 140).contiguous()
    n = torch.tensor([2240, 2240], dtype=torch.int32, device=DEV)
    whole, lse = paged.paged_attention(cache, q, tables, n, return_lse=True)
    parts = [paged.paged_attention(cache, q, t.contiguous(), torch.full_like(n, m), return_lse=True)
             for t, m in ((tables[:, :50], 800), (tables[:, 50:], 1440))]
    both = torch.logaddexp(parts[0][1], parts[1][1])
    joined = sum(o.float() * (z - both).exp()[..., None] for o, z in parts)
    assert torch.allclose(both, lse, rtol=0, atol=1e-4)
    # each of three results is off by a rounding of itself and of its weights, of values below 5
    assert (joined - whole.float()).abs().max() <= 5 * 4 * 2.0 ** -8


def test_attention_reports_bad_pages_and_lengths():
    cache = paged.PagedKVCache.allocate(8, 16, 1, 64, device=DEV)
    fill(cache)
    q = torch.randn(2, 2, 64, device=DEV).bfloat16()
    good = torch.tensor([[0, 1, 2], [3, 4, 5]], dtype=torch.int32, device=DEV)
    lengths = torch.tensor([40, 48], dtype=torch.int32, device=DEV)
    want = paged.paged_attention(cache, q, good, lengths)
    for value in (-1, 8, 2 ** 31 - 1, -2 ** 31, -2, -3):
        tables = good.clone()
        tables[1, 1] = value
        got = paged.paged_attention(cache, q, tables, lengths)
        ok, info = F.status_read(0)
        assert not ok and info[:2] == [_capi.STATUS_BAD_PAGE, 1] and 16 <= info[2] < 32 and info[3] == value
        assert torch.equal(got[0], want[0])
        # its rows are left out: as if request 1 had pages 3 and 5 alone
        other = paged.paged_attention(cache, q[1:], torch.tensor([[3, 5]], dtype=torch.int32, device=DEV), lengths[:1] - 8)
        assert (got[1].float() - other[0].float()).abs().max() <= 5 * 4 * 2.0 ** -8
    for value, like in ((-1, 0), (49, 48), (2 ** 31 - 1, 48), (-2 ** 31, 0)):
        got = paged.paged_attention(cache, q, good, torch.tensor([40, value], dtype=torch.int32, device=DEV))
        ok, info = F.status_read(0)
        assert not ok and info == [_capi.STATUS_SIZE_MISMATCH, 1, 0, value]
        assert torch.equal(got, paged.paged_attention(cache, q, good, torch.tensor([40, like], dtype=torch.int32, device=DEV)))
        assert F.status_read(0)[0]


def test_attention_beyond_4_gb_of_cache():
    """Rows whose offset passes 32 bits, on pages far apart."""
    pages = 300_000     # twice as many x 16 rows x 512 bytes: 4.9 GB each of K and V
    cache = paged.PagedKVCache.allocate(2 * pages, 16, 1, 256, device=DEV)
    tables = torch.tensor([[2 * pages - 1, 0, pages + 12345, 2 * pages - 2, 7]], dtype=torch.int32, device=DEV)
    slots = (tables[0, :, None].long() * 16 + torch.arange(16, device=DEV)).flatten()
    k, v = (torch.randn(80, 1, 256, device=DEV).bfloat16() for _ in range(2))
    paged.rotary_append(cache, None, k, v, slots)
    assert torch.equal(cache.k[2 * pages - 1, :, 0], k[:16, 0]) and torch.equal(cache.v[2 * pages - 2, :, 0], v[48:64, 0])
    check_attention(cache, torch.randn(1, 4, 256, device=DEV).bfloat16(), tables, torch.tensor([77], dtype=torch.int32, device=DEV))


@pytest.mark.parametrize("page,bits", [(16, None), (64, None), (8, None), (64, 8), (32, 4)])
def test_attention_without_a_table_or_a_request(page, bits):
    cache = paged.PagedKVCache.allocate(2, page, 1, 64, bit_rate=bits, device=DEV)
    q = torch.randn(3, 2, 64, device=DEV).bfloat16()
    out, lse = paged.paged_attention(cache, q, torch.zeros(3, 0, dtype=torch.int32, device=DEV),
                                     torch.zeros(3, dtype=torch.int32, device=DEV), return_lse=True)
    assert (out == 0).all() and (lse == -math.inf).all() and F.status_read(0)[0]
    out = paged.paged_attention(cache, q[:0], torch.zeros(0, 4, dtype=torch.int32, device=DEV),
                                torch.zeros(0, dtype=torch.int32, device=DEV))
    assert out.shape == (0, 2, 64)


# ---- together ----------------------------------------------------------------

class Server:
    """A few requests served step by step, with everything held on the device; and the same in 64 bits on the host."""

    def __init__(self, bits, kind, batch=5, heads=8, kv=2, dim=64, page=8, pages=200, capacity=256):
        self.dtype, self.dim, self.heads, self.kv, self.page = TYPES[kind], dim, heads, kv, page
        self.cache = paged.PagedKVCache.allocate(pages, page, kv, dim, dtype=self.dtype, bit_rate=None if bits == 16 else bits,
                                                 device=DEV)
        i = dict(dtype=torch.int32, device=DEV)
        self.lengths, self.new = torch.zeros(batch, **i), torch.zeros(batch, **i)
        self.tables = torch.full((batch, 40), -1, **i)
        self.free, self.num_free = torch.randperm(pages, device=DEV).to(torch.int32), torch.tensor([pages], **i)
        self.qkv = torch.zeros(capacity, (heads + 2 * kv) * dim, dtype=self.dtype, device=DEV)
        self.table = angles(400, dim)
        self.capacity, self.batch = capacity, batch
        self.last = torch.zeros(batch, heads, dim, dtype=self.dtype, device=DEV)

    def step(self):
        s = paged.paged_slots(self.lengths, self.new, self.tables, self.free, self.num_free, self.page, self.capacity)
        H, K = self.heads * self.dim, self.kv * self.dim
        q, k, v = (x.view(self.capacity, -1, self.dim) for x in self.qkv.split([H, K, K], 1))
        turned = paged.rotary_append(self.cache, q, k, v, s.slots, s.positions, self.table)
        newest = (s.offsets[1:] - 1).clamp(min=0).long()
        out = paged.paged_attention(self.cache, turned[newest], self.tables, s.lengths)
        self.lengths.copy_(s.lengths)
        self.num_free.copy_(s.num_free)
        return out, s, turned


@pytest.mark.parametrize("bits,kind", [(16, "bf16"), (8, "f16"), (4, "bf16")])
def test_serving_steps(bits, kind):
    torch.manual_seed(bits)
    rng = np.random.default_rng(bits)
    srv = Server(bits, kind)
    history = [[] for _ in range(srv.batch)]
    for step in range(12):
        new = rng.integers(0, 50, srv.batch) if step == 0 else rng.integers(0, 2, srv.batch)
        srv.new.copy_(torch.from_numpy(new.astype(np.int32)))
        srv.qkv.normal_()
        out, s, turned_q = srv.step()
        assert F.status_read(0)[0]
        # every row is where the table says, once
        live = s.slots[:int(new.sum())]
        assert (live >= 0).all() and live.unique().numel() == live.numel() and (s.slots[int(new.sum()):] == -1).all()
        at = 0
        for b in range(srv.batch):
            history[b] += [int(x) for x in live[at:at + new[b]]]
            at += int(new[b])
        held = [x for h in history for x in h]
        assert len(set(held)) == len(held)
        newest = (s.offsets[1:] - 1).clamp(min=0).long()
        got, _ = check_attention(srv.cache, turned_q[newest], srv.tables, srv.lengths)
        assert torch.equal(got, out)
    assert [len(h) for h in history] == srv.lengths.tolist()


def test_a_captured_step_is_replayed():
    """Two graphs of one server's step on two streams in turn, against the same steps without graphs."""
    a, b = Server(8, "bf16"), Server(8, "bf16")
    b.free.copy_(a.free)
    for srv in (a, b):
        srv.new.fill_(1)
        srv.qkv.copy_(torch.randn(srv.qkv.shape, generator=torch.Generator(DEV).manual_seed(3), device=DEV))
        srv.step()
    graphs, outs = [], []
    for _ in range(2):
        lengths, num_free, tables = a.lengths.clone(), a.num_free.clone(), a.tables.clone()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(a.step()[0])
        graphs.append(g)
        a.lengths.copy_(lengths)
        a.num_free.copy_(num_free)
        a.tables.copy_(tables)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for i in range(8):
        x = torch.randn(a.qkv.shape, generator=torch.Generator(DEV).manual_seed(i), device=DEV)
        for srv in (a, b):
            srv.qkv.copy_(x)
            srv.new.copy_(torch.tensor([1, 0, 1, 3, i % 2], dtype=torch.int32))
        torch.cuda.synchronize()
        with torch.cuda.stream(streams[i % 2]):
            graphs[i % 2].replay()
        torch.cuda.synchronize()
        want = b.step()[0]
        assert torch.equal(outs[i % 2], want)
        assert torch.equal(a.tables, b.tables) and torch.equal(a.lengths, b.lengths) and torch.equal(a.num_free, b.num_free)
    assert F.status_read(0)[0]


def test_calls_that_overlap():
    """Attention over different caches and batches on several streams at once: each its own results."""
    rng = np.random.default_rng(5)
    calls = []
    for i, (bits, kind) in enumerate(((16, "bf16"), (8, "f16"), (4, "bf16"), (16, "f16"))):
        cache = make_cache(200, 16, 2, 128, bits, TYPES[kind])
        fill(cache, i)
        lengths = torch.from_numpy(rng.integers(0, 3000, 3).astype(np.int32)).to(DEV)
        tables = torch.from_numpy(rng.integers(0, 200, (3, 200)).astype(np.int32)).to(DEV)
        q = torch.randn(3, 16, 128, device=DEV).to(TYPES[kind])
        calls.append((cache, q, tables, lengths))
    want = [paged.paged_attention(*c) for c in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in calls]
    got = [[] for _ in calls]
    for _ in range(20):
        for c, s, g in zip(calls, streams, got):
            with torch.cuda.stream(s):
                g.append(paged.paged_attention(*c))
    torch.cuda.synchronize()
    for w, g in zip(want, got):
        assert all(torch.equal(w, x) for x in g)


def test_results_into_given_memory():
    cache = paged.PagedKVCache.allocate(8, 16, 1, 64, device=DEV)
    fill(cache)
    q = torch.randn(2, 2, 64, device=DEV).bfloat16()
    tables = torch.tensor([[0, 1, 2], [3, 4, 5]], dtype=torch.int32, device=DEV)
    lengths = torch.tensor([40, 3], dtype=torch.int32, device=DEV)
    want = paged.paged_attention(cache, q, tables, lengths)
    big = torch.full((6, 2, 64), 7.0, device=DEV).bfloat16()
    assert paged.paged_attention(cache, q, tables, lengths, out=big[2:4]).data_ptr() == big[2:4].data_ptr()
    assert torch.equal(big[2:4], want) and (big[:2] == 7).all() and (big[4:] == 7).all()
    same = q.clone()      # in place: a head's query is read before its result is written
    turned_q = paged.rotary_append(cache, q, q[:, :1], q[:, :1], torch.tensor([-1, -1], device=DEV),
                                   torch.tensor([3, 5], dtype=torch.int32, device=DEV), angles(9, 64))
    paged.rotary_append(cache, same, q[:, :1], q[:, :1], torch.tensor([-1, -1], device=DEV),
                        torch.tensor([3, 5], dtype=torch.int32, device=DEV), angles(9, 64), q_out=same)
    assert torch.equal(same, turned_q)
    with pytest.raises(_capi.Fbgemmb200Error, match="overlaps"):
        paged.paged_attention(cache, same, tables, lengths, out=same)
    big = torch.empty(3, 2, 64, device=DEV).bfloat16()
    with pytest.raises(_capi.Fbgemmb200Error, match="overlaps"):
        paged.rotary_append(cache, big[:2], q[:, :1], q[:, :1], torch.tensor([-1, -1], device=DEV), q_out=big[1:])


@pytest.mark.parametrize("bits,kind,kv", [(16, "bf16", 2), (8, "f16", 2), (4, "bf16", 8)])
def test_attention_of_more_short_items_than_blocks(bits, kind, kv):
    """Warps take several whole items each, or share one with the next; some have no rows."""
    rng = np.random.default_rng(bits)
    lengths = rng.integers(0, 130, 250).tolist()
    lengths[:4] = [0, 0, 130, 1]
    tables, pages = place(lengths, 16, rng)
    cache = make_cache(pages, 16, kv, 128, bits, TYPES[kind])
    fill(cache)
    q = torch.randn(len(lengths), 3 * kv, 128, device=DEV).to(TYPES[kind])
    check_attention(cache, q, torch.from_numpy(tables).to(DEV), torch.tensor(lengths, dtype=torch.int32, device=DEV))


@pytest.mark.parametrize("bits,kind", [(16, "f16"), (4, "bf16")])
def test_attention_of_the_most_heads(bits, kind):
    """16384 query heads over one cached head: 256 tiles of heads."""
    cache = make_cache(40, 16, 1, 32, bits, TYPES[kind])
    fill(cache)
    tables = torch.randperm(40, device=DEV).to(torch.int32).view(2, 20)
    q = torch.randn(2, 16384, 32, device=DEV).to(TYPES[kind])
    check_attention(cache, q, tables, torch.tensor([100, 311], dtype=torch.int32, device=DEV))


def test_slots_from_several_threads():
    """Batches of several sizes at once, each with another need of shared memory."""
    def work(i):
        torch.cuda.set_device(0)
        batch, ok = 16384 - 2500 * i, True
        lengths = torch.full((batch,), 3, dtype=torch.int32, device=DEV)
        for _ in range(50):
            out = paged.paged_slots(lengths, torch.ones_like(lengths), torch.zeros(batch, 1, dtype=torch.int32, device=DEV),
                                    lengths[:0], torch.zeros(1, dtype=torch.int32, device=DEV), 16, batch)
            ok &= bool((out.slots == 3).all())
        return ok

    with ThreadPoolExecutor(4) as pool:
        assert all(pool.map(work, range(4)))
