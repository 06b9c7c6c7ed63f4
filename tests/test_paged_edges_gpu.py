"""The paged key-value cache on the GPU at its edges: memory that ends with the
last row, tables without a good page, numbers at the ends of their ranges, the
forms that only large calls take."""
import math
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

import fbgemm_b200 as F
from fbgemm_b200 import _capi, paged

import test_paged_gpu as known
from test_paged_gpu import DEV, TYPES, check_attention, fill, values

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


# ---- what is read ------------------------------------------------------------

@pytest.mark.parametrize("dim,bits,pitch", [(64, 8, 80), (48, 8, 64), (128, 4, 80), (32, 4, 32), (96, 16, 208), (112, 8, 124), (160, 4, 88)])
@pytest.mark.parametrize("pages,page", [(1, 1), (3, 1), (5, 8), (2, 16)])
def test_memory_ends_with_the_last_row(dim, bits, pitch, pages, page):
    """Rows further apart than they are long, and nothing behind the last one."""
    heads, bit_rate = 2 if page > 1 else 1, None if bits == 16 else bits
    n = paged.row_bytes(dim, bit_rate)
    rows = pages * page * heads
    at = 512                                         # the last row ends where the tensor's memory does
    size = at + (rows - 1) * pitch + n
    shape, strides = (pages, page, heads, n), (page * heads * pitch, heads * pitch, pitch, 1)
    made = []
    for _ in range(2):
        x = torch.full((size,), 0xFF, dtype=torch.uint8, device=DEV).as_strided(shape, strides, at)
        made.append(x if bits != 16 else x.view(torch.float16))
    cache = paged.PagedKVCache(*made, bit_rate=bit_rate)
    fill(cache)
    q = torch.randn(2, 4, dim, device=DEV).half()
    tables = torch.arange(pages - 1, -1, -1, dtype=torch.int32, device=DEV)[None].expand(2, pages).contiguous()
    check_attention(cache, q, tables, torch.tensor([pages * page, 1], dtype=torch.int32, device=DEV))


# ---- a copy that does not come -----------------------------------------------

@pytest.fixture
def no_copy_in_time():
    lib = _capi.lib()

    def limit(nanoseconds):
        return lib.fbgemm_b200_set_copy_limit(nanoseconds)

    before = limit(10 ** 9)
    yield limit
    limit(before)


@pytest.mark.parametrize("bits", [16, 8, 4])
@pytest.mark.parametrize("batch,rows,heads,dim", [(1, 40, 4, 64), (2, 1500, 8, 128), (1, 20_000, 8, 128), (130, 700, 16, 128), (3, 900, 12, 256)])
def test_a_copy_that_does_not_come_in_time(no_copy_in_time, bits, batch, rows, heads, dim):
    """Every wait runs out at once: the call ends, says so, and leaves nothing behind for the next one."""
    cache = paged.PagedKVCache.allocate(150, 16, 2 if heads < 12 else 1, dim, dtype=torch.float16,
                                        bit_rate=None if bits == 16 else bits, device=DEV)
    fill(cache)
    q = torch.randn(batch, heads, dim, device=DEV).half()
    tables = torch.randint(0, 150, (batch, -(-rows // 16)), device=DEV, dtype=torch.int32)
    lengths = torch.full((batch,), rows, dtype=torch.int32, device=DEV)
    want = paged.paged_attention(cache, q, tables, lengths)
    assert F.status_read(0)[0]
    assert no_copy_in_time(0) == 10 ** 9
    paged.paged_attention(cache, q, tables, lengths)
    ok, info = F.status_read(0)
    assert not ok and info[0] == _capi.STATUS_COPY_TIMEOUT and 0 <= info[1] < batch and info[2:] == [0, 0]
    assert no_copy_in_time(10 ** 9) == 0
    assert torch.equal(paged.paged_attention(cache, q, tables, lengths), want) and F.status_read(0)[0]


# ---- nothing left of a request -----------------------------------------------

# items that are whole ones of a warp, of a block, of a cluster; that neighbours share; that the chip shares
LEFT = [(1, 16, 2, 1), (3, 60, 4, 1), (2, 1500, 8, 2), (1, 20_000, 8, 2), (300, 100, 8, 2), (300, 700, 16, 2), (60, 2500, 24, 1)]


@pytest.mark.parametrize("batch,rows,heads,kv", LEFT)
@pytest.mark.parametrize("bits,page", [(16, 16), (16, 8), (8, 64), (8, 4), (4, 32)])
def test_a_request_whose_pages_are_all_bad(batch, rows, heads, kv, bits, page):
    """Its rows are left out, so there are none: zeros and -inf.  The other requests are as they were."""
    pages = 3200 // page
    cache = paged.PagedKVCache.allocate(pages, page, kv, 64, dtype=torch.bfloat16, bit_rate=None if bits == 16 else bits, device=DEV)
    fill(cache)
    q = torch.randn(batch, heads, 64, device=DEV).bfloat16()
    tables = torch.randint(0, pages, (batch, -(-rows // page)), device=DEV, dtype=torch.int32)
    lengths = torch.full((batch,), rows, dtype=torch.int32, device=DEV)
    want, want_lse = paged.paged_attention(cache, q, tables, lengths, return_lse=True)
    assert F.status_read(0)[0]
    hit = torch.zeros(batch, dtype=torch.bool)
    hit[::7] = True
    hit = hit.to(DEV)
    for value in (-1, pages):
        bad = torch.where(hit[:, None], value, tables)
        got, lse = paged.paged_attention(cache, q, bad, lengths, return_lse=True)
        ok, info = F.status_read(0)
        assert not ok and info[0] == _capi.STATUS_BAD_PAGE and info[1] % 7 == 0 and info[3] == value
        assert (got[hit] == 0).all() and (lse[hit] == -math.inf).all()
        assert torch.equal(got[~hit], want[~hit]) and torch.equal(lse[~hit], want_lse[~hit])
    # one row left: its value
    bad[0, -1] = tables[0, -1]
    last = (rows - 1) % page
    lengths[0] = rows - last
    got, lse = paged.paged_attention(cache, q[:1], bad[:1], lengths[:1], return_lse=True)
    F.status_read(0)
    one, one_lse = paged.paged_attention(cache, q[:1], tables[:1, -1:].contiguous(), torch.ones_like(lengths[:1]), return_lse=True)
    assert torch.equal(got, one) and torch.equal(lse, one_lse)


@pytest.mark.parametrize("bits", [16, 8, 4])
def test_a_window_over_bad_pages_alone(bits):
    cache = paged.PagedKVCache.allocate(8, 16, 2, 64, bit_rate=None if bits == 16 else bits, device=DEV)
    fill(cache)
    q = torch.randn(2, 4, 64, device=DEV).bfloat16()
    tables = torch.tensor([[0, 1, 8, -1], [2, 3, 4, 5]], dtype=torch.int32, device=DEV)
    lengths = torch.tensor([60, 60], dtype=torch.int32, device=DEV)
    for window in (1, 12, 13, 28):
        got, lse = paged.paged_attention(cache, q, tables, lengths, window=window, return_lse=True)
        ok, info = F.status_read(0)
        assert not ok and info[:2] == [_capi.STATUS_BAD_PAGE, 0] and 60 - window <= info[2] < 60
        assert (got[0] == 0).all() and (lse[0] == -math.inf).all()
        want = paged.paged_attention(cache, q[1:], tables[1:], lengths[1:], window=window)
        assert F.status_read(0)[0] and (got[1].float() - want[0].float()).abs().max() <= 5 * 2 * 2.0 ** -8   # (another split)


@pytest.mark.parametrize("rows", [10, 60, 1500, 20_000])
def test_scores_that_are_all_minus_infinity(rows):
    """Rows that are there, unlike none: 0 / 0, as in the formula; with one finite score among them that row's value."""
    cache = paged.PagedKVCache.allocate(1250, 16, 1, 64, dtype=torch.bfloat16, device=DEV)
    fill(cache)
    cache.k.zero_()
    cache.k[..., 0] = -math.inf
    q = torch.ones(1, 4, 64, device=DEV).bfloat16()
    tables = torch.arange(1250, dtype=torch.int32, device=DEV)[None]
    tables = tables[:, :-(-rows // 16)].contiguous()
    lengths = torch.tensor([rows], dtype=torch.int32, device=DEV)
    got, lse = paged.paged_attention(cache, q, tables, lengths, return_lse=True)
    assert got.isnan().all() and (lse == -math.inf).all()
    if rows > 100:
        tables[0, :3] = -1                     # some rows left out, the others as before
        got, lse = paged.paged_attention(cache, q, tables, lengths, return_lse=True)
        assert got.isnan().all() and (lse == -math.inf).all() and not F.status_read(0)[0]
    at = rows - 2
    cache.k[at // 16, at % 16, 0, 0] = 0
    got, lse = paged.paged_attention(cache, q, tables, lengths, return_lse=True)
    F.status_read(0)
    assert torch.equal(got[0], cache.v[at // 16, at % 16].expand(4, 64)) and (lse.abs() <= 2.0 ** -20).all()


# ---- numbers at the ends of their ranges -------------------------------------

@pytest.mark.parametrize("scale", [1.0, 0.125, 2.0, 2.0 ** 20])
@pytest.mark.parametrize("rows", [1, 77, 1500, 9000])
def test_queries_of_the_whole_range_of_bf16(rows, scale):
    """8-bit keys so small that the scores of queries up to 2^123 are ordinary; smaller queries beside them."""
    cache = paged.PagedKVCache.allocate(600, 16, 1, 64, bit_rate=8, device=DEV)
    fill(cache)
    codes = torch.randint(0, 256, (600, 16, 1, 64), device=DEV, dtype=torch.uint8)
    cache.k[..., :64] = codes
    cache.k[..., 64:] = torch.tensor([2.0 ** -120, -127.0 * 2.0 ** -120], device=DEV).view(torch.uint8)
    q = torch.randn(2, 10, 64, device=DEV)
    q[:, :3] *= 2.0 ** 114 / scale      # scores of 114 - 120 binary places, 8 columns' worth of 73 on average: about 9
    q[:, 3] *= 2.0 ** 118 / scale
    q[1, 4] *= 2.0 ** -100
    q[1, 5] *= 2.0 ** 100
    tables = torch.randint(0, 600, (2, -(-rows // 16)), device=DEV, dtype=torch.int32)
    out, lse = check_attention(cache, q.bfloat16(), tables, torch.tensor([rows, max(1, rows - 5)], dtype=torch.int32, device=DEV), scale=scale)
    assert out.isfinite().all() and lse.isfinite().all()


@pytest.mark.parametrize("bits", [8, 4])
def test_the_largest_queries_beside_quantized_rows(bits):
    """Scores of 2^120 and more: the largest takes all the weight."""
    cache = paged.PagedKVCache.allocate(4, 16, 1, 64, bit_rate=bits, device=DEV)
    fill(cache)
    q = torch.randn(1, 8, 64, device=DEV) * 2.0 ** 117
    q[0, 4:] *= 2.0 ** 3
    q = q.bfloat16()
    tables = torch.arange(4, dtype=torch.int32, device=DEV)[None]
    out, lse = paged.paged_attention(cache, q, tables, torch.tensor([60], dtype=torch.int32, device=DEV), scale=0.125, return_lse=True)
    assert F.status_read(0)[0]
    (k, _), (v, (step, code, _)) = (values(x.reshape(64, -1)[:60], bits, 64) for x in (cache.k, cache.v))
    score = q[0].double() @ k.T * 0.125
    top, at = score.max(-1)
    # (a score is off by 2^-18 of the sum of its terms' sizes; the second largest is further away)
    second = score.scatter(-1, at[:, None], -math.inf).amax(-1)
    assert ((top - second) > 2.0 ** -18 * (q[0].double().abs() @ k.abs().T).amax(-1) * 0.125 * 4).all()
    # One weight of 1, which enters times the row's scale as fp16: off by 2^-11 of scale * (code - middle), the rest of the value,
    # bias + scale * middle, is added in fp32 (sums of whole codes: 2^-18 of the largest value), and the sum is rounded once.
    weight = 2.0 ** -11 * (step * code)[at].abs()
    assert ((out[0].double() - v[at]).abs() <= 2.0 ** -8 * v[at].abs() + weight + 2.0 ** -18 * v.abs().max()).all()
    assert ((lse[0].double() - top).abs() <= 2.0 ** -18 * (q[0].double().abs() @ k.abs().T).amax(-1) * 0.125).all()


def rows_of(cache, n, k, v):
    """Stores n rows of single keys and values one behind another; the block table that names them."""
    paged.rotary_append(cache, None, k, v, torch.arange(n, device=DEV))
    assert F.status_read(0)[0]
    return torch.arange(-(-n // cache.page_size), dtype=torch.int32, device=DEV)[None]


@pytest.mark.parametrize("page", [16, 8])
@pytest.mark.parametrize("rows", [1, 50, 700, 5000])
@pytest.mark.parametrize("bits,kind", [(16, "f16"), (16, "bf16"), (8, "f16"), (4, "bf16")])
def test_equal_scores_far_from_zero(bits, kind, rows, page):
    """Scores of 2^20 to 2^30, all the same: the mean of the values, for every size of the scores' last place."""
    dtype = TYPES[kind]
    cache = paged.PagedKVCache.allocate(-(-rows // page), page, 1, 64, dtype=dtype, bit_rate=None if bits == 16 else bits, device=DEV)
    v = (torch.rand(rows, 1, 64, device=DEV) + 1).to(dtype)
    tables = rows_of(cache, rows, torch.full_like(v, 32.0), v)
    stored, parts = values(cache.v.reshape(-1, cache.v.shape[-1])[:rows], bits, 64)
    mean = stored.mean(0)
    # Equal weights of powers of two, exact, beside 16-bit rows; beside quantized ones times the row's scale as fp16 (2^-11 of scale *
    # (code - middle)).  Sums of rows / 16 steps and of joins, of whole codes beside quantized rows: 2^-22 each of what is summed.
    most = stored.abs().mean(0) if parts is None else (parts[0] * 2 ** bits + parts[2].abs()).mean(0)
    rounded = 0 if parts is None else 2.0 ** -11 * (parts[0] * parts[1].abs()).mean(0)
    bound = 2.0 ** -8 * mean.abs() + (rows / 16 + 64) * 2.0 ** -22 * most + rounded
    lengths = torch.tensor([rows], dtype=torch.int32, device=DEV)
    for power in range(20, 31):
        for sign in (1.0, -1.0):
            q = torch.full((1, 3, 64), 32.0 * sign, device=DEV).to(dtype)
            scale = 2.0 ** (power - 16)          # 64 columns of 2^10 each
            out, lse = paged.paged_attention(cache, q, tables, lengths, scale=scale, return_lse=True)
            assert ((out[0].double() - mean).abs() <= bound).all(), (power, sign)
            want = sign * 2.0 ** power + math.log(rows)
            assert ((lse.double() - want).abs() <= 2.0 ** -21 * abs(want)).all(), (power, sign)


@pytest.mark.parametrize("bits,kind", [(16, "f16"), (16, "bf16"), (8, "f16"), (8, "bf16")])
def test_scores_that_rise_by_single_steps_far_from_zero(bits, kind):
    """A running maximum whose last places are worth 2 to 32: weights stay numbers, and the result among the values."""
    dtype, rows = TYPES[kind], 1000
    cache = paged.PagedKVCache.allocate(63, 16, 1, 64, dtype=dtype, bit_rate=None if bits == 16 else bits, device=DEV)
    v = (torch.rand(rows, 1, 64, device=DEV) + 1).to(dtype)
    k = torch.zeros_like(v)
    tables = rows_of(cache, rows, k, v)
    lengths = torch.tensor([rows], dtype=torch.int32, device=DEV)
    row = torch.arange(rows, device=DEV)
    for power in range(22, 31):
        for step in (1, 2, 3, 4, 5, 6, 8):
            q = torch.zeros(1, 2, 64, device=DEV)
            if bits == 16:      # column 0: the common size; column 1: the steps
                q[..., 0], q[..., 1] = 2.0 ** 15, 1.0
                k[:, 0, 0], k[:, 0, 1] = 2.0 ** (power - 15), (row % 256 * 4 * step).to(dtype)
                tables = rows_of(cache, rows, k, v)
            else:               # codes of 0 and the row's bias
                bias = (2.0 ** power + row % 256 * 4 * step).float()
                flat = cache.k.permute(0, 2, 1, 3)[:, 0]          # [pages, page, row]
                flat[..., :68] = 0
                flat[..., 68:] = torch.nn.functional.pad(bias, (0, 8)).view(63, 16, 1).view(torch.uint8)
                q[..., 0] = 1.0
            out, lse = paged.paged_attention(cache, q.to(dtype), tables, lengths, scale=1.0, return_lse=True)
            # (a value of [1, 2] stored with an error of 2^-8, two roundings of 2^-8 each)
            assert ((out >= 1 - 3 * 2.0 ** -8) & (out <= 2 + 6 * 2.0 ** -8)).all(), (power, step)
            top = 2.0 ** power + 255 * 4 * step
            assert ((lse - top).abs() <= 2.0 ** -16 * top).all(), (power, step)


@pytest.mark.parametrize("page", [16, 8])
@pytest.mark.parametrize("rows", [1, 50, 1500, 9000])
@pytest.mark.parametrize("bits", [16, 8])
def test_the_largest_values(bits, rows, page):
    """Values near bf16's end: their mean is a number, though their sum is none."""
    cache = paged.PagedKVCache.allocate(-(-rows // page), page, 1, 64, bit_rate=None if bits == 16 else bits, device=DEV)
    lengths = torch.tensor([rows, max(1, rows // 2)], dtype=torch.int32, device=DEV)
    q = torch.randn(2, 4, 64, device=DEV).bfloat16()
    # the largest of all, by columns of one sign (8-bit rows: all of one sign, so that the row's range is a number), equal weights
    v = torch.full((rows, 1, 64), torch.finfo(torch.bfloat16).max, device=DEV).bfloat16()
    if bits == 16:
        v[..., ::2] *= -1
    tables = rows_of(cache, rows, torch.zeros_like(v), v).expand(2, -1).contiguous()
    out = paged.paged_attention(cache, q, tables, lengths)
    assert F.status_read(0)[0] and torch.equal(out, v[:1].expand(2, 4, 64))
    # half of that, all signs, all weights
    v = ((torch.rand(rows, 1, 64, device=DEV) - 0.5) * 2.0 ** 127).bfloat16()
    tables = rows_of(cache, rows, torch.randn(rows, 1, 64, device=DEV).bfloat16(), v).expand(2, -1).contiguous()
    out, lse = check_attention(cache, q, tables, lengths)
    assert out.isfinite().all()


@pytest.mark.parametrize("bits", [16, 8])
def test_small_values(bits):
    """Values of 1e-20 keep their bits."""
    cache = paged.PagedKVCache.allocate(100, 16, 1, 64, bit_rate=None if bits == 16 else bits, device=DEV)
    n = 1600
    fill(cache)
    scale = 2.0 ** -66
    if bits == 16:
        cache.v.mul_(scale)
        big = cache.v.float() / scale
    else:
        at = cache.v[..., 64:]
        at.copy_((at.contiguous().view(torch.float32) * scale).view(torch.uint8))
    q = torch.randn(1, 4, 64, device=DEV).bfloat16()
    tables = torch.arange(100, dtype=torch.int32, device=DEV)[None]
    lengths = torch.tensor([n], dtype=torch.int32, device=DEV)
    out = paged.paged_attention(cache, q, tables, lengths)
    if bits == 16:
        cache.v.copy_(big)
    else:
        at.copy_((at.contiguous().view(torch.float32) / scale).view(torch.uint8))
    # (every step is by the same powers of two)
    assert torch.equal(out.float() / scale, paged.paged_attention(cache, q, tables, lengths).float())


# ---- the form of rotary_append that many tokens take (a warp a token) --------

MANY = [
    # tokens, heads, kv_heads, dim, rot, sections, interleaved, bits, type, page, order, pitch
    (2047, 4, 2, 64, 64, (8, 10, 14), False, 8, "bf16", 16, "heads", None),     # (the last size of the other form)
    (2048, 7, 1, 256, 256, None, True, 16, "f16", 32, "pages last", None),
    (2049, 4, 2, 64, 64, None, False, 16, "bf16", 16, "heads", None),
    (2050, 10, 5, 80, 80, (10, 20, 10), True, 8, "bf16", 8, "tokens", 92),
    (2051, 3, 1, 128, 128, (16, 24, 24), False, 8, "f16", 64, "tokens", None),
    (2053, 6, 2, 64, 0, None, False, 4, "f16", 16, "heads", None),              # nothing is turned
    (2055, 0, 2, 112, 112, None, False, 16, "bf16", 16, "heads", None),         # no queries
    (3001, 1, 1, 32, 16, None, False, 4, "f16", 1, "tokens", 20),
    (2501, 9, 3, 208, 96, (0, 40, 0, 8), True, 8, "f16", 16, "heads", 220),
    (4097, 5, 3, 96, 48, None, True, 4, "bf16", 16, "heads", None),
]


@pytest.mark.parametrize("case", MANY, ids=lambda c: "-".join(str(x) for x in c))
def test_append_of_many_tokens(oracle, case):
    known.test_append(oracle, *case)


def test_append_of_many_tokens_reports_what_is_outside():
    n = 2051
    cache = known.make_cache(140, 16, 2, 64, 8, torch.float16)
    k = torch.randn(n, 2, 64, device=DEV).half()
    before = cache.k.clone(), cache.v.clone()
    table = known.angles(10, 64)
    for token in (0, 1027, n - 1):
        for value in (10, -1, 2 ** 31 - 1):
            slots = torch.full((n,), -1, device=DEV)
            slots[token] = 3
            positions = torch.zeros(n, dtype=torch.int32, device=DEV)
            positions[token] = value
            q = paged.rotary_append(cache, k, k, k, slots, positions, table)
            ok, info = F.status_read(0)
            assert not ok and info == [_capi.STATUS_BAD_INDEX, token, 0, value]
            assert torch.equal(q, k)                       # position 0 and the one outside: unturned
        for value in (140 * 16, -2, 2 ** 62):
            slots = torch.full((n,), -1, device=DEV)
            slots[token] = value
            paged.rotary_append(cache, k, k, k, slots, torch.zeros_like(positions), table)
            ok, info = F.status_read(0)
            assert not ok and info[:2] == [_capi.STATUS_BAD_PAGE, token]
    assert torch.equal(cache.k, before[0]) and torch.equal(cache.v, before[1]) and F.status_read(0)[0]


@pytest.mark.parametrize("bits", [16, 4])
def test_append_of_many_tokens_in_place(bits):
    n = 2051
    made = [known.make_cache(140, 16, 2, 96, bits, torch.bfloat16) for _ in range(2)]
    q, k, v = (torch.randn(n, heads, 96, device=DEV).bfloat16() for heads in (5, 2, 2))
    slots = torch.randperm(140 * 16, device=DEV)[:n]
    positions = torch.randint(0, 300, (n,), device=DEV, dtype=torch.int32)
    want = paged.rotary_append(made[0], q, k, v, slots, positions, known.angles(300, 96))
    assert paged.rotary_append(made[1], q, k, v, slots, positions, known.angles(300, 96), q_out=q) is q
    assert torch.equal(q, want) and torch.equal(made[0].k.view(torch.uint8), made[1].k.view(torch.uint8))
    assert torch.equal(made[0].v.view(torch.uint8), made[1].v.view(torch.uint8)) and F.status_read(0)[0]


# ---- every row once ----------------------------------------------------------

COUNTS = [
    # lengths, heads, kv_heads, dim, bits, page, window
    ([300_001, 5, 250_000, 0, 40_000], 8, 8, 64, 16, 16, 0),
    ([300_001, 5, 250_000, 0, 40_000], 8, 8, 64, 8, 64, 0),
    ([300_001, 5, 250_000, 0, 40_000], 32, 16, 64, 16, 16, 0),      # workers of either size
    ([300_001, 5, 250_000, 0, 40_000], 16, 16, 64, 8, 64, 0),
    ([9000, 30_011] * 20, 8, 4, 128, 8, 8, 0),
    ([20_001, 9000] * 40, 8, 1, 256, 16, 32, 0),
    ([300, 77] * 100, 4, 4, 64, 16, 16, 0),                         # (few units, although the table has room for more)
    ([300_001, 5, 250_000, 0, 40_000], 8, 8, 64, 4, 8, 0),
    ([200_003, 90_000, 70], 34, 2, 128, 16, 32, 0),                 # two warps to a worker
    ([100_001, 150_000], 20, 1, 256, 8, 32, 0),                     # and units of 16 rows
    ([131_072], 32, 8, 128, 16, 16, 0),
    ([260_000, 260_000], 8, 8, 64, 16, 64, 131_071),
    ([4000] * 3, 8, 8, 128, 16, 16, 0),                             # clusters
    ([100, 3000, 0, 777] * 40, 16, 4, 128, 4, 32, 0),               # items shared by neighbours
]


@pytest.mark.parametrize("lengths,heads,kv,dim,bits,page,window", COUNTS)
def test_every_row_enters_once(lengths, heads, kv, dim, bits, page, window):
    """Keys of 0: all weights are 1, and the sum of them is the number of rows.  Values are one of 64 columns' unit, by parts of the
    request: a unit of 16 rows that is lost, or another's twice, is seen at any length."""
    cache = paged.PagedKVCache.allocate(128, page, kv, dim, dtype=torch.float16, bit_rate=None if bits == 16 else bits, device=DEV)
    one = 1.0 if bits == 16 else (2 ** bits - 1) / 2 ** bits         # scales of powers of two: no weight is rounded
    v = torch.zeros(128 * page, kv, dim, device=DEV).half()
    column = torch.arange(128, device=DEV).repeat_interleave(page) % 64
    v[torch.arange(128 * page, device=DEV), :, column] = one
    paged.rotary_append(cache, None, torch.zeros_like(v), v, torch.arange(128 * page, device=DEV))
    width = -(-max(max(lengths), 20_000) // page)
    tables = torch.full((len(lengths), width), -1, dtype=torch.int32)
    want = torch.zeros(len(lengths), 64, dtype=torch.float64)
    rows = torch.tensor([min(n, window) if window else n for n in lengths])
    for b, n in enumerate(lengths):
        pages = -(-n // page)
        part = torch.arange(pages) * 64 // max(pages, 1)
        tables[b, :pages] = (part + 64 * torch.randint(0, 2, (pages,))).int()
        t = torch.arange(n - int(rows[b]), n)
        want[b] = torch.bincount(part[t // page], minlength=64).double()
    q = torch.randn(len(lengths), heads, dim, device=DEV).half()
    out, lse = paged.paged_attention(cache, q, tables.to(DEV), torch.tensor(lengths, dtype=torch.int32, device=DEV), window=window,
                                     return_lse=True)
    assert F.status_read(0)[0]
    some = rows > 0
    # whole numbers below 2^24 are exact sums; a logarithm of up to 16 and its sum with 0 are rounded by 2^-21 each
    assert ((lse.double().cpu()[some] - rows[some].double().log()[:, None]).abs() <= 2.0 ** -20).all()
    got, want = out.double().cpu()[some], want[some] / rows[some, None] * one
    # one rounding to fp16, and sums (of centred codes: of all rows) within 2^-20 of the whole
    assert ((got[..., :64] - want[:, None]).abs() <= 2.0 ** -11 * want[:, None] + 2.0 ** -20).all()
    assert (got[..., 64:].abs() <= 2.0 ** -20).all() and (out.cpu()[~some] == 0).all()


@pytest.mark.parametrize("bits,kind,page", [(16, "bf16", 16), (8, "f16", 64), (8, "bf16", 8)])
def test_attention_of_many_long_items(bits, kind, page):
    """Long lines of many items: a second set of workers takes the last quarter, and ends items that the first began."""
    rng = np.random.default_rng(bits)
    pages = 3000 // page
    cache = known.make_cache(pages, page, 16, 64, bits, TYPES[kind])
    fill(cache)
    lengths = [200_001, 5, 150_000, 0, 40_000]
    tables = torch.from_numpy(rng.integers(0, pages, (5, 200_001 // page + 1)).astype(np.int32)).to(DEV)
    q = torch.randn(5, 32, 64, device=DEV).to(TYPES[kind])
    check_attention(cache, q, tables, torch.tensor(lengths, dtype=torch.int32, device=DEV))


# ---- what may stand before a call in a graph ---------------------------------

def test_captured_behind_copies_and_other_streams():
    """In a graph behind a copy, a fill, a kernel of another stream and another call: the call waits for all of them."""
    cache = paged.PagedKVCache.allocate(400, 16, 2, 64, device=DEV)
    fill(cache)
    tables = torch.randint(0, 400, (3, 200), device=DEV, dtype=torch.int32)
    n = torch.tensor([3100, 40, 900], dtype=torch.int32, device=DEV)
    source = torch.zeros(3, 4, 64, device=DEV).bfloat16()
    q, lengths, other = torch.zeros_like(source), torch.zeros_like(n), torch.cuda.Stream()
    big = torch.zeros(64 << 20, device=DEV)
    width = [tables, tables[:, :64].contiguous()]      # shared by the chip; by clusters
    outs = []

    def step():
        for t in width:
            lengths.copy_(n)                              # a copy before it
            q.copy_(source)
            first = paged.paged_attention(cache, q, t, lengths.clamp(max=t.shape[1] * 16), return_lse=True)
            lengths.zero_()                               # a fill before it
            empty = paged.paged_attention(cache, q, t, lengths, return_lse=True)
            other.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(other):
                big.add_(1)                               # some 80 us, then what is read
                lengths.copy_(n)
                lengths.clamp_(max=t.shape[1] * 16)
            torch.cuda.current_stream().wait_stream(other)
            again = paged.paged_attention(cache, q, t, lengths, return_lse=True)
            q.neg_()
            third = paged.paged_attention(cache, q, t, lengths, return_lse=True)
            fourth = paged.paged_attention(cache, third[0], t, lengths, return_lse=True)   # a call that reads a call's result
            outs.append((first, empty, again, third, fourth))

    source.normal_()
    step()
    torch.cuda.synchronize()
    outs.clear()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step()
    captured = list(outs)
    for _ in range(3):
        source.normal_()
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        got = [[(o.clone(), z.clone()) for o, z in x] for x in captured]
        outs.clear()
        for t in width:                                   # one call at a time
            m = n.clamp(max=t.shape[1] * 16)
            want = []
            for x, lens in ((source, m), (source, torch.zeros_like(n)), (source, m), (-source, m)):
                want.append(paged.paged_attention(cache, x.clone(), t, lens, return_lse=True))
                torch.cuda.synchronize()
            want.append(paged.paged_attention(cache, want[-1][0], t, m, return_lse=True))
            torch.cuda.synchronize()
            for (o, z), (o2, z2) in zip(got.pop(0), want):
                assert torch.equal(o, o2) and torch.equal(z, z2)
    assert F.status_read(0)[0]


FIRST_CALLS = """
import torch
from fbgemm_b200 import paged
cache = paged.PagedKVCache.allocate(40, 16, 2, 64, device="cuda:0")
i = dict(dtype=torch.int32, device="cuda:0")
q = torch.randn(2, 4, 64, device="cuda:0").bfloat16()
tables, lengths, free, num_free = torch.arange(8, **i).view(2, 4), torch.tensor([60, 3], **i), torch.arange(8, 40, **i), torch.tensor([32], **i)
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    s = paged.paged_slots(lengths, torch.ones_like(lengths), tables, free, num_free, 16, 4)
    turned = paged.rotary_append(cache, q, q[:, :2], q[:, :2], s.slots[:2])
    out = paged.paged_attention(cache, turned, tables, s.lengths)
g.replay()
torch.cuda.synchronize()
want = paged.paged_attention(cache, turned, tables, s.lengths)
assert s.slots.tolist() == [3 * 16 + 12, 4 * 16 + 3, -1, -1] and torch.equal(out, want) and want.abs().max() > 0
print("captured")
"""


def test_the_first_calls_of_a_process_are_captured():
    res = subprocess.run([sys.executable, "-c", FIRST_CALLS], capture_output=True, text=True, timeout=100, cwd=ROOT)
    assert res.returncode == 0 and res.stdout == "captured\n", res.stderr


# ---- one rounding ------------------------------------------------------------

ROUNDED = [
    # lengths, heads, kv_heads, dim, bits, type, page, window
    ([1, 2, 5, 40], 8, 2, 64, 16, "bf16", 16, 0), ([1, 2, 5, 40], 8, 2, 64, 16, "f16", 16, 0),
    ([1, 2, 5, 40], 8, 2, 64, 8, "f16", 8, 0), ([1, 2, 5, 40], 8, 2, 64, 4, "f16", 16, 0),
    ([3000, 77, 900], 8, 2, 128, 16, "bf16", 16, 0), ([3000, 77, 900], 32, 2, 128, 16, "f16", 32, 500),
    ([3000, 77, 900], 12, 1, 256, 16, "bf16", 32, 0), ([3000, 77, 900], 20, 1, 128, 16, "bf16", 4, 0),
    ([3000, 77, 900], 8, 2, 128, 8, "f16", 32, 0), ([3000, 77, 900], 32, 2, 128, 8, "bf16", 16, 0),
    ([3000, 77, 900], 12, 1, 256, 8, "f16", 64, 0), ([3000, 77, 900], 4, 1, 48, 8, "f16", 2, 0),
    ([3000, 77, 900], 8, 2, 128, 4, "f16", 32, 0), ([3000, 77, 900], 32, 2, 128, 4, "bf16", 16, 0),
    ([3000, 77, 900], 12, 1, 256, 4, "f16", 64, 300), ([3000, 77, 900], 4, 1, 96, 4, "f16", 8, 0),
    ([100, 20, 300] * 60, 8, 4, 64, 8, "f16", 16, 0), ([100, 20, 300] * 60, 8, 4, 64, 16, "bf16", 16, 0),
]


@pytest.mark.parametrize("lengths,heads,kv,dim,bits,kind,page,window", ROUNDED)
@pytest.mark.parametrize("sharp", [0.5, 4.0])
def test_weights_are_as_good_as_their_sum(lengths, heads, kv, dim, bits, kind, page, window, sharp):
    """The result is the formula's, rounded once to its type: what 16-bit weights would add on top is not there."""
    dtype = TYPES[kind]
    tables, pages = known.place(lengths, page, np.random.default_rng(1))
    cache = paged.PagedKVCache.allocate(pages, page, kv, dim, dtype=dtype, bit_rate=None if bits == 16 else bits, device=DEV)
    fill(cache)
    q = (torch.randn(len(lengths), heads, dim, device=DEV) * sharp).to(dtype)
    tables = torch.from_numpy(tables).to(DEV)
    out = paged.paged_attention(cache, q, tables, torch.tensor(lengths, dtype=torch.int32, device=DEV), window=window)
    assert F.status_read(0)[0]
    off, once, n = 0.0, 0.0, 0
    for b, length in list(enumerate(lengths))[:12]:
        t = torch.arange(max(0, length - window) if window else 0, length, device=DEV)
        where = tables[b, t // page].long()
        k, v = (values(x[where, t % page], bits, dim)[0] for x in (cache.k, cache.v))
        s = dim ** -0.5 * torch.einsum("kgd,tkd->kgt", q[b].double().view(kv, -1, dim), k)
        o = torch.einsum("kgt,tkd->kgd", torch.softmax(s, -1), v).reshape(heads, dim)
        off += float((out[b].double() - o).square().sum())
        once += float((o.to(dtype).double() - o).square().sum())
        n += o.numel()
    # A rounding's error is even over half a step, which holds bf16's 2^-9 and fp16's 2^-12 of a value on average; what else there is (fp32
    # sums, weights of 16 bits and more: 2^-14 beside bf16 rows, 2^-19 otherwise, of values below 5 and independent of it) adds less
    # than a tenth of that to the root of the squares.
    assert off ** 0.5 <= 1.1 * once ** 0.5 + 2.0 ** -20 * n ** 0.5, (off ** 0.5, once ** 0.5)


@pytest.mark.parametrize("page", [16, 8])
@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("rows", [1, 40, 3000])
def test_infinite_values(rows, kind, page):
    """An infinity among 16-bit values is the result of its column, two of either sign a NaN, whatever the weights."""
    dtype = TYPES[kind]
    cache = paged.PagedKVCache.allocate(-(-rows // page), page, 1, 64, dtype=dtype, device=DEV)
    v = torch.randn(rows, 1, 64, device=DEV).to(dtype)
    v[rows // 2, 0, 3] = math.inf
    v[rows - 1, 0, 17] = -math.inf
    v[0, 0, 40], v[rows - 1, 0, 40] = -math.inf, math.inf
    q = torch.randn(1, 8, 64, device=DEV).to(dtype)
    for k in (torch.zeros_like(v), torch.randn(rows, 1, 64, device=DEV).to(dtype)):      # weights of powers of two, and others
        tables = rows_of(cache, rows, k, v)
        out = paged.paged_attention(cache, q, tables, torch.tensor([rows], dtype=torch.int32, device=DEV))[0]
        assert (out[:, 3] == math.inf).all() and (out[:, 17] == -math.inf).all()
        assert out[:, 40].isnan().all() if rows > 1 else (out[:, 40] == math.inf).all()
        others = [c for c in range(64) if c not in (3, 17, 40)]
        assert out[:, others].isfinite().all()
