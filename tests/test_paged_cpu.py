"""The paged key-value cache without a GPU: what is refused, and how the
attention is split over workers."""
import copy
import ctypes as C
import os
import pickle
import subprocess

import pytest
import torch

from fbgemm_b200 import _capi, build, paged
from fbgemm_b200 import embedding as E

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_rule_of_the_split(tmp_path):
    exe = str(tmp_path / "paged_rule_test")
    cuda = os.path.join(os.path.dirname(os.path.dirname(build._nvcc())), "include")
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-I", build.CSRC, "-I", build.INCLUDE, "-I", cuda,
                    os.path.join(ROOT, "tests", "cpp", "paged_rule_test.cc"), "-o", exe], check=True)
    res = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert res.returncode == 0, res.stdout


def cache(dim=64, bit_rate=None, pages=3, page=4, heads=2, dtype=torch.float16):
    n = paged.row_bytes(dim, bit_rate) if bit_rate else dim
    x = [torch.zeros(pages, page, heads, n, dtype=torch.uint8 if bit_rate else dtype) for _ in range(2)]
    return paged.PagedKVCache(*x, bit_rate=bit_rate)


def test_struct_layouts_match_the_header():
    assert C.sizeof(_capi.PagedCache) == 48 + 5 * 4 + 4
    assert _capi.PagedCache.page_size.offset == 48 and _capi.PagedCache.bit_rate.offset == 64
    assert C.sizeof(_capi.Rotary) == 16 + 7 * 4 + 4 and _capi.Rotary.section_end.offset == 28


@pytest.mark.parametrize("dim,bit_rate", [(16, None), (80, None), (256, None), (16, 8), (112, 8), (256, 8), (32, 4), (96, 4)])
def test_caches_that_are_taken(dim, bit_rate):
    c = cache(dim, bit_rate)
    assert (c.head_dim, c.page_size, c.num_pages, c.kv_heads) == (dim, 4, 3, 2)
    for other in (copy.copy(c), copy.deepcopy(c), pickle.loads(pickle.dumps(c))):   # a copy describes its own tensors
        assert other._struct.k == other.k.data_ptr() and other._address != c._address
        assert other.head_dim == dim and other.bit_rate == bit_rate
    a = paged.PagedKVCache.allocate(3, 4, 2, dim, dtype=torch.bfloat16, bit_rate=bit_rate, device="cpu")
    assert a.head_dim == dim and (bit_rate is None or a._struct.slot_stride % 16 == 0)


@pytest.mark.parametrize("make", [
    lambda: cache(24), lambda: cache(272), lambda: cache(48, 4), lambda: cache(8, 8), lambda: cache(page=3), lambda: cache(page=131072, pages=1),
    lambda: cache(dtype=torch.float32),
    lambda: paged.PagedKVCache(torch.zeros(2, 4, 2, 64).half(), torch.zeros(2, 4, 2, 32).half()),
    lambda: paged.PagedKVCache(torch.zeros(2, 4, 2, 64).half(), torch.zeros(2, 4, 64, 2).half().transpose(2, 3)),
    lambda: paged.PagedKVCache(torch.zeros(2, 4, 2, 72, dtype=torch.uint8), torch.zeros(2, 4, 2, 72, dtype=torch.uint8), bit_rate=2),
    lambda: paged.PagedKVCache(torch.zeros(2, 4, 2, 4, dtype=torch.uint8), torch.zeros(2, 4, 2, 4, dtype=torch.uint8), bit_rate=8),
    lambda: paged.PagedKVCache(*[torch.zeros(2 * 4 * 2 * 64 + 1).half()[1:].view(2, 4, 2, 64)] * 2),            # 2-byte aligned
    lambda: paged.PagedKVCache(*[torch.zeros(2, 4, 2, 68).half()[..., :64]] * 2),                             # rows 136 bytes apart
    lambda: paged.PagedKVCache(*[torch.zeros(2, 4, 2, 74, dtype=torch.uint8)[..., :72]] * 2, bit_rate=8),     # 74 bytes apart
    lambda: paged.PagedKVCache(*[torch.zeros(1, 1, 1, 64).half().expand(2, 4, 2, 64)] * 2),                   # all rows one
    lambda: paged.PagedKVCache(*[torch.zeros(0, 4, 2, 64).half()] * 2),
])
def test_caches_that_are_refused(make):
    with pytest.raises((ValueError, TypeError, _capi.Fbgemmb200Error)):
        make()


def attention_arguments(**kw):
    a = dict(cache=cache(), q=torch.zeros(2, 4, 64).half(), block_tables=torch.zeros(2, 3, dtype=torch.int32),
             lengths=torch.ones(2, dtype=torch.int32))
    a.update(kw)
    return a


@pytest.mark.parametrize("bad", [
    dict(q=torch.zeros(2, 4, 64)), dict(q=torch.zeros(2, 4, 64).bfloat16()), dict(q=torch.zeros(2, 4, 32).half()),
    dict(q=torch.zeros(8, 64).half()), dict(q=torch.zeros(2, 64, 4).half().transpose(1, 2)),
    dict(block_tables=torch.zeros(2, 3, dtype=torch.int64)), dict(block_tables=torch.zeros(3, 3, dtype=torch.int32)),
    dict(block_tables=torch.zeros(3, 2, dtype=torch.int32).T), dict(lengths=torch.ones(2)), dict(lengths=torch.ones(3, dtype=torch.int32)),
    dict(lengths=torch.ones(4, dtype=torch.int32)[::2]),
    dict(),   # host tensors: there is no CPU path
])
def test_attention_refuses(bad):
    with pytest.raises((ValueError, TypeError)):
        paged.paged_attention(**attention_arguments(**bad))


def append_arguments(**kw):
    a = dict(cache=cache(), q=torch.zeros(5, 4, 64).half(), k=torch.zeros(5, 2, 64).half(), v=torch.zeros(5, 2, 64).half(),
             slots=torch.zeros(5, dtype=torch.int64), positions=torch.zeros(5, dtype=torch.int32), cos_sin=torch.zeros(9, 64))
    a.update(kw)
    return a


@pytest.mark.parametrize("bad", [
    dict(k=torch.zeros(5, 2, 64)), dict(k=torch.zeros(5, 2, 64).bfloat16()), dict(v=torch.zeros(5, 2, 64).bfloat16()),
    dict(v=torch.zeros(4, 2, 64).half()), dict(k=torch.zeros(5, 4, 64).half()), dict(q=torch.zeros(5, 4, 32).half()),
    dict(slots=torch.zeros(5, dtype=torch.int32)), dict(slots=torch.zeros(4, dtype=torch.int64)),
    dict(positions=None), dict(positions=torch.zeros(5, dtype=torch.int64)), dict(positions=torch.zeros(4, dtype=torch.int32)),
    dict(cos_sin=torch.zeros(9, 64).double()), dict(cos_sin=None), dict(cos_sin=torch.zeros(64, 9).T),
    dict(sections=[16, 16]), dict(positions=torch.zeros(2, 5, dtype=torch.int32), sections=[16, 8]),
    dict(positions=torch.zeros(2, 5, dtype=torch.int32), sections=[40, -8]),
    dict(positions=torch.zeros(5, 5, dtype=torch.int32), sections=[8, 8, 8, 4, 4]),
    dict(q=None, q_out=torch.zeros(5, 4, 64).half()), dict(q_out=torch.zeros(5, 4, 64)),
    dict(),   # host tensors
])
def test_append_refuses(bad):
    with pytest.raises((ValueError, TypeError)):
        paged.rotary_append(**append_arguments(**bad))


def slots_arguments(**kw):
    i = dict(dtype=torch.int32)
    a = dict(lengths=torch.zeros(2, **i), new_tokens=torch.ones(2, **i), block_tables=torch.zeros(2, 3, **i),
             free_pages=torch.zeros(8, **i), num_free=torch.ones(1, **i), page_size=16, capacity=4)
    a.update(kw)
    return a


@pytest.mark.parametrize("bad", [
    dict(lengths=torch.zeros(2, dtype=torch.int64)), dict(new_tokens=torch.ones(3, dtype=torch.int32)),
    dict(block_tables=torch.zeros(3, 3, dtype=torch.int32)), dict(num_free=torch.ones(2, dtype=torch.int32)),
    dict(num_free=torch.ones(1)), dict(free_pages=torch.zeros(2, 4, dtype=torch.int32)), dict(),
])
def test_slots_refuses(bad):
    with pytest.raises((ValueError, TypeError)):
        paged.paged_slots(**slots_arguments(**bad))


class Stand:
    """A context that no call gets as far as using."""
    memory = C.create_string_buffer(1 << 16)
    handle = C.addressof(memory)


def c_cache(**kw):
    a = dict(k=1 << 20, v=1 << 21, num_pages=4, page_stride=16 * 2 * 128, slot_stride=2 * 128, head_stride=128, page_size=16,
             kv_heads=2, head_dim=64, in_dtype=2, bit_rate=0)
    a.update(kw)
    return _capi.PagedCache(**a)


@pytest.mark.parametrize("bad", [
    dict(k=0), dict(v=(1 << 21) + 8), dict(num_pages=0), dict(num_pages=1 << 31), dict(page_size=0), dict(page_size=24),
    dict(page_size=1 << 17), dict(kv_heads=0), dict(head_dim=0), dict(head_dim=40), dict(head_dim=512), dict(in_dtype=1),
    dict(in_dtype=4), dict(in_dtype=0, bit_rate=2), dict(head_stride=120), dict(head_stride=-128), dict(slot_stride=112),
])
def test_c_cache_check_refuses(bad):
    assert _capi.lib().fbgemm_b200_paged_cache_check(C.byref(c_cache(**bad))) == _capi.EINVAL
    assert _capi.last_error() != ""


def test_c_cache_check_takes():
    for good in (dict(), dict(in_dtype=3), dict(in_dtype=0, bit_rate=8, head_stride=72, slot_stride=144, page_stride=16 * 144),
                 dict(num_pages=1, page_stride=0), dict(kv_heads=1, head_stride=0), dict(page_size=1, slot_stride=0)):
        assert _capi.lib().fbgemm_b200_paged_cache_check(C.byref(c_cache(**good))) == 0, good


@pytest.mark.parametrize("bad", [
    dict(ctx=None), dict(slot=-1), dict(slot=_capi.USER_SLOTS), dict(batch=-1), dict(q_heads=3), dict(q_heads=0), dict(dtype=0),
    dict(dtype=2), dict(q=0), dict(q=8), dict(q_token=4), dict(tables=0), dict(width=-1), dict(width=1 << 28), dict(lengths=0),
    dict(window=-1), dict(out=0), dict(out=8), dict(workspace=0), dict(workspace_bytes=100),
])
def test_c_attention_refuses(bad):
    a = dict(ctx=Stand.handle, batch=2, q_heads=4, dtype=1, q=1 << 20, q_token=256, tables=1 << 20, width=1000, lengths=1 << 20,
             window=0, out=1 << 24, workspace=1 << 20, workspace_bytes=1 << 30, slot=0)
    a.update(bad)
    rc = _capi.lib().fbgemm_b200_paged_attention(
        a["ctx"], C.byref(c_cache()), a["batch"], a["q_heads"], a["dtype"], a["q"], a["q_token"], 64, a["tables"], a["width"], 1000,
        a["lengths"], 0.125, a["window"], a["out"], None, a["workspace"], a["workspace_bytes"], a["slot"], None)
    assert rc == _capi.EINVAL and _capi.last_error() != ""


@pytest.mark.parametrize("bad", [
    dict(ctx=None), dict(tokens=-1), dict(dtype=2), dict(q=8), dict(k=0), dict(v=4), dict(token=12), dict(slots=0),
    dict(positions=0), dict(rot_dim=8), dict(rot_dim=80), dict(rot_dim=40), dict(axes=0), dict(axes=5), dict(ends=(16, 0, 0, 0)),
    dict(axes=2, ends=(40, 32, 0, 0)), dict(max_pos=0), dict(cos_sin=0), dict(q_heads=0),
])
def test_c_append_refuses(bad):
    a = dict(ctx=Stand.handle, tokens=2, dtype=1, q=1 << 20, k=1 << 20, v=1 << 20, token=128, slots=1 << 20, positions=1 << 20,
             rot_dim=64, axes=1, ends=(32, 0, 0, 0), max_pos=4, cos_sin=1 << 20, q_heads=4)
    a.update(bad)
    r = _capi.Rotary(cos_sin=a["cos_sin"], max_pos=a["max_pos"], rot_dim=a["rot_dim"], axes=a["axes"],
                     section_end=(C.c_int32 * 4)(*a["ends"]))
    rc = _capi.lib().fbgemm_b200_rotary_append(
        a["ctx"], C.byref(c_cache()), a["tokens"], a["q_heads"], a["dtype"], a["q"], a["token"], 64, a["k"], 128, 64, a["v"], 128, 64,
        1 << 24, a["slots"], a["positions"], 0, C.byref(r), 0, None)
    assert rc == _capi.EINVAL and _capi.last_error() != ""


def overlapping(rc):
    return rc == _capi.EINVAL and "overlap" in _capi.last_error()


# Two rows of four heads of 64 16-bit values: 1024 bytes at 1 << 20, or with rows 1024 elements apart 2560.
@pytest.mark.parametrize("token,out", [(256, 0), (256, 1008), (256, -1008), (1024, 0), (1024, 2544), (-256, -512)])
def test_c_attention_refuses_results_over_queries(token, out):
    call = _capi.lib().fbgemm_b200_paged_attention
    assert overlapping(call(Stand.handle, C.byref(c_cache()), 2, 4, 1, 1 << 20, token, 64, 1 << 22, 8, 8, 1 << 22, 0.125, 0,
                            (1 << 20) + out, None, None, 0, 0, None))


@pytest.mark.parametrize("q,token,head,k,v", [
    (-16, 256, 64, 1 << 23, 1 << 23), (1008, 256, 64, 1 << 23, 1 << 23),
    (0, 264, 64, 1 << 23, 1 << 23), (0, 256, 72, 1 << 23, 1 << 23), (0, 0, 64, 1 << 23, 1 << 23),   # not the same rows
    (0, 256, 64, 1008, 1 << 23), (0, 256, 64, 1 << 23, -496), (1 << 23, 256, 64, 0, 1 << 23)])
def test_c_append_refuses_results_over_what_it_reads(q, token, head, k, v):
    r = _capi.Rotary(cos_sin=1 << 22, max_pos=4, rot_dim=64, axes=1, section_end=(C.c_int32 * 4)(32, 0, 0, 0))
    at = 1 << 20
    assert overlapping(_capi.lib().fbgemm_b200_rotary_append(
        Stand.handle, C.byref(c_cache()), 2, 4, 1, at + q, token, head, at + k, 128, 64, at + v, 128, 64, at, 1 << 22, 1 << 22, 0,
        C.byref(r), 0, None))


def test_c_append_refuses_keys_and_values_in_one_place():
    rc = _capi.lib().fbgemm_b200_rotary_append(Stand.handle, C.byref(c_cache(v=1 << 20)), 2, 0, 1, None, 0, 0, 1 << 22, 128, 64,
                                               1 << 22, 128, 64, None, 1 << 22, None, 0, None, 0, None)
    assert rc == _capi.EINVAL and "same memory" in _capi.last_error()


@pytest.mark.parametrize("bad", [
    dict(ctx=None), dict(batch=0), dict(batch=_capi.PAGED_MAX_BATCH + 1), dict(page_size=12), dict(page_size=0), dict(width=-1),
    dict(width=1 << 27), dict(capacity=-1), dict(free_capacity=-1), dict(stride=7), dict(lengths=0), dict(tables=0), dict(slots=0),
    dict(free_pages=0), dict(num_free=0),
])
def test_c_slots_refuses(bad):
    a = dict(ctx=Stand.handle, batch=2, lengths=1 << 20, tables=1 << 20, width=8, stride=8, free_pages=1 << 20, free_capacity=4,
             num_free=1 << 20, page_size=16, capacity=4, slots=1 << 20)
    a.update(bad)
    x = 1 << 20
    rc = _capi.lib().fbgemm_b200_paged_slots(a["ctx"], a["batch"], a["lengths"], x, a["tables"], a["width"], a["stride"],
                                             a["free_pages"], a["free_capacity"], a["num_free"], a["page_size"], a["capacity"],
                                             a["slots"], x, x, x, x, x, 0, None)
    assert rc == _capi.EINVAL and _capi.last_error() != ""


def test_nothing_to_do_is_no_call():
    assert _capi.lib().fbgemm_b200_paged_attention(Stand.handle, C.byref(c_cache()), 0, 4, 1, None, 0, 0, None, 0, 0, None, 1.0, 0,
                                                   None, None, None, 0, 0, None) == 0
    assert _capi.lib().fbgemm_b200_rotary_append(Stand.handle, C.byref(c_cache()), 0, 4, 1, None, 0, 0, None, 0, 0, None, 0, 0,
                                                 None, None, None, 0, None, 0, None) == 0
    assert E is paged.E


def test_numbers_and_arrays_are_no_tensors():
    for wrong in (5, 1.5, None, [1]):
        for call, arguments, name in ((paged.paged_attention, attention_arguments, "q"),
                                      (paged.paged_attention, attention_arguments, "block_tables"),
                                      (paged.paged_attention, attention_arguments, "lengths"),
                                      (paged.rotary_append, append_arguments, "k"), (paged.rotary_append, append_arguments, "slots"),
                                      (paged.paged_slots, slots_arguments, "lengths"), (paged.paged_slots, slots_arguments, "num_free")):
            with pytest.raises((TypeError, AttributeError)):
                call(**arguments(**{name: wrong}))


def test_sizes_beyond_32_bits_are_refused():
    many = torch.zeros(1, dtype=torch.int32).expand(1, 1).as_strided((2, 2 ** 31), (0, 0))
    for call, arguments, bad in ((paged.paged_attention, attention_arguments, dict(window=2 ** 31)),
                                 (paged.paged_attention, attention_arguments, dict(window=-1)),
                                 (paged.paged_attention, attention_arguments, dict(block_tables=many)),
                                 (paged.paged_slots, slots_arguments, dict(page_size=2 ** 33)),
                                 (paged.paged_slots, slots_arguments, dict(block_tables=many))):
        with pytest.raises(ValueError):
            call(**arguments(**bad))
