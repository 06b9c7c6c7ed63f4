"""The paged key-value cache at its edges, without a GPU."""
import os
import re
import subprocess

import pytest
import torch

from fbgemm_b200 import _capi, build, paged

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_rules_at_the_edges(tmp_path):
    exe = str(tmp_path / "paged_edges_test")
    cuda = os.path.join(os.path.dirname(os.path.dirname(build._nvcc())), "include")
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-I", build.CSRC, "-I", build.INCLUDE, "-I", cuda,
                    os.path.join(ROOT, "tests", "cpp", "paged_edges_test.cc"), "-o", exe], check=True)
    res = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert res.returncode == 0, res.stdout


def test_status_codes_are_the_headers():
    header = open(os.path.join(build.INCLUDE, "fbgemm_b200", "embedding_c_api.h")).read()
    codes = dict(re.findall(r"#define FBGEMM_B200_(STATUS_[A-Z_]+) (\d+) ", header))
    assert codes["STATUS_COPY_TIMEOUT"] == "8"
    for name, value in codes.items():
        assert getattr(_capi, name, int(value)) == int(value), name
    assert _capi.STATUS_COPY_TIMEOUT == 8


@pytest.mark.parametrize("wrong", [-1, 10 ** 9 + 1, 2 ** 32])
def test_copy_limit_refuses(wrong):
    lib = _capi.lib()
    assert lib.fbgemm_b200_set_copy_limit(wrong) == _capi.EINVAL and "nanoseconds" in _capi.last_error()
    assert lib.fbgemm_b200_set_copy_limit(10 ** 9) == 10 ** 9


def append_with(sections):
    x = torch.zeros(5, 2, 64).half()
    cache = paged.PagedKVCache(torch.zeros(3, 4, 2, 64).half(), torch.zeros(3, 4, 2, 64).half())
    return paged.rotary_append(cache, x, x, x, torch.zeros(5, dtype=torch.int64), torch.zeros(len(sections), 5, dtype=torch.int32),
                               torch.zeros(9, 64), sections=sections)


@pytest.mark.parametrize("sections", [(2 ** 32 + 32,), (16, 2 ** 32 + 16), (2 ** 31, 32), (2 ** 62, 2 ** 62), (2 ** 64, 32)])
def test_sections_beyond_32_bits_are_refused(sections):
    with pytest.raises((ValueError, OverflowError), match="sections|too (big|large)"):
        append_with(sections)


@pytest.mark.parametrize("slot", [2 ** 32, 2 ** 31, -2 ** 32, -1])
def test_status_slots_beyond_32_bits_are_refused(slot):
    i = dict(dtype=torch.int32)
    x = torch.zeros(5, 2, 64).half()
    cache = paged.PagedKVCache(torch.zeros(3, 4, 2, 64).half(), torch.zeros(3, 4, 2, 64).half())
    with pytest.raises(ValueError, match="slot"):
        paged.paged_slots(torch.zeros(2, **i), torch.ones(2, **i), torch.zeros(2, 3, **i), torch.zeros(8, **i), torch.ones(1, **i), 16, 4,
                          slot=slot)
    with pytest.raises(ValueError, match="slot"):
        paged.rotary_append(cache, x, x, x, torch.zeros(5, dtype=torch.int64), slot=slot)
    with pytest.raises(ValueError, match="slot"):
        paged.paged_attention(cache, x, torch.zeros(5, 3, **i), torch.ones(5, **i), slot=slot)
