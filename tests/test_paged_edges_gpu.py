"""The paged key-value cache on the GPU at its edges: memory that ends with the
last row, tables without a good page, numbers at the ends of their ranges, the
forms that only large calls take."""
import numpy as np
import pytest
import torch

from fbgemm_b200 import paged

from test_paged_gpu import DEV, TYPES, check_attention, fill

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def seeded():
    torch.manual_seed(1234)


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
