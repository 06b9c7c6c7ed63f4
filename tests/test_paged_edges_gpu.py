"""The paged key-value cache on the GPU at its edges: memory that ends with the
last row, tables without a good page, numbers at the ends of their ranges, the
forms that only large calls take."""
import pytest
import torch

import fbgemm_b200 as F
from fbgemm_b200 import _capi, paged

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
