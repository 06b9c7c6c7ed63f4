"""A serving step over a key-value cache in pages, on the GPU.

The K and V rows of many requests lie in pages of a cache: 16-bit rows, or the
fused 8- and 4-bit rows that the row-wise quantizers build and the lookups
read.  A request's pages are named by its row of a block table.  One step is

    step = paged_slots(lengths, new_tokens, block_tables, free_pages, num_free, page_size, capacity)
    q = rotary_append(cache, q, k, v, step.slots, step.positions, cos_sin)      # in every layer
    out = paged_attention(cache, q, block_tables, step.lengths)                 # one new token per request

``paged_slots`` gives out pages and slots from the requests' lengths (beside
the scan that turns bag lengths into offsets), ``rotary_append`` turns queries
and keys and stores the new rows (beside the quantizers), ``paged_attention``
gathers, dequantizes and pools each request's rows with the weights of a
softmax (beside the pooled lookups).  The reference's operators of this kind are
fbgemm_gpu/experimental/gen_ai/src/kv_cache; layouts and arithmetic are this
library's own.

All calls are asynchronous on torch's current stream of the tensors' device,
allocate through torch only, and may be captured into a CUDA graph (the first
calls of a process too, once a ``PagedKVCache`` on the device has been made).
They are for serving: no result carries a gradient.  What they find wrong in
the tensors' contents shows in status slot ``slot``
(``fbgemm_b200.status_read``).
"""
from __future__ import annotations

import ctypes as C
from itertools import accumulate
from typing import NamedTuple

import torch

from . import embedding as E

_DTYPE = {torch.float16: 1, torch.bfloat16: 2}      # FBGEMM_B200_OUT_F16, _BF16
_CONTIGUOUS = torch.contiguous_format
_IN_DTYPE = {torch.float16: 2, torch.bfloat16: 3}   # FBGEMM_B200_IN_F16, _BF16


def row_bytes(head_dim: int, bit_rate: int | None) -> int:
    """Bytes of one cached row: 16-bit values, or codes with fp32 (8-bit rows) or fp16 (4-bit rows) scale and bias."""
    if bit_rate is None:
        return 2 * head_dim
    if bit_rate not in (8, 4):
        raise ValueError("bit_rate must be 8, 4 or None (16-bit rows)")
    return head_dim + 8 if bit_rate == 8 else head_dim // 2 + 4


class PagedKVCache:
    """The K and V rows of one layer: ``k`` and ``v`` of shape [pages, page_size,
    kv_heads, row], laid out alike and in any order of memory with whole rows.
    ``bit_rate`` None: rows of head_dim float16 or bfloat16 values, 16-byte
    aligned.  8 or 4: uint8, fused quantized rows, 4-byte aligned (a multiple of
    16 bytes apart they are read fastest).  ``k`` and ``v`` do not overlap.  Holds
    the tensors, not a copy."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor, bit_rate: int | None = None):
        if k.dim() != 4 or k.shape != v.shape or k.dtype != v.dtype:
            raise ValueError("k and v are [pages, page_size, kv_heads, row], of one shape and type")
        if bit_rate is None:
            if k.dtype not in _DTYPE:
                raise TypeError("16-bit rows are float16 or bfloat16 (quantized rows: uint8 and a bit_rate)")
            head_dim = k.shape[3]
        else:
            if k.dtype != torch.uint8:
                raise TypeError("quantized rows are uint8")
            head_dim = k.shape[3] - 8 if bit_rate == 8 else (k.shape[3] - 4) * 2
            row_bytes(max(head_dim, 0), bit_rate)
        strides = [k.stride(i) if k.shape[i] > 1 else 0 for i in range(4)]
        if strides != [v.stride(i) if v.shape[i] > 1 else 0 for i in range(4)] or strides[3] > 1:
            raise ValueError("k and v are laid out alike, their rows without gaps")
        if k.get_device() != v.get_device():
            raise ValueError("k and v lie on one device")
        self._k, self._v = k, v
        self.bit_rate = bit_rate
        self.dtype = k.dtype if bit_rate is None else None
        self.num_pages, self.page_size, self.kv_heads = k.shape[:3]
        self.head_dim = head_dim
        self.device = k.device
        self._index = k.get_device()
        size = k.element_size()
        self._struct = E._capi.PagedCache(
            k=k.data_ptr(), v=v.data_ptr(), num_pages=self.num_pages, page_stride=strides[0] * size,
            slot_stride=strides[1] * size, head_stride=strides[2] * size, page_size=self.page_size, kv_heads=self.kv_heads,
            head_dim=head_dim, in_dtype=0 if bit_rate else _IN_DTYPE[k.dtype], bit_rate=bit_rate or 0)
        self._address = C.addressof(self._struct)
        self._workspace = {}   # (batch, query heads, type, width, window) -> bytes
        E._capi.check(E._capi.lib().fbgemm_b200_paged_cache_check(C.byref(self._struct)), "PagedKVCache")
        _context(self._index)  # made here if this is the device's first: a capture does not let it allocate

    @classmethod
    def allocate(cls, num_pages: int, page_size: int, kv_heads: int, head_dim: int, dtype=torch.bfloat16,
                 bit_rate: int | None = None, device="cuda", row_alignment: int = 16) -> "PagedKVCache":
        """A cleared cache.  A head's rows of a page follow one another, as one request reads them; quantized rows are
        padded to ``row_alignment`` bytes."""
        n = row_bytes(head_dim, bit_rate)
        if bit_rate is None:
            shape, dtype = (num_pages, kv_heads, page_size, head_dim), dtype
            rows = [torch.zeros(shape, dtype=dtype, device=device) for _ in range(2)]
        else:
            pitch = (n + row_alignment - 1) // row_alignment * row_alignment
            shape = (num_pages, kv_heads, page_size, pitch)
            rows = [torch.zeros(shape, dtype=torch.uint8, device=device)[..., :n] for _ in range(2)]
        return cls(*(x.permute(0, 2, 1, 3) for x in rows), bit_rate=bit_rate)

    @property
    def k(self) -> torch.Tensor:
        return self._k

    @property
    def v(self) -> torch.Tensor:
        return self._v

    def __reduce__(self):   # a copy describes its own tensors
        return PagedKVCache, (self._k, self._v, self.bit_rate)

    def _workspace_bytes(self, batch: int, heads: int, dtype, width: int, window: int) -> int:
        key = batch, heads, dtype, width, window
        n = self._workspace.get(key)
        if n is None:
            if dtype not in _DTYPE or self._index < 0:
                return 0    # (the call itself refuses)
            rc = E._capi.lib().fbgemm_b200_paged_attention_workspace(
                _context(self._index), C.byref(self._struct), batch, heads, _DTYPE[dtype], width, window)
            n = E._capi.check(rc, "fbgemm_b200_paged_attention_workspace")
            if len(self._workspace) >= 1024:    # (a width for every step of long generations)
                self._workspace.clear()
            self._workspace[key] = n
        return n


def _context(device: int):
    """The context's address; None for host tensors, which the call refuses."""
    return E._handle_of(device) if device >= 0 else None


def _stream(device: int):
    return E._current_stream(device) if device >= 0 else None


class PagedSlots(NamedTuple):
    """What ``paged_slots`` returns, all on the device."""
    slots: torch.Tensor       # int64 [capacity]: page * page_size + place in the page; -1 behind the last row
    positions: torch.Tensor   # int32 [capacity]: the row's place in its request; 0 behind the last row
    requests: torch.Tensor    # int32 [capacity]: whose row it is; -1 behind the last row
    offsets: torch.Tensor     # int32 [batch + 1]: each request's first row
    lengths: torch.Tensor     # int32 [batch]: lengths + new_tokens
    num_free: torch.Tensor    # int32 [1]: pages left


def paged_slots(lengths: torch.Tensor, new_tokens: torch.Tensor, block_tables: torch.Tensor, free_pages: torch.Tensor,
                num_free: torch.Tensor, page_size: int, capacity: int, slot: int = 0) -> PagedSlots:
    """Room for ``new_tokens[b]`` more rows in each request that holds
    ``lengths[b]`` (int32; negative counts are 0).

    Pages that the new rows need come from the top of the stack
    ``free_pages[:num_free]``, requests in order, and are entered into
    ``block_tables`` (int32 [batch, pages], in place; no other entry changes).
    The maps have ``capacity`` rows: the new rows, request after request, and
    padding behind them.  A last page that is not full is continued, so it must
    not be shared with another request.  1 to 16384 requests.

    All or nothing: if pages, table columns or capacity run out, no page and no
    slot is given out (``slots`` all -1, lengths and num_free as they were) and
    the status record is {6, first request that does not fit, its new length,
    num_free}.  Give the outputs' ``lengths`` and ``num_free`` to the next step;
    they are not the inputs' memory."""
    batch = lengths.shape[0]
    device = lengths.device
    slots = torch.empty(capacity, dtype=torch.int64, device=device)
    rest = torch.empty(2 * capacity + 2 * batch + 2, dtype=torch.int32, device=device)
    dev = lengths.get_device()
    rc = E._capi.paged().paged_slots(_context(dev), lengths, new_tokens, block_tables, free_pages, num_free, page_size, capacity,
                                      slots, rest, slot, _stream(dev))
    E._capi.check(rc, "fbgemm_b200_paged_slots")
    return PagedSlots(slots, *rest.split_with_sizes((capacity, capacity, batch + 1, batch, 1)))


def rotary_append(cache: PagedKVCache, q: torch.Tensor | None, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor,
                  positions: torch.Tensor | None = None, cos_sin: torch.Tensor | None = None, *, sections=None,
                  interleaved: bool = False, q_out: torch.Tensor | None = None, slot: int = 0) -> torch.Tensor | None:
    """Turns the heads of ``q`` [tokens, heads, head_dim] and ``k`` [tokens,
    kv_heads, head_dim] by their positions, stores ``k`` and ``v`` in rows
    ``slots`` (int64 [tokens], distinct; -1: not stored) of the cache, and returns
    the turned ``q`` (None if ``q`` is).

    ``cos_sin``: float32 [max_pos, rot_dim], a position's rot_dim / 2 cosines and
    then its sines; the first rot_dim columns of a head (a multiple of 16) turn,
    in pairs half of rot_dim apart, or next to each other if ``interleaved``.
    None: nothing is turned, ``q`` is copied.  ``positions``: int32 [tokens], or [axes,
    tokens] with ``sections``, the number of pairs of each axis in turn (time,
    height, width).  The arithmetic is fp32 with one rounding: to 16 bits, or to
    the codes, scale and bias that ``FloatToFused...Quantized...`` give for the
    same fp32 row, byte for byte.  ``q_out``, contiguous, takes the turned queries; it
    may be ``q`` itself, and overlaps nothing else that is read.

    A position outside the table leaves its token's query unturned and its rows
    unstored (status {1, token, 0, position}); a slot outside the cache stores
    nothing (status {7, token, 0, slot})."""
    if q is None:
        if q_out is not None:
            raise ValueError("q_out without q")
    elif q_out is None:
        q_out = torch.empty_like(q, memory_format=_CONTIGUOUS)
    if cos_sin is None:
        if positions is not None or sections is not None:
            raise ValueError("positions and sections go with cos_sin")
    elif positions is None:
        raise ValueError("cos_sin goes with positions")
    ends = None
    if sections is not None:
        if not 1 <= len(sections) <= 4 or min(sections) < 0:
            raise ValueError("sections are the pairs of 1 to 4 axes")
        ends = tuple(accumulate(sections))
    dev = cache._index
    rc = E._capi.paged().rotary_append(_context(dev), cache._address, dev, q, k, v, q_out, slots, positions, cos_sin,
                                        interleaved, ends, slot, _stream(dev))
    E._capi.check(rc, "fbgemm_b200_rotary_append")
    return q_out


def paged_attention(cache: PagedKVCache, q: torch.Tensor, block_tables: torch.Tensor, lengths: torch.Tensor,
                    scale: float | None = None, window: int = 0, out: torch.Tensor | None = None, return_lse: bool = False,
                    slot: int = 0):
    """Attention of one new token per request over its rows of the cache.

    ``q``: [batch, heads, head_dim] float16 or bfloat16 (a 16-bit cache's type),
    ``heads`` a multiple of the cache's, query head h reading cached head
    h // (heads / kv_heads).  ``block_tables``: int32 [batch, pages], row t of
    request b in page ``block_tables[b, t // page_size]``.  ``lengths``: int32
    [batch], rows of each request with the new token's own.  ``scale``: of the
    scores, head_dim ** -0.5 by default.  ``window``: rows that a token sees, the
    last ones (0: all).  Returns [batch, heads, head_dim] in q's type, and with
    ``return_lse`` the float32 [batch, heads] logarithms of the sums of
    exp(scale * q.k), by which results over parts of the rows are joined.  A
    request without rows gets zeros and -inf.  ``out``, contiguous, takes the
    result; it does not overlap ``q``.

    Scores, sums and the output are fp32 until the output's one rounding; the
    weights enter the sum over rows as two 16-bit numbers each (bfloat16 beside a
    bfloat16 cache: 16 bits; float16 beside others: 22 bits, beside quantized rows
    with bfloat16 queries 11; beside quantized rows times the row's scale, each row
    off by up to 2**-35 of the widest row's range).  A page outside the cache
    is left out (status {7, request, row, page}; all of a request's pages: a
    request without rows); a length that is negative or
    beyond the table is brought within it (status {3, request, 0, length})."""
    if out is None:
        out = torch.empty_like(q, memory_format=_CONTIGUOUS)
    batch, heads = q.shape[:2]
    lse = lengths.new_empty((batch, heads), dtype=torch.float32) if return_lse else None
    # The call's own workspace: calls on several streams, captured ones too, share nothing.
    workspace, n = None, cache._workspace_bytes(batch, heads, q.dtype, block_tables.shape[-1], window)
    if n:
        workspace = torch.empty(n, dtype=torch.uint8, device=cache.device)
    dev = cache._index
    rc = E._capi.paged().paged_attention(_context(dev), cache._address, dev, q, block_tables, lengths, scale, window, out, lse,
                                          workspace, n, slot, _stream(dev))
    E._capi.check(rc, "fbgemm_b200_paged_attention")
    return (out, lse) if return_lse else out
