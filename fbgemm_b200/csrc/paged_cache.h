// The paged key-value cache: what its kernels share (paged_slots_kernels.cu, rotary_append_kernels.cu,
// paged_attention.cuh) and the rule by which the attention is split.
#pragma once

#include <cuda_runtime.h>

#include <cstddef>
#include <cstdint>

#include "fbgemm_b200/embedding_c_api.h"

namespace fbgemm_b200 {

#ifdef __CUDACC__
#define FBGEMM_B200_HD __host__ __device__ __forceinline__
#else
#define FBGEMM_B200_HD inline
#endif

// ---- how the attention is split (also compiled on the host by its test) -----------------------------------------------
//
// A request's rows are cut into units of `unit` rows, the last one short; every (request, cached head, head tile) has
// units_of() of them, at least one, so that a request without rows is somebody's too.  All units stand in one line,
// request after request, head after head, and each worker (a warp, or several that share rows) takes the same number of
// neighbours: the chip is filled whatever the lengths are, long requests are split, short ones share a worker.

// Rows [first, end) that a request's new token sees: `length` rows in the cache, the last `window` of them (0: all).
struct RowSpan {
  int32_t first, end;
};
FBGEMM_B200_HD RowSpan span_of(int32_t length, int32_t window, int64_t most) {
  int64_t end = length < 0 ? 0 : length;
  end = end > most ? most : end;
  const int64_t first = window > 0 && end > window ? end - window : 0;
  return RowSpan{(int32_t)first, (int32_t)end};
}

// Units are counted from a multiple of 32 rows, so that 16 rows of a step lie in one page of 16 or more, and 32 in one of 32.
FBGEMM_B200_HD int32_t aligned_first(RowSpan s) {
  return s.first & ~31;
}
FBGEMM_B200_HD int32_t units_of(RowSpan s, int32_t unit) {
  const int32_t n = (int32_t)(((int64_t)s.end - aligned_first(s) + unit - 1) / unit);
  return n > 0 ? n : 1;
}

// Who takes which units.  The first `workers` take `big` units each.  SMs are not equally fast at bringing rows (three quarters to
// one and an eighth of the mean rate, by where they lie), so where memory is what warps wait for (two_sizes) the last quarter of
// the line is left to as many workers again, `small` units each, whose blocks start where others have ended.
struct UnitSplit {
  int64_t big, small, workers;
  FBGEMM_B200_HD int64_t first(int64_t worker) const {
    return worker <= workers ? worker * big : workers * big + (worker - workers) * small;
  }
  FBGEMM_B200_HD int64_t worker_of(int64_t unit) const {
    return unit < workers * big || small == 0 ? unit / big : workers + (unit - workers * big) / small;
  }
  FBGEMM_B200_HD int64_t units_of(int64_t worker) const { return worker < workers ? big : small; }
};
constexpr int64_t kUnitsForTwo = 40;  // units per worker from which on there are workers of either size
// Whether a call may have workers of either size.  With them over without, 30, 42, 60 and 100 units a worker: 128 columns, 4 heads to a
// cached one, 128 items 1.01 0.98 0.97 0.96 (16-bit rows), 0.99 0.96 0.96 0.98 (8-bit); 256 items of 64 or 96 columns 1.01 to 1.05,
// 1.00 to 1.02, 0.97 to 0.99, 0.98 to 1.01; of 256 columns 1.03 to 1.08, 0.99 to 1.06, 0.99 to 1.02, 0.97 to 0.99; 32 requests of
// 16384 8-bit rows (74 units) 0.98.  Few items are joined by parts: 64 items 1.03 1.00 0.98 0.96 and 1.00 0.98 0.98 0.98, 32 items
// 1.07 1.02 1.00 1.00, 8 items 1.17 1.12 1.10 1.01.  Where instructions are what warps wait for, all SMs are as fast, and the second start
// costs 10 to 20 us: 4-bit rows 1.13 to 1.30, 1.12 to 1.23, 1.10 to 1.17, 1.05 to 1.10 (1.03 still at 148 units), 16 heads of a warp and
// 32 of two 1.09 to 1.25, 1.07 to 1.21, 1.03 to 1.16, 1.00 to 1.11.
FBGEMM_B200_HD bool two_sizes(int32_t bits, int32_t tile_heads, int64_t items, int64_t most_units, int64_t workers) {
  return bits != 4 && tile_heads <= 8 && items >= 64 && most_units >= kUnitsForTwo * workers;
}
FBGEMM_B200_HD UnitSplit split_units(int64_t total, int64_t workers, bool two) {
  UnitSplit s;
  s.workers = workers;
  s.big = (total + workers - 1) / workers;
  s.small = 0;
  if (two && s.big >= kUnitsForTwo) {
    s.big = s.big * 3 / 4;
    s.small = (total - workers * s.big + workers - 1) / workers;
  }
  s.big = s.big > 0 ? s.big : 1;
  return s;
}

// What a block's neighbouring workers have together, and how many of them have any; nothing behind the last unit (a block of the
// second set where there is none).
struct BlockShare {
  int64_t units;
  int32_t active;
};
FBGEMM_B200_HD BlockShare block_share(const UnitSplit& s, int64_t block, int32_t workers, int64_t total) {
  const int64_t first = s.first(block * workers), per = s.units_of(block * workers);
  const int64_t end = first + workers * per < total ? first + workers * per : total;
  BlockShare r = {0, 0};
  if (per > 0 && end > first) {
    r.units = end - first;
    r.active = (int32_t)((r.units + per - 1) / per);
  }
  return r;
}

// Blocks that take an item, as far as the host knows its length: one for 512 rows, as many as that takes for more, as long as
// all of them are on the chip at once; and more, up to eight, down to 64 rows each, while every one has an SM to itself.  0: the
// units are shared by the whole chip, which takes a second launch and a workspace.  Us by one block a head, by two, by
// eight, shared by the chip, one request of 8 heads: 1000 rows 18.7, 13.3, 8.2, 11.2; 2000 rows 33.2, -, 10.1, 11.5.  With more
// items than blocks, a block each and shared: 208 requests of up to 30 16-bit rows 20.2 and 12.3, 128 of 100 17.1 and 14.1, 208
// of 500 45.5 and 50.1, of 8-bit rows 40.8 and 38.4.  (A block an item up to 2048 rows: 42 instead of 32 for 64 requests of 64 to
// 2000 rows.)
FBGEMM_B200_HD int32_t blocks_of_item(int64_t most_rows, int64_t items, int64_t blocks) {
  int32_t n = 1;
  while (n < 8 && ((most_rows > 512 * n && items * 2 * n <= blocks) || (most_rows >= 128 * n && items * 2 * n <= blocks / 3))) {
    n *= 2;
  }
  return items <= blocks && most_rows <= 512 * n ? n : 0;
}

// Bytes of a row's 16-byte piece `piece`: what the copies of pages below 16 rows read, so that nothing behind a row is read
// (strides may be padded without padding behind the last row).
FBGEMM_B200_HD int32_t piece_bytes(int32_t row_bytes, int32_t piece) {
  const int32_t n = row_bytes - 16 * piece;
  return n < 0 ? 0 : n < 16 ? n : 16;
}

// ---- kernel parameters ------------------------------------------------------------------------------------------------

struct PagedSlotsParams {
  const int32_t* lengths;
  const int32_t* fresh;      // new tokens of each request
  int32_t* tables;
  int64_t table_stride;      // elements between requests
  const int32_t* free_pages;
  const int32_t* num_free;
  int64_t* slots;
  int32_t* positions;
  int32_t* requests;
  int32_t* offsets;
  int32_t* lengths_out;
  int32_t* num_free_out;
  int32_t* status;
  int32_t batch, width, free_capacity, page_shift, capacity;
};
cudaError_t launch_paged_slots(const PagedSlotsParams& p, cudaStream_t stream);

struct RotaryAppendParams {
  const void *q, *k, *v;                       // 16-bit types, 16-byte aligned rows
  int64_t q_token, q_head, k_token, k_head, v_token, v_head;  // bytes
  void* q_out;                                 // [tokens, heads, dim], null: q is not rotated
  const int64_t* slots;
  const int32_t* positions;                    // [axes, tokens], null: nothing is rotated
  int64_t positions_stride;                    // elements between axes
  const float* cos_sin;                        // [max_pos, rot]: cosines, sines
  int64_t max_pos;
  uint8_t *k_cache, *v_cache;
  int64_t page_stride, slot_stride, head_stride, num_slots;   // bytes; rows in all pages
  int32_t* status;
  int64_t tokens;
  int32_t heads, kv_heads, dim, rot, page_shift, axes;
  int32_t section_end[4];                      // pairs [section_end[a - 1], section_end[a]) turn by axis a
  int32_t interleaved, bf16, bits;             // bits: 16, 8 or 4
  bool angles_aligned;                         // cos_sin to 16 bytes
};
cudaError_t launch_rotary_append(const RotaryAppendParams& p, cudaStream_t stream);

struct PagedAttentionParams {
  const uint8_t *k, *v;
  int64_t page_stride, slot_stride, head_stride;  // bytes
  const uint8_t* q;
  int64_t q_token, q_head;                        // bytes
  const int32_t* tables;
  int64_t table_stride;
  const int32_t* lengths;
  void* out;                                      // [batch, heads, dim]
  float* lse;                                     // [batch, heads] or null
  float* parts;                                   // partial results, two per worker
  int4* open;                                     // per worker: the item that it began and others end
  int32_t* status;
  uint32_t copy_limit;                            // nanoseconds that a copy of the kernel's own is waited for
  int64_t most_rows;                              // rows that a block table names
  float scale_log2;                               // softmax scale * log2(e)
  int32_t num_pages, page_shift, batch, kv_heads, group, head_tiles, dim, window, workers;  // workers of the first size
  bool aligned;                                   // rows are 16-byte aligned
  bool tall;                                      // pages of 32 rows or more
  bool two;                                       // there are workers of either size
  int32_t cluster;                                // 0: the chip shares all units; else blocks that take an item
};

// Which kernel a cache takes (paged_attention_variants.cuh).
struct PagedAttentionShape {
  int32_t bits;       // 16, 8, 4
  bool bf16;          // of q, the output and 16-bit rows
  int32_t dim;
  int32_t group;      // query heads per cached head
  bool fast;          // rows 16-byte aligned, 16 or more to a page
};
struct PagedAttentionPlan {
  int32_t unit;        // rows per unit
  int32_t tile_heads;  // query heads of a tile
  int32_t head_tiles;
  int32_t blocks;
  int32_t workers;
  size_t part_floats;  // of one partial result
};
PagedAttentionPlan plan_paged_attention(const PagedAttentionShape& s, int64_t sms);
// `split`: an item may be shared by workers, whose results are then joined by a second launch.
cudaError_t launch_paged_attention(const PagedAttentionShape& s, const PagedAttentionPlan& plan, const PagedAttentionParams& p,
                                   bool split, cudaStream_t stream);

}  // namespace fbgemm_b200
