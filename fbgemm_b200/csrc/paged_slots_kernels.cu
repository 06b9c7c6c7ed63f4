// Block tables and slot maps of a step, from the requests' lengths: request b holds L_b rows of a paged cache and gets
// n_b more.  With pages of P rows it needs ceil((L_b + n_b) / P) - ceil(L_b / P) fresh pages, which come from the top of
// a stack of free ones, requests in order; new row t of request b goes to slot table[b][t / P] * P + t % P.
//
// All or nothing: if the stack, a table's columns or the maps' capacity run out, nothing is given out (every slot is -1)
// and the first request that does not fit is recorded.
//
// One launch, bound by its latency: a few kilobytes are read and 16 bytes written per row.  Every block scans the
// requests' counts itself into shared memory (8 bytes a request; a scan of its own launch costs more than reading them
// again from L2) and then fills its stretch of the maps, each row finding its request by bisection.  What a block reads
// no block writes: fresh pages are looked up in the stack, not in the table that they are being written to.  256 requests
// of one new row take 3.7 us, 71 thousand rows of 64 requests 5.4, of which their bytes would take 0.2: the launch, the scan's
// reads and barriers, the bisection and the reads of length and page behind it, one after the other.
#include "internal.h"
#include "paged_cache.h"

namespace fbgemm_b200 {

namespace {

constexpr int kThreads = 512;
constexpr int kRowsPerBlock = 4 * kThreads;

// Exclusive sums of two values per thread across the block; totals to *ta, *tb.
__device__ __forceinline__ void block_exclusive_sums(int64_t& a, int64_t& b, int64_t* ta, int64_t* tb) {
  __shared__ int64_t sums[2][kThreads / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int64_t ia = a, ib = b;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int64_t ua = __shfl_up_sync(0xffffffffu, ia, d), ub = __shfl_up_sync(0xffffffffu, ib, d);
    if (lane >= d) {
      ia += ua;
      ib += ub;
    }
  }
  if (lane == 31) {
    sums[0][warp] = ia;
    sums[1][warp] = ib;
  }
  __syncthreads();
  int64_t before_a = 0, before_b = 0, all_a = 0, all_b = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) {
    const int64_t sa = sums[0][w], sb = sums[1][w];
    if (w < warp) {
      before_a += sa;
      before_b += sb;
    }
    all_a += sa;
    all_b += sb;
  }
  a = before_a + ia - a;
  b = before_b + ib - b;
  *ta = all_a;
  *tb = all_b;
}

struct Counts {
  int64_t length, fresh;  // rows in the cache, rows to come
  int64_t have, want;     // pages of either
};
__device__ __forceinline__ Counts counts_of(const PagedSlotsParams& p, int b) {
  Counts c;
  c.length = max(p.lengths[b], 0);
  c.fresh = max(p.fresh[b], 0);
  const int64_t up = ((int64_t)1 << p.page_shift) - 1;
  c.have = (c.length + up) >> p.page_shift;
  c.want = (c.length + c.fresh + up) >> p.page_shift;
  return c;
}

__global__ void __launch_bounds__(kThreads) paged_slots_kernel(const PagedSlotsParams p) {
  extern __shared__ int32_t smem[];
  int32_t* const start = smem;               // [batch + 1] first row of each request in the maps
  int32_t* const taken = smem + p.batch + 1; // [batch] pages that the requests before take
  __shared__ int bad;
  const int tid = threadIdx.x;
  if (tid == 0) {
    bad = 0x7fffffff;
  }
  const int chunk = (p.batch + kThreads - 1) / kThreads;
  const int b0 = min(tid * chunk, p.batch), b1 = min(b0 + chunk, p.batch);
  int64_t pages = 0, rows = 0;
  for (int b = b0; b < b1; ++b) {
    const Counts c = counts_of(p, b);
    pages += c.want - c.have;
    rows += c.fresh;
  }
  int64_t all_pages, all_rows;
  block_exclusive_sums(pages, rows, &all_pages, &all_rows);
  const int32_t num_free = *p.num_free;
  const int64_t at_hand = num_free < 0 || num_free > p.free_capacity ? -1 : num_free;  // -1: not the height of this stack
  for (int b = b0; b < b1; ++b) {
    const Counts c = counts_of(p, b);
    start[b] = (int32_t)rows;   // (read only if all rows fit into the capacity)
    taken[b] = (int32_t)pages;
    pages += c.want - c.have;
    rows += c.fresh;
    if (pages > at_hand || rows > p.capacity || c.want > p.width) {
      atomicMin(&bad, b);
      break;
    }
  }
  if (tid == 0) {
    start[p.batch] = (int32_t)all_rows;
  }
  __syncthreads();
  const bool fits = bad == 0x7fffffff;

  if (blockIdx.x == 0) {
    for (int b = tid; b < p.batch; b += kThreads) {
      p.offsets[b] = fits ? start[b] : 0;
      p.lengths_out[b] = fits ? (int32_t)(counts_of(p, b).length + counts_of(p, b).fresh) : p.lengths[b];
    }
    if (tid == 0) {
      p.offsets[p.batch] = fits ? start[p.batch] : 0;
      *p.num_free_out = fits ? (int32_t)(num_free - all_pages) : num_free;
      if (!fits && atomicCAS(p.status, 0, FBGEMM_B200_STATUS_NO_PAGES) == 0) {
        const Counts c = counts_of(p, bad);
        p.status[1] = bad;
        p.status[2] = (int32_t)min(c.length + c.fresh, (int64_t)0x7fffffff);
        p.status[3] = num_free;
      }
    }
  }

  const int64_t row0 = (int64_t)blockIdx.x * kRowsPerBlock;
#pragma unroll
  for (int i = 0; i < kRowsPerBlock / kThreads; ++i) {
    const int64_t at = row0 + tid + i * kThreads;
    if (at >= p.capacity) {
      break;
    }
    const int32_t r = (int32_t)at;
    int64_t slot = -1;
    int32_t position = 0, request = -1;
    if (fits && r < all_rows) {
      int lo = 0, hi = p.batch - 1;  // the last request that starts at or before row r; the ones after it that are empty start behind r
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (start[mid] <= r) {
          lo = mid;
        } else {
          hi = mid - 1;
        }
      }
      request = lo;
      const Counts c = counts_of(p, lo);
      position = (int32_t)(c.length + (r - start[lo]));
      const int page_at = position >> p.page_shift, within = position & ((1 << p.page_shift) - 1);
      int32_t* const entry = p.tables + lo * p.table_stride + page_at;
      int32_t page;
      if (page_at >= c.have) {
        page = p.free_pages[num_free - 1 - (taken[lo] + (page_at - c.have))];
        if (within == 0) {
          *entry = page;
        }
      } else {
        page = *entry;
      }
      if (page >= 0) {
        slot = ((int64_t)page << p.page_shift) + within;
      }
    }
    p.slots[r] = slot;
    p.positions[r] = position;
    p.requests[r] = request;
  }
}

}  // namespace

cudaError_t launch_paged_slots(const PagedSlotsParams& p, cudaStream_t stream) {
  const int64_t blocks = p.capacity > kRowsPerBlock ? ((int64_t)p.capacity + kRowsPerBlock - 1) / kRowsPerBlock : 1;
  const int smem = (2 * p.batch + 1) * 4;
  if (smem > 40 * 1024) {  // (always to the most there can be: calls from several threads would undercut each other)
    constexpr int kMost = (2 * FBGEMM_B200_PAGED_MAX_BATCH + 1) * 4;
    const cudaError_t e = cudaFuncSetAttribute(paged_slots_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMost);
    if (e != cudaSuccess) {
      return e;
    }
  }
  paged_slots_kernel<<<(unsigned)blocks, kThreads, smem, stream>>>(p);
  g_launch_count.fetch_add(1, std::memory_order_relaxed);
  return cudaGetLastError();
}

}  // namespace fbgemm_b200
