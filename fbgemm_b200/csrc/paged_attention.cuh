// Attention of one new token per request over a paged cache:
//   o = sum_t p_t v_t,  p = softmax_t(scale q.k_t),  t over the rows that the token sees,
// for rows of 16-bit values or fused 8- and 4-bit rows (codes c_t, scale s_t and bias b_t), where
//   q.k_t = s_t (q.c_t) + b_t sum(q)   and   o = sum_t (p_t s_t) c_t + sum_t p_t b_t
// so that the codes themselves are multiplied and a row's scale and bias cost a few operations per score.
//
// Bound by memory: a cached row is read once and used for the `group` query heads that share it, 2 operations per byte
// and head.  That is too much for the fp32 units (8 heads on 4-bit rows: 200 TFLOP/s at the memory's rate) and little for
// the tensor units.  The large tensor instructions read shared memory, where codes would have to be written back as numbers
// first; the small ones take registers.  The rows are M and the heads N of m16n8k16: S^T = K Q^T takes 16 rows and 8 heads,
// O^T = V^T P^T 16 columns and 8 heads, nothing is padded at 8 heads.  P^T is turned to the second product's layout by movmatrix.
//
// At 44 GB/s per SM and a microsecond of latency about 44 KB have to be on their way to every SM all the time.  Each
// warp has a ring of half tiles (16 or 32 rows of K, or of V) in shared memory that it fills by asynchronous copies of
// its own, several ahead of the one it works on: 147 KB per SM at 128 columns.  (With the rows on their way to registers a
// warp had two half tiles in flight at most: 97 us for 64 requests of up to 8192 16-bit rows, 92 for 128 of up to 4096 4-bit
// rows.)  Pages of 16 rows and more hold all 16 rows of a step: one lane asks for a step by a tensor copy, whatever the strides (FAST;
// copies of 16 bytes by all lanes cost half of all instructions, 102 us for one request of 131072 16-bit rows);
// smaller pages and unaligned rows are copied in pieces of 16 or 4 bytes.  Rows that the token does not see are masked, in
// the tiles that have some.
//
// ldmatrix reads K without conflicts (16-bit rows are swizzled, quantized ones an odd multiple of 16 bytes apart), and
// turns V, for 16-bit values and for pairs of 8-bit and fours of 4-bit codes alike: a register holds the same columns of
// two rows, and their codes become two fp16 numbers by a mask or a byte permutation that puts them into the lowest
// bits: subnormal numbers, c 2^-24 (4-bit codes in the upper half of a byte, c 2^-20), which the products take exactly.
// The power of two is made up for once per score and result.  (The products align a subnormal as if its first bit were
// set: 4-bit codes in the lowest 4 bits cost 6 bits of the sums, and results that were off by 1e-3.)
//
// One pass with a running maximum and sum per head in fp32 (in registers, per warp).  A tile's largest score is looked
// for across lanes only if one exceeds the running maximum by more than 2^kSlack.  Weights are rounded to 16 bits for the
// second product: bf16 beside bf16 rows; fp16 otherwise (2^10 times as large, so that weights down to 2^-24 of the largest keep all 11
// bits), with the quantized rows' scales taken relative to the largest power of two seen so far.  Where that rounding is as coarse as
// the output's, what it leaves out enters as a second 16-bit number.  (Alone: errors against 64 bits of up to 1.55 times those of the
// output's rounding, 2.1e-3 for 1.7e-3 over 64 requests of up to 8192 bf16 rows.  The second number's products take 1 to 3 % of the
// time, 9 % over 128 requests of 1000 4-bit rows.)  Beside 16-bit rows the first is rounded towards zero, and the second is not 0 unless
// the weight is: so an infinite value stays one (no inf - inf, no 0 inf).  Beside quantized rows and a bf16 output, eight times as coarse
// as fp16 weights, codes are weighed about the middle of their range instead (sum w (c - 128) = sum w c - 128 sum w, with the rounded
// w), which keeps the weights' roundings to the values' own size (8-bit rows, 32 requests of up to 16384: 130 us, 135 with two numbers).
//
// Work is split over the chip by paged_cache.h's rule: a worker is a warp (or the HW warps that share rows), and nothing
// makes warps wait for one another, so that what a warp does between two items (its results out, the next queries in) is
// covered by the other warps of the SM; its ring runs on into the next item meanwhile.  (Blocks that joined their warps'
// results item by item took 77 us for 128 requests of 64 to 4096 4-bit rows.)  An item that several workers share is
// left as partial results, and a second launch (paged_attention_join) adds them up in a fixed order; a block whose workers
// all work on one item joins theirs first.  Short items are left to a block each, or to a cluster of two, four or eight that
// joins its results through distributed shared memory: one launch.
//
// Measured over 32 requests of 16384 rows of 8 heads of 128 columns: 16-bit rows 323 to 326 us, 6.6 TB/s, what a plain copy
// reaches.  8-bit rows 207 us, 0.84 of that rate, and 4-bit ones 141, 0.62 (beside fp16 queries 153): a tile is half or a
// quarter of the bytes and no fewer instructions (about 750 of a warp for 32 4-bit rows, three warps a scheduler, one instruction in two cycles),
// whose chain from the scores through the weights to the sums is what a tile takes.  Below some 100 us a fixed 15 us shows:
// 4 until the first rows are there, the slowest SM's 10 behind the mean one, and the join.
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cfloat>

#include "internal.h"
#include "paged_cache.h"

namespace fbgemm_b200 {

// The rows at `rows` (K's or V's) as a tensor [page][slot][head][columns] for copies of 16 rows of a head: 16-bit columns in
// swizzled boxes of 64, quantized rows as 4-byte words in boxes of `box`, whose end is filled with zeros, `height` rows high
// (paged_attention_dispatch.cu).
cudaError_t encode_rows(CUtensorMap* map, const uint8_t* rows, const PagedAttentionParams& p, bool swizzled, int box, int height,
                        int bits, int tail_bytes);

namespace paged {

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
constexpr uint32_t kLateCopy = 1000000;  // nanoseconds that a copy which is late gets once more
constexpr int kByItem = 6;  // workers to an item from which on the join goes by items

// A weight is exp2(score - maximum so far), at most 2^kSlack.  fp16 numbers are 2^10 times that, 2^14 at most, and with a scale of
// less than 2 below 2^15 (quantized rows: V's scales hold the power of two).  Sums over 2^31 rows of bf16's or fp32's largest values
// are to stay numbers until they are divided by the sum of the weights: bf16 weights are 2^-36 of it, and quantized rows' sums
// are kept times as much.
constexpr float kSlack = 4.f;
constexpr float kSmall = 1.f / 68719476736.f;  // 2^-36
template <typename S, bool BF16>
struct Weights {
  static constexpr float kWeight = BF16 ? kSmall : 1024.f;                          // beside 16-bit rows
  static constexpr float kResult = S::BITS == 16 ? 1.f / kWeight : 1.f / kSmall;    // of what the sums are divided by
};
constexpr float kFar = 1152921504606846976.f;  // 2^60
constexpr float kLn2 = 0.6931471805599453f;
constexpr unsigned kAll = 0xffffffffu;

// ---- instructions -----------------------------------------------------------------------------------------------------

template <bool BF16>
__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                    uint32_t b1) {
  if constexpr (BF16) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  } else {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
}

// An 8 x 8 matrix of 16-bit values, row i in lanes 4i .. 4i + 3, to its transpose.
__device__ __forceinline__ uint32_t transposed(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

__device__ __forceinline__ float exp2_of(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// a in the low half; towards zero if DOWN.
template <bool BF16, bool DOWN = false>
__device__ __forceinline__ uint32_t pack(float a, float b) {
  uint32_t r;
  if constexpr (BF16 && DOWN) {
    asm("cvt.rz.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
  } else if constexpr (BF16) {
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
  } else if constexpr (DOWN) {
    asm("cvt.rz.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
  } else {
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
  }
  return r;
}

// Four 8 x 8 matrices of 16-bit values; lane 8 i + j has the address of row j of matrix i.
__device__ __forceinline__ void load_matrices(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(at)
               : "memory");
}
__device__ __forceinline__ void load_turned(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(at)
               : "memory");
}

// 16 or 4 bytes to shared memory, past the first cache where that is possible; only `bytes` of them are read, zeros for the
// others.
__device__ __forceinline__ void copy16(uint32_t to, const uint8_t* from, uint32_t bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copy4(uint32_t to, const uint8_t* from, uint32_t bytes) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
}

// ---- tensor copies ----------------------------------------------------------------------------------------------------

__device__ __forceinline__ void barrier_init(uint32_t bar) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void barrier_expect(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool barrier_try(uint32_t bar, uint32_t parity) {
  uint32_t done;
  asm volatile("{\n.reg .pred p;\nmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\nselp.u32 %0, 1, 0, p;\n}"
               : "=r"(done)
               : "r"(bar), "r"(parity)
               : "memory");
  return done;
}
__device__ __forceinline__ uint64_t nanoseconds() {
  uint64_t t;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
  return t;
}
// Waits for a phase of the barrier, for `limit` nanoseconds at most.  False: it did not come.
__device__ __forceinline__ bool barrier_wait(uint32_t bar, uint32_t parity, uint32_t limit) {
  if (!barrier_try(bar, parity)) {
    const uint64_t since = nanoseconds();
    while (!barrier_try(bar, parity)) {
      if (nanoseconds() - since > limit) {
        return false;
      }
    }
  }
  return true;
}
__device__ __forceinline__ void copy_box(uint32_t to, const CUtensorMap* map, int column, int head, int slot, int page,
                                         uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(
          to),
      "l"(map), "r"(column), "r"(head), "r"(slot), "r"(page), "r"(bar)
      : "memory");
}

// ---- the blocks of a cluster --------------------------------------------------------------------------------------------

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release;\nbarrier.cluster.wait.acquire;" ::: "memory");
}
// Where block `rank` of the cluster has what lies at `at` here.
__device__ __forceinline__ uint32_t in_block(uint32_t at, int rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(at), "r"(rank));
  return r;
}
__device__ __forceinline__ float load_remote(uint32_t at) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ float4 load_remote4(uint32_t at) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(at) : "memory");
  return v;
}

// Nibbles i and i + 4 of a word as subnormal fp16, c 2^-20.  (The even ones by a product: the units for shifts and masks
// are the busier ones.)
__device__ __forceinline__ uint32_t nibbles(uint32_t w, int i) {
  const uint32_t x = i < 2 ? w : w >> 8;
  if (i % 2 == 1) {
    return x & 0x00f000f0u;
  }
  uint32_t r;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(x & 0x000f000fu), "r"(0x4c004c00u));  // times 16
  return r;
}

__device__ __forceinline__ float2 halves(uint32_t w) {
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}

// ---- what a kernel variant is -----------------------------------------------------------------------------------------

// BITS of a cached value, DP columns (dim rounded up to 64, 128 or 256), NT tiles of 8 query heads in a warp, HW warps that
// take further heads of the same rows.
template <int BITS_, int DP_, int NT_, int HW_>
struct Shape {
  static constexpr int BITS = BITS_, DP = DP_, NT = NT_, HW = HW_;
  static constexpr int kTail = BITS == 8 ? 8 : BITS == 4 ? 4 : 0;   // bytes of a row's scale and bias
  static constexpr int kPieces = (DP * BITS / 8 + kTail + 15) / 16; // 16-byte pieces of a row
  static constexpr int PITCH = (kPieces | 1) * 16;                  // between rows in shared memory (not swizzled ones)
  static constexpr int kBlocks16 = DP * BITS / 128;                 // 16-byte blocks of a row's columns
  static constexpr int SUB = PITCH > 144 ? 1 : 2;                   // 16-row steps of a tile
  static constexpr int ROWS = 16 * SUB;                             // of a warp's tile
  static constexpr bool kSwizzled = BITS == 16;                     // by tensor copies: boxes of 16 rows of 128 bytes
  static constexpr int kBoxes = kSwizzled ? DP / 64 : 1;            // of a step
  static constexpr int kBoxBytes = 16 * (kSwizzled ? 128 : PITCH);
  static constexpr bool kTall = SUB == 2 && kBoxes == 1;            // two steps' boxes may be one, of a page of 32 rows
  static constexpr int SLOT = ROWS * PITCH;                         // bytes of a half tile
  static constexpr int SLOT_FAST = SUB * kBoxes * kBoxBytes;
  static constexpr int UNIT = ROWS;
  static constexpr int kWorkers = kWarps / HW;                      // of a block
  static constexpr int KSTEPS = DP / 16;
  static constexpr int MT = DP / 16;                                // 16-column tiles of the output
  static constexpr int kWarpHeads = 8 * NT;
  static constexpr int kHeads = kWarpHeads * HW;
  static constexpr int kPartFloats = kHeads * (DP + 2);
  // Blocks of an SM by registers (output 4 NT MT, queries 2 NT KSTEPS, scores, and about 70 more), and ring slots of a warp
  // by shared memory.  (128 requests of up to 4096 4-bit rows, before the join went by workers there: 68 us with three blocks, 79
  // with two, 77 with four, whose registers do not suffice.)
  static constexpr int kRegisters = 4 * NT * MT + 2 * NT * KSTEPS + 4 * NT * SUB;
  static constexpr int kBlocks = kRegisters <= 90 ? 3 : 2;
  static constexpr int kFit = 222 * 1024 / (kBlocks * kWarps * SLOT);
  static constexpr int SLOTS = kFit > 6 ? 6 : kFit;
  static constexpr int kShared = kWarps * SLOTS * SLOT + 1024;      // (aligned for swizzled boxes)
  static_assert(SLOT >= SLOT_FAST, "one size for both");
  static_assert(SLOTS >= 3, "two half tiles on their way");
  static_assert(kWarps * SLOTS * SLOT_FAST >= (kWorkers + 1) * kPartFloats * 4, "results take the rings' place");
};

// ---- the kernel -------------------------------------------------------------------------------------------------------

// FAST: pages of 16 rows or more, rows 16-byte aligned, by tensor copies.
template <typename S, bool BF16, bool FAST>
__global__ void __launch_bounds__(kThreads, S::kBlocks)
paged_attention_kernel(const PagedAttentionParams p, const __grid_constant__ CUtensorMap k_map,
                       const __grid_constant__ CUtensorMap v_map) {
  constexpr int BITS = S::BITS, NT = S::NT, SUB = S::SUB;
  constexpr bool kQuantized = BITS != 16;
  constexpr bool kMmaBf16 = !kQuantized && BF16;
  constexpr bool kRest = !(kQuantized && BF16);   // weights enter with what their rounding leaves out
  constexpr bool kCentred = kQuantized && !kRest;
  constexpr float kMiddle = BITS == 8 ? 128.f : 8.f;
  constexpr float kWeight = Weights<S, BF16>::kWeight, kResult = Weights<S, BF16>::kResult;
  constexpr float kCode = BITS == 4 ? 1.f / 1048576.f : 1.f / 16777216.f;  // what a code of 1 is to the products
  constexpr unsigned kFull = S::ROWS == 32 ? kAll : (1u << (S::ROWS & 31)) - 1;
  constexpr int kSlot = FAST ? S::SLOT_FAST : S::SLOT;
  extern __shared__ __align__(1024) uint8_t smem_start[];
  uint8_t* const smem = smem_start + (-(uint32_t)__cvta_generic_to_shared(smem_start) & 1023);  // swizzled boxes: 1024 bytes
  __shared__ uint64_t sm_bars[kWarps][S::SLOTS];
  __shared__ unsigned sm_seen[kWarps][S::SLOTS];  // rows of a half tile that the token sees
  __shared__ int64_t sm_sums[kWarps];
  __shared__ int32_t sm_request[S::kWorkers];
  __shared__ int64_t sm_unit[S::kWorkers];

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c = lane & 3;
  const int head_warp = warp % S::HW;
  const int per_request = p.kv_heads * p.head_tiles;
  uint8_t* const ring = smem + warp * (S::SLOTS * kSlot);
  const uint32_t bars = (uint32_t)__cvta_generic_to_shared(&sm_bars[warp][0]);
  if (FAST && lane < S::SLOTS) {
    barrier_init(bars + 8 * lane);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (FAST && tid < 2) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(tid ? &v_map : &k_map) : "memory");
  }
  // The join may come to its SMs from here on; what it reads before it waits for this launch (the lengths) was there by now.
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  int left;                         // units still to be worked on
  int64_t last_unit = 0;
  UnitSplit split = {1, 0, 1};
  int64_t total = 0;
  const int worker = blockIdx.x * S::kWorkers + warp / S::HW;
  const int rank = p.cluster ? blockIdx.x % p.cluster : 0;  // of this block in its cluster
  int block_item = 0, block_active = S::kWorkers;           // the item of blocks that join their results, workers that have some
  if (p.cluster) {
    // -- a cluster of blocks takes an item, its workers equal shares of it
    const int at = blockIdx.x / p.cluster, request = at / per_request;
    const int units = units_of(span_of(p.lengths[request], p.window, p.most_rows), S::UNIT);
    const int workers = p.cluster * S::kWorkers, share = (units + workers - 1) / workers;
    const int first = share * (rank * S::kWorkers + warp / S::HW);
    left = max(min(share, units - first), 0);
    block_item = at - request * per_request;
    block_active = min(max((units - share * rank * S::kWorkers + share - 1) / share, 0), S::kWorkers);
    if (tid < S::kWorkers) {
      sm_request[tid] = request;
      sm_unit[tid] = (int64_t)block_item * units + min(share * (rank * S::kWorkers + tid), units - 1);
    }
    __syncthreads();
  } else {
    // -- the units of this block's workers, and the requests that their first ones belong to
    const int chunk = (p.batch + kThreads - 1) / kThreads;
    const int b0 = min(tid * chunk, p.batch), b1 = min(b0 + chunk, p.batch);
    auto units_of_request = [&](int b) {
      return (int64_t)units_of(span_of(p.lengths[b], p.window, p.most_rows), S::UNIT) * per_request;
    };
    int64_t sum = 0;
    for (int b = b0; b < b1; ++b) {
      sum += units_of_request(b);
    }
    int64_t before = sum;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int64_t up = __shfl_up_sync(kAll, before, d);
      before += lane >= d ? up : 0;
    }
    if (lane == 31) {
      sm_sums[warp] = before;
    }
    if (tid < S::kWorkers) {
      sm_request[tid] = 0;
      sm_unit[tid] = 0;
    }
    __syncthreads();
    before -= sum;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      before += w < warp ? sm_sums[w] : 0;
      total += sm_sums[w];
    }
    split = split_units(total, p.workers, p.two);
#pragma unroll
    for (int w = 0; w < S::kWorkers; ++w) {
      const int64_t first = split.first((int64_t)blockIdx.x * S::kWorkers + w);
      if (first >= before && first < before + sum) {
        int64_t from = before;
        for (int b = b0; b < b1; ++b) {
          const int64_t n = units_of_request(b);
          if (first < from + n) {
            sm_request[w] = b;
            sm_unit[w] = first - from;
            break;
          }
          from += n;
        }
      }
    }
    __syncthreads();
    const int64_t first_unit = split.first(worker);
    last_unit = min(first_unit + split.units_of(worker), total);
    left = (int)max(last_unit - first_unit, (int64_t)0);
  }

  const int row_bytes = p.dim * BITS / 8 + S::kTail;
  const uint32_t ring_at = (uint32_t)__cvta_generic_to_shared(ring);
  const uint32_t ring_end = ring_at + S::SLOTS * kSlot;
  // ldmatrix: K's matrices are rows 0 - 7 and 8 - 15 of a block of columns, then of the next; V's two blocks of rows 0 - 7,
  // then of 8 - 15.
  constexpr bool kSwizzled = FAST && S::kSwizzled;
  constexpr int kRow = kSwizzled ? 128 : S::PITCH;
  const uint32_t k_lane = ((lane & 7) + (lane & 8)) * kRow, k_odd = lane >> 4;
  const uint32_t v_lane = ((lane & 7) + ((lane >> 4) << 3)) * kRow, v_odd = (lane >> 3) & 1;
  const uint32_t tail_lane = g * S::PITCH + p.dim * BITS / 8;
  // (b even: this lane's block b or b + 1 of step s; in a swizzled box block x of row r is at x ^ (r % 8))
  auto matrix_at = [&](uint32_t half, uint32_t row, uint32_t odd, int s, int b) {
    if constexpr (kSwizzled) {
      return half + row + (s * S::kBoxes + b / 8) * S::kBoxBytes + ((((b % 8) | odd) ^ (lane & 7)) << 4);
    } else {
      return half + row + 16 * s * S::PITCH + 16 * (b + odd);
    }
  };

  // The ring: what is filled next and what is worked on.
  uint32_t fill_at = ring_at, at = ring_at;
  int fill_slot = 0, slot = 0;
  uint32_t phase = 0;
  bool lost = false;  // a copy did not come in time: the warp leaves

  // A place in the line of units: tile u of an item (a cached head and a tile of its query heads) of a request.
  struct Place {
    int request, item, u, units;
    RowSpan span;
  };
  auto enter = [&](Place& w, int request) {
    w.request = request;
    w.span = span_of(p.lengths[request], p.window, p.most_rows);
    w.units = units_of(w.span, S::UNIT);
  };
  auto next_item = [&](Place& w) {  // (the caller knows that there is one)
    w.u = 0;
    if (++w.item == per_request) {
      w.item = 0;
      enter(w, w.request + 1);
    }
  };
  Place now, ahead;
  enter(now, sm_request[warp / S::HW]);
  now.item = (int)(sm_unit[warp / S::HW] / now.units);
  now.u = (int)(sm_unit[warp / S::HW] - (int64_t)now.item * now.units);
  ahead = now;
  // Whether all of the block's units are of one item: it joins its results itself.
  bool together = false, block_begins = false, block_ends = false;
  if (p.cluster) {
    together = block_begins = block_ends = true;
  } else if constexpr (S::kWorkers > 1) {
    const BlockShare share = block_share(split, blockIdx.x, S::kWorkers, total);
    const int units = units_of(span_of(p.lengths[sm_request[0]], p.window, p.most_rows), S::UNIT);
    const int u = (int)(sm_unit[0] % units);
    together = share.active > 1 && u + share.units <= units;
    block_begins = u == 0;
    block_ends = u + share.units == units;
    block_item = (int)(sm_unit[0] / units);
    block_active = share.active;
  }

  // -- half tiles come in turn: K and V of a tile, then of the next.  SLOTS - 1 are on their way, and the pages of the tile
  // behind them.
  int to_read = left;           // tiles whose pages have not been read
  constexpr int kPages = FAST ? SUB : 1;
  int32_t page[kPages], page_next[kPages];  // FAST: every lane knows the pages of the steps, else those of its own row
  int row_fill = 0, row_next = aligned_first(ahead.span) + ahead.u * S::ROWS;  // the tile's first row
  int head_fill = 0, head_next = ahead.item / p.head_tiles, head_ahead = head_next;  // its cached head
  unsigned seen = 0, seen_next = 0;         // its rows that the token sees
  int request_next = 0;
  bool fill_more = false;
  int64_t off = 0;
  const int32_t* table = p.tables + ahead.request * p.table_stride;
  const int page_mask = (1 << p.page_shift) - 1;
  const bool tall = S::kTall && p.tall;
  int row_ahead = row_next;
  auto read_pages = [&] {
    if (to_read <= 0) {
      return;
    }
    const int row = row_ahead;
    row_next = row;
    head_next = head_ahead;
    request_next = ahead.request;
    seen_next = kFull;
    if (row < ahead.span.first) {  // (by less than 32)
      seen_next &= ~0u << (ahead.span.first - row);
    }
    if (ahead.span.end - row < S::ROWS) {
      seen_next &= ahead.span.end > row ? kFull >> (S::ROWS - (ahead.span.end - row)) : 0u;
    }
#pragma unroll
    for (int s = 0; s < kPages; ++s) {
      if (FAST && s > 0 && tall) {
        break;
      }
      const unsigned rows_of = FAST ? (tall ? seen_next : (seen_next >> (16 * s)) & 0xffffu)
                                    : (seen_next >> lane) & (lane < S::ROWS);  // that this page is needed for
      page_next[s] = rows_of ? __ldg(table + ((row + (FAST ? 16 * s : lane)) >> p.page_shift)) : 0;
    }
    row_ahead += S::ROWS;
    if (++ahead.u == ahead.units && to_read > 1) {
      next_item(ahead);
      head_ahead = ahead.item / p.head_tiles;
      row_ahead = aligned_first(ahead.span);
      table = p.tables + ahead.request * p.table_stride;
    }
  };
  auto report_page = [&](int request, int row, int32_t number) {
    if (atomicCAS(p.status, 0, FBGEMM_B200_STATUS_BAD_PAGE) == 0) {
      p.status[1] = request;
      p.status[2] = row;
      p.status[3] = number;
    }
  };
  auto next_tile = [&] {
    fill_more = to_read > 0;
    if (!fill_more) {
      return;
    }
    row_fill = row_next;
    head_fill = head_next;
    seen = seen_next;
#pragma unroll
    for (int s = 0; s < kPages; ++s) {
      page[s] = page_next[s];
    }
    if constexpr (FAST) {
      bool good = true;
      if (S::kTall && tall) {
        page[SUB - 1] = page[0];
      }
#pragma unroll
      for (int s = 0; s < SUB; ++s) {
        good = good && (uint32_t)page[s] < (uint32_t)p.num_pages;
      }
      if (!good) {
#pragma unroll
        for (int s = 0; s < SUB; ++s) {
          if ((uint32_t)page[s] >= (uint32_t)p.num_pages) {
            const unsigned lost = (seen >> (16 * s)) & 0xffffu;
            if (lane == 0 && lost) {
              report_page(request_next, row_fill + 16 * s + __ffs(lost) - 1, page[s]);
            }
            seen &= ~(0xffffu << (16 * s));
          }
        }
      }
    } else {
      const bool there = lane < S::ROWS && ((seen >> (lane & 31)) & 1);
      const bool good = there && (uint32_t)page[0] < (uint32_t)p.num_pages;
      if (there && !good) {
        report_page(request_next, row_fill + lane, page[0]);
      }
      seen = __ballot_sync(kAll, good);
      off = good ? page[0] * p.page_stride + ((row_fill + lane) & page_mask) * p.slot_stride : 0;
    }
    --to_read;
    read_pages();
  };
  auto fill = [&](bool is_v) {
    if (!is_v) {
      next_tile();
    }
    if (fill_more) {
      if (lane == 0 && !is_v) {
        sm_seen[warp][fill_slot] = seen;
      }
      if constexpr (FAST) {
        if (lane == 0) {
          const uint32_t bar = bars + 8 * fill_slot;
          const CUtensorMap* const map = is_v ? &v_map : &k_map;
          if (S::kTall && tall) {
            barrier_expect(bar, seen ? SUB * S::kBoxBytes : 0);
            if (seen) {
              copy_box(fill_at, map, 0, head_fill, row_fill & page_mask, page[0], bar);
            }
          } else {
            int steps = SUB;
            if (seen != kFull) {
              steps = 0;
#pragma unroll
              for (int s = 0; s < SUB; ++s) {
                steps += ((seen >> (16 * s)) & 0xffffu) != 0;
              }
            }
            barrier_expect(bar, steps * (S::kBoxes * S::kBoxBytes));
#pragma unroll
            for (int s = 0; s < SUB; ++s) {
              if ((seen >> (16 * s)) & 0xffffu) {
#pragma unroll
                for (int x = 0; x < S::kBoxes; ++x) {
                  copy_box(fill_at + (s * S::kBoxes + x) * S::kBoxBytes, map, 64 * x, head_fill, (row_fill + 16 * s) & page_mask,
                           page[s], bar);
                }
              }
            }
          }
        }
      } else {
        const uint8_t* const rows = (is_v ? p.v : p.k) + head_fill * p.head_stride;
        if (p.aligned) {
          constexpr int kRounds = (S::ROWS * S::kPieces + 31) / 32;
#pragma unroll 4
          for (int j = 0; j < kRounds; ++j) {
            const int n = lane + 32 * j, r = n / S::kPieces, piece = n - r * S::kPieces;
            const int64_t row = __shfl_sync(kAll, off, min(r, S::ROWS - 1));
            if (r < S::ROWS) {  // (zeros behind the row's end)
              const int bytes = (seen >> r) & 1 ? piece_bytes(row_bytes, piece) : 0;
              copy16(fill_at + r * S::PITCH + piece * 16, rows + row + (bytes ? piece * 16 : 0), bytes);
            }
          }
        } else if (lane < S::ROWS) {
          const uint32_t bytes = (seen >> lane) & 1 ? 4 : 0;
          for (int n = 0; n < row_bytes; n += 4) {
            copy4(fill_at + lane * S::PITCH + n, rows + off + n, bytes);
          }
        }
      }
      fill_at += kSlot;
      ++fill_slot;
      if (fill_at == ring_end) {
        fill_at = ring_at;
        fill_slot = 0;
      }
    }
    if constexpr (!FAST) {
      asm volatile("cp.async.commit_group;" ::: "memory");
    }
  };
  // The half tile that is worked on next is there, and the one before has been read by all lanes.  False: it did not come in
  // time, as far as this lane can tell.
  auto arrived = [&] {
    bool came = true;
    if constexpr (FAST) {
      came = barrier_wait(bars + 8 * slot, phase, p.copy_limit);
    } else {
      asm volatile("cp.async.wait_group %0;" ::"n"(S::SLOTS - 2) : "memory");
    }
    __syncwarp();
    return came;
  };
  // A half tile did not come in time, the one at `from` or one behind it.  No copy is asked for any more, so that no barrier is
  // armed again whose phase has not ended, and those that were asked for are waited for once more: one that comes up to
  // kLateCopy later still finds its memory there.
  auto give_up = [&](int from, uint32_t parity) {
    if (lane == 0 && atomicCAS(p.status, 0, FBGEMM_B200_STATUS_COPY_TIMEOUT) == 0) {
      p.status[1] = now.request;
      p.status[2] = p.status[3] = 0;
    }
    lost = true;
    fill_more = false;
    to_read = 0;
    do {  // (at least one, at most all)
      barrier_wait(bars + 8 * from, parity, kLateCopy);
      if (++from == S::SLOTS) {
        from = 0;
        parity ^= 1;
      }
    } while (from != fill_slot);
    __syncwarp();
  };
  read_pages();
#pragma unroll
  for (int h = 0; h < S::SLOTS - 1; ++h) {
    fill(h & 1);
  }
  int4 opened = make_int4(0, 0, 0, 0);
  const bool idle = left == 0;
  if (FAST && p.copy_limit == 0 && !idle) {
    give_up(slot, phase);
  }

  // -- item after item
  while (left > 0) {
    const int request = now.request, item = now.item;
    const bool begins = now.u == 0, ends = now.units - now.u <= left;
    const int tiles = lost ? 0 : ends ? now.units - now.u : left;
    const int kv_head = item / p.head_tiles, first_head = (item - kv_head * p.head_tiles) * S::kHeads + head_warp * S::kWarpHeads;
    const int heads = min(p.group - first_head, S::kWarpHeads);  // of this warp, may be none
    const int q_head0 = kv_head * p.group + first_head;
    if (begins && item == 0 && head_warp == 0 && lane == 0) {
      const int32_t length = p.lengths[request];
      if ((length < 0 || length > p.most_rows) && atomicCAS(p.status, 0, FBGEMM_B200_STATUS_SIZE_MISMATCH) == 0) {
        p.status[1] = request;
        p.status[2] = 0;
        p.status[3] = length;
      }
    }

    // -- queries as the products take them: head g of a tile in lanes 4g .. 4g + 3, columns in the order of K's registers.
    // Columns of 16 bits: 2c, 2c + 1 and 2c + 8, 2c + 9 of a step of 16.  8-bit codes: 4c .. 4c + 3 of a step.  4-bit codes:
    // 8c .. 8c + 7 of two steps.
    uint32_t qf[NT][S::KSTEPS][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int head = 8 * n + g;
      const bool there = head < heads;
      const uint8_t* q = p.q + request * p.q_token + (there ? q_head0 + head : 0) * p.q_head;
      if constexpr (BITS == 4) {
#pragma unroll
        for (int k = 0; k < S::KSTEPS; k += 2) {
          const int column = 16 * k + 8 * c;
          uint4 v = make_uint4(0, 0, 0, 0);
          if (there && column < p.dim) {
            v = *reinterpret_cast<const uint4*>(q + 2 * column);
          }
          qf[n][k][0] = v.x;
          qf[n][k][1] = v.y;
          qf[n][k + 1][0] = v.z;
          qf[n][k + 1][1] = v.w;
        }
      } else {
#pragma unroll
        for (int k = 0; k < S::KSTEPS; ++k) {
          const int column = 16 * k + (BITS == 16 ? 2 : 4) * c;
          qf[n][k][0] = qf[n][k][1] = 0;
          if (there && 16 * k < p.dim) {
            qf[n][k][0] = *reinterpret_cast<const uint32_t*>(q + 2 * column);
            qf[n][k][1] = *reinterpret_cast<const uint32_t*>(q + 2 * column + (BITS == 16 ? 16 : 4));
          }
        }
      }
    }

    float factor[NT][2], q_sum[NT][2];  // heads 2c and 2c + 1
    // Heads (a bit of 2 n + x each) of queries so large that their factor is no fp32 number: 2^-60 of it is kept, and their
    // scores are multiplied twice.
    unsigned far = 0;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float scale_head = 1.f, sum_head = 0.f;
      if constexpr (kQuantized) {
        // Beside fp16 codes the queries are fp16 too; bf16 ones may lie outside its range, so each head is moved by a power
        // of two.
        auto two = [&](uint32_t x) {
          return BF16 ? make_float2(__uint_as_float(x << 16), __uint_as_float(x & 0xffff0000u)) : halves(x);
        };
        float most = 0.f;
#pragma unroll
        for (int k = 0; k < S::KSTEPS; ++k) {
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const float2 f = two(qf[n][k][j]);
            most = fmaxf(most, fmaxf(fabsf(f.x), fabsf(f.y)));
          }
        }
        most = fmaxf(most, __shfl_xor_sync(kAll, most, 1));
        most = fmaxf(most, __shfl_xor_sync(kAll, most, 2));
        const int e = (int)(__float_as_uint(most) >> 23);  // 127 + exponent
        int move = e == 0 || e == 255 ? 0 : 137 - e;       // the largest comes to lie in [2^10, 2^11)
        move = min(move, 126);
        const float up = __uint_as_float((uint32_t)(127 + move) << 23);
        scale_head = __uint_as_float((uint32_t)(127 - move) << 23);
#pragma unroll
        for (int k = 0; k < S::KSTEPS; ++k) {
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const float2 f = two(qf[n][k][j]);
            const float x = __fmul_rn(f.x, up), y = __fmul_rn(f.y, up);
            sum_head += x + y;
            qf[n][k][j] = pack<false>(x, y);
          }
        }
        sum_head += __shfl_xor_sync(kAll, sum_head, 1);
        sum_head += __shfl_xor_sync(kAll, sum_head, 2);
      }
      if constexpr (BITS == 4) {
#pragma unroll
        for (int k = 0; k < S::KSTEPS; k += 2) {  // columns (0,4), (1,5) and (2,6), (3,7)
          const uint32_t w0 = qf[n][k][0], w1 = qf[n][k][1], w2 = qf[n][k + 1][0], w3 = qf[n][k + 1][1];
          qf[n][k][0] = __byte_perm(w0, w2, 0x5410);
          qf[n][k][1] = __byte_perm(w0, w2, 0x7632);
          qf[n][k + 1][0] = __byte_perm(w1, w3, 0x5410);
          qf[n][k + 1][1] = __byte_perm(w1, w3, 0x7632);
        }
      }
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int from = 4 * (2 * c + x);
        const float scale_x = __shfl_sync(kAll, scale_head, from);
        factor[n][x] = __fmul_rn(scale_x, p.scale_log2);
        if constexpr (kQuantized) {
          factor[n][x] = __fmul_rn(factor[n][x], 1.f / kCode);
          if (BF16 && isinf(factor[n][x])) {
            factor[n][x] = __fmul_rn(__fmul_rn(__fmul_rn(scale_x, 1.f / kFar), p.scale_log2), 1.f / kCode);
            far |= 1u << (2 * n + x);
          }
          q_sum[n][x] = __fmul_rn(__shfl_sync(kAll, sum_head, from), kCode);
        }
      }
    }

    const bool any_far = kQuantized && BF16 && __any_sync(kAll, far != 0);
    float o[NT][S::MT][4];
    // m: what weights are relative to, base = m, or 0 before the first; l: their sum over this lane's rows; of the rounded weights
    // w_sum (centred codes), of the weights times the rows' biases bias_sum
    float m[NT][2], base[NT][2], l[NT][2], w_sum[NT][2], bias_sum[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int i = 0; i < S::MT; ++i) {
        o[n][i][0] = o[n][i][1] = o[n][i][2] = o[n][i][3] = 0.f;
      }
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        m[n][x] = -INFINITY;
        base[n][x] = 0.f;
        l[n][x] = w_sum[n][x] = bias_sum[n][x] = 0.f;
      }
    }
    // V's scales are taken relative to 2^(exponent - 127) = 2^10 / v_unit, and are below scale_limit, twice that.
    int exponent = 11;
    float v_unit = __uint_as_float(253u << 23), scale_limit = __uint_as_float(12u << 23);

    auto advance = [&] {
      at += kSlot;
      ++slot;
      if (at == ring_end) {
        at = ring_at;
        slot = 0;
        phase ^= 1;
      }
    };
    auto tail_of = [&](uint32_t half, int s, int r) {
      const uint32_t from = half + tail_lane + (16 * s + 8 * r) * S::PITCH;
      if constexpr (BITS == 8) {
        float2 v;
        asm volatile("ld.shared.v2.f32 {%0,%1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(from) : "memory");
        return v;
      } else {
        uint32_t w;
        asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w) : "r"(from) : "memory");
        return halves(w);
      }
    };

    unsigned any_seen = 0;
    for (int i = 0; i < tiles; ++i) {
      // -- scores
      bool late = !arrived();
      fill(S::SLOTS % 2 == 0);  // (into the half before, which has come)
      float sc[NT][SUB][4];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int s = 0; s < SUB; ++s) {
          sc[n][s][0] = sc[n][s][1] = sc[n][s][2] = sc[n][s][3] = 0.f;
        }
      }
#pragma unroll
      for (int s = 0; s < SUB; ++s) {
#pragma unroll
        for (int b = 0; b < S::kBlocks16; b += 2) {
          uint32_t r[4];
          load_matrices(r, matrix_at(at, k_lane, k_odd, s, b));
          if constexpr (BITS == 16) {
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              mma<kMmaBf16>(sc[n][s], r[0], r[1], r[2], r[3], qf[n][b / 2][0], qf[n][b / 2][1]);
            }
          } else {
#pragma unroll
            for (int h = 0; h < 2; ++h) {  // r[2h]: block b + h of rows g, r[2h + 1]: of rows g + 8
              if constexpr (BITS == 8) {
                const uint32_t a0 = __byte_perm(r[2 * h], 0, 0x4140), a2 = __byte_perm(r[2 * h], 0, 0x4342);
                const uint32_t a1 = __byte_perm(r[2 * h + 1], 0, 0x4140), a3 = __byte_perm(r[2 * h + 1], 0, 0x4342);
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                  mma<false>(sc[n][s], a0, a1, a2, a3, qf[n][b + h][0], qf[n][b + h][1]);
                }
              } else {
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                  const uint32_t a0 = nibbles(r[2 * h], 2 * j), a2 = nibbles(r[2 * h], 2 * j + 1);
                  const uint32_t a1 = nibbles(r[2 * h + 1], 2 * j), a3 = nibbles(r[2 * h + 1], 2 * j + 1);
#pragma unroll
                  for (int n = 0; n < NT; ++n) {
                    mma<false>(sc[n][s], a0, a1, a2, a3, qf[n][2 * (b + h) + j][0], qf[n][2 * (b + h) + j][1]);
                  }
                }
              }
            }
          }
        }
      }
#pragma unroll
      for (int s = 0; s < SUB; ++s) {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const float2 sb = kQuantized ? tail_of(at, s, r) : make_float2(1.f, 0.f);
#pragma unroll
          for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              float& v = sc[n][s][2 * r + x];
              if constexpr (kQuantized) {
                v = __fmaf_rn(sb.x, v, __fmul_rn(sb.y, q_sum[n][x]));
              }
              v = __fmul_rn(v, factor[n][x]);
            }
          }
        }
      }
      if (any_far) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
          for (int s = 0; s < SUB; ++s) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              sc[n][s][j] = __fmul_rn(sc[n][s][j], (far >> (2 * n + j % 2)) & 1 ? kFar : 1.f);
            }
          }
        }
      }
      const unsigned rows_seen = sm_seen[warp][slot];
      any_seen |= rows_seen;
      if (rows_seen != kFull) {
#pragma unroll
        for (int s = 0; s < SUB; ++s) {
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const bool there = (rows_seen >> (16 * s + 8 * r + g)) & 1;
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              sc[n][s][2 * r] = there ? sc[n][s][2 * r] : -INFINITY;
              sc[n][s][2 * r + 1] = there ? sc[n][s][2 * r + 1] : -INFINITY;
            }
          }
        }
      }
      advance();

      // -- weights
      late |= !arrived();
      if (kSwizzled && rows_seen != kFull) {  // whatever else the page holds: weights of 0 do not make up for infinities
        for (int n = lane; n < S::SLOT_FAST / 16; n += 32) {
          const int row = (n / 8) % 16 + 16 * (n / (S::kBoxes * 128));
          if (!((rows_seen >> row) & 1)) {
            asm volatile("st.shared.v4.u32 [%0], {%1,%1,%1,%1};" ::"r"(at + 16 * n), "r"(0) : "memory");
          }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
      }
      bool more = FAST && late;
      float top[NT][2];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          top[n][x] = fmaxf(sc[n][0][x], sc[n][0][2 + x]);
#pragma unroll
          for (int s = 1; s < SUB; ++s) {
            top[n][x] = fmaxf(top[n][x], fmaxf(sc[n][s][x], sc[n][s][2 + x]));
          }
          more |= top[n][x] - m[n][x] > kSlack;  // (a difference of close numbers is exact)
        }
      }
      float2 v_sb[SUB][2];
      float largest = 0.f;
      if constexpr (kQuantized) {
#pragma unroll
        for (int s = 0; s < SUB; ++s) {
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            v_sb[s][r] = tail_of(at, s, r);
          }
        }
        if (rows_seen != kFull) {
#pragma unroll
          for (int s = 0; s < SUB; ++s) {
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              if (!((rows_seen >> (16 * s + 8 * r + g)) & 1)) {
                v_sb[s][r] = make_float2(0.f, 0.f);
              }
            }
          }
        }
#pragma unroll
        for (int s = 0; s < SUB; ++s) {
          largest = fmaxf(largest, fmaxf(fabsf(v_sb[s][0].x), fabsf(v_sb[s][1].x)));
        }
        more |= largest >= scale_limit;
      }
      if (__any_sync(kAll, more)) {
        if (FAST && __any_sync(kAll, late)) {  // (this tile's halves from K's on: V's is at `slot`)
          give_up(slot == 0 ? S::SLOTS - 1 : slot - 1, slot == 0 ? phase ^ 1 : phase);
          break;
        }
        float fade_scale = 1.f;
        if constexpr (kQuantized) {
          const int to = (int)min(__reduce_max_sync(kAll, __float_as_uint(largest) >> 23), 253u);
          if (to > exponent) {
            fade_scale = to - exponent > 126 ? 0.f : __uint_as_float((uint32_t)(127 - (to - exponent)) << 23);
            exponent = to;
            scale_limit = __uint_as_float((uint32_t)(exponent + 1) << 23);
            v_unit = __uint_as_float((uint32_t)(264 - exponent) << 23);
          }
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            float t = top[n][x];
            t = fmaxf(t, __shfl_xor_sync(kAll, t, 4));
            t = fmaxf(t, __shfl_xor_sync(kAll, t, 8));
            t = fmaxf(t, __shfl_xor_sync(kAll, t, 16));
            t = fmaxf(t, m[n][x]);
            const float b = t == -INFINITY ? 0.f : t;  // nothing seen yet: every weight is 0
            // (a largest score of +inf: inf - inf, so that the row becomes NaN as in the formula)
            const float fade = m[n][x] == t ? 1.f : exp2_of(m[n][x] - b);
            m[n][x] = t;
            base[n][x] = b;
            l[n][x] = __fmul_rn(l[n][x], fade);
            const float f = __fmul_rn(fade, fade_scale);
            if constexpr (kQuantized) {
              bias_sum[n][x] = __fmul_rn(bias_sum[n][x], fade);
              w_sum[n][x] = __fmul_rn(w_sum[n][x], f);
            }
#pragma unroll
            for (int k = 0; k < S::MT; ++k) {
              o[n][k][x] = __fmul_rn(o[n][k][x], f);
              o[n][k][2 + x] = __fmul_rn(o[n][k][2 + x], f);
            }
          }
        }
      }
      fill(S::SLOTS % 2 != 0);  // (into K's half, which has come, as that question has shown)
      uint32_t wt[NT][SUB][2], rest[NT][SUB][2];
#pragma unroll
      for (int s = 0; s < SUB; ++s) {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const float vs = kQuantized ? __fmul_rn(v_sb[s][r].x, v_unit) : 1.f;
          const float vb = __fmul_rn(kCentred ? __fmaf_rn(kMiddle, v_sb[s][r].x, v_sb[s][r].y) : v_sb[s][r].y, kSmall);
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            float e[2];
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              e[x] = exp2_of(sc[n][s][2 * r + x] - base[n][x]);
              l[n][x] += e[x];
              if constexpr (kQuantized) {
                bias_sum[n][x] = __fmaf_rn(e[x], vb, bias_sum[n][x]);
                e[x] = __fmul_rn(e[x], vs);
              } else {
                e[x] = __fmul_rn(e[x], kWeight);
              }
            }
            const uint32_t w = pack<kMmaBf16, !kQuantized>(e[0], e[1]);
            const float2 held = kMmaBf16 ? make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)) : halves(w);
            wt[n][s][r] = transposed(w);
            if constexpr (kRest) {
              uint32_t left_out = pack<kMmaBf16>(e[0] - held.x, e[1] - held.y);
              if constexpr (!kQuantized) {
                left_out |= __vminu2(w, 0x00010001u);  // (the last bit, where the weight is not 0)
              }
              rest[n][s][r] = transposed(left_out);
            } else {
              w_sum[n][0] += held.x;
              w_sum[n][1] += held.y;
            }
          }
        }
      }

      // -- the weighted sum
#pragma unroll
      for (int s = 0; s < SUB; ++s) {
#pragma unroll
        for (int b = 0; b < S::kBlocks16; b += 2) {
          uint32_t r[4];
          load_turned(r, matrix_at(at, v_lane, v_odd, s, b));
          if constexpr (BITS == 16) {
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              mma<kMmaBf16>(o[n][b / 2], r[0], r[1], r[2], r[3], wt[n][s][0], wt[n][s][1]);
              mma<kMmaBf16>(o[n][b / 2], r[0], r[1], r[2], r[3], rest[n][s][0], rest[n][s][1]);
            }
          } else {
#pragma unroll
            for (int h = 0; h < 2; ++h) {  // r[h]: block b + h of rows 2c, 2c + 1, r[2 + h]: of rows 2c + 8, 2c + 9
              if constexpr (BITS == 8) {
                const uint32_t a0 = r[h] & 0x00ff00ffu, a1 = __byte_perm(r[h], 0, 0x4341);
                const uint32_t a2 = r[2 + h] & 0x00ff00ffu, a3 = __byte_perm(r[2 + h], 0, 0x4341);
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                  mma<false>(o[n][b + h], a0, a1, a2, a3, wt[n][s][0], wt[n][s][1]);
                  if constexpr (kRest) {
                    mma<false>(o[n][b + h], a0, a1, a2, a3, rest[n][s][0], rest[n][s][1]);
                  }
                }
              } else {
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                  const uint32_t a0 = nibbles(r[h], 2 * j), a1 = nibbles(r[h], 2 * j + 1);
                  const uint32_t a2 = nibbles(r[2 + h], 2 * j), a3 = nibbles(r[2 + h], 2 * j + 1);
#pragma unroll
                  for (int n = 0; n < NT; ++n) {
                    mma<false>(o[n][2 * (b + h) + j], a0, a1, a2, a3, wt[n][s][0], wt[n][s][1]);
                    if constexpr (kRest) {
                      mma<false>(o[n][2 * (b + h) + j], a0, a1, a2, a3, rest[n][s][0], rest[n][s][1]);
                    }
                  }
                }
              }
            }
          }
        }
      }
      advance();
    }

    // -- this warp's result: whole, or a part of one.  No row at all, or none on a page of the cache: zeros, and -inf as the
    // maximum.  Rows whose scores are all -inf: 0 / 0, as in the formula; the lowest finite maximum tells other parts that there
    // are such.
    const bool none = any_seen == 0;
    float scale_l[NT][2], scale_o[NT][2], add_o[NT][2];
    const bool whole = begins && ends && !together;
    const float unit = kQuantized ? __uint_as_float((uint32_t)exponent << 23) : 1.f;  // 2^10 / v_unit
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        float sum_l = l[n][x], sum_b = bias_sum[n][x];
        if constexpr (kCentred) {
          sum_b = __fmaf_rn(__fmul_rn(__fmul_rn(w_sum[n][x], kSmall / 1024.f), unit), -kMiddle, sum_b);
        }
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) {
          sum_l += __shfl_xor_sync(kAll, sum_l, d);
          if constexpr (kQuantized) {
            sum_b += __shfl_xor_sync(kAll, sum_b, d);
          }
        }
        const float inv = !whole ? 1.f : none ? 0.f : __fdiv_rn(kResult, sum_l);
        scale_l[n][x] = sum_l;
        scale_o[n][x] = inv;
        add_o[n][x] = sum_b;
      }
    }
    float* const part = whole      ? nullptr
                        : together ? reinterpret_cast<float*>(smem) + (warp / S::HW) * S::kPartFloats
                                   : p.parts + (2 * (int64_t)worker + begins) * S::kPartFloats;
    if (together) {
      __syncthreads();  // (all rings have been read)
    }
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int h = 8 * n + 2 * c + x;
        if (h >= heads) {
          continue;
        }
        const int64_t row = (int64_t)request * p.kv_heads * p.group + q_head0 + h;
        const int in_part = head_warp * S::kWarpHeads + h;
        if (g == 0) {
          if (!whole) {
            part[in_part] = m[n][x] == -INFINITY && !none ? -FLT_MAX : m[n][x];
            part[S::kHeads + in_part] = scale_l[n][x];
          } else if (p.lse) {
            p.lse[row] = none ? -INFINITY : __fmaf_rn(base[n][x], kLn2, logf(scale_l[n][x]));
          }
        }
        uint16_t* const out = static_cast<uint16_t*>(p.out) + row * p.dim;
        float* const to = part + 2 * S::kHeads + in_part * S::DP;
#pragma unroll
        for (int t = 0; t < S::MT; ++t) {
          float a = o[n][t][x], b = o[n][t][2 + x];
          if constexpr (kQuantized) {
            a = __fmaf_rn(__fmul_rn(a, kSmall / 1024.f / kCode), unit, add_o[n][x]);
            b = __fmaf_rn(__fmul_rn(b, kSmall / 1024.f / kCode), unit, add_o[n][x]);
          }
          // 16-bit rows: columns g and g + 8 of a step of 16; quantized ones: two columns side by side
          const int column = BITS == 16 ? 16 * t + g : BITS == 8 ? 16 * t + 2 * g : 32 * (t / 2) + 4 * g + 2 * (t % 2);
          if (whole) {
            if (column < p.dim) {
              const uint32_t r = pack<BF16>(__fmul_rn(a, scale_o[n][x]), __fmul_rn(b, scale_o[n][x]));
              if constexpr (BITS == 16) {
                out[column] = (uint16_t)r;
                out[column + 8] = (uint16_t)(r >> 16);
              } else {
                *reinterpret_cast<uint32_t*>(out + column) = r;
              }
            }
          } else if constexpr (BITS == 16) {
            to[column] = a;
            to[column + 8] = b;
          } else {
            *reinterpret_cast<float2*>(to + column) = make_float2(a, b);
          }
        }
      }
    }
    if (begins && !ends && !(together && block_ends)) {  // others end what this worker began: it names them
      const int64_t last = last_unit - left + now.units - 1;
      opened = make_int4((int)(split.worker_of(last) - worker), request, item, 0);
    }
    left = lost ? 0 : left - tiles;
    if (left > 0) {
      next_item(now);
    }
  }
  if (p.open && head_warp == 0 && lane == 0) {
    p.open[worker] = opened;
  }
  if (together) {
    if (idle) {  // (it has met no barrier yet)
      __syncthreads();
    }
    __syncthreads();
    const int kv_head = block_item / p.head_tiles, first_head = (block_item - kv_head * p.head_tiles) * S::kHeads;
    const int heads = min(p.group - first_head, S::kHeads);
    const float* const parts = reinterpret_cast<const float*>(smem);
    auto results_out = [&](int h, int column, float4 v, float top, float sum_l) {
      const bool none = top == -INFINITY;
      const float inv = none ? 0.f : __fdiv_rn(kResult, sum_l);
      const int64_t row = ((int64_t)sm_request[0] * p.kv_heads + kv_head) * p.group + first_head + h;
      if (column < p.dim) {
        *reinterpret_cast<uint2*>(static_cast<uint8_t*>(p.out) + (row * p.dim + column) * 2) =
            make_uint2(pack<BF16>(__fmul_rn(v.x, inv), __fmul_rn(v.y, inv)),
                       pack<BF16>(__fmul_rn(v.z, inv), __fmul_rn(v.w, inv)));
      }
      if (column == 0 && p.lse) {
        p.lse[row] = none ? -INFINITY : __fmaf_rn(top, kLn2, logf(sum_l));
      }
    };
    const bool whole = block_begins && block_ends;
    // A part of an item goes to where the join looks for it, or to the end of the workers' results for the cluster's blocks.
    float* const part = p.cluster > 1 ? reinterpret_cast<float*>(smem) + S::kWorkers * S::kPartFloats
                                      : p.parts + (2 * (int64_t)blockIdx.x * S::kWorkers + block_begins) * S::kPartFloats;
    for (int n = tid; n < heads * (S::DP / 4); n += kThreads) {
      const int h = n / (S::DP / 4), column = n % (S::DP / 4) * 4;
      float top = -INFINITY;
      for (int w = 0; w < block_active; ++w) {
        top = fmaxf(top, parts[w * S::kPartFloats + h]);
      }
      const float from = top == -INFINITY ? 0.f : top;
      float sum_l = 0.f;
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int w = 0; w < block_active; ++w) {
        const float f = exp2_of(parts[w * S::kPartFloats + h] - from);
        const float4 x = *reinterpret_cast<const float4*>(parts + w * S::kPartFloats + 2 * S::kHeads + h * S::DP + column);
        sum_l = __fmaf_rn(f, parts[w * S::kPartFloats + S::kHeads + h], sum_l);
        v.x = __fmaf_rn(f, x.x, v.x);
        v.y = __fmaf_rn(f, x.y, v.y);
        v.z = __fmaf_rn(f, x.z, v.z);
        v.w = __fmaf_rn(f, x.w, v.w);
      }
      if (whole && p.cluster <= 1) {
        results_out(h, column, v, top, sum_l);
      } else {
        *reinterpret_cast<float4*>(part + 2 * S::kHeads + h * S::DP + column) = v;
        if (column == 0) {
          part[h] = top;
          part[S::kHeads + h] = sum_l;
        }
      }
    }
    if (p.cluster > 1) {  // the blocks' results, each block a share of the columns
      cluster_sync();
      const uint32_t mine = (uint32_t)__cvta_generic_to_shared(part);
      for (int n = tid + rank * kThreads; n < heads * (S::DP / 4); n += p.cluster * kThreads) {
        const int h = n / (S::DP / 4), column = n % (S::DP / 4) * 4;
        float top = -INFINITY;
        for (int r = 0; r < p.cluster; ++r) {
          top = fmaxf(top, load_remote(in_block(mine + 4 * h, r)));
        }
        const float from = top == -INFINITY ? 0.f : top;
        float sum_l = 0.f;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int r = 0; r < p.cluster; ++r) {
          const float f = exp2_of(load_remote(in_block(mine + 4 * h, r)) - from);
          const float4 x = load_remote4(in_block(mine + 4 * (2 * S::kHeads + h * S::DP + column), r));
          sum_l = __fmaf_rn(f, load_remote(in_block(mine + 4 * (S::kHeads + h), r)), sum_l);
          v.x = __fmaf_rn(f, x.x, v.x);
          v.y = __fmaf_rn(f, x.y, v.y);
          v.z = __fmaf_rn(f, x.z, v.z);
          v.w = __fmaf_rn(f, x.w, v.w);
        }
        results_out(h, column, v, top, sum_l);
      }
      cluster_sync();  // (a block's memory is there until all have read it)
    }
    if (!whole) {  // the other workers' parts: nothing
      for (int n = tid; n < (block_active - 1) * S::kHeads; n += kThreads) {
        float* const other = p.parts + 2 * ((int64_t)blockIdx.x * S::kWorkers + 1 + n / S::kHeads) * S::kPartFloats;
        other[n % S::kHeads] = -INFINITY;
        other[S::kHeads + n % S::kHeads] = 0.f;
      }
    }
  }
}

// Adds up the parts of items that several workers share, in their order: a block takes a few heads of an item, TEAM warps a
// head.  BY_ITEM: block x takes item x, whose workers follow from the lengths as in the kernel before (few items, many
// workers each: 4 us for one request of 131072 rows of four heads; a pass over all workers' records took 38).
// Otherwise block x takes the item that worker x began, if others end it: no scan of the lengths and no block for whole items.
// (By item from six workers an item on: 128 requests of 1000 4-bit rows, under two workers an item, 55 us by item, 48 by
// worker; 36 of 8-bit rows, five an item, 28.7 and 26; 32 of 16384 rows, seven an item, 150.0 and 150.7.)
template <typename S, bool BF16, bool BY_ITEM, int TEAM>
__global__ void __launch_bounds__(kThreads) paged_attention_join(const PagedAttentionParams p) {
  constexpr int kTeams = kWarps / TEAM, kCols = S::DP / 32;
  __shared__ float sm_o[kTeams][TEAM][S::DP];
  __shared__ float sm_m[kTeams][TEAM], sm_l[kTeams][TEAM];
  __shared__ int64_t sm_sums[2][kWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, team = warp / TEAM, mate = warp % TEAM;
  int worker = blockIdx.x, n, request, item;
  if constexpr (BY_ITEM) {
    // (the lengths are not the kernel's before: they were there when it began)
    const int per_request = p.kv_heads * p.head_tiles;
    request = blockIdx.x / per_request;
    item = blockIdx.x - request * per_request;
    int64_t before = 0, total = 0;
    for (int b = threadIdx.x; b < p.batch; b += kThreads) {
      const int64_t units = units_of(span_of(p.lengths[b], p.window, p.most_rows), S::UNIT);
      total += units;
      before += b < request ? units : 0;
    }
    const int64_t units = units_of(span_of(p.lengths[request], p.window, p.most_rows), S::UNIT);
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) {
      total += __shfl_xor_sync(kAll, total, d);
      before += __shfl_xor_sync(kAll, before, d);
    }
    if (lane == 0) {
      sm_sums[0][warp] = total;
      sm_sums[1][warp] = before;
    }
    __syncthreads();
    total = before = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      total += sm_sums[0][w] * per_request;
      before += sm_sums[1][w] * per_request;
    }
    const UnitSplit split = split_units(total, p.workers, p.two);
    const int64_t start = before + item * units, end = start + units;
    worker = (int)split.worker_of(start);
    n = (int)split.worker_of(end - 1) - worker + 1;
    const int block = worker / S::kWorkers * S::kWorkers;
    if (start == split.first(block) && end == min(split.first(block) + S::kWorkers * split.units_of(block), total)) {
      n = 1;  // the whole of what a block had, and joined
    }
    asm volatile("griddepcontrol.wait;" ::: "memory");  // (by every block: none of this launch ends before the other)
  } else {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int4 opened = p.open[worker];
    n = opened.x + 1;
    request = opened.y;
    item = opened.z;
  }
  if (n == 1) {
    return;
  }
  const int kv_head = item / p.head_tiles, first_head = (item - kv_head * p.head_tiles) * S::kHeads;
  const int heads = min(p.group - first_head, S::kHeads);
  auto part_of = [&](int i) {  // what the worker began, then what the next ones ended
    return p.parts + (2 * ((int64_t)worker + i) + (i == 0)) * S::kPartFloats;
  };
  for (int h0 = blockIdx.y * kTeams; h0 < heads; h0 += gridDim.y * kTeams) {
    const int h = h0 + team;
    float v[kCols], sum_l = 0.f, top = -INFINITY;
#pragma unroll
    for (int j = 0; j < kCols; ++j) {
      v[j] = 0.f;
    }
    for (int i0 = mate * 32; h < heads && i0 < n; i0 += TEAM * 32) {  // 32 parts at a time, each lane one's maximum and sum
      const int i = i0 + lane;
      float m = -INFINITY, l = 0.f;
      if (i < n) {
        m = part_of(i)[h];
        l = part_of(i)[S::kHeads + h];
      }
      float t = m;
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) {
        t = fmaxf(t, __shfl_xor_sync(kAll, t, d));
      }
      t = fmaxf(t, top);
      const float base = t == -INFINITY ? 0.f : t;
      const float fade = top == t ? 1.f : exp2_of(top - base);
      top = t;
      const float f = exp2_of(m - base);
      sum_l = __fmul_rn(sum_l, fade);
#pragma unroll
      for (int j = 0; j < kCols; ++j) {
        v[j] = __fmul_rn(v[j], fade);
      }
      // (joined in their block: nothing is left in the others' parts)
      unsigned todo = __ballot_sync(kAll, i < n && !(m == -INFINITY && l == 0.f));
      while (todo) {
        float2 x[4][kCols / 2];
        float fs[4], ls[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int from = todo ? __ffs(todo) - 1 : -1;
          todo &= todo - 1;
          fs[k] = from < 0 ? 0.f : __shfl_sync(kAll, f, from & 31);
          ls[k] = from < 0 ? 0.f : __shfl_sync(kAll, l, from & 31);
#pragma unroll
          for (int j = 0; j < kCols / 2; ++j) {
            x[k][j] = make_float2(0.f, 0.f);
            if (from >= 0) {
              x[k][j] = *reinterpret_cast<const float2*>(part_of(i0 + from) + 2 * S::kHeads + h * S::DP + 64 * j + 2 * lane);
            }
          }
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          sum_l = __fmaf_rn(fs[k], ls[k], sum_l);
#pragma unroll
          for (int j = 0; j < kCols / 2; ++j) {
            v[2 * j] = __fmaf_rn(fs[k], x[k][j].x, v[2 * j]);
            v[2 * j + 1] = __fmaf_rn(fs[k], x[k][j].y, v[2 * j + 1]);
          }
        }
      }
    }
    if constexpr (TEAM > 1) {
      if (lane == 0) {
        sm_m[team][mate] = top;
        sm_l[team][mate] = sum_l;
      }
#pragma unroll
      for (int j = 0; j < kCols; j += 2) {
        *reinterpret_cast<float2*>(&sm_o[team][mate][32 * j + 2 * lane]) = make_float2(v[j], v[j + 1]);
      }
      __syncthreads();
    }
    if (h < heads && mate == 0) {
      if constexpr (TEAM > 1) {
        float all = top;
#pragma unroll
        for (int w = 1; w < TEAM; ++w) {
          all = fmaxf(all, sm_m[team][w]);
        }
        const float base = all == -INFINITY ? 0.f : all;
        const float own = exp2_of(top - base);
        sum_l = __fmul_rn(sum_l, own);
#pragma unroll
        for (int j = 0; j < kCols; ++j) {
          v[j] = __fmul_rn(v[j], own);
        }
#pragma unroll
        for (int w = 1; w < TEAM; ++w) {
          const float f = exp2_of(sm_m[team][w] - base);
          sum_l = __fmaf_rn(f, sm_l[team][w], sum_l);
#pragma unroll
          for (int j = 0; j < kCols; j += 2) {
            const float2 x = *reinterpret_cast<const float2*>(&sm_o[team][w][32 * j + 2 * lane]);
            v[j] = __fmaf_rn(f, x.x, v[j]);
            v[j + 1] = __fmaf_rn(f, x.y, v[j + 1]);
          }
        }
        top = all;
      }
      const int64_t row = ((int64_t)request * p.kv_heads + kv_head) * p.group + first_head + h;
      const float inv = top == -INFINITY ? 0.f : __fdiv_rn(Weights<S, BF16>::kResult, sum_l);  // (no row on a page of the cache: zeros)
#pragma unroll
      for (int j = 0; j < kCols; j += 2) {
        const int column = 32 * j + 2 * lane;
        if (column < p.dim) {
          *reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(p.out) + (row * p.dim + column) * 2) =
              pack<BF16>(__fmul_rn(v[j], inv), __fmul_rn(v[j + 1], inv));
        }
      }
      if (lane == 0 && p.lse) {
        p.lse[row] = __fmaf_rn(top == -INFINITY ? 0.f : top, kLn2, logf(sum_l));
      }
    }
    if constexpr (TEAM > 1) {
      __syncthreads();
    }
  }
}

// ---- launches ---------------------------------------------------------------------------------------------------------

template <typename S>
PagedAttentionPlan plan_of(int group, int64_t sms) {
  PagedAttentionPlan r;
  r.unit = S::UNIT;
  r.tile_heads = S::kHeads;
  r.head_tiles = (group + S::kHeads - 1) / S::kHeads;
  r.blocks = (int32_t)(sms * S::kBlocks);
  r.workers = r.blocks * S::kWorkers;
  r.part_floats = S::kPartFloats;
  return r;
}

// Sets attributes of a kernel once per device.
template <typename F>
cudaError_t once_per_device(std::atomic<uint64_t>& done, F&& set) {
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  const uint64_t bit = 1ull << (device & 63);
  if (e == cudaSuccess && (device > 63 || !(done.load(std::memory_order_relaxed) & bit))) {
    e = set();
    if (e == cudaSuccess) {
      done.fetch_or(bit, std::memory_order_relaxed);
    }
  }
  return e;
}
template <typename Kernel>
cudaError_t prefer_shared(Kernel kernel, std::atomic<uint64_t>& done) {
  return once_per_device(done, [=] {
    return cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
  });
}
// (More than 48 KB have to be asked for.)
template <typename Kernel>
cudaError_t allow_shared(Kernel kernel, int bytes, std::atomic<uint64_t>& done) {
  return once_per_device(done, [=] {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
    return e != cudaSuccess ? e : cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  });
}

template <typename S, bool BF16, bool FAST>
cudaError_t launch_of(const PagedAttentionPlan& plan, const PagedAttentionParams& p, bool split, cudaStream_t stream) {
  static std::atomic<uint64_t> asked{0};
  cudaError_t e = allow_shared(paged_attention_kernel<S, BF16, FAST>, S::kShared, asked);
  CUtensorMap maps[2] = {};
  if (FAST && e == cudaSuccess) {
    for (int i = 0; i < 2 && e == cudaSuccess; ++i) {
      e = encode_rows(&maps[i], i ? p.v : p.k, p, S::kSwizzled, S::kSwizzled ? 64 : S::PITCH / 4, S::kTall && p.tall ? 32 : 16,
                      S::BITS, S::kTail);
    }
  }
  if (e != cudaSuccess) {
    return e;
  }
  // Blocks come to their SM while the launch before ends, and wait there for its results.
  cudaLaunchAttribute attrs[2];
  attrs[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attrs[0].val.programmaticStreamSerializationAllowed = 1;
  attrs[1].id = cudaLaunchAttributeClusterDimension;
  attrs[1].val.clusterDim.x = (unsigned)p.cluster;
  attrs[1].val.clusterDim.y = attrs[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3((unsigned)(p.cluster ? (int64_t)p.batch * p.kv_heads * p.head_tiles * p.cluster
                                   : p.two   ? 2 * plan.blocks
                                             : plan.blocks));
  config.blockDim = dim3(kThreads);
  config.dynamicSmemBytes = S::kShared;
  config.stream = stream;
  config.attrs = attrs;
  config.numAttrs = p.cluster > 1 ? 2 : 1;
  e = cudaLaunchKernelEx(&config, paged_attention_kernel<S, BF16, FAST>, p, maps[0], maps[1]);
  g_launch_count.fetch_add(1, std::memory_order_relaxed);
  if (e != cudaSuccess || !split) {
    return e;
  }
  const int64_t items = (int64_t)p.batch * p.kv_heads * p.head_tiles;
  config.dynamicSmemBytes = 0;
  config.numAttrs = 1;
  // (all kernels with the same share of the SM for shared memory: it is not changed between them)
  if (items * kByItem <= plan.workers) {
    config.gridDim = dim3((unsigned)items, (unsigned)(p.group < S::kHeads ? p.group : S::kHeads));
    static std::atomic<uint64_t> known{0};
    e = prefer_shared(paged_attention_join<S, BF16, true, kWarps>, known);
    if (e == cudaSuccess) {
      e = cudaLaunchKernelEx(&config, paged_attention_join<S, BF16, true, kWarps>, p);
    }
  } else {
    config.gridDim = dim3((unsigned)(p.two ? 2 * plan.workers : plan.workers), (unsigned)(S::kHeads / 8));
    static std::atomic<uint64_t> known{0};
    e = prefer_shared(paged_attention_join<S, BF16, false, 1>, known);
    if (e == cudaSuccess) {
      e = cudaLaunchKernelEx(&config, paged_attention_join<S, BF16, false, 1>, p);
    }
  }
  g_launch_count.fetch_add(1, std::memory_order_relaxed);
  return e;
}

}  // namespace paged
}  // namespace fbgemm_b200
