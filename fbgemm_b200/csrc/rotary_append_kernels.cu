// Rotary positions, and the new rows' way into the paged cache: of every token, each query and key head is turned pair
// by pair, (a, b) -> (a cos - b sin, b cos + a sin), pair i by the angle of the position on the axis that i belongs to
// (time, height and width of a picture's tokens; text has one axis).  Turned queries go out in their own type; keys and values
// go to row slots[t] of the cache, rounded once: to 16 bits, or as fused 8- or 4-bit rows with the codes, scale and
// bias that the row-wise quantizers (row_coder.cuh) give for the same fp32 row, byte for byte.  A slot of -1 is a row of
// padding: nothing is stored for it.
//
// Bound by memory: every value is read once and written once.  A group of 4, 8 or 16 lanes takes a head; each lane
// holds 16 of its values, two chunks of 16 bytes that contain both ends of every pair (half a head apart, or next to
// each other), so that turning needs no exchange and a row's minimum and maximum two to four.  A token's heads share the
// lanes' cosines and sines, which are read once per block.
#include <cuda_bf16.h>

#include "internal.h"
#include "paged_cache.h"
#include "row_coder.cuh"

namespace fbgemm_b200 {

namespace {

constexpr int kThreads = 128;

struct Half16 {
  using type = __half;
  static __device__ __forceinline__ float2 wide(uint32_t v) {
    return __half22float2(*reinterpret_cast<const __half2*>(&v));
  }
  static __device__ __forceinline__ uint32_t narrow(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
};
struct Bf16 {
  using type = __nv_bfloat16;
  static __device__ __forceinline__ float2 wide(uint32_t v) {
    return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
  }
  static __device__ __forceinline__ uint32_t narrow(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
};

template <typename T>
__device__ __forceinline__ void load8(float* x, const uint8_t* p) {
  const uint4 v = *reinterpret_cast<const uint4*>(p);
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = T::wide(w[i]);
    x[2 * i] = f.x;
    x[2 * i + 1] = f.y;
  }
}
template <typename T>
__device__ __forceinline__ void store8(uint8_t* p, const float* x) {
  *reinterpret_cast<uint4*>(p) =
      make_uint4(T::narrow(x[0], x[1]), T::narrow(x[2], x[3]), T::narrow(x[4], x[5]), T::narrow(x[6], x[7]));
}

// Block x: a token; block y: a share of its heads (queries, then keys, then values).
template <typename T, int BITS, int LANES>
__global__ void __launch_bounds__(kThreads) rotary_append_kernel(const RotaryAppendParams p) {
  const int64_t t = blockIdx.x;
  const int lane = threadIdx.x % LANES;
  const bool active = lane * 16 < p.dim;
  const int chunks = p.rot / 16;  // chunks of eight in half of the turned part
  const bool turns = p.cos_sin != nullptr && lane < chunks;
  const int c0 = lane < chunks ? lane : 2 * lane;                   // (2 * chunks + 2 * (lane - chunks))
  const int c1 = lane < chunks ? lane + chunks : 2 * lane + 1;

  const int64_t slot = p.slots[t];
  bool keep = slot >= 0 && slot < p.num_slots;
  bool known = true;
  float cosine[8], sine[8];
  if (p.cos_sin != nullptr) {
    int32_t position[4];
    int64_t outside = 0;
#pragma unroll
    for (int a = 0; a < 4; ++a) {
      position[a] = a < p.axes ? p.positions[a * p.positions_stride + t] : 0;
      if (position[a] < 0 || position[a] >= p.max_pos) {
        known = false;
        outside = position[a];
        position[a] = 0;
      }
    }
    if (!known) {
      keep = false;
      if (threadIdx.x == 0 && blockIdx.y == 0 && atomicCAS(p.status, 0, FBGEMM_B200_STATUS_BAD_INDEX) == 0) {
        p.status[1] = (int32_t)t;
        p.status[2] = 0;
        p.status[3] = (int32_t)outside;
      }
    }
    if (turns) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int pair = p.interleaved ? 4 * (e < 4 ? c0 : c1) + (e & 3) : 8 * lane + e;
        const int axis = (pair >= p.section_end[0]) + (pair >= p.section_end[1]) + (pair >= p.section_end[2]);
        const int32_t at = axis == 0 ? position[0] : axis == 1 ? position[1] : axis == 2 ? position[2] : position[3];
        const float* row = p.cos_sin + (int64_t)at * p.rot;
        cosine[e] = known ? __ldg(row + pair) : 1.f;
        sine[e] = known ? __ldg(row + p.rot / 2 + pair) : 0.f;
      }
    }
  }
  if ((slot < -1 || slot >= p.num_slots) && threadIdx.x == 0 && blockIdx.y == 0 &&
      atomicCAS(p.status, 0, FBGEMM_B200_STATUS_BAD_PAGE) == 0) {
    p.status[1] = (int32_t)t;
    p.status[2] = 0;
    p.status[3] = (int32_t)slot;
  }

  const int queries = p.q_out != nullptr ? p.heads : 0;
  const int rows = queries + 2 * p.kv_heads;
  const int64_t cache_row =
      keep ? (slot >> p.page_shift) * p.page_stride + (slot & ((1 << p.page_shift) - 1)) * p.slot_stride : 0;
  const int step = gridDim.y * (kThreads / LANES);
  // (all lanes of a warp go round together: the quantizers exchange values)
  for (int first = blockIdx.y * (kThreads / LANES); first < rows; first += step) {
    const int r = first + threadIdx.x / LANES;
    const int kind = r < queries ? 0 : r < queries + p.kv_heads ? 1 : 2;
    const int head = kind == 0 ? r : kind == 1 ? r - queries : r - queries - p.kv_heads;
    const bool here = active && r < rows && (kind == 0 || keep);
    float a[8], b[8];
    if (here) {
      const uint8_t* x = kind == 0   ? static_cast<const uint8_t*>(p.q) + t * p.q_token + head * p.q_head
                         : kind == 1 ? static_cast<const uint8_t*>(p.k) + t * p.k_token + head * p.k_head
                                     : static_cast<const uint8_t*>(p.v) + t * p.v_token + head * p.v_head;
      load8<T>(a, x + 16 * c0);
      load8<T>(b, x + 16 * c1);
      if (turns && kind != 2) {
        if (p.interleaved) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float u = a[2 * e], v = a[2 * e + 1], w = b[2 * e], z = b[2 * e + 1];
            a[2 * e] = __fsub_rn(__fmul_rn(u, cosine[e]), __fmul_rn(v, sine[e]));
            a[2 * e + 1] = __fadd_rn(__fmul_rn(v, cosine[e]), __fmul_rn(u, sine[e]));
            b[2 * e] = __fsub_rn(__fmul_rn(w, cosine[4 + e]), __fmul_rn(z, sine[4 + e]));
            b[2 * e + 1] = __fadd_rn(__fmul_rn(z, cosine[4 + e]), __fmul_rn(w, sine[4 + e]));
          }
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float u = a[e], v = b[e];
            a[e] = __fsub_rn(__fmul_rn(u, cosine[e]), __fmul_rn(v, sine[e]));
            b[e] = __fadd_rn(__fmul_rn(v, cosine[e]), __fmul_rn(u, sine[e]));
          }
        }
      }
    }
    if (here && kind == 0) {
      uint8_t* o = static_cast<uint8_t*>(p.q_out) + (t * p.heads + head) * (int64_t)p.dim * 2;
      store8<T>(o + 16 * c0, a);
      store8<T>(o + 16 * c1, b);
    }
    if constexpr (BITS == 16) {
      if (here && kind != 0) {
        uint8_t* o = (kind == 1 ? p.k_cache : p.v_cache) + cache_row + head * p.head_stride;
        store8<T>(o + 16 * c0, a);
        store8<T>(o + 16 * c1, b);
      }
    } else {
      // NaN: left out by fminf and fmaxf unless the whole row is, as in the quantizers
      float lo = __int_as_float(0x7fffffff), hi = lo;
      if (here) {
        lo = hi = a[0];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          lo = fminf(fminf(lo, a[e]), b[e]);
          hi = fmaxf(fmaxf(hi, a[e]), b[e]);
        }
      }
#pragma unroll
      for (int d = LANES / 2; d > 0; d >>= 1) {
        lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, d));
        hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, d));
      }
      if (here && kind != 0) {
        Coder<BITS, BITS == 8> coder;
        coder.init(lo, hi);
        uint8_t* o = (kind == 1 ? p.k_cache : p.v_cache) + cache_row + head * p.head_stride;
        uint32_t w[2][BITS / 4];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const float* x = c ? b : a;
#pragma unroll
          for (int i = 0; i < BITS / 4; ++i) {
            w[c][i] = 0;
#pragma unroll
            for (int e = 0; e < 32 / BITS; ++e) {
              w[c][i] |= coder.code(x[i * (32 / BITS) + e]) << (e * BITS);
            }
          }
        }
        // (rows are 4-byte aligned; most caches lay them further apart)
        uint8_t* o0 = o + c0 * BITS;
        uint8_t* o1 = o + c1 * BITS;
        if constexpr (BITS == 8) {
          if (reinterpret_cast<uintptr_t>(o) % 8 == 0) {
            *reinterpret_cast<uint2*>(o0) = make_uint2(w[0][0], w[0][1]);
            *reinterpret_cast<uint2*>(o1) = make_uint2(w[1][0], w[1][1]);
          } else {
            reinterpret_cast<uint32_t*>(o0)[0] = w[0][0];
            reinterpret_cast<uint32_t*>(o0)[1] = w[0][1];
            reinterpret_cast<uint32_t*>(o1)[0] = w[1][0];
            reinterpret_cast<uint32_t*>(o1)[1] = w[1][1];
          }
        } else {
          *reinterpret_cast<uint32_t*>(o0) = w[0][0];
          *reinterpret_cast<uint32_t*>(o1) = w[1][0];
        }
        if (lane == 0) {
          uint32_t* sb = reinterpret_cast<uint32_t*>(o + p.dim * BITS / 8);
          sb[0] = coder.sb[0];
          if constexpr (BITS == 8) {
            sb[1] = coder.sb[1];
          }
        }
      }
    }
  }
}

template <typename T, int BITS>
void launch(const RotaryAppendParams& p, cudaStream_t stream) {
  const int lanes = p.dim <= 64 ? 4 : p.dim <= 128 ? 8 : 16;
  const int rows = (p.q_out ? p.heads : 0) + 2 * p.kv_heads;
  const int rounds = (rows + kThreads / lanes - 1) / (kThreads / lanes);
  const dim3 grid((unsigned)p.tokens, (unsigned)(p.tokens < 1024 ? rounds : 1));
  (lanes == 4   ? rotary_append_kernel<T, BITS, 4>
   : lanes == 8 ? rotary_append_kernel<T, BITS, 8>
                : rotary_append_kernel<T, BITS, 16>)<<<grid, kThreads, 0, stream>>>(p);
}

}  // namespace

cudaError_t launch_rotary_append(const RotaryAppendParams& p, cudaStream_t stream) {
  if (p.bf16) {
    (p.bits == 16 ? launch<Bf16, 16> : p.bits == 8 ? launch<Bf16, 8> : launch<Bf16, 4>)(p, stream);
  } else {
    (p.bits == 16 ? launch<Half16, 16> : p.bits == 8 ? launch<Half16, 8> : launch<Half16, 4>)(p, stream);
  }
  g_launch_count.fetch_add(1, std::memory_order_relaxed);
  return cudaGetLastError();
}

}  // namespace fbgemm_b200
