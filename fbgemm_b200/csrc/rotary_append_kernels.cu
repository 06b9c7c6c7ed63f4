// Rotary positions, and the new rows' way into the paged cache: of every token, each query and key head is turned pair
// by pair, (a, b) -> (a cos - b sin, b cos + a sin), pair i by the angle of the position on the axis that i belongs to
// (time, height and width of a picture's tokens; text has one axis).  Turned queries go out in their own type; keys and values
// go to row slots[t] of the cache, rounded once: to 16 bits, or as fused 8- or 4-bit rows with the codes, scale and
// bias that the row-wise quantizers (row_coder.cuh) give for the same fp32 row, byte for byte.  A slot of -1 is a row of
// padding: nothing is stored for it.
//
// Bound by memory: every value is read once and written once.  A group of 4, 8 or 16 lanes takes a head; each lane
// holds 16 of its values, two chunks of 16 bytes that contain both ends of every pair (half a head apart, or next to
// each other), so that turning needs no exchange and a row's minimum and maximum two to four.  The heads of a token share
// the lanes' cosines and sines: with many tokens a warp takes a whole token, so that their address arithmetic is done
// once for all its heads, and the next heads are on their way meanwhile; with few the heads go to as many warps as there are.  (A block per
// token, the quantizer's arithmetic run by the warps of query heads too: 55 us for 8192 tokens of 32 + 2 x 8 heads into
// 8-bit rows, issue bound; this 40, of which 29 are the bytes: 0.72 of a copy's rate, 63 % of the issue slots taken, and with one
// head ahead 32 KB an SM on their way.  16-bit rows 37 for 31, 4-bit ones 38 for 28.)
#include <cuda_bf16.h>

#include "internal.h"
#include "paged_cache.h"
#include "row_coder.cuh"

namespace fbgemm_b200 {

namespace {

constexpr int kThreads = 128;
constexpr int64_t kWarpTokens = 2048;

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
__device__ __forceinline__ void widen8(float* x, const uint4& v) {
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

// Cosines or sines of N pairs in a row of the table, from `pair` on; the pairs of an axis turn by the position on it.
template <int N>
__device__ __forceinline__ void load_angles(float* x, const RotaryAppendParams& p, const int32_t (&position)[4], int pair, int skip) {
  auto axis_of = [&](int i) { return (i >= p.section_end[0]) + (i >= p.section_end[1]) + (i >= p.section_end[2]); };
  auto row_of = [&](int axis) {
    const int32_t at = axis == 0 ? position[0] : axis == 1 ? position[1] : axis == 2 ? position[2] : position[3];
    return p.cos_sin + (int64_t)at * p.rot + skip;
  };
  const int axis = axis_of(pair);
  if (p.angles_aligned && axis == axis_of(pair + N - 1)) {
    const float* row = row_of(axis) + pair;
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const float4 v = __ldg(reinterpret_cast<const float4*>(row + i));
      x[i] = v.x;
      x[i + 1] = v.y;
      x[i + 2] = v.z;
      x[i + 3] = v.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      x[i] = __ldg(row_of(axis_of(pair + i)) + pair + i);
    }
  }
}

// WARP: a warp takes a token.  Otherwise block x takes token x, block y a share of its heads (queries, then keys, then
// values).
template <typename T, int BITS, int LANES, bool WARP>
__global__ void __launch_bounds__(kThreads, 8) rotary_append_kernel(const RotaryAppendParams p) {
  constexpr int kGroups = (WARP ? 32 : kThreads) / LANES;  // heads at a time
  const int64_t t = WARP ? (int64_t)blockIdx.x * (kThreads / 32) + threadIdx.x / 32 : blockIdx.x;
  if (t >= p.tokens) {
    return;  // (whole warps)
  }
  const int lane = threadIdx.x % LANES, group = threadIdx.x % (WARP ? 32 : kThreads) / LANES;
  const bool active = lane * 16 < p.dim;
  const int chunks = p.rot / 16;  // chunks of eight in half of the turned part
  const bool turns = p.cos_sin != nullptr && lane < chunks;
  const int c0 = lane < chunks ? lane : 2 * lane;                   // (2 * chunks + 2 * (lane - chunks))
  const int c1 = lane < chunks ? lane + chunks : 2 * lane + 1;
  const bool reports = WARP ? threadIdx.x % 32 == 0 : threadIdx.x == 0 && blockIdx.y == 0;

  const int queries = p.q_out != nullptr ? p.heads : 0;
  const int rows = queries + 2 * p.kv_heads;
  const int first = WARP ? 0 : blockIdx.y * kGroups, step = WARP ? kGroups : gridDim.y * kGroups;
  auto read = [&](int r, uint4& x, uint4& y) {
    if (active && r < rows) {
      const uint8_t* from = r < queries                ? static_cast<const uint8_t*>(p.q) + t * p.q_token + r * p.q_head
                            : r < queries + p.kv_heads ? static_cast<const uint8_t*>(p.k) + t * p.k_token + (r - queries) * p.k_head
                                                       : static_cast<const uint8_t*>(p.v) + t * p.v_token +
                                                             (r - queries - p.kv_heads) * p.v_head;
      x = *reinterpret_cast<const uint4*>(from + 16 * c0);
      y = *reinterpret_cast<const uint4*>(from + 16 * c1);
    }
  };
  uint4 next_x = make_uint4(0, 0, 0, 0), next_y = next_x;
  read(first + group, next_x, next_y);

  const int64_t slot = p.slots[t];
  bool keep = slot >= 0 && slot < p.num_slots;
  float cosine[8], sine[8];
  if (p.cos_sin != nullptr) {
    int32_t position[4];
    int64_t outside = 0;
    bool known = true;
#pragma unroll
    for (int a = 0; a < 4; ++a) {
      position[a] = a < p.axes ? p.positions[a * p.positions_stride + t] : 0;
      if (position[a] < 0 || position[a] >= p.max_pos) {
        known = false;
        outside = position[a];
        position[a] = 0;
      }
    }
    if (turns) {
      if (p.interleaved) {
        load_angles<4>(cosine, p, position, 4 * c0, 0);
        load_angles<4>(cosine + 4, p, position, 4 * c1, 0);
        load_angles<4>(sine, p, position, 4 * c0, p.rot / 2);
        load_angles<4>(sine + 4, p, position, 4 * c1, p.rot / 2);
      } else {
        load_angles<8>(cosine, p, position, 8 * lane, 0);
        load_angles<8>(sine, p, position, 8 * lane, p.rot / 2);
      }
    }
    if (!known) {
      keep = false;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        cosine[e] = 1.f;
        sine[e] = 0.f;
      }
      if (reports && atomicCAS(p.status, 0, FBGEMM_B200_STATUS_BAD_INDEX) == 0) {
        p.status[1] = (int32_t)t;
        p.status[2] = 0;
        p.status[3] = (int32_t)outside;
      }
    }
  }
  if ((slot < -1 || slot >= p.num_slots) && reports && atomicCAS(p.status, 0, FBGEMM_B200_STATUS_BAD_PAGE) == 0) {
    p.status[1] = (int32_t)t;
    p.status[2] = 0;
    p.status[3] = (int32_t)slot;
  }
  const int64_t cache_row =
      keep ? (slot >> p.page_shift) * p.page_stride + (slot & ((1 << p.page_shift) - 1)) * p.slot_stride : 0;

  // (all lanes of a warp go round together: the quantizers exchange values)
  for (int r0 = first; r0 < rows; r0 += step) {
    const int r = r0 + group;
    const int kind = r < queries ? 0 : r < queries + p.kv_heads ? 1 : 2;
    const int head = kind == 0 ? r : kind == 1 ? r - queries : r - queries - p.kv_heads;
    const bool here = active && r < rows && (kind == 0 || keep);
    float a[8], b[8];
    widen8<T>(a, next_x);
    widen8<T>(b, next_y);
    read(r + step, next_x, next_y);
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
    if (kind == 0) {
      if (here) {
        uint8_t* o = static_cast<uint8_t*>(p.q_out) + (t * p.heads + head) * (int64_t)p.dim * 2;
        store8<T>(o + 16 * c0, a);
        store8<T>(o + 16 * c1, b);
      }
    }
    if constexpr (BITS == 16) {
      if (here && kind != 0) {
        uint8_t* o = (kind == 1 ? p.k_cache : p.v_cache) + cache_row + head * p.head_stride;
        store8<T>(o + 16 * c0, a);
        store8<T>(o + 16 * c1, b);
      }
    } else {
      if (!__any_sync(0xffffffffu, kind != 0)) {
        continue;
      }
      // NaN: left out by fminf and fmaxf unless the whole row is, as in the quantizers
      float lo = __int_as_float(0x7fffffff), hi = lo;
      if (active) {
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

template <typename T, int BITS, int LANES>
void launch_lanes(const RotaryAppendParams& p, cudaStream_t stream) {
  const int rows = (p.q_out ? p.heads : 0) + 2 * p.kv_heads;
  const int at_a_time = kThreads / LANES;
  // A warp per token once that fills the chip; before, its heads go to several warps.  (8-bit rows of 32 + 2 x 8 heads: 1024
  // tokens 8.4 us with their heads apart, 2048 10.8 and 8192 40 a warp each, 55 with their heads apart.)
  if (p.tokens >= kWarpTokens) {
    rotary_append_kernel<T, BITS, LANES, true>
        <<<(unsigned)((p.tokens + kThreads / 32 - 1) / (kThreads / 32)), kThreads, 0, stream>>>(p);
  } else {
    const dim3 grid((unsigned)p.tokens, (unsigned)((rows + at_a_time - 1) / at_a_time));
    rotary_append_kernel<T, BITS, LANES, false><<<grid, kThreads, 0, stream>>>(p);
  }
}

template <typename T, int BITS>
void launch(const RotaryAppendParams& p, cudaStream_t stream) {
  (p.dim <= 64 ? launch_lanes<T, BITS, 4> : p.dim <= 128 ? launch_lanes<T, BITS, 8> : launch_lanes<T, BITS, 16>)(p, stream);
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
