// How the row-wise quantizers code a row (quantize_kernels.cu, rotary_append_kernels.cu), operation for operation as the
// scalar reference does: 8-bit + fp32 scale,bias src/QuantUtils.cc:677-718, N-bit + fp16 scale,bias src/QuantUtils.cc:534-611.
#pragma once

#include <cuda_fp16.h>

#include <cstdint>

namespace fbgemm_b200 {

// Scale, bias and codes of one row from its minimum and maximum.
template <int BITS, bool FP32_SB>
struct Coder {
  float mn, inv;
  uint32_t sb[FP32_SB ? 2 : 1];  // scale, bias as they are stored

  __device__ __forceinline__ void init(float lo, float hi) {
    if constexpr (FP32_SB) {
      mn = lo;
      const float range = __fsub_rn(hi, lo);
      sb[0] = __float_as_uint(__fdiv_rn(range, 255.0f));
      sb[1] = __float_as_uint(lo);
      inv = __fdiv_rn(255.0f, __fadd_rn(range, 1e-8f));
    } else {
      constexpr int QMAX = (1 << BITS) - 1;
      // the bias is stored as fp16: round the minimum first
      const __half mn_h = __float2half_rn(lo);
      mn = __half2float(mn_h);
      const float range = __fsub_rn(hi, mn);
      // The scale is stored as fp16 too; quantize with the value a reader will see.
      __half scale_h = __float2half_rn(range == 0.f ? 1.0f : __fdiv_rn(range, (float)QMAX));
      float scale = __half2float(scale_h);
      if (scale == 0.f) {
        scale = 1.0f;
        scale_h = __ushort_as_half((unsigned short)0x3C00);
      }
      inv = __fdiv_rn(1.0f, scale);
      if (isinf(inv)) {
        inv = 1.0f;
        scale_h = __ushort_as_half((unsigned short)0x3C00);
      }
      sb[0] = (uint32_t)__half_as_ushort(scale_h) | ((uint32_t)__half_as_ushort(mn_h) << 16);
    }
  }
  __device__ __forceinline__ uint32_t code(float x) const {
    const int q = __float2int_rn(__fmul_rn(__fsub_rn(x, mn), inv));
    if constexpr (FP32_SB) {
      return (uint32_t)q & 0xffu;
    } else {
      return (uint32_t)max(0, min(q, (1 << BITS) - 1));
    }
  }
};

}  // namespace fbgemm_b200
