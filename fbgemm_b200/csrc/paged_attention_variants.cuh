// The variants of paged_attention.cuh by row width and query heads per cached head: rows of up to 64, 128 and 256
// columns; 8 heads in a warp, 16 where the output of 16 fits the registers (up to 128 columns), and twice as many in two
// warps that read the same rows at about the same time, the second from the caches.  More heads than that are an item of
// their own, which reads the rows again.
#pragma once

#include "paged_attention.cuh"

namespace fbgemm_b200 {
namespace paged {

template <int BITS, typename F>
auto with_shape(int dim, int group, F&& f) {
  if (dim > 128) {
    return group > 8 ? f(Shape<BITS, 256, 1, 2>()) : f(Shape<BITS, 256, 1, 1>());
  }
  if (dim > 64) {
    return group > 16 ? f(Shape<BITS, 128, 2, 2>()) : group > 8 ? f(Shape<BITS, 128, 2, 1>()) : f(Shape<BITS, 128, 1, 1>());
  }
  return group > 16 ? f(Shape<BITS, 64, 2, 2>()) : group > 8 ? f(Shape<BITS, 64, 2, 1>()) : f(Shape<BITS, 64, 1, 1>());
}

}  // namespace paged

// One translation unit's part of the dispatch: the plan (p null) or the launch.
using PagedVariants = cudaError_t (*)(const PagedAttentionShape&, int64_t sms, PagedAttentionPlan*, const PagedAttentionParams*,
                                      bool split, cudaStream_t);
cudaError_t paged_attention_f16(const PagedAttentionShape&, int64_t, PagedAttentionPlan*, const PagedAttentionParams*, bool,
                                cudaStream_t);
cudaError_t paged_attention_bf16(const PagedAttentionShape&, int64_t, PagedAttentionPlan*, const PagedAttentionParams*, bool,
                                 cudaStream_t);
cudaError_t paged_attention_8(const PagedAttentionShape&, int64_t, PagedAttentionPlan*, const PagedAttentionParams*, bool,
                              cudaStream_t);
cudaError_t paged_attention_4(const PagedAttentionShape&, int64_t, PagedAttentionPlan*, const PagedAttentionParams*, bool,
                              cudaStream_t);

#define FBGEMM_B200_PAGED_16(NAME, IS_BF16)                                                                                  \
  cudaError_t NAME(const PagedAttentionShape& s, int64_t sms, PagedAttentionPlan* plan, const PagedAttentionParams* p,       \
                   bool split, cudaStream_t stream) {                                                                        \
    return paged::with_shape<16>(s.dim, s.group, [&](auto shape) {                                                           \
      using S = decltype(shape);                                                                                             \
      if (!p) {                                                                                                              \
        *plan = paged::plan_of<S>(s.group, sms);                                                                             \
        return cudaSuccess;                                                                                                  \
      }                                                                                                                      \
      return s.fast ? paged::launch_of<S, IS_BF16, true>(*plan, *p, split, stream)                                           \
                    : paged::launch_of<S, IS_BF16, false>(*plan, *p, split, stream);                                         \
    });                                                                                                                      \
  }

#define FBGEMM_B200_PAGED_QUANTIZED(NAME, ROW_BITS)                                                                          \
  cudaError_t NAME(const PagedAttentionShape& s, int64_t sms, PagedAttentionPlan* plan, const PagedAttentionParams* p,       \
                   bool split, cudaStream_t stream) {                                                                        \
    return paged::with_shape<ROW_BITS>(s.dim, s.group, [&](auto shape) {                                                     \
      using S = decltype(shape);                                                                                             \
      if (!p) {                                                                                                              \
        *plan = paged::plan_of<S>(s.group, sms);                                                                             \
        return cudaSuccess;                                                                                                  \
      }                                                                                                                      \
      return s.fast ? (s.bf16 ? paged::launch_of<S, true, true>(*plan, *p, split, stream)                                    \
                              : paged::launch_of<S, false, true>(*plan, *p, split, stream))                                  \
                    : (s.bf16 ? paged::launch_of<S, true, false>(*plan, *p, split, stream)                                   \
                              : paged::launch_of<S, false, false>(*plan, *p, split, stream));                                \
    });                                                                                                                      \
  }

}  // namespace fbgemm_b200
