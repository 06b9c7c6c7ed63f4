// Which variant of paged_attention.cuh a call takes: by the rows' format and alignment, the columns and the query heads
// per cached head.
#include "paged_attention_variants.cuh"

namespace fbgemm_b200 {

namespace {

PagedVariants variants_of(const PagedAttentionShape& s) {
  return s.bits == 8 ? paged_attention_8 : s.bits == 4 ? paged_attention_4 : s.bf16 ? paged_attention_bf16 : paged_attention_f16;
}

}  // namespace

cudaError_t encode_rows(CUtensorMap* map, const uint8_t* rows, const PagedAttentionParams& p, bool swizzled, int box, int height,
                        int bits, int tail_bytes) {
  using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                              const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
  static std::atomic<Encode> known{nullptr};
  Encode encode = known.load(std::memory_order_relaxed);
  if (!encode) {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult found;
    const cudaError_t e = cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &found);
    if (e != cudaSuccess || found != cudaDriverEntryPointSuccess) {
      return e != cudaSuccess ? e : cudaErrorNotSupported;
    }
    encode = reinterpret_cast<Encode>(f);
    known.store(encode, std::memory_order_relaxed);
  }
  const int word = swizzled ? 2 : 4;
  const cuuint64_t columns = (cuuint64_t)(p.dim * bits / 8 + tail_bytes) / word;
  // A dimension of one has no stride of its own: any multiple of 16 will do.
  const cuuint64_t dims[4] = {columns, (cuuint64_t)p.kv_heads, (cuuint64_t)1 << p.page_shift, (cuuint64_t)p.num_pages};
  const cuuint64_t strides[3] = {(cuuint64_t)(p.kv_heads > 1 ? p.head_stride : 16), (cuuint64_t)p.slot_stride,
                                 (cuuint64_t)(p.num_pages > 1 ? p.page_stride : 16)};
  const cuuint32_t boxes[4] = {(cuuint32_t)box, 1, (cuuint32_t)height, 1};
  const cuuint32_t steps[4] = {1, 1, 1, 1};
  const CUresult r = encode(map, swizzled ? CU_TENSOR_MAP_DATA_TYPE_UINT16 : CU_TENSOR_MAP_DATA_TYPE_UINT32, 4,
                            const_cast<uint8_t*>(rows), dims, strides, boxes, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
                            swizzled ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_NONE,
                            CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

PagedAttentionPlan plan_paged_attention(const PagedAttentionShape& s, int64_t sms) {
  PagedAttentionPlan plan = {};
  variants_of(s)(s, sms, &plan, nullptr, false, nullptr);
  return plan;
}

cudaError_t launch_paged_attention(const PagedAttentionShape& s, const PagedAttentionPlan& plan, const PagedAttentionParams& p,
                                   bool split, cudaStream_t stream) {
  PagedAttentionPlan copy = plan;
  return variants_of(s)(s, 0, &copy, &p, split, stream);
}

}  // namespace fbgemm_b200
