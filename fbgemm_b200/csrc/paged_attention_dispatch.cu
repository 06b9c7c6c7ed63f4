// Which variant of paged_attention.cuh a call takes: by the rows' format and alignment, the columns and the query heads
// per cached head.
#include "paged_attention_variants.cuh"

namespace fbgemm_b200 {

namespace {

PagedVariants variants_of(const PagedAttentionShape& s) {
  return s.bits == 8 ? paged_attention_8 : s.bits == 4 ? paged_attention_4 : s.bf16 ? paged_attention_bf16 : paged_attention_f16;
}

}  // namespace

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
