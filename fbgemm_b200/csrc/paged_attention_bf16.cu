// paged_attention.cuh for rows of bf16 values.
#include "paged_attention_variants.cuh"

namespace fbgemm_b200 {
FBGEMM_B200_PAGED_16(paged_attention_bf16, true)
}  // namespace fbgemm_b200
