// paged_attention.cuh for fused 4-bit rows.
#include "paged_attention_variants.cuh"

namespace fbgemm_b200 {
FBGEMM_B200_PAGED_QUANTIZED(paged_attention_4, 4)
}  // namespace fbgemm_b200
