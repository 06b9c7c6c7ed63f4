// paged_attention.cuh for fused 8-bit rows.
#include "paged_attention_variants.cuh"

namespace fbgemm_b200 {
FBGEMM_B200_PAGED_QUANTIZED(paged_attention_8, 8)
}  // namespace fbgemm_b200
