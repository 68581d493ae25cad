// Attention of one new token, bf16 queries on an fp8 cache.
#include "dq_attention.h"

namespace dq {
int attention_bf16_fp8(const AttnArgs& a, hipStream_t stream) { return attention_of_type<bf16_t, CACHE_FP8>(a, stream); }
}  // namespace dq
