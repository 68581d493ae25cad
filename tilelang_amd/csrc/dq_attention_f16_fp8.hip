// Attention of one new token, fp16 queries on an fp8 cache.
#include "dq_attention.h"

namespace dq {
int attention_f16_fp8(const AttnArgs& a, hipStream_t stream) { return attention_of_type<half_t, CACHE_FP8>(a, stream); }
}  // namespace dq
