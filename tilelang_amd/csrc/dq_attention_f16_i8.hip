// Attention of one new token, fp16 queries on an int8 cache.
#include "dq_attention.h"

namespace dq {
int attention_f16_i8(const AttnArgs& a, hipStream_t stream) { return attention_of_type<half_t, CACHE_I8>(a, stream); }
}  // namespace dq
