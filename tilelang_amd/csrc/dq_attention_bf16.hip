// Attention of one new token, bf16 queries on a bf16 cache.
#include "dq_attention.h"

namespace dq {
int attention_bf16(const AttnArgs& a, hipStream_t stream) { return attention_of_type<bf16_t, CACHE_BF16>(a, stream); }
}  // namespace dq
