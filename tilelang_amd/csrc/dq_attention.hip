// Attention of one new token: which kernel, how many splits, and the join of the splits' results.
#include "dq_attention.h"

#include <algorithm>

namespace dq {

int attention_f16(const AttnArgs& a, hipStream_t stream);
int attention_f16_fp8(const AttnArgs& a, hipStream_t stream);
int attention_f16_i8(const AttnArgs& a, hipStream_t stream);
int attention_bf16(const AttnArgs& a, hipStream_t stream);
int attention_bf16_fp8(const AttnArgs& a, hipStream_t stream);
int attention_bf16_i8(const AttnArgs& a, hipStream_t stream);

namespace {

// One workgroup a (sequence, head): o = sum_s 2^(m_s - m) o_s / sum_s 2^(m_s - m) l_s, the splits in their order.
template <class T>
__global__ __launch_bounds__(64) void attention_join_kernel(const AttnArgs a) {
  const size_t at = (size_t)blockIdx.y * a.heads + blockIdx.x;
  const float* const ml = a.part_ml + 2 * at * a.splits;
  const int D = a.shape.head_dim;
  float most = -INFINITY;
  for (int s = 0; s < a.splits; ++s) most = fmaxf(most, ml[2 * s]);
  const float sink = a.sinks ? a.sinks[blockIdx.x] * 1.44269504088896341f : -INFINITY;
  const float base = fmaxf(most, sink);
  float x[4] = {}, sum = weight(sink, base);
  for (int s = 0; s < a.splits; ++s) {
    const float w = weight(ml[2 * s], base);
    sum += w * ml[2 * s + 1];
    if (ml[2 * s] == -INFINITY) continue;  // nothing was written there
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int d = threadIdx.x + 64 * i;
      if (d < D) x[i] += w * a.part_o[(at * a.splits + s) * D + d];
    }
  }
  const float inv = sum > 0.f ? 1.f / sum : (sum == 0.f ? 0.f : sum);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int d = threadIdx.x + 64 * i;
    if (d < D) reinterpret_cast<T*>(a.out)[at * D + d] = (T)(x[i] * inv);
  }
  if (a.lse && threadIdx.x == 0) a.lse[at] = base == -INFINITY ? -INFINITY : (base + log2f(sum)) * 0.693147180559945309f;
}

}  // namespace

// Splits of a sequence's tokens: about four workgroups a compute unit, none of fewer than a tile a wave.
static int attention_splits(int sequences, int heads, int kv_heads, long capacity) {
  const int head_blocks = (heads / kv_heads + 15) / 16;
  const long have = (long)sequences * kv_heads * head_blocks, want = (1024 + have - 1) / have;
  const long most = (capacity + kAttnTile * kAttnWaves - 1) / (kAttnTile * kAttnWaves);
  return (int)std::max(1l, std::min(want, most));
}

size_t attention_workspace_bytes(int sequences, int heads, int kv_heads, int head_dim, long capacity) {
  const int splits = attention_splits(sequences, heads, kv_heads, capacity);
  return splits == 1 ? 0 : (size_t)sequences * heads * splits * (head_dim + 2) * 4;
}

bool attention_head_dim(int d) { return d == 64 || d == 80 || d == 96 || d == 112 || d == 128 || d == 160 || d == 192 || d == 256; }

int attention_decode(const void* Q, const void* KCache, const void* VCache, const float* KScale, const float* VScale,
                     const int* PageTable, const int* Lengths, const float* Sinks, void* Out, float* Lse, void* Workspace,
                     float scale, int sequences, int heads, int kv_heads, int head_dim, int pages, int page_shift, int max_pages,
                     int window, int bf16, int format, hipStream_t stream) {
  AttnArgs a = {};
  a.q = Q, a.cache[0] = KCache, a.cache[1] = VCache, a.scale[0] = KScale, a.scale[1] = VScale;
  a.table = PageTable, a.lengths = Lengths, a.sinks = Sinks, a.out = Out, a.lse = Lse;
  a.score_scale = scale * 1.44269504088896341f;
  a.sequences = sequences, a.heads = heads, a.max_pages = max_pages, a.window = window;
  a.head_blocks = (heads / kv_heads + 15) / 16;
  a.shape = {pages, kv_heads, page_shift, head_dim};
  a.splits = attention_splits(sequences, heads, kv_heads, (long)max_pages << page_shift);
  a.part_o = (float*)Workspace;
  a.part_ml = a.part_o + (size_t)sequences * heads * a.splits * head_dim;
  int rc;
  switch (format) {
    case CACHE_FP8: rc = bf16 ? attention_bf16_fp8(a, stream) : attention_f16_fp8(a, stream); break;
    case CACHE_I8: rc = bf16 ? attention_bf16_i8(a, stream) : attention_f16_i8(a, stream); break;
    default: rc = bf16 ? attention_bf16(a, stream) : attention_f16(a, stream);
  }
  if (rc != 0 || a.splits == 1) return rc;
  if (bf16) attention_join_kernel<bf16_t><<<dim3(heads, sequences), 64, 0, stream>>>(a);
  else attention_join_kernel<half_t><<<dim3(heads, sequences), 64, 0, stream>>>(a);
  DQ_CHECK_HIP(hipGetLastError());
  return 0;
}

}  // namespace dq
