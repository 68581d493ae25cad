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

// A column that lies in several pieces, a head at a time: o = sum_i 2^(m_i - m) o_i / sum_i 2^(m_i - m) l_i, in a fixed order.
// Eight groups of 32 lanes, four elements (and at more than 128 four more) a lane.  SPREAD (few columns, maybe hundreds of
// pieces): a workgroup a head, its groups take the pieces in turn and are added at the end.  Else (many columns, few
// pieces): a workgroup a column, a group a head.
constexpr int kJoinGroups = 8;
template <class T, bool SPREAD>
__global__ __launch_bounds__(256) void attention_join_kernel(const AttnArgs a) {
  const int columns = a.shape.kv_heads * a.head_blocks, sequence = blockIdx.x / columns, column = blockIdx.x - sequence * columns;
  const int first = a.pieces[2 * (size_t)blockIdx.x], count = a.pieces[2 * (size_t)blockIdx.x + 1] - first + 1;
  if (count <= 1) return;  // written by the workgroup that had it whole
  const int D = a.shape.head_dim, group = a.heads / a.shape.kv_heads, kv_head = column / a.head_blocks, block = column - kv_head * a.head_blocks;
  __shared__ float4_t so[SPREAD ? kJoinGroups : 1][kMaxHeadDim / 4];
  __shared__ float ss[kJoinGroups];
  const int lane = threadIdx.x & 31, part = threadIdx.x >> 5;
  const int rows = min(a.rows, group - block * a.rows);
  for (int row = SPREAD ? blockIdx.y : part; row < rows; row += SPREAD ? gridDim.y : kJoinGroups) {
    const int head = kv_head * group + block * a.rows + row;
    auto at = [&](int i) { return ((size_t)(first + i) * 2 + (i == 0)) * a.rows + row; };
    float most = -INFINITY;
    for (int i = lane; i < count; i += 32) most = fmaxf(most, a.part_ml[2 * at(i)]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor(most, o));
    const float sink = a.sinks ? a.sinks[head] * 1.44269504088896341f : -INFINITY;
    const float base = fmaxf(most, sink);
    float4_t x[2] = {};
    float sum = 0.f;
#pragma unroll 4
    for (int i = SPREAD ? part : 0; i < count; i += SPREAD ? kJoinGroups : 1) {
      const size_t k = at(i);
      const float w = weight(a.part_ml[2 * k], base);
      sum += w * a.part_ml[2 * k + 1];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int d = 4 * lane + 128 * j;
        if (d < D) x[j] += w * *reinterpret_cast<const float4_t*>(a.part_o + k * D + d);
      }
    }
    if constexpr (SPREAD) {
#pragma unroll
      for (int j = 0; j < 2; ++j)
        if (4 * lane + 128 * j < D) so[part][lane + 32 * j] = x[j];
      if (lane == 0) ss[part] = sum;
      __syncthreads();
      if (part == 0) {
        sum = 0.f;
        x[0] = x[1] = float4_t{};
#pragma unroll
        for (int p = 0; p < kJoinGroups; ++p) {
          sum += ss[p];
#pragma unroll
          for (int j = 0; j < 2; ++j)
            if (4 * lane + 128 * j < D) x[j] += so[p][lane + 32 * j];
        }
      }
    }
    if (!SPREAD || part == 0) {
      sum += weight(sink, base);
      const float inv = sum > 0.f ? 1.f / sum : (sum == 0.f ? 0.f : sum);
      const size_t to = (size_t)sequence * a.heads + head;
      typedef T T4 __attribute__((ext_vector_type(4)));
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int d = 4 * lane + 128 * j;
        if (d < D) *reinterpret_cast<T4*>(reinterpret_cast<T*>(a.out) + to * D + d) = T4{(T)(x[j][0] * inv), (T)(x[j][1] * inv), (T)(x[j][2] * inv), (T)(x[j][3] * inv)};
      }
      if (a.lse && lane == 0) a.lse[to] = base == -INFINITY ? -INFINITY : (base + log2f(sum)) * 0.693147180559945309f;
    }
    if (SPREAD) __syncthreads();
  }
}

template <class T>
void launch_join(const AttnArgs& a, hipStream_t stream) {
  const int columns = a.sequences * a.shape.kv_heads * a.head_blocks;
  // a workgroup a compute unit, or a head where that makes no more than eight of them
  if ((long)columns * a.rows <= 8 * kComputeUnits) attention_join_kernel<T, true><<<dim3(columns, a.rows), 256, 0, stream>>>(a);
  else attention_join_kernel<T, false><<<columns, 256, 0, stream>>>(a);
}

}  // namespace

// A launch's workgroups and what they need to leave pieces of heads: as many as the chip holds at once, and no more than
// pay.  tokens: that a sequence can have, or that its window shows.
struct AttnPlan {
  int head_blocks, rows, workgroups;
  bool joins;
  size_t floats() const { return (size_t)workgroups * 2 * rows; }
};
static AttnPlan attention_plan(int sequences, int heads, int kv_heads, int head_dim, int format, long capacity, int window) {
  AttnPlan p;
  const int group = heads / kv_heads;
  p.head_blocks = (group + 15) / 16;
  p.rows = std::min(group, 16);
  // (a window may begin and end inside a tile)
  const long tokens = window > 0 && window + kAttnTile - 1 < capacity ? window + kAttnTile - 1 : capacity;
  const long units = ((tokens + kAttnTile - 1) / kAttnTile + kAttnWaves - 1) / kAttnWaves, columns = (long)sequences * kv_heads * p.head_blocks;
  p.joins = units > kWholeUnits;
  p.workgroups = (int)std::min<long>(kComputeUnits * attention_per_unit(head_dim, format), p.joins ? columns * units : columns);
  return p;
}

// Units are counted in 31 bits.
bool attention_fits(int sequences, int heads, int kv_heads, long capacity) {
  const double units = (double)sequences * kv_heads * ((heads / kv_heads + 15) / 16) * (capacity / kAttnUnit + 3);
  return units < 2147483647.0;
}

size_t attention_workspace_bytes(int sequences, int heads, int kv_heads, int head_dim, int format, long capacity, int window) {
  const AttnPlan p = attention_plan(sequences, heads, kv_heads, head_dim, format, capacity, window);
  return p.joins ? (p.floats() * (head_dim + 2) + (size_t)sequences * kv_heads * p.head_blocks * 2) * 4 : 0;
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
  const AttnPlan p = attention_plan(sequences, heads, kv_heads, head_dim, format, (long)max_pages << page_shift, window);
  a.head_blocks = p.head_blocks, a.rows = p.rows, a.workgroups = p.workgroups;
  a.shape = {pages, kv_heads, page_shift, head_dim};
  if (p.joins) {
    a.part_o = (float*)Workspace;
    a.part_ml = a.part_o + p.floats() * head_dim;
    a.pieces = (int*)(a.part_ml + p.floats() * 2);
  }
  int rc;
  switch (format) {
    case CACHE_FP8: rc = bf16 ? attention_bf16_fp8(a, stream) : attention_f16_fp8(a, stream); break;
    case CACHE_I8: rc = bf16 ? attention_bf16_i8(a, stream) : attention_f16_i8(a, stream); break;
    default: rc = bf16 ? attention_bf16(a, stream) : attention_f16(a, stream);
  }
  if (rc != 0 || !p.joins) return rc;
  if (bf16) launch_join<bf16_t>(a, stream);
  else launch_join<half_t>(a, stream);
  DQ_CHECK_HIP(hipGetLastError());
  return 0;
}

}  // namespace dq
