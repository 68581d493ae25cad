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
typedef float float2_t __attribute__((ext_vector_type(2)));
template <class T, bool SPREAD>
__global__ __launch_bounds__(256) void attention_join_kernel(const AttnArgs a) {
  const int columns = a.shape.kv_heads * a.head_blocks, sequence = blockIdx.x / columns, column = blockIdx.x - sequence * columns;
  const int first = a.pieces[2 * (size_t)blockIdx.x], count = a.pieces[2 * (size_t)blockIdx.x + 1] - first + 1;
  if (count <= 1) return;  // written by the workgroup that had it whole
  const int D = a.shape.head_dim, group = a.heads / a.shape.kv_heads, kv_head = column / a.head_blocks, block = column - kv_head * a.head_blocks;
  __shared__ float4_t so[SPREAD ? kJoinGroups : 1][kMaxHeadDim / 4];
  __shared__ float2_t ss[kJoinGroups];
  const int lane = threadIdx.x & 31, part = threadIdx.x >> 5;
  const int rows = min(a.rows, group - block * a.rows);
  for (int row = SPREAD ? blockIdx.y : part; row < rows; row += SPREAD ? gridDim.y : kJoinGroups) {
    const int head = kv_head * group + block * a.rows + row;
    // four pieces at a time: their loads together, then the running maximum and sums
    float m = -INFINITY, sum = 0.f;
    float4_t x[2] = {};
    constexpr int kStep = SPREAD ? kJoinGroups : 1;
    for (int i0 = SPREAD ? part : 0; i0 < count; i0 += 4 * kStep) {
      float2_t ml[4];
      float4_t o[4][2];
#pragma unroll
      for (int p = 0; p < 4; ++p) {
        const int i = min(i0 + p * kStep, count - 1);
        const size_t k = ((size_t)(first + i) * 2 + (i == 0)) * a.rows + row;
        ml[p] = *reinterpret_cast<const float2_t*>(a.part_ml + 2 * k);
        if (i0 + p * kStep >= count) ml[p] = float2_t{-INFINITY, 0.f};
#pragma unroll
        for (int j = 0; j < 2; ++j)
          if (4 * lane + 128 * j < D) o[p][j] = *reinterpret_cast<const float4_t*>(a.part_o + k * D + 4 * lane + 128 * j);
      }
      const float to = fmaxf(fmaxf(m, fmaxf(ml[0][0], ml[1][0])), fmaxf(ml[2][0], ml[3][0]));
      const float keep = weight(m, to);
      m = to, sum *= keep;
#pragma unroll
      for (int j = 0; j < 2; ++j) x[j] *= keep;
#pragma unroll
      for (int p = 0; p < 4; ++p) {
        const float w = weight(ml[p][0], to);
        sum += w * ml[p][1];
#pragma unroll
        for (int j = 0; j < 2; ++j)
          if (4 * lane + 128 * j < D && i0 + p * kStep < count) x[j] += w * o[p][j];
      }
    }
    if constexpr (SPREAD) {
#pragma unroll
      for (int j = 0; j < 2; ++j)
        if (4 * lane + 128 * j < D) so[part][lane + 32 * j] = x[j];
      if (lane == 0) ss[part] = float2_t{m, sum};
      __syncthreads();
      if (part == 0) {
        m = -INFINITY, sum = 0.f;
        x[0] = x[1] = float4_t{};
#pragma unroll
        for (int p = 0; p < kJoinGroups; ++p) m = fmaxf(m, ss[p][0]);
#pragma unroll
        for (int p = 0; p < kJoinGroups; ++p) {
          const float w = weight(ss[p][0], m);
          sum += w * ss[p][1];
#pragma unroll
          for (int j = 0; j < 2; ++j)
            if (4 * lane + 128 * j < D) x[j] += w * so[p][lane + 32 * j];
        }
      }
    }
    if (!SPREAD || part == 0) {
      const float sink = a.sinks ? a.sinks[head] * 1.44269504088896341f : -INFINITY;
      const float base = fmaxf(m, sink), keep = weight(m, base);
      sum = sum * keep + weight(sink, base);
#pragma unroll
      for (int j = 0; j < 2; ++j) x[j] *= keep;
      const float inv = sum > 0.f ? 1.f / sum : (sum == 0.f ? 0.f : sum);
      const size_t to = (size_t)sequence * a.heads + head;
      typedef T T4 __attribute__((ext_vector_type(4)));
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int d = 4 * lane + 128 * j;
        if (d < D) *reinterpret_cast<T4*>(reinterpret_cast<T*>(a.out) + to * D + d) = T4{(T)(x[j][0] * inv), (T)(x[j][1] * inv), (T)(x[j][2] * inv), (T)(x[j][3] * inv)};
      }
      if (a.lse && lane == 0) a.lse[to] = log_of_sum(base, sum);
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

// A launch's workgroups and what they need to leave pieces of heads: attention_per_unit a compute unit, and no more than there
// can be units; where no column can be cut, one a column.  tokens: that a sequence can have, or that its window shows.
struct AttnPlan {
  int head_blocks, rows, workgroups;
  bool joins;
  size_t floats() const { return (size_t)workgroups * 2 * rows; }
};
static AttnPlan attention_plan(int sequences, int heads, int kv_heads, int head_dim, int format, long capacity, int window) {
  AttnPlan p;
  const int group = heads / kv_heads;
  const int row_blocks = attention_row_blocks(group);
  p.head_blocks = (group + 16 * row_blocks - 1) / (16 * row_blocks);
  p.rows = std::min(group, 16 * row_blocks);
  // (a window may begin and end inside a tile)
  const long tokens = window > 0 ? std::min((long)window + kAttnTile - 1, capacity) : capacity;
  const long units = ((tokens + kAttnTile - 1) / kAttnTile + kAttnWaves - 1) / kAttnWaves, columns = (long)sequences * kv_heads * p.head_blocks;
  // Columns of up to 16 units stay whole where there are enough of them: 1024 of 2000 tokens, fp8, 86 us, cut 114; 256 of 2000,
  // bf16, 43 and 46; 128 of 1000 17 and 20; 64 of 1000 as before, 8 of 1000 13.9 and 11.2.
  p.joins = units > (columns >= 128 ? 16 : kWholeUnits);
  p.workgroups = (int)(p.joins ? std::min<long>(kComputeUnits * attention_per_unit(head_dim, row_blocks, format), columns * units) : columns);
  return p;
}

// Costs are counted in 31 bits, and a column may be a workgroup.
bool attention_fits(int sequences, int heads, int kv_heads, long capacity) {
  const double columns = (double)sequences * kv_heads * ((heads / kv_heads + 15) / 16);
  return columns < 8388608.0 && columns * (capacity / kAttnUnit + 1 + kColumnCost) < 2147483647.0;
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
