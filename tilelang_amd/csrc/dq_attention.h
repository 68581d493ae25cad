// Attention of one new token over the paged key-value cache (layout: dq_kv.h), the cache's length split over workgroups.
//
// For a query head n and the tokens t that it sees:
//     s_t = scale q_n . k_t,   m = max_t s_t,   o = sum_t e^(s_t - m) v_t / sum_t e^(s_t - m)
// in one pass over keys and values: a wave keeps the running maximum, sum and o of its tokens and, when the maximum grows,
// scales what it has.  Partial results (m, sum, o) of waves and of workgroups are joined by the same rule, in a fixed order.
//
// The heads that share a key-value head are the columns of the matrix instruction (16x16x32, fp32 sums), 16 at a time:
//     S^T[token, head] = K[token, d] Q^T[d, head]          two instructions' rows: 32 tokens
//     O^T[d, head]    += V^T[d, token] P^T[token, head]
// The row of the first product that a lane group g = lane / 16 gets back is its own choice of token, so K's rows are
// taken in an order that hands group g the tokens 8 g .. 8 g + 7: these are the eight tokens that the second product wants
// from the same lane, P^T never leaves its registers.  V^T's operand needs eight tokens of one d in a lane; a lane loads
// eight tokens' rows at its own few d instead (a whole row of V is 16 lanes side by side) and turns the piece with byte
// permutes, so neither product passes through LDS and no wave waits for another inside the loop.
//
// A quantised cache is multiplied as fp16: a code is exact there; a query is scaled by a power of two so that its largest element
// lies in [2^14, 2^15), where bf16's range is no issue; a token's scale multiplies its score in fp32.  A weight times its
// value's scale, w_t = p_t c_t, may lie anywhere: o is kept relative to a power of two of its own, the running maximum of a
// head's w_t, as the sum is relative to the running maximum of its scores.
#pragma once

#include "dq_kv.h"

namespace dq {

constexpr int kAttnWaves = 4;
constexpr int kAttnTile = 32;  // tokens a wave takes at once

struct AttnArgs {
  const void* q;           // [sequences][heads][head_dim]
  const void* cache[2];
  const float* scale[2];
  const int* table;        // [sequences][max_pages]
  const int* lengths;      // [sequences]
  const float* sinks;      // [heads] or null
  void* out;               // [sequences][heads][head_dim]
  float* lse;              // [sequences][heads] or null
  float* part_o;           // [sequences][heads][splits][head_dim]
  float* part_ml;          // [sequences][heads][splits][2]
  float score_scale;       // scale * log2(e)
  int sequences, heads, max_pages, window, splits, head_blocks;
  CacheShape shape;
};

typedef float float2_t_ __attribute__((ext_vector_type(2)));

// ---- which elements of a row a lane holds ----------------------------------------------------------------------
// Keys (and queries): k-step s of 32 elements, group g has eight of them.  16 bit: 32 s + 8 g.  8 bit: a lane loads 16
// codes at 64 p + 16 g for steps 2 p and 2 p + 1; what is left of D behind the last 64 goes as in 16 bit.
template <int D, bool WIDE>
__device__ __forceinline__ constexpr int key_element(int step, int g) {
  const int pair = step >> 1;
  if (!WIDE && 64 * (pair + 1) <= D) return 64 * pair + 16 * g + 8 * (step & 1);
  return 32 * step + 8 * g;
}

// Values: D in blocks of 16 E elements, lane r of 16 has E of each at r E.
template <int D>
struct ValueBlocks {
  static constexpr int e(int i) {
    int rest = D / 16;
    for (int k = 0;; ++k) {
      const int e = rest >= 8 ? 8 : rest >= 4 ? 4 : rest >= 2 ? 2 : rest;
      if (k == i) return e;
      rest -= e;
    }
  }
  static constexpr int start(int i) {
    int at = 0;
    for (int k = 0; k < i; ++k) at += 16 * e(k);
    return at;
  }
  static constexpr int count() {
    int n = 0, rest = D / 16;
    while (rest > 0) {
      rest -= rest >= 8 ? 8 : rest >= 4 ? 4 : rest >= 2 ? 2 : rest;
      ++n;
    }
    return n;
  }
  // dwords of one token that a lane holds of blocks before i
  static constexpr int dword(int i, int bytes) {
    int n = 0;
    for (int k = 0; k < i; ++k) n += (e(k) * bytes + 3) / 4;
    return n;
  }
};

template <class T>
__device__ __forceinline__ float4_t mfma16(typename Vec8<T>::type a, typename Vec8<T>::type b, float4_t c) {
  if constexpr (__is_same(T, half_t)) return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// Four codes (a dword) -> four fp16, exact.
template <int FORMAT>
__device__ __forceinline__ void codes4_to_half(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if constexpr (FORMAT == CACHE_FP8) {
    lo = as_u32(__builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, false));
    hi = as_u32(__builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, true));
  } else {
    // code + 128 in the last byte of an fp16 whose last place is 1: 1024 + 128 + code
    const uint32_t u = w ^ 0x80808080u;
    const half2_t bias = {(half_t)1152.f, (half_t)1152.f};
    lo = as_u32(as_half2(__builtin_amdgcn_perm(0x64646464u, u, 0x04010400u)) - bias);
    hi = as_u32(as_half2(__builtin_amdgcn_perm(0x64646464u, u, 0x04030402u)) - bias);
  }
}

__device__ __forceinline__ float max_over_groups(float x) {
  x = fmaxf(x, __shfl_xor(x, 16));
  return fmaxf(x, __shfl_xor(x, 32));
}
__device__ __forceinline__ float sum_over_groups(float x) {
  x += __shfl_xor(x, 16);
  return x + __shfl_xor(x, 32);
}

// 2^(m - to), 0 where there is nothing (m = -inf), whatever `to` is
__device__ __forceinline__ float weight(float m, float to) { return m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - to); }

// T: queries and output; FORMAT: the cache; D: head_dim; NT: blocks of 16 heads that a workgroup takes
template <class T, int FORMAT, int D, int NT>
__global__ __launch_bounds__(64 * kAttnWaves, 2) void attention_kernel(const AttnArgs a) {
  constexpr bool kWide = cache_is_16bit(FORMAT);
  using C = typename std::conditional<kWide, T, half_t>::type;  // what the products are taken in
  typedef typename Vec8<C>::type C8;
  constexpr int kBytes = kWide ? 2 : 1;
  constexpr int kSteps = (D + 31) / 32;
  using VB = ValueBlocks<D>;
  constexpr int kVDwords = VB::dword(VB::count(), kBytes);
  constexpr int kAcc = D / 16;
  constexpr int kKeyDwords = kWide ? 4 : 2;  // of one k-step

  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
  const int split = blockIdx.x, kv_head = blockIdx.y / a.head_blocks, head_block = blockIdx.y - kv_head * a.head_blocks;
  const int sequence = blockIdx.z;
  const int group = a.heads / a.shape.kv_heads;  // heads that share kv_head

  const int capacity = a.max_pages << a.shape.page_shift;
  const int length = min(max(a.lengths[sequence], 0), capacity);
  const int first_token = a.window > 0 ? max(0, length - a.window) : 0;
  const int tile0 = first_token / kAttnTile, tiles_all = (length + kAttnTile - 1) / kAttnTile - tile0;
  // this split's tiles, whole rounds of the workgroup's waves
  const int per = ((tiles_all + a.splits - 1) / a.splits + kAttnWaves - 1) / kAttnWaves * kAttnWaves;
  const int begin = tile0 + split * per, end = min(begin + per, tile0 + tiles_all);

  // ---- queries: the second operand of the first product, held for the whole walk -----------------------------
  C8 q[NT][kSteps];
  float q_scale[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int row = (head_block * NT + t) * 16 + n;
    const T* const qrow = reinterpret_cast<const T*>(a.q) + ((size_t)sequence * a.heads + (size_t)kv_head * group + row) * D;
    float f[kSteps][8];
    float most = 0.f;
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      const int d = key_element<D, kWide>(s, g);
      typename Vec8<T>::type h = {};
      if (row < group && d < D) h = *reinterpret_cast<const typename Vec8<T>::type*>(qrow + d);
      if constexpr (kWide) {
        q[t][s] = h;
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) f[s][i] = (float)h[i], most = fmaxf(most, fabsf(f[s][i]));
      }
    }
    q_scale[t] = a.score_scale;
    if constexpr (!kWide) {
      most = max_over_groups(most);
      const int e = most > 0.f ? 14 - ilogbf(most) : 0;  // 2^e * most in [2^14, 2^15)
      const int shift = min(max(e, -126), 126);
      q_scale[t] = ldexpf(a.score_scale, -shift);
#pragma unroll
      for (int s = 0; s < kSteps; ++s)
#pragma unroll
        for (int i = 0; i < 8; ++i) q[t][s][i] = (C)ldexpf(f[s][i], shift);
    }
  }

  float4_t acc[NT][kAcc];
  float m[NT], l[NT];
  float o_ref[NT];  // acc is o / 2^o_ref (quantised caches; else 2^m)
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    m[t] = -INFINITY, l[t] = 0.f, o_ref[t] = -INFINITY;
#pragma unroll
    for (int i = 0; i < kAcc; ++i) acc[t][i] = float4_t{0.f, 0.f, 0.f, 0.f};
  }

  const int place_mask = (1 << a.shape.page_shift) - 1;
  const int* const table = a.table + (size_t)sequence * a.max_pages;

  for (int tile = begin + wave; tile < end; tile += kAttnWaves) {
    // the eight tokens whose keys (values) this lane reads, their page, whether it is there
    const int k_first = tile * kAttnTile + (n >> 2) * 8, v_first = tile * kAttnTile + g * 8;
    int k_page = -1, v_page = -1;
    if (k_first < length) k_page = table[k_first >> a.shape.page_shift];
    if (v_first < length) v_page = table[v_first >> a.shape.page_shift];
    const bool k_there = (unsigned)k_page < (unsigned)a.shape.pages, v_there = (unsigned)v_page < (unsigned)a.shape.pages;
    const size_t k_row = cache_row(a.shape, k_there ? k_page : 0, kv_head, (k_first & place_mask) + (n & 3));
    const size_t v_row = cache_row(a.shape, v_there ? v_page : 0, kv_head, v_first & place_mask);
    const char* const kp = reinterpret_cast<const char*>(a.cache[0]) + k_row * (D * kBytes);
    const char* const vp = reinterpret_cast<const char*>(a.cache[1]) + v_row * (D * kBytes);

    uint32_t kr[2][kSteps][kKeyDwords];
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        const char* const p = kp + t * 4 * D * kBytes + key_element<D, kWide>(s, g) * kBytes;
        if constexpr (!kWide) {
          if (64 * ((s >> 1) + 1) <= D) {
            if (s & 1) continue;
            const uint4_t w = *reinterpret_cast<const uint4_t*>(p);
            kr[t][s][0] = w[0], kr[t][s][1] = w[1], kr[t][s + 1][0] = w[2], kr[t][s + 1][1] = w[3];
            continue;
          }
          uint2_t w = {0u, 0u};
          if (32 * (s + 1) <= D || key_element<D, kWide>(s, g) < D) w = *reinterpret_cast<const uint2_t*>(p);
          kr[t][s][0] = w[0], kr[t][s][1] = w[1];
        } else {
          uint4_t w = {0u, 0u, 0u, 0u};
          if (32 * (s + 1) <= D || key_element<D, kWide>(s, g) < D) w = *reinterpret_cast<const uint4_t*>(p);
#pragma unroll
          for (int i = 0; i < 4; ++i) kr[t][s][i] = w[i];
        }
      }
    uint32_t vr[8][kVDwords];
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int b = 0; b < VB::count(); ++b) {
        constexpr int kNone = 0;
        (void)kNone;
        const int e = VB::e(b), at = VB::dword(b, kBytes);
        const char* const p = vp + (j * D + VB::start(b) + n * e) * kBytes;
        const int bytes = e * kBytes;
        if (bytes == 16) {
          const uint4_t w = *reinterpret_cast<const uint4_t*>(p);
          vr[j][at] = w[0], vr[j][at + 1] = w[1], vr[j][at + 2] = w[2], vr[j][at + 3] = w[3];
        } else if (bytes == 8) {
          const uint2_t w = *reinterpret_cast<const uint2_t*>(p);
          vr[j][at] = w[0], vr[j][at + 1] = w[1];
        } else if (bytes == 4) {
          vr[j][at] = *reinterpret_cast<const uint32_t*>(p);
        } else if (bytes == 2) {
          vr[j][at] = *reinterpret_cast<const uint16_t*>(p);
        } else {
          vr[j][at] = *reinterpret_cast<const uint8_t*>(p);
        }
      }
    float ks[8], vs[8];
    if constexpr (!kWide) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float4_t kq = *reinterpret_cast<const float4_t*>(a.scale[0] + v_row + 4 * i), vq = *reinterpret_cast<const float4_t*>(a.scale[1] + v_row + 4 * i);
#pragma unroll
        for (int j = 0; j < 4; ++j) ks[4 * i + j] = kq[j], vs[4 * i + j] = vq[j];
      }
    }

    // the tokens v_first + j that take part
    const int low = max(first_token - v_first, 0), high = v_there ? min(length - v_first, 8) : 0;
    const bool whole = __all(low == 0 && high == 8);
    if (!whole) {
      // what lies in dead places may be anything: its values count as zeros, not as zero times them
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (j >= low && j < high) continue;
#pragma unroll
        for (int i = 0; i < kVDwords; ++i) vr[j][i] = 0u;
        if constexpr (!kWide) ks[j] = 0.f, vs[j] = 0.f;
      }
    }

    // ---- scores ---------------------------------------------------------------------------------------------
    float p[NT][8];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      C8 kf[kSteps];
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        uint4_t w;
        if constexpr (kWide) {
          w = uint4_t{kr[t][s][0], kr[t][s][1], kr[t][s][2], kr[t][s][3]};
        } else {
          uint32_t h[4];
          codes4_to_half<FORMAT>(kr[t][s][0], h[0], h[1]);
          codes4_to_half<FORMAT>(kr[t][s][1], h[2], h[3]);
          w = uint4_t{h[0], h[1], h[2], h[3]};
        }
        kf[s] = __builtin_bit_cast(C8, w);
      }
#pragma unroll
      for (int b = 0; b < NT; ++b) {
        float4_t sc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < kSteps; ++s) sc = mfma16<C>(kf[s], q[b][s], sc);
#pragma unroll
        for (int i = 0; i < 4; ++i) p[b][4 * t + i] = sc[i];
      }
    }
    // ---- running maximum and sum ----------------------------------------------------------------------------
#pragma unroll
    for (int b = 0; b < NT; ++b) {
      float most = -INFINITY;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        p[b][j] *= q_scale[b];
        if constexpr (!kWide) p[b][j] *= ks[j];
        if (!whole && (j < low || j >= high)) p[b][j] = -INFINITY;
        most = fmaxf(most, p[b][j]);
      }
      most = fmaxf(m[b], max_over_groups(most));
      const float base = most == -INFINITY ? 0.f : most;
      float shrink = weight(m[b], base);
      m[b] = most;
      l[b] *= shrink;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        p[b][j] = __builtin_amdgcn_exp2f(p[b][j] - base);
        l[b] += p[b][j];
      }
      if constexpr (!kWide) {
        float top = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) p[b][j] *= vs[j], top = fmaxf(top, p[b][j]);
        top = max_over_groups(top);
        const float ref = fmaxf(o_ref[b], top > 0.f ? base + (float)__builtin_amdgcn_frexp_expf(top) : -INFINITY);
        const float factor = ref == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(base - ref);
        shrink = weight(o_ref[b], ref);
        o_ref[b] = ref;
#pragma unroll
        for (int j = 0; j < 8; ++j) p[b][j] *= factor;
      }
#pragma unroll
      for (int i = 0; i < kAcc; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k) acc[b][i][k] *= shrink;
    }
    C8 pf[NT];
#pragma unroll
    for (int b = 0; b < NT; ++b)
#pragma unroll
      for (int j = 0; j < 8; ++j) pf[b][j] = (C)p[b][j];
    // ---- values ---------------------------------------------------------------------------------------------
    int at_acc = 0;
#pragma unroll
    for (int blk = 0; blk < VB::count(); ++blk) {
      const int e_count = VB::e(blk), at = VB::dword(blk, kBytes);
      if constexpr (kWide) {
#pragma unroll
        for (int e = 0; e < e_count; ++e) {
          uint4_t w;
#pragma unroll
          for (int i = 0; i < 4; ++i)
            w[i] = __builtin_amdgcn_perm(vr[2 * i + 1][at + (e >> 1)], vr[2 * i][at + (e >> 1)], (e & 1) ? 0x07060302u : 0x05040100u);
#pragma unroll
          for (int b = 0; b < NT; ++b) acc[b][at_acc + e] = mfma16<C>(__builtin_bit_cast(C8, w), pf[b], acc[b][at_acc + e]);
        }
      } else {
#pragma unroll
        for (int dw = 0; dw < (e_count + 3) / 4; ++dw) {
          uint4_t tr[2];  // byte e of four tokens
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const uint4_t w = {vr[4 * half][at + dw], vr[4 * half + 1][at + dw], vr[4 * half + 2][at + dw], vr[4 * half + 3][at + dw]};
            tr[half] = transpose4x4_bytes(w);
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            if (4 * dw + e >= e_count) break;
            uint32_t h[4];
            codes4_to_half<FORMAT>(tr[0][e], h[0], h[1]);
            codes4_to_half<FORMAT>(tr[1][e], h[2], h[3]);
            const uint4_t w = {h[0], h[1], h[2], h[3]};
#pragma unroll
            for (int b = 0; b < NT; ++b)
              acc[b][at_acc + 4 * dw + e] = mfma16<C>(__builtin_bit_cast(C8, w), pf[b], acc[b][at_acc + 4 * dw + e]);
          }
        }
      }
      at_acc += e_count;
    }
  }

  // ---- the waves' results, joined in their order -----------------------------------------------------------------
  __shared__ float sm[kAttnWaves][16 * NT][3];
  extern __shared__ float so[];  // [waves][16 heads][D + 4]
  constexpr int kRow = D + 4;
#pragma unroll
  for (int b = 0; b < NT; ++b) {
    l[b] = sum_over_groups(l[b]);
    if (g == 0) sm[wave][16 * b + n][0] = m[b], sm[wave][16 * b + n][1] = l[b], sm[wave][16 * b + n][2] = kWide ? m[b] : o_ref[b];
  }
  for (int b = 0; b < NT; ++b) {
    __syncthreads();
    int at_acc = 0;
#pragma unroll
    for (int blk = 0; blk < VB::count(); ++blk) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < VB::e(blk); ++e) {
          const int d = VB::start(blk) + (4 * g + i) * VB::e(blk) + e;
          so[(wave * 16 + n) * kRow + d] = acc[b][at_acc + e][i];
        }
      at_acc += VB::e(blk);
    }
    __syncthreads();
    // 16 lanes a head
    const int row = threadIdx.x >> 4, head_in_group = (head_block * NT + b) * 16 + row;
    if (head_in_group < group) {
      const int head = kv_head * group + head_in_group;
      float most = -INFINITY;
#pragma unroll
      for (int w = 0; w < kAttnWaves; ++w) most = fmaxf(most, sm[w][16 * b + row][0]);
      const float sink = a.splits == 1 && a.sinks ? a.sinks[head] * 1.44269504088896341f : -INFINITY;
      const float base = fmaxf(most, sink);
      float factor[kAttnWaves], sum = weight(sink, base);
#pragma unroll
      for (int w = 0; w < kAttnWaves; ++w) {
        factor[w] = weight(sm[w][16 * b + row][2], base);
        sum += weight(sm[w][16 * b + row][0], base) * sm[w][16 * b + row][1];
      }
      const size_t at = (size_t)sequence * a.heads + head;
      if (a.splits == 1) {
        const float inv = sum > 0.f ? 1.f / sum : (sum == 0.f ? 0.f : sum);
        for (int d = threadIdx.x & 15; d < D; d += 16) {
          float x = 0.f;
#pragma unroll
          for (int w = 0; w < kAttnWaves; ++w) x += factor[w] * so[(w * 16 + row) * kRow + d];
          reinterpret_cast<T*>(a.out)[at * D + d] = (T)(x * inv);
        }
        if (a.lse && (threadIdx.x & 15) == 0)
          a.lse[at] = base == -INFINITY ? -INFINITY : (base + log2f(sum)) * 0.693147180559945309f;
      } else {
        const size_t part = at * a.splits + split;
        if (most != -INFINITY) {
          for (int d = threadIdx.x & 15; d < D; d += 16) {
            float x = 0.f;
#pragma unroll
            for (int w = 0; w < kAttnWaves; ++w) x += factor[w] * so[(w * 16 + row) * kRow + d];
            a.part_o[part * D + d] = x;
          }
        }
        if ((threadIdx.x & 15) == 0) a.part_ml[2 * part] = most, a.part_ml[2 * part + 1] = sum;
      }
    }
  }
}

template <class T, int FORMAT, int D, int NT>
int launch_attention(const AttnArgs& a, hipStream_t stream) {
  constexpr int kLds = kAttnWaves * 16 * (D + 4) * 4;
  if constexpr (kLds > 65536 - 4096) {
    static bool raised[kMaxDevices];
    if (raise_lds_limit<kLds>(attention_kernel<T, FORMAT, D, NT>, raised) != 0) return -1;
  }
  attention_kernel<T, FORMAT, D, NT><<<dim3(a.splits, a.shape.kv_heads * a.head_blocks, a.sequences), 64 * kAttnWaves, kLds, stream>>>(a);
  DQ_CHECK_HIP(hipGetLastError());
  return 0;
}

template <class T, int FORMAT>
int attention_of_type(const AttnArgs& a, hipStream_t stream) {
  switch (a.shape.head_dim) {
    case 64: return launch_attention<T, FORMAT, 64, 1>(a, stream);
    case 80: return launch_attention<T, FORMAT, 80, 1>(a, stream);
    case 96: return launch_attention<T, FORMAT, 96, 1>(a, stream);
    case 112: return launch_attention<T, FORMAT, 112, 1>(a, stream);
    case 128: return launch_attention<T, FORMAT, 128, 1>(a, stream);
    case 160: return launch_attention<T, FORMAT, 160, 1>(a, stream);
    case 192: return launch_attention<T, FORMAT, 192, 1>(a, stream);
    case 256: return launch_attention<T, FORMAT, 256, 1>(a, stream);
    default: DQ_FAIL("attention: no kernel for a head of %d", a.shape.head_dim);
  }
}

}  // namespace dq
