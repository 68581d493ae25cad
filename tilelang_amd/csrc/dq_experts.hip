// The experts' products at a few rows an expert: a workgroup has 16 weight rows of the gate and the 16 of the up projection (or 32
// weight rows) of one expert and multiplies them with up to 16 of its rows at a time.
//
// What bounds it is the weights' way out of memory: every expert that has rows is read once.  K is cut over the workgroup's waves,
// whose sums meet in LDS.  A lane reads 16 bytes of a weight row at a time, 32 k; the matrix instruction's k are labelled
// 32 g + 8 j + e for its lane group g and the j-th of four instructions, for both operands, so that the weights go into it as
// they lie and the activations of a lane are 64 contiguous bytes.
#include "dq_experts.h"

namespace dq {

int experts_tiles(const experts::Args& a, int mxfp4, bool up, int tile_rows, hipStream_t stream);

namespace {

using experts::Args;

constexpr int kStep = 128;  // k of a step: 32 a lane group

// The `nth` expert that has rows, or false.  Every wave finds it by itself.
__device__ __forceinline__ bool nth_expert(const Args& a, int nth, int& expert, int& begin, int& end) {
  const int lane = threadIdx.x & 63;
  for (int base = 0; base < a.experts; base += 64) {
    int b = 0, e = 0;
    if (base + lane < a.experts) experts::rows_of(a, base + lane, b, e);
    unsigned long long has = __ballot(e > b);
    const int count = __popcll(has);
    if (nth < count) {
      for (; nth > 0; --nth) has &= has - 1;
      const int at = __builtin_ctzll(has);
      expert = base + at;
      begin = __builtin_amdgcn_readlane(b, at);
      end = __builtin_amdgcn_readlane(e, at);
      return true;
    }
    nth -= count;
  }
  return false;
}

template <class W, bool UP, int WAVES>
__global__ __launch_bounds__(WAVES * 64) void rows_kernel(const Args a) {
  using T = typename W::T;
  typedef T vec __attribute__((ext_vector_type(8)));
  __shared__ float4_t sums[WAVES][2][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int g = lane >> 4, c = lane & 15;
  int expert, begin, end;
  if (!nth_expert(a, blockIdx.y, expert, begin, end)) return;
  const int rows = (UP ? 2 : 1) * a.N;  // weight rows of an expert
  const int n0 = blockIdx.x * (UP ? 16 : 32);
  size_t w_row[2];
  w_row[0] = (size_t)expert * rows + n0 + c;
  w_row[1] = w_row[0] + (UP ? a.N : 16);
  const size_t row_bytes = (size_t)a.K >> 1;

  for (int r0 = begin; r0 < end; r0 += 16) {
    const int row = r0 + c;
    const bool there = row < end;
    const T* x = (const T*)a.A;
    if (there) {
      int at = row;
      if constexpr (UP) at = min((unsigned)a.Order[row] / (unsigned)a.top_k, (unsigned)a.tokens - 1);
      x += (size_t)at * a.K;
    }
    float4_t acc[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
    for (int k0 = wave * kStep; k0 < a.K; k0 += WAVES * kStep) {
      const int k = k0 + 32 * g;
      const bool inside = k < a.K;  // (K is a multiple of 32)
      vec xv[4];
      uint4_t words[2];
      typename W::Raw raw[2];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        xv[j] = vec{};
        if (there && inside) xv[j] = *reinterpret_cast<const vec*>(x + k + 8 * j);
      }
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        words[t] = uint4_t{};
        const int ks = inside ? k : 0;
        if (inside) words[t] = *reinterpret_cast<const uint4_t*>(a.B + w_row[t] * row_bytes + (k >> 1));
        raw[t] = W::fetch(a, w_row[t], ks);
      }
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const typename W::Scale s = W::scale(raw[t]);
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[t] = W::mfma(__builtin_bit_cast(typename W::frag, xv[j]), W::decode(words[t][j], s), acc[t]);
      }
    }
    if (r0 != begin) __syncthreads();  // (the sums before are read)
    sums[wave][0][lane] = acc[0];
    sums[wave][1][lane] = acc[1];
    __syncthreads();
    // one value a thread: [tile][lane][4]
    const float* const all = (const float*)sums;
    if constexpr (UP) {
      for (int i = threadIdx.x; i < 256; i += WAVES * 64) {
        const int m = i >> 4, n = i & 15, at = ((m >> 2) * 16 + n) * 4 + (m & 3);
        float v[2] = {0.f, 0.f};
#pragma unroll
        for (int w = 0; w < WAVES; ++w) v[0] += all[w * 512 + at], v[1] += all[w * 512 + 256 + at];
        if (a.Bias != nullptr) {
          const T* bias = (const T*)a.Bias + (size_t)expert * rows + n0 + n;
          v[0] += (float)bias[0];
          v[1] += (float)bias[a.N];
        }
        if (r0 + m < end) ((T*)a.Out)[(size_t)(r0 + m) * a.N + n0 + n] = (T)(experts::activate(v[0], a.gelu) * v[1]);
      }
    } else {
      for (int i = threadIdx.x; i < 512; i += WAVES * 64) {
        const int m = i >> 5, n = i & 31, at = (n >> 4) * 256 + ((m >> 2) * 16 + (n & 15)) * 4 + (m & 3);
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) v += all[w * 512 + at];
        if (a.Bias != nullptr) v += (float)((const T*)a.Bias)[(size_t)expert * rows + n0 + n];
        if (r0 + m < end) {
          const unsigned pair = a.Order[r0 + m];
          if (pair < (unsigned)a.pairs) a.Parts[(size_t)pair * a.N + n0 + n] = v * a.Weights[pair];
        }
      }
    }
  }
}

// A token's pairs added, in the order of its choices, onto the residual.
template <class T>
__global__ __launch_bounds__(256) void sum_kernel(const Args a) {
  typedef T vec4 __attribute__((ext_vector_type(4)));
  const size_t at = ((size_t)blockIdx.x * 256 + threadIdx.x) * 4;
  const size_t token = at / a.N;
  const int n = (int)(at - token * a.N);
  if (token >= (size_t)a.tokens) return;
  float4_t v = {0.f, 0.f, 0.f, 0.f};
  for (int j = 0; j < a.top_k; ++j) {
    const size_t pair = token * a.top_k + j;
    if ((unsigned)a.Ids[pair] - (unsigned)a.first < (unsigned)a.experts) v += *reinterpret_cast<const float4_t*>(a.Parts + pair * a.N + n);
  }
  if (a.Residual != nullptr) {
    const vec4 r = *reinterpret_cast<const vec4*>((const T*)a.Residual + at);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] += (float)r[i];
  }
  vec4 o;
#pragma unroll
  for (int i = 0; i < 4; ++i) o[i] = (T)v[i];
  *reinterpret_cast<vec4*>((T*)a.Out + at) = o;
}

template <class T>
int sum(const Args& a, hipStream_t stream) {
  const size_t threads = (size_t)a.tokens * a.N / 4;
  hipLaunchKernelGGL((sum_kernel<T>), dim3((unsigned)((threads + 255) / 256)), dim3(256), 0, stream, a);
  DQ_CHECK_HIP(hipGetLastError());
  return 0;
}

template <class W, bool UP>
int product(const Args& a, hipStream_t stream) {
  constexpr int kWaves = 4;
  const int most = a.experts < a.pairs ? a.experts : a.pairs;  // experts that can have rows
  hipLaunchKernelGGL((rows_kernel<W, UP, kWaves>), dim3(a.N / (UP ? 16 : 32), most), dim3(kWaves * 64), 0, stream, a);
  DQ_CHECK_HIP(hipGetLastError());
  if constexpr (!UP) return sum<typename W::T>(a, stream);
  return 0;
}

// Rows of a tile of the matrix pipe's kernel, or 0: few rows an expert.
int tile_rows(const Args& a, int mxfp4) {
  if (a.K < 128) return 0;
  const long mean = a.pairs / (a.experts < a.pairs ? a.experts : a.pairs);
  if (mean < 48) return 0;
  const bool tall = mxfp4 || a.group_shift > 5;
  return tall && mean >= 512 ? 256 : 128;
}

template <bool UP>
int by_format(const Args& a, int mxfp4, hipStream_t stream) {
  if (const int rows = tile_rows(a, mxfp4)) {
    if (const int rc = experts_tiles(a, mxfp4, UP, rows, stream)) return rc;
    if constexpr (!UP) return mxfp4 ? sum<bf16_t>(a, stream) : sum<half_t>(a, stream);
    return 0;
  }
  if (mxfp4) return product<experts::Mxfp4, UP>(a, stream);
  return a.Z != nullptr ? product<experts::Uint4<true>, UP>(a, stream) : product<experts::Uint4<false>, UP>(a, stream);
}

}  // namespace

size_t experts_down_workspace_bytes(int tokens, int top_k, int N) { return (size_t)tokens * top_k * N * 4; }

int experts_up(const Args& a, int mxfp4, hipStream_t stream) { return by_format<true>(a, mxfp4, stream); }
int experts_down(const Args& a, int mxfp4, hipStream_t stream) { return by_format<false>(a, mxfp4, stream); }

}  // namespace dq
