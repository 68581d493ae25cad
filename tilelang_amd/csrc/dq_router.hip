// The router's logits: Logits[t][e] = X[t] . W[e] + bias, for some tokens and up to 1024 experts, fp16 or bf16 -> fp32.
//
// A product of so few columns that tiles of a GEMM leave most of the chip idle and walk K alone.  Here a workgroup has up to 16 MB tokens
// and 16 NB experts, and K is cut over its waves: wave w takes blocks w, w + WAVES, ... of 128 k, whose operands it loads from memory (or
// the L2 cache) into the registers that the matrix instruction reads, 64 bytes of a row a lane group, all of a block at once.  The
// waves' sums meet in LDS and are added in their order.
//
// What bounds it is a CU's load unit, about 41 bytes a nanosecond for one workgroup, and 8.7 TB/s for all: at few tokens a workgroup has
// fewer than 16 tokens and experts, whose rows the others of the matrix instruction repeat (repeated rows are one load), at many more,
// for fewer loads a product.  Measured, K = 4096, 128 experts, us, 16 x 16 / 32 x 16 / 32 x 32 / 64 x 32: 16 tokens 8.8 / 9.7 / 13.2 / 15.3;
// 1024 tokens 16.9 / 12.8 / 16.2 / 23.2; 4096 tokens 62 / 46 / 30 / 24 (the tiled GEMM of call_gemm_plain: 33.5, 34.3 and 34.3).
#include "dq_kv.h"

#include <algorithm>

namespace dq {

namespace {

constexpr int kBlock = 128;  // k

template <class T>
struct Mfma16;
template <>
struct Mfma16<half_t> {
  using frag = half8_t;
  __device__ static __forceinline__ float4_t mfma(frag a, frag b, float4_t c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
};
template <>
struct Mfma16<bf16_t> {
  using frag = bf16x8_t;
  __device__ static __forceinline__ float4_t mfma(frag a, frag b, float4_t c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
};

template <class T, int MB, int NB, int WAVES>
__global__ __launch_bounds__(WAVES * 64) void router_kernel(const T* __restrict__ X, const T* __restrict__ W, const T* __restrict__ Bias,
                                                             float* __restrict__ Logits, int tokens, int experts, int K, int own_tokens, int own_experts) {
  using frag = typename Mfma16<T>::frag;
  __shared__ float4_t sums[WAVES][MB * NB][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, r = lane & 15;
  const int t0 = blockIdx.x * own_tokens, t1 = min(t0 + own_tokens, tokens), e0 = blockIdx.y * own_experts, e1 = min(e0 + own_experts, experts);
  // (rows beyond the last repeat it; what they give is not stored)
  const T *a[MB], *b[NB];
#pragma unroll
  for (int i = 0; i < MB; ++i) a[i] = X + (size_t)min(t0 + 16 * i + r, t1 - 1) * K + 8 * g;
#pragma unroll
  for (int j = 0; j < NB; ++j) b[j] = W + (size_t)min(e0 + 16 * j + r, e1 - 1) * K + 8 * g;
  float4_t acc[MB][NB] = {};
  // (unsigned: with K next to 2^31 the step beyond it passes that)
  for (unsigned k0 = wave * kBlock; k0 < (unsigned)K; k0 += WAVES * kBlock) {
    frag x[4][MB], w[4][NB];
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      // (K is a multiple of 32: a step is there as a whole or not at all)
      const unsigned k = k0 + 32 * s;
      if (k < (unsigned)K) {
#pragma unroll
        for (int i = 0; i < MB; ++i) x[s][i] = *reinterpret_cast<const frag*>(a[i] + k);
#pragma unroll
        for (int j = 0; j < NB; ++j) w[s][j] = *reinterpret_cast<const frag*>(b[j] + k);
      } else {
#pragma unroll
        for (int i = 0; i < MB; ++i) x[s][i] = frag{};
#pragma unroll
        for (int j = 0; j < NB; ++j) w[s][j] = frag{};
      }
    }
#pragma unroll
    for (int s = 0; s < 4; ++s)
#pragma unroll
      for (int i = 0; i < MB; ++i)
#pragma unroll
        for (int j = 0; j < NB; ++j) acc[i][j] = Mfma16<T>::mfma(x[s][i], w[s][j], acc[i][j]);
  }
#pragma unroll
  for (int i = 0; i < MB; ++i)
#pragma unroll
    for (int j = 0; j < NB; ++j) sums[wave][i * NB + j][lane] = acc[i][j];
  __syncthreads();
  // a wave a block of 16 x 16: lane (g, r) has expert r of it, tokens 4 g .. 4 g + 3
  for (int block = wave; block < MB * NB; block += WAVES) {
    const int i = block / NB, j = block % NB, e = e0 + 16 * j + r;
    float4_t v = sums[0][block][lane];
#pragma unroll
    for (int n = 1; n < WAVES; ++n) v += sums[n][block][lane];
    if (e >= e1) continue;
    const float add = Bias == nullptr ? 0.f : (float)Bias[e];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int t = t0 + 16 * i + 4 * g + q;
      if (t < t1) Logits[(size_t)t * experts + e] = v[q] + add;
    }
  }
}

struct Call {
  const void *X, *W, *Bias;
  float* Logits;
  int tokens, experts, K;
  hipStream_t stream;
};

template <class T, int MB, int NB, int WAVES>
int launch(const Call& c, int own_tokens, int own_experts) {
  hipLaunchKernelGGL((router_kernel<T, MB, NB, WAVES>), dim3((c.tokens + own_tokens - 1) / own_tokens, (c.experts + own_experts - 1) / own_experts), dim3(WAVES * 64),
                     0, c.stream, (const T*)c.X, (const T*)c.W, (const T*)c.Bias, c.Logits, c.tokens, c.experts, c.K, own_tokens, own_experts);
  DQ_CHECK_HIP(hipGetLastError());
  return 0;
}

template <class T>
int by_size(const Call& c) {
  // what a split would take, in bytes of one workgroup's rows of K
  auto workgroups = [&](int t, int e) { return (double)((c.tokens + t - 1) / t) * ((c.experts + e - 1) / e); };
  auto cost = [&](int t, int e) { return (std::min(t, c.tokens) + std::min(e, c.experts)) * std::max(1.0, workgroups(t, e) * 41 / 8700); };
  const double small = cost(16, 16), tall = cost(32, 16), square = cost(32, 32), large = cost(64, 32);
  if (large < std::min(small, std::min(tall, square))) return launch<T, 4, 2, 8>(c, 64, 32);
  if (square < std::min(small, tall)) return launch<T, 2, 2, 8>(c, 32, 32);
  if (tall < small) return launch<T, 2, 1, 16>(c, 32, 16);
  // the larger side halved while there are no more workgroups than CUs
  int t = std::min(16, c.tokens), e = std::min(16, c.experts);
  while (std::max(t, e) > 2) {
    const int t2 = t >= e ? (t + 1) / 2 : t, e2 = t >= e ? e : (e + 1) / 2;
    if (workgroups(t2, e2) > 256) break;
    t = t2, e = e2;
  }
  return launch<T, 1, 1, 16>(c, t, e);
}

}  // namespace

int router_logits(const void* X, const void* W, const void* Bias, float* Logits, int tokens, int experts, int K, int bf16, hipStream_t stream) {
  const Call c{X, W, Bias, Logits, tokens, experts, K, stream};
  return bf16 ? by_size<bf16_t>(c) : by_size<half_t>(c);
}

}  // namespace dq
