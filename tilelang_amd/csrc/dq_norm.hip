// Root-mean-square norm with the residual's addition: h = x + r, y = w h / sqrt(mean h^2 + eps), and y as it is or as int8 codes
// with a scale a row.
//
// A row stays in registers between the sum of its squares and its product (8-bit output: and its largest magnitude), so that
// everything is read once and written once: what bounds it is memory, or, at a few rows, one pass through it.  A row belongs to
// LANES lanes, NV pieces of eight elements each, piece i of lane l at 8 (i LANES + l).  LANES is 16 or 64, several rows a workgroup
// and no barrier, or all of a workgroup of 256 or 1024, whose waves meet in LDS once a reduction.
//
// Measured: 7999 x 5120 bf16 with a residual 63 us, 5.2 TB/s, what a copy reaches here; 2048 x 8192 fp16 with a residual to int8 23.5 us,
// 5.0 TB/s; one row of 4096 2.3 to 2.5 us, of which an empty launch is 2.0.
#include "dq_kv.h"

namespace dq {

namespace {

// Sum or largest of a value over LANES neighbouring lanes (of one wave); every lane gets it.
template <int LANES, bool MAX>
__device__ __forceinline__ float over_lanes(float v) {
#pragma unroll
  for (int d = 1; d < LANES; d *= 2) {
    const float o = __shfl_xor(v, d, 64);
    v = MAX ? fmaxf(v, o) : v + o;
  }
  return v;
}

// ... over the row's lanes.  `slots`: a float a wave, used once.
template <int LANES, bool MAX>
__device__ __forceinline__ float over_row(float v, float* slots) {
  if constexpr (LANES <= 64) {
    return over_lanes<LANES, MAX>(v);
  } else {
    v = over_lanes<64, MAX>(v);
    if ((threadIdx.x & 63) == 0) slots[threadIdx.x >> 6] = v;
    __syncthreads();
    float all = slots[0];
#pragma unroll
    for (int i = 1; i < LANES / 64; ++i) all = MAX ? fmaxf(all, slots[i]) : all + slots[i];
    return all;
  }
}

template <class T, int LANES, int NV, bool RESIDUAL, bool INT8>
__global__ __launch_bounds__(LANES <= 64 ? 256 : LANES) void norm_kernel(const T* __restrict__ X, const T* __restrict__ Residual,
                                                                         const T* __restrict__ Weight, void* __restrict__ Y, T* __restrict__ Sum,
                                                                         float* __restrict__ Scale, int rows, int dim, long row_stride, float eps) {
  using vec = typename Vec8<T>::type;
  constexpr int kRows = LANES <= 64 ? 256 / LANES : 1;  // a workgroup's
  __shared__ float slots[4][16];
  const int lane = threadIdx.x % LANES;
  const long row = ((long)blockIdx.y * gridDim.x + blockIdx.x) * kRows + threadIdx.x / LANES;
  if (row >= rows) return;  // (one row a workgroup where there is a barrier)
  const int pieces = dim >> 3;

  vec xv[NV], rv[NV], wv[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int at = i * LANES + lane;
    if (at < pieces) {
      xv[i] = *reinterpret_cast<const vec*>(X + row * row_stride + 8 * at);
      if constexpr (RESIDUAL) rv[i] = *reinterpret_cast<const vec*>(Residual + row * dim + 8 * at);
    }
  }
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int at = i * LANES + lane;
    if (at < pieces) wv[i] = *reinterpret_cast<const vec*>(Weight + 8 * at);
  }
  float h[NV][8];
  float squares = 0.f, largest = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int at = i * LANES + lane;
#pragma unroll
    for (int e = 0; e < 8; ++e) h[i][e] = 0.f;
    if (at < pieces) {
      vec s;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        h[i][e] = (float)xv[i][e];
        if constexpr (RESIDUAL) h[i][e] += (float)rv[i][e], s[e] = (T)h[i][e];
        squares = fmaf(h[i][e], h[i][e], squares);
      }
      // the sum is rounded on its way out; the norm is of the sum before that
      if constexpr (RESIDUAL) *reinterpret_cast<vec*>(Sum + row * dim + 8 * at) = s;
    }
  }
  squares = over_row<LANES, false>(squares, slots[0]);
  float mean = squares / (float)dim, factor = 1.f;
  if (__builtin_isinf(mean)) {
    // squares beyond fp32's range (bf16 alone reaches that): the same with every element 2^-70 of itself
    constexpr float kDown = 0x1p-70f;
    squares = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) squares = fmaf(h[i][e] * kDown, h[i][e] * kDown, squares);
    squares = over_row<LANES, false>(squares, slots[1]);
    mean = squares / (float)dim;  // (2^-140 eps is nothing beside it)
    eps = 0.f;
    factor = kDown;
  }
  const float inverse = factor / sqrtf(mean + eps);
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int at = i * LANES + lane;
    if (at < pieces) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        h[i][e] = h[i][e] * inverse * (float)wv[i][e];
        if constexpr (INT8) largest = fmaxf(largest, __builtin_isnan(h[i][e]) ? __builtin_inff() : fabsf(h[i][e]));
      }
      if constexpr (!INT8) {
        vec y;
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = (T)h[i][e];
        *reinterpret_cast<vec*>((T*)Y + row * dim + 8 * at) = y;
      }
    }
  }
  if constexpr (INT8) {
    largest = over_row<LANES, true>(largest, slots[2]);
    // a row with an infinity or a NaN: codes of zero under a scale that is NaN, so that it reads back as NaN
    const bool broken = __builtin_isinf(largest);
    const float scale = 127.f / fmaxf(largest, 1e-5f);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int at = i * LANES + lane;
      if (at < pieces) {
        uint2_t codes = {0u, 0u};
        if (!broken) {
          float c[8];
          // (a product a hair over 127 is rounded to 127: no clamp)
#pragma unroll
          for (int e = 0; e < 8; ++e) c[e] = h[i][e] * scale;
          codes[0] = quantise4<CACHE_I8>(c[0], c[1], c[2], c[3]);
          codes[1] = quantise4<CACHE_I8>(c[4], c[5], c[6], c[7]);
        }
        *reinterpret_cast<uint2_t*>((int8_t*)Y + row * dim + 8 * at) = codes;
      }
    }
    if (lane == 0) Scale[row] = broken ? __builtin_nanf("") : scale;
  }
}

struct NormArgs {
  const void *X, *Residual, *Weight;
  void *Y, *Sum;
  float* Scale;
  int rows, dim;
  long row_stride;
  float eps;
  hipStream_t stream;
};

template <class T, int LANES, int NV, bool RESIDUAL, bool INT8>
int launch(const NormArgs& a) {
  constexpr int kRows = LANES <= 64 ? 256 / LANES : 1;
  const unsigned blocks = ((unsigned)a.rows + kRows - 1) / kRows, wide = blocks < (1u << 20) ? blocks : 1u << 20;  // (a launch takes 2^32 threads a dimension)
  hipLaunchKernelGGL((norm_kernel<T, LANES, NV, RESIDUAL, INT8>), dim3(wide, (blocks + wide - 1) / wide), dim3(LANES <= 64 ? 256 : LANES), 0, a.stream,
                     (const T*)a.X, (const T*)a.Residual, (const T*)a.Weight, a.Y, (T*)a.Sum, a.Scale, a.rows, a.dim, a.row_stride, a.eps);
  DQ_CHECK_HIP(hipGetLastError());
  return 0;
}

template <class T, bool RESIDUAL, bool INT8>
int by_size(const NormArgs& a) {
  const int pieces = a.dim >> 3;
  if (pieces <= 16) return launch<T, 16, 1, RESIDUAL, INT8>(a);
  if (pieces <= 64) return launch<T, 64, 1, RESIDUAL, INT8>(a);
  if (pieces <= 256) return launch<T, 256, 1, RESIDUAL, INT8>(a);
  if (pieces <= 512) return launch<T, 256, 2, RESIDUAL, INT8>(a);
  if (pieces <= 1024) return launch<T, 256, 4, RESIDUAL, INT8>(a);
  if (pieces <= 2048) return launch<T, 1024, 2, RESIDUAL, INT8>(a);
  return launch<T, 1024, 4, RESIDUAL, INT8>(a);
}

}  // namespace

int rms_norm(const void* X, const void* Residual, const void* Weight, void* Y, void* Sum, float* Scale, int rows, int dim, long row_stride,
             int int8, int bf16, float eps, hipStream_t stream) {
  const NormArgs a{X, Residual, Weight, Y, Sum, Scale, rows, dim, row_stride, eps, stream};
#define DQ_NORM(T_) (Residual ? (int8 ? by_size<T_, true, true>(a) : by_size<T_, true, false>(a)) : (int8 ? by_size<T_, false, true>(a) : by_size<T_, false, false>(a)))
  return bf16 ? DQ_NORM(bf16_t) : DQ_NORM(half_t);
#undef DQ_NORM
}

}  // namespace dq
