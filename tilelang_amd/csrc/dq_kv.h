// What the kernels around the paged key-value cache share: its types and where a token lies in it.
//
// Keys and values: [pages][kv_heads][page_size][head_dim], a head's page one contiguous piece; in 8 bits with fp32
// scales [pages][kv_heads][page_size], one a token and head.  page_size is a power of two from 8 on, so eight tokens
// that start at a multiple of eight lie one behind the other.  Offsets are 64-bit: a cache of 288 GB has more than 2^32
// elements.
#pragma once

#include "dq_common.h"

namespace dq {

enum CacheFormat : int {
  CACHE_F16 = 0,
  CACHE_BF16 = 1,
  CACHE_FP8 = 2,  // OCP e4m3, largest 448
  CACHE_I8 = 3,   // -127 .. 127
};
constexpr bool cache_is_16bit(int format) { return format <= CACHE_BF16; }

// A head whose largest magnitude is below this is stored as zeros: the factor 448 / a stays finite.
constexpr float kSmallestHead = 0x1p-100f;

constexpr int kMaxHeadDim = 256;  // of the cache's heads
constexpr int kMaxRotaryHead = 512;

struct CacheShape {
  int pages, kv_heads, page_shift, head_dim;
};

// The row (token and head) of a place in the cache: times head_dim the offset of its elements, itself that of its scale.
__device__ __forceinline__ size_t cache_row(const CacheShape& c, int page, int head, int place) {
  return ((((size_t)page * c.kv_heads + head) << c.page_shift) + place);
}

template <class T>
__device__ __forceinline__ float to_float(T x) {
  return (float)x;
}

template <class T>
struct Vec8 {
  typedef T type __attribute__((ext_vector_type(8)));
};

// Eight e4m3 codes (two dwords) or eight int8 codes as fp32.
template <int FORMAT>
__device__ __forceinline__ void codes8_to_float(uint2_t w, float (&f)[8]) {
  typedef float float2_t __attribute__((ext_vector_type(2)));
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if constexpr (FORMAT == CACHE_FP8) {
      const float2_t lo = __builtin_amdgcn_cvt_pk_f32_fp8(w[i], false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(w[i], true);
      f[4 * i] = lo[0], f[4 * i + 1] = lo[1], f[4 * i + 2] = hi[0], f[4 * i + 3] = hi[1];
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) f[4 * i + j] = (float)(int8_t)(w[i] >> (8 * j));
    }
  }
}

// Four floats of magnitude at most 448 (127) -> codes, round to nearest even.
template <int FORMAT>
__device__ __forceinline__ uint32_t quantise4(float a, float b, float c, float d) {
  if constexpr (FORMAT == CACHE_FP8) {
    uint32_t w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return __builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
  } else {
    // 1.5 * 2^23 + x: the sum's last byte is x rounded to the nearest even integer
    constexpr float kMagic = 12582912.f;
    const uint32_t ia = __builtin_bit_cast(uint32_t, a + kMagic), ib = __builtin_bit_cast(uint32_t, b + kMagic);
    const uint32_t ic = __builtin_bit_cast(uint32_t, c + kMagic), id = __builtin_bit_cast(uint32_t, d + kMagic);
    const uint32_t ab = __builtin_amdgcn_perm(ib, ia, 0x0C0C0400u), cd = __builtin_amdgcn_perm(id, ic, 0x04000C0Cu);
    return ab | cd;
  }
}

}  // namespace dq
