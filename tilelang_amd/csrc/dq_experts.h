// What the kernels of the experts' products share: their arguments, and the two weight formats.
//
// Rows are the pairs (token, choice) in the order of their experts: rows Starts[e] .. Starts[e + 1] - 1 are expert e's, row r is
// pair Order[r] = token * top_k + choice.  "Up" multiplies a row's token with the expert's gate and up weights and leaves
// act(gate) * up; "down" multiplies a row with the expert's weights and adds what belongs to a token, by its weights.
#pragma once

#include "dq_fp4_codes.h"

namespace dq {
namespace experts {

struct Args {
  const void* A;       // up: [tokens][K]; down: [pairs][K]
  const uint8_t* B;    // [experts][up: 2 N, down: N][K / 2]
  const void* S;       // scales [experts][rows][K / group]
  const void* Z;       // zero points, or nullptr
  const void* Bias;    // [experts][rows], or nullptr
  const int* Order;    // [pairs]
  const int* Starts;   // [experts + 1]
  const int* Ids;      // down: [pairs], an expert `first` on
  const float* Weights;  // down: [pairs]
  const void* Residual;  // down: [tokens][N], or nullptr
  void* Out;           // up: [pairs][N]; down: [tokens][N]
  float* Parts;        // down: fp32 [slices][pairs][N], a pair's product, of a slice of K
  int tokens, experts, top_k, pairs, N, K, group_shift, gelu, first, slices;
  int routed;  // choices are of so many experts, of which these are some: what to expect here, no more
};

// Activations and weights of a product: uint4 codes x fp16, as the dense W4A16 kernels have them (rounded to fp16), and e2m1 x bf16.
template <bool ZEROS, int SHIFT>
struct Uint4 {
  using T = half_t;
  using frag = half8_t;
  static constexpr bool kZeros = ZEROS;
  static constexpr int kShift = SHIFT, kScaleBytes = 2;  // 2 ^ kShift k share a scale
  static constexpr int MODE = ZEROS ? W4_ZEROS_ORIGINAL : W4_SCALE;
  struct Scale { half_t s, addend; };
  // (the bits of a scale and a zero point)
  __device__ static __forceinline__ Scale scale(unsigned s, unsigned z) {
    const half_t f = __builtin_bit_cast(half_t, (unsigned short)s);
    return {f, w4_cvt_addend<MODE>(f, __builtin_bit_cast(half_t, (unsigned short)z))};
  }
  // eight activations in the order that a word's codes are decoded in
  __device__ static __forceinline__ uint4_t order(uint4_t d) {
    return {__builtin_amdgcn_perm(d[1], d[0], 0x05040100u), __builtin_amdgcn_perm(d[3], d[2], 0x05040100u),
            __builtin_amdgcn_perm(d[1], d[0], 0x07060302u), __builtin_amdgcn_perm(d[3], d[2], 0x07060302u)};
  }
  __device__ static __forceinline__ frag decode(uint32_t w, const Scale& s) { return decode_w4_cvt<MODE, false, false>(w, s.s, s.addend); }
  __device__ static __forceinline__ float4_t mfma(frag a, frag b, float4_t c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
};

struct Mxfp4 {
  using T = bf16_t;
  using frag = bf16x8_t;
  static constexpr bool kZeros = false;
  static constexpr int kShift = 5, kScaleBytes = 1;
  using Scale = float;
  __device__ static __forceinline__ Scale scale(unsigned e, unsigned) { return scale_to_f32((int)e, 0); }
  __device__ static __forceinline__ uint4_t order(uint4_t d) { return d; }
  __device__ static __forceinline__ frag decode(uint32_t w, const Scale& s) { return cvt_e2m1x8(w, s); }
  __device__ static __forceinline__ float4_t mfma(frag a, frag b, float4_t c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
};

// x / (1 + e^-x), and the tanh form of x times the normal distribution's integral up to x: 1/2 (1 + tanh u) = 1 / (1 + e^-2u).
__device__ __forceinline__ float activate(float x, int gelu) {
  const float u = gelu ? 1.5957691216057308f * (x + 0.044715f * x * x * x) : x;
  const float y = x / (1.f + expf(-u));
  return u < -87.f ? (x != x ? x : 0.f) : y;  // (e^-u is beyond fp32, x times its inverse below)
}

// The rows of an expert, whatever Starts holds: inside of the pairs.
__device__ __forceinline__ void rows_of(const Args& a, int e, int& begin, int& end) {
  begin = min(max(a.Starts[e], 0), a.pairs);
  end = min(max(a.Starts[e + 1], begin), a.pairs);
}

// K that is an odd number of blocks of 64, or a row's scales that are: rows of scales begin between dwords
inline bool odd_rows(int mxfp4, int K, int group_shift) { return (K / 64) % 2 != 0 || (!mxfp4 && ((K >> group_shift) & 1) != 0); }

}  // namespace experts
}  // namespace dq
