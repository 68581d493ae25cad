// MXFP4 x bf16 policy of the dequantize GEMMs of dq_gemm_core.h and dq_gemm_kwaves.h.
#pragma once

#include "dq_fp4_codes.h"
#include "dq_gemm_core.h"

namespace dq {

namespace {

using gemm::Params;

struct Bf16Mfma {
  static constexpr int kKPerBlock = 64;
  using frag_t = bf16x8_t;
  using acc_t = float16_t;
  __device__ static __forceinline__ acc_t mfma(frag_t a, frag_t b, acc_t c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
};

// ---- MXFP4 x bf16 -------------------------------------------------------------------------------
// Scale[N, K/32] uint8, p.p0 = 127 - scale_bias.  Lane group g owns one 32-k scale block per tile.
template <int FMT, bool HAS_BIAS>
struct MxPolicy : Bf16Mfma, gemm::PlainA {
  static constexpr int kBRowBytes = 32;
  static constexpr bool kOneOrder = true;  // the header's promise of a row's bits
  static constexpr gemm::RowsCost kRowCosts[4] = {{4.3, 1.2, 10.4}, {5.15, 1.1, 12.8}, {-3.2, 14.7, 15.0}, {-7.2, 26.3, 16.3}};
  static constexpr bool kTransposed = false;
  using out_t = bf16_t;
  using ScaleRaw = int;
  static constexpr int kScaleDma = 1;  // one scale byte per 32 k travels by DMA in the direct-to-LDS kernel
  // by dwords, so only from where a dword lies: Scale may start at any byte, and the register-staged kernel reads bytes
  static bool dma_ok(const Params& p) { return ((size_t)p.S & 3) == 0; }
  struct Scale { float f; uint32_t add; };
  __device__ static __forceinline__ ScaleRaw fetch_scale(const Params& p, int row, int kb, int g) {
    return ((const uint8_t*)p.S)[(size_t)row * (p.K >> 5) + kb * 2 + g];
  }
  __device__ static __forceinline__ Scale prep_scale(ScaleRaw e, const Params& p) {
    Scale s;
    if constexpr (FMT == FP4_SIMPLE) {
      int ex = 126 + e + p.p0 - 127;
      ex = ex < 0 ? 0 : (ex > 252 ? 252 : ex);  // E adds up to 3
      s.add = ((uint32_t)ex << 7) * 0x00010001u;
      s.f = 0.f;
    } else {
      s.f = scale_to_f32(e, p.p0);
      s.add = 0;
    }
    return s;
  }
  __device__ static __forceinline__ frag_t decode(const uint32_t* w, int j, const Scale& s) {
    if constexpr (FMT == FP4_E2M1) return cvt_e2m1x8(w[j], s.f);
    else if constexpr (FMT == FP4_TWIDDLING) return cvt_e2m1x8(twiddled_to_plain(w[j]), s.f);
    else return __builtin_bit_cast(frag_t, simple_fp4x8<7>(w[j], s.add));
  }
  __device__ static __forceinline__ out_t finish(uint32_t raw, const Params& p, int m, int n) {
    float v = __builtin_bit_cast(float, raw);
    // reference: C = bf16(float(acc) + float(Bias))
    if constexpr (HAS_BIAS) v += (float)((const bf16_t*)p.Bias)[(size_t)m * p.N + n];
    return (bf16_t)v;
  }
};

}  // namespace

}  // namespace dq
