// The experts' products at many rows an expert: the direct-to-LDS GEMM of dq_gemm_core.h on tiles of 64 or 128 rows of one expert
// by 256 of its weight rows (up: 128 of the gate and the 128 of the up projection that go with them, in blocks of 32, so that a
// lane has both sums of a value; down: or a slice of K of them, each slice with fp32 results of its own, which the sums of the tokens
// add in their order).
//
// How many tiles there are is known on the device alone.  The grid has as many workgroups as there can be, every one counts the
// experts' tiles and those beyond them end; the others go over the XCDs in runs, expert by expert, so that an XCD finds an expert's
// rows and weights in its own L2 cache.  Rows of "up" are gathered where they are loaded: a lane's source address is its row's own.
// What bounds it is the matrix pipe: 4096 tokens, two of 8 experts, uint4, 14336 x 4096 "up" 1.75 ms, 1.1 PFLOP/s, 4096 x 14336 "down"
// 1.02 ms, 0.94 (1088 tiles on the 512 places of two workgroups a CU: the last 64 have the chip for themselves).
#include "dq_experts.h"
#include "dq_gemm_mx.h"
#include "dq_gemm_w4.h"

namespace dq {

namespace {

using experts::Args;

struct TileParams : gemm::Params {
  Args a;
  int begin, expert, slice;  // of the tile
};

template <class Base, bool UP>
struct ExpertsPolicy : Base {
  static constexpr bool kGrouped = true;
  using params_t = TileParams;
  using acc_t = typename Base::acc_t;
  using T = typename Base::out_t;
  static constexpr int kColumns = UP ? 128 : 256;  // of the output, in a tile

  __device__ static bool take_tile(TileParams& p, int bid, int tile_rows, int& m0, int& n0) {
    const Args& a = p.a;
    const int lane = threadIdx.x & 63;
    auto tiles_of = [&](int e, int& begin, int& rows) {
      int end = 0;
      begin = 0;
      if (e < a.experts) experts::rows_of(a, e, begin, end);
      rows = end - begin;
      return (rows + tile_rows - 1) / tile_rows;
    };
    int begin, rows, all = 0;
    for (int base = 0; base < a.experts; base += 64) all += tiles_of(base + lane, begin, rows);
#pragma unroll
    for (int d = 1; d < 64; d *= 2) all += __shfl_xor(all, d, 64);
    // runs of tiles an XCD (workgroup id mod 8)
    const int tiles_n = p.tiles_n * (UP ? 1 : a.slices);  // and slices of K
    const int tiles = __builtin_amdgcn_readfirstlane(all) * tiles_n;
    const int x = bid & 7, i = bid >> 3, share = tiles >> 3, more = tiles & 7;
    if (i >= share + (x < more ? 1 : 0)) return false;
    const int pid = x * share + min(x, more) + i;
    int row_tile = pid / tiles_n, before = 0;
    for (int base = 0;; base += 64) {
      const int n = tiles_of(base + lane, begin, rows);
      int upto = n;
#pragma unroll
      for (int d = 1; d < 64; d *= 2) {
        const int o = __shfl_up(upto, d, 64);
        if (lane >= d) upto += o;
      }
      const unsigned long long beyond = __ballot(before + upto > row_tile);
      if (beyond != 0) {
        const int at = __builtin_ctzll(beyond);
        p.expert = base + at;
        p.begin = __builtin_amdgcn_readlane(begin, at);
        p.M = __builtin_amdgcn_readlane(rows, at);
        const int tiles_m = __builtin_amdgcn_readlane(n, at);
        // the expert's tiles in bands of four tile rows, column by column inside a band
        const int local = pid - (before + __builtin_amdgcn_readlane(upto, at) - tiles_m) * tiles_n;
        const int band = 4 * tiles_n, first = local / band * 4, in_band = local % band, high = min(tiles_m - first, 4);
        m0 = (first + in_band % high) * tile_rows;
        n0 = in_band / high;
        break;
      }
      before += __builtin_amdgcn_readlane(upto, 63);
    }
    p.slice = 0;
    if constexpr (!UP) {
      p.slice = n0 % a.slices;
      n0 /= a.slices;
    }
    n0 *= kColumns;
    const size_t weight_rows = (size_t)p.expert * p.N;
    p.B = (const unsigned char*)p.B + weight_rows * (a.K >> 1);
    const size_t scales = weight_rows * (a.K >> a.group_shift) * (Base::kScaleDma == 1 ? 1 : 2);
    p.S = (const unsigned char*)p.S + scales;
    if constexpr (Base::kScaleDma == 3) p.Z = (const unsigned char*)p.Z + scales;
    if constexpr (!UP) p.A = (const unsigned char*)p.A + ((size_t)p.begin + m0) * a.K * 2;
    if constexpr (!UP) {
      // whole units of 256 k: a row's scales of one begin at a dword, whatever its groups
      const int units = a.K >> 8, k0 = units * p.slice / a.slices << 8;
      if (p.slice + 1 < a.slices) p.K = units * (p.slice + 1) / a.slices << 8;
      p.K -= k0;
      p.A = (const unsigned char*)p.A + (size_t)k0 * 2;
      p.B = (const unsigned char*)p.B + (k0 >> 1);
      const int groups = Base::kScaleDma == 1 ? k0 >> 5 : k0 >> a.group_shift << 1;  // bytes
      p.S = (const unsigned char*)p.S + groups;
      if constexpr (Base::kScaleDma == 3) p.Z = (const unsigned char*)p.Z + groups;
    }
    p.tiles_m = m0;
    return true;
  }
  __device__ static __forceinline__ unsigned a_row(const TileParams& p, int m) {
    if constexpr (UP) return min((unsigned)p.a.Order[p.begin + m] / (unsigned)p.a.top_k, (unsigned)p.a.tokens - 1);
    else return (unsigned)(m - p.tiles_m);
  }
  // (N is a multiple of 32: a block of 32 columns is there as a whole or not at all, and one that is not repeats the first)
  __device__ static __forceinline__ unsigned b_row(const TileParams& p, int n0, int row) {
    const int block = row >> 5, n = n0 + (UP ? block >> 1 : block) * 32;
    return (unsigned)((n < p.a.N ? n : n0) + (row & 31) + (UP && (block & 1) ? p.a.N : 0));
  }

  template <int MB, int NB>
  __device__ static void store(const TileParams& p, acc_t (&acc)[MB][NB], unsigned char* smem, int wave, int lane, int m0, int n0, int wn) {
    constexpr int kStride = 36;
    float* const slab = reinterpret_cast<float*>(smem) + wave * (32 * kStride);
    const Args& a = p.a;
    const int g = lane >> 5, r = lane & 31;
    const T* const bias = a.Bias == nullptr ? nullptr : (const T*)a.Bias + (size_t)p.expert * p.N;
#pragma unroll
    for (int mb = 0; mb < MB; ++mb) {
      if (m0 + mb * 32 >= p.M) break;
      if constexpr (UP) {
#pragma unroll
        for (int q = 0; q < NB / 2; ++q) {
          const int n = n0 + (wn * (NB / 2) + q) * 32;
          if (n >= a.N) break;
          float gate_bias = 0.f, up_bias = 0.f;
          if (bias != nullptr) gate_bias = (float)bias[n + r], up_bias = (float)bias[a.N + n + r];
#pragma unroll
          for (int i = 0; i < 16; ++i)
            slab[(8 * (i >> 2) + 4 * g + (i & 3)) * kStride + r] =
                experts::activate(acc[mb][2 * q][i] + gate_bias, a.gelu) * (acc[mb][2 * q + 1][i] + up_bias);
          __builtin_amdgcn_wave_barrier();
#pragma unroll
          for (int it = 0; it < 2; ++it) {
            const int row = (lane + 64 * it) >> 2, piece = lane & 3, m = m0 + mb * 32 + row;
            const float4_t lo = *reinterpret_cast<const float4_t*>(slab + row * kStride + piece * 8);
            const float4_t hi = *reinterpret_cast<const float4_t*>(slab + row * kStride + piece * 8 + 4);
            if (m < p.M) {
              T o[8];
#pragma unroll
              for (int e = 0; e < 4; ++e) o[e] = (T)lo[e], o[4 + e] = (T)hi[e];
              uint4_t bits;
              __builtin_memcpy(&bits, o, 16);
              *reinterpret_cast<uint4_t*>((T*)a.Out + ((size_t)p.begin + m) * a.N + n + piece * 8) = bits;
            }
          }
          __builtin_amdgcn_wave_barrier();
        }
      } else {
        unsigned pair[4];
        float weight[4];
#pragma unroll
        for (int it = 0; it < 4; ++it) {
          const int m = m0 + mb * 32 + ((lane + 64 * it) >> 3);
          pair[it] = m < p.M ? (unsigned)a.Order[p.begin + m] : ~0u;
          weight[it] = pair[it] < (unsigned)a.pairs ? a.Weights[pair[it]] : 0.f;
        }
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
          const int n = n0 + (wn * NB + nb) * 32;
          if (n >= a.N) break;
          const float add = bias == nullptr || p.slice != 0 ? 0.f : (float)bias[n + r];
#pragma unroll
          for (int i = 0; i < 16; ++i) slab[(8 * (i >> 2) + 4 * g + (i & 3)) * kStride + r] = acc[mb][nb][i] + add;
          __builtin_amdgcn_wave_barrier();
#pragma unroll
          for (int it = 0; it < 4; ++it) {
            const int row = (lane + 64 * it) >> 3, piece = lane & 7;
            const float4_t v = *reinterpret_cast<const float4_t*>(slab + row * kStride + piece * 4);
            if (pair[it] < (unsigned)a.pairs) *reinterpret_cast<float4_t*>(a.Parts + ((size_t)p.slice * a.pairs + pair[it]) * a.N + n + piece * 4) = v * weight[it];
          }
          __builtin_amdgcn_wave_barrier();
        }
      }
    }
  }
};

template <class P, int kMBW, bool kOdd>
int launch_tiles(const TileParams& p, int workgroups, hipStream_t stream) {
  // three stages of rows and weights and the rings of scales, or the epilogue's slabs
  constexpr int kPipe = 3 * (32 * kMBW * gemm::kARowBytes + gemm::BN * P::kBRowBytes) + 8 * 1024, kSlabs = 4 * 32 * 36 * 4;
  constexpr int kLds = kPipe > kSlabs ? kPipe : kSlabs;
  static_assert(P::kBRowBytes == 32 && kLds <= 80 * 1024, "LDS budget of two workgroups a CU");
  auto kern = gemm::gemm_kernel_dma<P, kMBW, 2, 1, 1, kOdd>;
  static bool raised[kMaxDevices];
  if (raise_lds_limit<kLds>(kern, raised)) return -1;
  hipLaunchKernelGGL(kern, dim3(workgroups), dim3(256), kLds, stream, p);
  DQ_CHECK_HIP(hipGetLastError());
  return 0;
}

template <class Base, bool UP>
int tiles(const Args& a, int tile_rows, hipStream_t stream) {
  using P = ExpertsPolicy<Base, UP>;
  TileParams p{};
  static_cast<gemm::Params&>(p) = gemm::make_params(a.A, a.B, a.S, a.Z, nullptr, a.Out, a.pairs, (UP ? 2 : 1) * a.N, a.K);
  p.a = a;
  p.p0 = Base::kScaleDma == 1 ? 0 : a.group_shift;  // MXFP4: E8M0 exponents as they are
  p.tiles_n = (a.N + P::kColumns - 1) / P::kColumns;
  // every expert's last tile may be a part of one
  const long row_tiles = a.pairs / tile_rows + (a.experts < a.pairs ? a.experts : a.pairs);
  const long all = (row_tiles * p.tiles_n * (UP ? 1 : a.slices) + 7) / 8 * 8;
  if (all >= 1l << 23) DQ_FAIL("experts: %d rows of %d columns: more tiles than a launch takes", a.pairs, a.N);  // (2^32 threads)
  const int workgroups = (int)all;
  const bool odd = experts::odd_rows(Base::kScaleDma == 1, a.K, a.group_shift);
#define DQ_TILES(BLOCKS_) (odd ? launch_tiles<P, BLOCKS_, true>(p, workgroups, stream) : launch_tiles<P, BLOCKS_, false>(p, workgroups, stream))
  return tile_rows == 64 ? DQ_TILES(2) : DQ_TILES(4);
#undef DQ_TILES
}

}  // namespace

// Tiles of 64 or 128 rows.
int experts_tiles(const Args& a, int mxfp4, bool up, int tile_rows, hipStream_t stream) {
  if (mxfp4) return up ? tiles<MxPolicy<FP4_E2M1, false>, true>(a, tile_rows, stream) : tiles<MxPolicy<FP4_E2M1, false>, false>(a, tile_rows, stream);
  if (a.Z != nullptr)
    return up ? tiles<W4F16Policy<W4_ZEROS_ORIGINAL, false>, true>(a, tile_rows, stream) : tiles<W4F16Policy<W4_ZEROS_ORIGINAL, false>, false>(a, tile_rows, stream);
  return up ? tiles<W4F16Policy<W4_SCALE, false>, true>(a, tile_rows, stream) : tiles<W4F16Policy<W4_SCALE, false>, false>(a, tile_rows, stream);
}

}  // namespace dq
