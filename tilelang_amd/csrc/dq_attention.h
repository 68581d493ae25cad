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
// Which token a row of the first product is, is free, so K's rows are taken in an order that hands the lane group g = lane / 16
// the tokens 8 g .. 8 g + 7: these are the eight that the second product wants from the same lanes, and P^T never leaves
// its registers.  V^T's operand is eight tokens of one d in a lane; a lane loads eight tokens' rows at its own few d instead
// (a whole row of V is 16 lanes side by side) and turns the piece with byte permutes.  K's operand, 16 bytes of each of 16
// rows, would take half a line of memory an instruction; keys come as they lie, whole lines, and go through an LDS corner of
// the wave's own.  No wave waits for another inside the loop.
//
// A quantised cache is multiplied as fp16: a code is exact there; a query is scaled by a power of two so that its largest element
// lies in [2^14, 2^15), where bf16's range is no issue; a token's scale multiplies its score in fp32.  A weight times its
// value's scale, w_t = p_t c_t, may lie anywhere: o is kept relative to a power of two of its own, the running maximum of a
// head's |w_t|, as the sum is relative to the running maximum of its scores; it is counted from that maximum, and from 2^-112 on, so
// that no factor is infinite where the token of the largest score has a value of zero.
//
// Weights go into the second product in two parts, what the product's type holds of one and what that left (some 22 bits in fp16, 16
// in bf16), so that they are rounded far below the result, which is rounded once, at the end.  Codes are finite, so there the first
// part is the nearest number; of a 16-bit cache it is the one toward zero, and the second is not zero where the first is not, so
// that an infinity among the values stays one.  (In one part, rounded to the cache's type: 1.6e-3 of the result off that of fp32
// weights, in two 1.9e-4; 131071 tokens, bf16, 88 us either way.)  In fp16 weights are taken times 2^kLift, the largest then about
// 2^15 of the 65504 that fp16 ends at: all are held to 2^-40 of the largest.  At 1 that was 2^-25, and thousands of tokens that
// light, beside a heavy one of a small value all that the result is made of, were lost.
//
// Bound by memory: eight heads on one key-value head do 8 operations a byte of a 16-bit cache, where the chip has some 300.
// 128 sequences of 8192 tokens, 8 heads of 128, int8: 347 us, 6.4 TB/s of the 6.9 that plain streamed reads of such pieces
// reach (when it took 355, keys and values not streamed took 397 and K's operand straight from memory 400); one sequence of 131071 tokens, bf16: 88 us,
// 5 of them the join.  Short calls are two launches of 4.3 us, or one where no column can be cut.
#pragma once

#include "dq_kv.h"

namespace dq {

constexpr int kAttnWaves = 4;
constexpr int kAttnTile = 32;                        // tokens that a wave takes at once
constexpr int kAttnUnit = kAttnTile * kAttnWaves;  // ... and a workgroup
constexpr int kComputeUnits = 256;

struct AttnArgs {
  const void* q;           // [sequences][heads][head_dim]
  const void* cache[2];
  const float* scale[2];
  const int* table;        // [sequences][max_pages]
  const int* lengths;      // [sequences]
  const float* sinks;      // [heads] or null
  void* out;               // [sequences][heads][head_dim]
  float* lse;              // [sequences][heads] or null
  float* part_o;           // [workgroups][2][rows][head_dim]
  float* part_ml;          // [workgroups][2][rows][2]
  int* pieces;             // [sequences][kv_heads * head_blocks][2]: the first and last workgroup that has a piece
  float score_scale;       // scale * log2(e)
  int sequences, heads, max_pages, window, head_blocks, rows, workgroups;
  CacheShape shape;
};

// The tokens of a sequence: [first, length), in tiles from tile0 on, in units of kAttnUnit tokens.
struct Span {
  int length, first, tile0, tiles, units;
};
__device__ __forceinline__ Span span_of(int length, int capacity, int window) {
  Span s;
  s.length = min(max(length, 0), capacity);
  s.first = window > 0 ? max(0, s.length - window) : 0;
  s.tile0 = s.first / kAttnTile;
  s.tiles = (s.length + kAttnTile - 1) / kAttnTile - s.tile0;
  s.units = (s.tiles + kAttnWaves - 1) / kAttnWaves;
  return s;
}

// How the work is shared out.  The tokens that a key-value head (a column) has of a sequence cost their units and two more: what
// a workgroup does before the first and after the last takes about as long (64 sequences of 0 to 16000 tokens, fp8: 158 us
// without, 127 with one, 124 with two or three; short windows 11.7, with three 13.0).  All costs in a row, sequence by
// sequence and in a sequence column by column, are cut into equal shares, one a workgroup, whatever the lengths are; a
// cut inside a column makes pieces of it, which the join adds up.  A column of up to kWholeUnits is not worth a join (one
// sequence of 512 tokens: cut 11.7 us, whole 7.5; of 1000 11.2 and 13.9): a cut there moves to its nearer end.
constexpr int kWholeUnits = 4, kColumnCost = 2;
struct Shares {
  unsigned each, more;  // the first `more` workgroups have one more
  __device__ __forceinline__ Shares(unsigned total, unsigned workgroups) : each(total / workgroups), more(total - total / workgroups * workgroups) {}
  __device__ __forceinline__ unsigned begin(unsigned w) const { return w * each + min(w, more); }
  __device__ __forceinline__ unsigned owner(unsigned u) const {
    const unsigned large = more * (each + 1);
    return u < large ? u / (each + 1) : more + (u - large) / max(each, 1u);
  }
};

struct Share {
  unsigned at, end;         // in costs
  int sequence, length;     // of the column at `at`
  unsigned sequence_begin;  // the sequence's first cost
};
struct ShareSearch {
  int scan[kAttnWaves];
  unsigned cut[2];
  int sequence, length;
  unsigned sequence_begin;
};

// Where a cut falls that lies in a sequence whose first cost is `begin`: inside a column, or at the nearer end of a short one.
__device__ __forceinline__ unsigned moved_cut(unsigned cut, unsigned begin, int units) {
  const unsigned cost = units + kColumnCost, off = (cut - begin) % cost;
  return units <= kWholeUnits ? cut - off + (2 * off >= cost ? cost : 0) : cut;
}

// The workgroup's share: a running sum of the sequences' costs, and the two cuts in it.  For all threads of the workgroup.
// Up to 64 sequences lie in a wave's lanes, and every wave finds the share by itself (a short call takes 0.4 us less).
__device__ __forceinline__ Share find_share(const AttnArgs& a, int capacity, int columns, int wave, int lane, ShareSearch& s, Shares& shares) {
  if (a.sequences <= 64) {
    const int length = lane < a.sequences ? a.lengths[lane] : 0;
    const int units = lane < a.sequences ? span_of(length, capacity, a.window).units : -kColumnCost;
    int sum = units + kColumnCost;  // inclusive
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int up = __shfl_up(sum, o);
      if (lane >= o) sum += up;
    }
    const int total = __builtin_amdgcn_readlane(sum, 63);
    shares = Shares((unsigned)total * columns, a.workgroups);
    Share share;
    unsigned cut[2];
#pragma unroll
    for (int side = 0; side < 2; ++side) {
      cut[side] = shares.begin(blockIdx.x + side);
      const int at = cut[side] / columns;
      if (at >= total) continue;  // behind everything
      const int b = __builtin_ctzll(__ballot(at < sum));
      const int b_units = __builtin_amdgcn_readlane(units, b);
      const unsigned b_end = (unsigned)__builtin_amdgcn_readlane(sum, b) * columns, b_begin = b_end - (unsigned)(b_units + kColumnCost) * columns;
      cut[side] = moved_cut(cut[side], b_begin, b_units);
      if (side == 0) {
        const bool next = cut[0] == b_end;
        share.sequence = b + next, share.sequence_begin = next ? b_end : b_begin;
        share.length = __builtin_amdgcn_readlane(length, min(b + next, 63));
      }
    }
    share.at = cut[0], share.end = cut[1];
    return share;
  }
  const int per_thread = (a.sequences + 64 * kAttnWaves - 1) / (64 * kAttnWaves);
  const int seq_begin = min((int)threadIdx.x * per_thread, a.sequences), seq_end = min(seq_begin + per_thread, a.sequences);
  int mine = 0, length_here = 0;  // (of the last of this thread's sequences: of its one, where a thread has one)
  for (int b = seq_begin; b < seq_end; ++b) length_here = a.lengths[b], mine += span_of(length_here, capacity, a.window).units + kColumnCost;
  int sum = mine;  // inclusive
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int up = __shfl_up(sum, o);
    if (lane >= o) sum += up;
  }
  if (lane == 63) s.scan[wave] = sum;
  __syncthreads();
  int total = 0;
#pragma unroll
  for (int w = 0; w < kAttnWaves; ++w) {
    if (w < wave) sum += s.scan[w];
    total += s.scan[w];
  }
  shares = Shares((unsigned)total * columns, a.workgroups);
#pragma unroll
  for (int side = 0; side < 2; ++side) {
    const unsigned cut = shares.begin(blockIdx.x + side);
    const int at = cut / columns;
    if (threadIdx.x == 0 && at >= total) s.cut[side] = cut;  // behind everything
    if (!(sum - mine <= at && at < sum)) continue;
    int b = seq_begin, before = sum - mine;
    for (;; ++b) {
      const int length = per_thread == 1 ? length_here : a.lengths[b];
      const int units = span_of(length, capacity, a.window).units, cost = units + kColumnCost;
      if (at >= before + cost) {
        before += cost;
        continue;
      }
      const unsigned begin = (unsigned)before * columns, moved = moved_cut(cut, begin, units);
      s.cut[side] = moved;
      if (side == 0) {
        const bool next = moved == begin + (unsigned)cost * columns;
        s.sequence = b + next, s.sequence_begin = next ? moved : begin;
        s.length = !next ? length : b + 1 < a.sequences ? a.lengths[b + 1] : 0;
      }
      break;
    }
  }
  __syncthreads();
  Share share;
  share.at = __builtin_amdgcn_readfirstlane(s.cut[0]), share.end = __builtin_amdgcn_readfirstlane(s.cut[1]);
  share.sequence = __builtin_amdgcn_readfirstlane(s.sequence), share.length = __builtin_amdgcn_readfirstlane(s.length);
  share.sequence_begin = __builtin_amdgcn_readfirstlane(s.sequence_begin);
  return share;
}

// ---- which elements of a row a lane holds ----------------------------------------------------------------------
// Keys (and queries): k-step s of 32 elements, group g has eight of them.  16 bit: 32 s + 8 g.  8 bit: a lane loads 16
// codes at 64 p + 16 g for steps 2 p and 2 p + 1; what is left of D behind the last 64 goes as in 16 bit.
template <int D, bool WIDE>
__device__ __forceinline__ constexpr int key_element(int step, int g) {
  const int pair = step >> 1;
  if (!WIDE && 64 * (pair + 1) <= D) return 64 * pair + 16 * g + 8 * (step & 1);
  return 32 * step + 8 * g;
}

// Values: D in blocks of up to 16 E elements, E = 8, 4 or 2, lane r of 16 has E of each at r E.  The last block may have
// fewer than 16 lanes (80, 96 and 112 wide, E = 8): the rest read the last one's and compute what nobody writes, which is
// cheaper than a second and third load a token (112 wide, fp8, 32 sequences of 8192 tokens: 89 us against 110).
template <int D>
struct ValueBlocks {
  static constexpr int e_of(int rest) { return rest > 64 ? 8 : rest > 32 ? 4 : 2; }
  static constexpr int start(int i) {
    int at = 0;
    for (int k = 0; k < i; ++k) at += 16 * e_of(D - at);
    return at;
  }
  static constexpr int e(int i) { return e_of(D - start(i)); }
  static constexpr int lanes(int i) { return D - start(i) >= 16 * e(i) ? 16 : (D - start(i)) / e(i); }
  static constexpr int count() {
    int n = 0;
    while (start(n) < D) ++n;
    return n;
  }
  // dwords of one token that a lane holds of blocks before i; accumulators of blocks before i
  static constexpr int dword(int i, int bytes) {
    int n = 0;
    for (int k = 0; k < i; ++k) n += (e(k) * bytes + 3) / 4;
    return n;
  }
  static constexpr int rows(int i) {
    int n = 0;
    for (int k = 0; k < i; ++k) n += e(k);
    return n;
  }
};

// f(0), f(1), .. f(N - 1), each a constant
template <int N, int I = 0, class F>
__device__ __forceinline__ void for_each(F&& f) {
  if constexpr (I < N) {
    f(std::integral_constant<int, I>{});
    for_each<N, I + 1>(f);
  }
}

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
    // code + 128 in the last byte of an fp16 whose last place is 1: 1024 + 128 + code, and 1152 off.  (Keys too: with the 1152 left in, and
    // 1152 * sum q taken off the product, the fp32 sum of queries with a mean runs so high that the score is what its rounding leaves.)
    const uint32_t u = w ^ 0x80808080u;
    lo = __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u), hi = __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u);
    const half2_t bias = {(half_t)1152.f, (half_t)1152.f};
    lo = as_u32(as_half2(lo) - bias), hi = as_u32(as_half2(hi) - bias);
  }
}

// Rows of 16 lanes change places pairwise, then the halves of the wave.  In assembly: of a builtin's two results the compiler
// uses one for both where a value is swapped with itself.  (Two wait states between a result and its swap.)
__device__ __forceinline__ float max_over_groups(float x) {
  float y = x;
  asm("s_nop 1\n\tv_permlane16_swap_b32 %0, %1" : "+v"(x), "+v"(y));
  x = fmaxf(x, y), y = x;
  asm("s_nop 1\n\tv_permlane32_swap_b32 %0, %1" : "+v"(x), "+v"(y));
  return fmaxf(x, y);
}
__device__ __forceinline__ float sum_over_groups(float x) {
  x += __shfl_xor(x, 16);
  return x + __shfl_xor(x, 32);
}

// Eight weights as two parts that add up to them; of a weight above 0 (2^-24 in fp16) both are, if the second has to be made so.
template <class C>
__device__ __forceinline__ void positive_parts(const float (&p)[8], typename Vec8<C>::type& first, typename Vec8<C>::type& second) {
#pragma unroll
  for (int j = 0; j < 8; j += 2) {
    float low[2];
    if constexpr (__is_same(C, half_t)) {
      const auto z = __builtin_amdgcn_cvt_pkrtz(p[j], p[j + 1]);
      first[j] = (half_t)z[0], first[j + 1] = (half_t)z[1];
      low[0] = fminf(p[j], 0x1p-24f), low[1] = fminf(p[j + 1], 0x1p-24f);
    } else {
      first[j] = __builtin_bit_cast(bf16_t, (uint16_t)(__builtin_bit_cast(uint32_t, p[j]) >> 16));
      first[j + 1] = __builtin_bit_cast(bf16_t, (uint16_t)(__builtin_bit_cast(uint32_t, p[j + 1]) >> 16));
      low[0] = p[j] * 0x1p-20f, low[1] = p[j + 1] * 0x1p-20f;
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) second[j + i] = (C)fmaxf(p[j + i] - (float)first[j + i], low[i]);
  }
}

// 2^(m - to), 0 where there is nothing (m = -inf), whatever `to` is
__device__ __forceinline__ float weight(float m, float to) { return m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - to); }

// The natural logarithm of 2^m * sum.  NaN where the sum is: scores that are NaN are no maximum, so m alone cannot tell a head all of
// whose scores are NaN (m = -inf, sum NaN) from one that sees no token (m = -inf, sum 0).
__device__ __forceinline__ float log_of_sum(float m, float sum) {
  return m == -INFINITY && sum == 0.f ? -INFINITY : (m + log2f(sum)) * 0.693147180559945309f;
}

// How many workgroups (of four waves) a compute unit is to have where the work is shared out: as few as keep enough of the
// cache in flight, for every one more is a column cut once more and has less in a row.  One of 16-bit rows of 160 bytes
// and more (32 sequences of 4096 tokens, 128 wide: one 84 us, two 90, three 106; 256 wide 91 and 122), two of shorter ones, whose
// tiles are small (64 wide 99, 91, 92, four 95; fp8 128 wide, 64 sequences, 113, 91, 106), and of 8 bits, whose waves have codes
// to convert, up to 256 wide (92 and 103; two blocks of 16 heads of more than 128 elements leave registers for one).
constexpr int attention_per_unit(int head_dim, int row_blocks, int format) {
  return head_dim > 64 && (cache_is_16bit(format) || head_dim > (row_blocks == 2 ? 128 : 192)) ? 1 : 2;
}

// How many of them the registers are to leave room for: more where they fit without spills, for columns that stay whole.
constexpr int attention_room(int head_dim, int row_blocks) {
  if (head_dim <= 64) return row_blocks == 1 ? 3 : 2;
  return head_dim > (row_blocks == 2 ? 128 : 192) ? 1 : 2;
}

// Blocks of 16 heads that a workgroup takes, with one read of the keys and values: two where more than 16 heads share them (32
// heads on one, 48 sequences of 6000 tokens, bf16, one block and two: 128 wide 55 and 37 us, 160 wide 67 and 45, 256 wide 103 and 82,
// some registers of which lie in memory; int8, from 160 wide on with one workgroup a compute unit in place of two: 128 wide 42 and 36,
// 160 wide 48 and 47, 256 wide 64 and 58).  One wave has both blocks: from 160 wide on that is one wave a SIMD, and nothing covers the way
// from keys through scores and exponentials to values, so these cases stay at 1.6 to 3.3 times their bytes.
constexpr int attention_row_blocks(int heads_a_column) { return heads_a_column > 16 ? 2 : 1; }

// A wave's LDS: 32 keys on their way into the operand's order, later 16 rows of its result.
constexpr int attention_wave_lds(int head_dim, int format) {
  const int bytes = head_dim * (cache_is_16bit(format) ? 2 : 1), keys = kAttnTile * (bytes / 16 | 1) * 16, result = 16 * (head_dim + 4) * 4;
  return keys > result ? keys : result;
}

// Whether a workgroup's heads are taken PACKED, see there: up to eight, where instructions and not memory bound the kernel, which
// is in narrow heads of 8 bits (64 sequences of 4000 tokens, eight heads on each of eight: int8, 64 wide, 66.6 -> 65.6 us, 80 wide 82 -> 78,
// 96 wide 82 -> 78, 112 wide 89 -> 86; fp8, 64 wide 54 -> 51, 112 wide 85 -> 83; with four heads on each, fp8, 128 wide 88 -> 88 and 16
// bits, 64 wide, 83 -> 83).
constexpr bool attention_packs(int heads_a_column, int head_dim, int format) { return heads_a_column <= 8 && head_dim < 128 && !cache_is_16bit(format); }

// What lane n ^ 8 of the 16 has; into lane n < 8 its four elements, behind its own four.
template <class T>
__device__ __forceinline__ T other_half(T x) { return dpp_move<0x128>(x); }
__device__ __forceinline__ float into_upper_half(float x, float upper) {  // lanes n >= 8 get lane n - 8's `upper`
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(__builtin_bit_cast(int, x), __builtin_bit_cast(int, upper), 0x128, 0xF, 0xC, false));
}
template <class C8>
__device__ __forceinline__ void both_halves(C8& x) {
  uint4_t w = __builtin_bit_cast(uint4_t, x);
  w[2] = other_half((uint32_t)w[0]), w[3] = other_half((uint32_t)w[1]);
  x = __builtin_bit_cast(C8, w);
}

// T: queries and output; FORMAT: the cache; D: head_dim; NT: blocks of 16 heads that a workgroup takes.  PACKED: of its 16
// columns at most eight are heads, so between the products lane n has the scores of head n & 7: n < 8 of its lane group's first
// four tokens, n >= 8 of the other four, and the softmax half the instructions.
template <class T, int FORMAT, int D, int NT, bool PACKED>
__global__ __launch_bounds__(64 * kAttnWaves, attention_room(D, NT)) void attention_kernel(const AttnArgs a) {
  static_assert(NT == 1 || !PACKED, "");
  constexpr int kEach = PACKED ? 4 : 8;  // tokens of a tile whose scores a lane has
  constexpr bool kWide = cache_is_16bit(FORMAT);
  using C = typename std::conditional<kWide, T, half_t>::type;  // what the products are taken in
  typedef typename Vec8<C>::type C8;
  constexpr float kLift = __is_same(C, half_t) ? 15.f : 0.f;  // weights are taken times 2^kLift
  constexpr int kBytes = kWide ? 2 : 1;
  constexpr int kSteps = (D + 31) / 32;
  using VB = ValueBlocks<D>;
  constexpr int kVDwords = VB::dword(VB::count(), kBytes);
  constexpr int kAcc = VB::rows(VB::count());
  constexpr int kKeyPieces = D * kBytes / 2;              // of 16 bytes, of eight tokens
  constexpr int kKeyLoads = (4 * kKeyPieces + 63) / 64;
  constexpr int kKeyPitch = (D * kBytes / 16 | 1) * 16;   // an odd number of pieces: 16 rows on 64 banks
  constexpr int kWaveLds = attention_wave_lds(D, FORMAT);

  constexpr int kRow = D + 4;                             // of a wave's result: 16 rows on 64 banks

  __shared__ float sm[kAttnWaves][16 * NT][3];  // a wave's m, l and the power of two, from 2^m, that its o is relative to (or -inf)
  __shared__ ShareSearch search;
  extern __shared__ __align__(16) char lds[];

  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
  const int lane_tokens = PACKED ? (n & 8) >> 1 : 0;  // where the kEach of eight begin
  char* const keys = lds + wave * kWaveLds;
  auto result = [&](int w, int row) { return reinterpret_cast<float*>(lds + w * kWaveLds) + row * kRow; };
  const int group = a.heads / a.shape.kv_heads;  // heads that share a key-value head
  const int columns = a.shape.kv_heads * a.head_blocks;
  const int capacity = a.max_pages << a.shape.page_shift;
  const int place_mask = (1 << a.shape.page_shift) - 1;

  Share share;
  Shares shares(0, 1);
  if (a.pieces) {
    share = find_share(a, capacity, columns, wave, lane, search, shares);
  } else {  // no column can be cut: one a workgroup
    share.sequence = blockIdx.x / columns, share.length = a.lengths[share.sequence], share.sequence_begin = 0;
    const unsigned cost = span_of(share.length, capacity, a.window).units + kColumnCost;
    share.at = (blockIdx.x - share.sequence * columns) * cost, share.end = share.at + cost;
  }

  while (share.at < share.end) {
    const Span span = span_of(share.length, capacity, a.window);
    const int sequence = share.sequence, cost = span.units + kColumnCost;
    const int column = (share.at - share.sequence_begin) / cost, from = (share.at - share.sequence_begin) - column * cost;
    const int to = min((unsigned)cost, from + (share.end - share.at));
    const unsigned column_begin = share.at - from;
    share.at += to - from;
    if (share.at == share.sequence_begin + (unsigned)cost * columns) {
      share.sequence_begin = share.at, ++share.sequence;
      if (share.at < share.end) share.length = a.lengths[share.sequence];
    }
    // the first kColumnCost of a column stand for no tokens; a share that ends there leaves it all to the next
    const int unit0 = max(from - kColumnCost, 0), units_here = max(to - kColumnCost, 0) - unit0;
    const bool complete = unit0 == 0 && to == cost;
    if (to <= kColumnCost && !complete) continue;
    const int kv_head = column / a.head_blocks, head_block = column - kv_head * a.head_blocks;
    const int begin = span.tile0 + unit0 * kAttnWaves, end = span.tile0 + min((unit0 + units_here) * kAttnWaves, span.tiles);
    const int length = span.length, first_token = span.first;
    const int* const table = a.table + (size_t)sequence * a.max_pages;

    // The page of a token; beyond the last one's, the last one's.  (Without a branch: the compiler counts the loads in flight
    // behind one as the fewer, and waits for the next keys before it uses these values.)
    const int last_token = max(length - 1, 0);
    auto page_of = [&](int token) { return table[min(token, last_token) >> a.shape.page_shift]; };
    auto row_of = [&](int page, int token) { return cache_row(a.shape, (unsigned)page < (unsigned)a.shape.pages ? page : 0, kv_head, token & place_mask); };

    uint4_t kraw[kKeyLoads];
    uint32_t vr[8][kVDwords];
    float ks[kEach], vs[kEach];
    // Eight tokens' keys are one piece of memory: a load takes 64 times 16 bytes of the tile as they lie, whole lines.
    auto load_keys = [&](int page, int tile) {  // page: that of the tokens 8 g ..
      const char* base[4];
#pragma unroll
      for (int e = 0; e < 4; ++e)
        base[e] = reinterpret_cast<const char*>(a.cache[0]) + row_of(__builtin_amdgcn_readlane(page, 16 * e), tile * kAttnTile + 8 * e) * (D * kBytes);
#pragma unroll
      for (int k = 0; k < kKeyLoads; ++k) {
        const int i = 64 * k + lane, lo = 64 * k / kKeyPieces, hi = min((64 * k + 63) / kKeyPieces, 3);
        const char* p = base[lo];
        int e = lo;
#pragma unroll
        for (int more = lo + 1; more <= hi; ++more)
          if (i >= more * kKeyPieces) p = base[more], e = more;
        if (64 * (k + 1) <= 4 * kKeyPieces || i < 4 * kKeyPieces)
          kraw[k] = __builtin_nontemporal_load(reinterpret_cast<const uint4_t*>(p + (i - e * kKeyPieces) * 16));
      }
    };
    // ... and goes through the wave's own LDS into the operand's order: row 16 t + n is that of lane n in product t.
    auto keys_to_lds = [&] {
#pragma unroll
      for (int k = 0; k < kKeyLoads; ++k) {
        const int i = 64 * k + lane;
        const int token = i / (D * kBytes / 16), piece = i - token * (D * kBytes / 16), r = token & 7;
        if (64 * (k + 1) <= 4 * kKeyPieces || i < 4 * kKeyPieces)
          *reinterpret_cast<uint4_t*>(keys + ((r >> 2) * 16 + (token >> 3) * 4 + (r & 3)) * kKeyPitch + piece * 16) = kraw[k];
      }
      asm volatile("" ::: "memory");  // read by other lanes; a wave's LDS accesses keep their order
    };
    auto load_values = [&](size_t row) {
      const char* const vp = reinterpret_cast<const char*>(a.cache[1]) + row * (D * kBytes);
#pragma unroll
      for (int j = 0; j < 8; ++j)
        for_each<VB::count()>([&](auto block) {
          constexpr int b = decltype(block)::value, e = VB::e(b), at = VB::dword(b, kBytes), bytes = e * kBytes, start = VB::start(b), lanes = VB::lanes(b);
          const char* const p = vp + (j * D + start + (lanes == 16 ? n : min(n, lanes - 1)) * e) * kBytes;
          if constexpr (bytes == 16) {
            const uint4_t w = __builtin_nontemporal_load(reinterpret_cast<const uint4_t*>(p));
            vr[j][at] = w[0], vr[j][at + 1] = w[1], vr[j][at + 2] = w[2], vr[j][at + 3] = w[3];
          } else if constexpr (bytes == 8) {
            const uint2_t w = __builtin_nontemporal_load(reinterpret_cast<const uint2_t*>(p));
            vr[j][at] = w[0], vr[j][at + 1] = w[1];
          } else if constexpr (bytes == 4) {
            vr[j][at] = __builtin_nontemporal_load(reinterpret_cast<const uint32_t*>(p));
          } else {
            vr[j][at] = __builtin_nontemporal_load(reinterpret_cast<const uint16_t*>(p));
          }
        });
    };
    auto load_scales = [&](size_t row) {
      if constexpr (!kWide) {
        if constexpr (PACKED) row += lane_tokens;
#pragma unroll
        for (int i = 0; i < kEach / 4; ++i) {
          const float4_t kq = *reinterpret_cast<const float4_t*>(a.scale[0] + row + 4 * i), vq = *reinterpret_cast<const float4_t*>(a.scale[1] + row + 4 * i);
#pragma unroll
          for (int j = 0; j < 4; ++j) ks[4 * i + j] = kq[j], vs[4 * i + j] = vq[j];
        }
      }
    };

    int tile = begin + wave;
    int page = page_of(tile * kAttnTile + g * 8), page_next = -1, page_after = -1;
    float sink_here[NT];  // (of the head that this thread joins at the end)
#pragma unroll
    for (int b = 0; b < NT; ++b) {
      const int in_group = (head_block * NT + b) * 16 + (int)(threadIdx.x >> 4);
      sink_here[b] = a.sinks && in_group < group ? a.sinks[kv_head * group + in_group] * 1.44269504088896341f : -INFINITY;
    }
    typename Vec8<T>::type q_raw[NT][kSteps];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int row = (head_block * NT + t) * 16 + n;
      const T* const qrow = reinterpret_cast<const T*>(a.q) + ((size_t)sequence * a.heads + (size_t)kv_head * group + row) * D;
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        const int d = key_element<D, kWide>(s, g);
        q_raw[t][s] = typename Vec8<T>::type{};
        if (row < group && d < D) q_raw[t][s] = *reinterpret_cast<const typename Vec8<T>::type*>(qrow + d);
      }
    }

    // The first tile's loads, and the page ids of the second: from here on keys, values and page ids are asked for a tile
    // ahead, each as soon as its registers are free.
    if (tile < end) {
      load_keys(page, tile);
      page_next = page_of((tile + kAttnWaves) * kAttnTile + g * 8);
      const size_t row = row_of(page, tile * kAttnTile + g * 8);
      load_scales(row);
      load_values(row);
    }

    // ---- queries: the second operand of the first product, held for the whole walk -----------------------------
    C8 q[NT][kSteps];
    float q_scale[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      q_scale[t] = a.score_scale;
      if constexpr (kWide) {
#pragma unroll
        for (int s = 0; s < kSteps; ++s) q[t][s] = q_raw[t][s];
      } else {
        float most = 0.f;
#pragma unroll
        for (int s = 0; s < kSteps; ++s)
#pragma unroll
          for (int i = 0; i < 8; ++i) most = fmaxf(most, fabsf((float)q_raw[t][s][i]));
        most = max_over_groups(most);
        const int e = most > 0.f ? 14 - ilogbf(most) : 0;  // 2^e * most in [2^14, 2^15)
        const int shift = min(max(e, -126), 126);
        q_scale[t] = ldexpf(a.score_scale, -shift);
#pragma unroll
        for (int s = 0; s < kSteps; ++s)
#pragma unroll
          for (int i = 0; i < 8; ++i) q[t][s][i] = (C)ldexpf((float)q_raw[t][s][i], shift);
        if constexpr (PACKED) {
          const float there = other_half(q_scale[t]);
          if (n >= 8) q_scale[t] = there;
        }
      }
    }

    float4_t acc[NT][kAcc];
    float m[NT], l[NT];
    float o_exp[NT];  // acc is o / 2^(m + o_exp - kLift) (quantised caches; else 2^(m - kLift))
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      m[t] = -INFINITY, l[t] = 0.f, o_exp[t] = -INFINITY;
#pragma unroll
      for (int i = 0; i < kAcc; ++i) acc[t][i] = float4_t{0.f, 0.f, 0.f, 0.f};
    }

    auto take = [&](auto last) {
      const int next = tile + kAttnWaves;
      const int v_first = tile * kAttnTile + g * 8;
      // the tokens v_first + j that take part
      const int low = max(first_token - v_first, 0), high = (unsigned)page < (unsigned)a.shape.pages ? min(length - v_first, 8) : 0;
      const bool whole = __all(low <= 0 && high == 8);

      // ---- scores ---------------------------------------------------------------------------------------------
      keys_to_lds();
      float p[NT][kEach];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        C8 kf[kSteps];
        uint4_t pair = {};
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
          const int d = key_element<D, kWide>(s, g);
          const char* const p = keys + (16 * t + n) * kKeyPitch + d * kBytes;
          uint4_t w = {0u, 0u, 0u, 0u};
          if constexpr (kWide) {
            if (32 * (s + 1) <= D || d < D) w = *reinterpret_cast<const uint4_t*>(p);
          } else {
            uint2_t c = {0u, 0u};
            if (64 * ((s >> 1) + 1) <= D) {
              if (s & 1) c = uint2_t{pair[2], pair[3]};
              else pair = *reinterpret_cast<const uint4_t*>(p), c = uint2_t{pair[0], pair[1]};
            } else if (32 * (s + 1) <= D || d < D) {
              c = *reinterpret_cast<const uint2_t*>(p);
            }
            uint32_t h[4];
            codes4_to_half<FORMAT>(c[0], h[0], h[1]);
            codes4_to_half<FORMAT>(c[1], h[2], h[3]);
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
          for (int i = 0; i < 4; ++i) {
            const float x = sc[i];
            if constexpr (!PACKED) p[b][4 * t + i] = x;
            else p[b][i] = t == 0 ? x : into_upper_half(p[b][i], x);
          }
        }
      }
      asm volatile("" ::: "memory");  // the next keys come behind these
      size_t next_row = 0;
      if constexpr (!decltype(last)::value) {
        load_keys(page_next, next);
        // (before the values, so that the wait for it waits for none of them)
        page_after = page_of((next + kAttnWaves) * kAttnTile + g * 8);
        next_row = row_of(page_next, next * kAttnTile + g * 8);
      }

      // ---- running maximum and sum ----------------------------------------------------------------------------
      if constexpr (!kWide) {
        if (!whole) {
#pragma unroll
          for (int j = 0; j < kEach; ++j)
            if (lane_tokens + j < low || lane_tokens + j >= high) ks[j] = 0.f, vs[j] = 0.f;
        }
      }
#pragma unroll
      for (int b = 0; b < NT; ++b) {
        float most = -INFINITY;
#pragma unroll
        for (int j = 0; j < kEach; ++j) {
          p[b][j] *= q_scale[b];
          if constexpr (!kWide) p[b][j] *= ks[j];
        }
        if (!whole) {
#pragma unroll
          for (int j = 0; j < kEach; ++j)
            if (lane_tokens + j < low || lane_tokens + j >= high) p[b][j] = -INFINITY;
        }
#pragma unroll
        for (int j = 0; j < kEach; ++j) most = fmaxf(most, p[b][j]);
        most = max_over_groups(most);
        if constexpr (PACKED) most = fmaxf(most, other_half(most));
        most = fmaxf(m[b], most);
        const float base = most == -INFINITY ? 0.f : most;
        float shrink = weight(m[b], base);
        const float grown = m[b] - base;
        m[b] = most;
        l[b] *= shrink;
#pragma unroll
        for (int j = 0; j < kEach; ++j) {
          p[b][j] = __builtin_amdgcn_exp2f(p[b][j] - base);
          l[b] += p[b][j];
        }
        if constexpr (!kWide) {
          float top = 0.f;
#pragma unroll
          for (int j = 0; j < kEach; ++j) p[b][j] *= vs[j], top = fmaxf(top, fabsf(p[b][j]));
          top = max_over_groups(top);
          if constexpr (PACKED) top = fmaxf(top, other_half(top));
          // (smaller ones than 2^kLowest are small beside it; where o_exp lies below it, these weights are all zero)
          constexpr int kLowest = -112;
          const float before = o_exp[b] + grown;
          o_exp[b] = fmaxf(before, top > 0.f ? (float)max(__builtin_amdgcn_frexp_expf(top), kLowest) : -INFINITY);
          const float factor = __builtin_amdgcn_exp2f(fminf(kLift - o_exp[b], kLift - kLowest));
          shrink = weight(before, o_exp[b]);
#pragma unroll
          for (int j = 0; j < kEach; ++j) p[b][j] *= factor;
        }
        if constexpr (kWide && kLift != 0.f) {
#pragma unroll
          for (int j = 0; j < kEach; ++j) p[b][j] *= 0x1p15f;
        }
        // (a head of no tokens yet has nothing to scale: 0 by whatever)
        if (__any(shrink != 1.f)) {
#pragma unroll
          for (int i = 0; i < kAcc; ++i)
#pragma unroll
            for (int k = 0; k < 4; ++k) acc[b][i][k] *= shrink;
        }
      }
      C8 pf[NT], rest[NT];  // the weights' two parts
#pragma unroll
      for (int b = 0; b < NT; ++b) {
        if constexpr (kWide) {
          positive_parts<C>(p[b], pf[b], rest[b]);
        } else {
#pragma unroll
          for (int j = 0; j < kEach; ++j) pf[b][j] = (C)p[b][j], rest[b][j] = (C)(p[b][j] - (float)pf[b][j]);
        }
        if constexpr (PACKED) {  // the columns from 8 on are no heads': whatever they sum up is not read
          both_halves(pf[b]), both_halves(rest[b]);
        }
      }
      if constexpr (!decltype(last)::value) load_scales(next_row);

      // ---- values ---------------------------------------------------------------------------------------------
      if (!whole) {
        // what lies in dead places may be anything: its values count as zeros, not as zero times them
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if (j >= low && j < high) continue;
#pragma unroll
          for (int i = 0; i < kVDwords; ++i) vr[j][i] = 0u;
        }
      }
      for_each<VB::count()>([&](auto block) {
        constexpr int blk = decltype(block)::value, e_count = VB::e(blk), at = VB::dword(blk, kBytes), at_acc = VB::rows(blk);
        if constexpr (kWide) {
#pragma unroll
          for (int e = 0; e < e_count; e += 2) {  // (two at a time: a product that another waits for lies further back)
            uint4_t w[2];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const uint32_t odd = vr[2 * i + 1][at + (e >> 1)], even = vr[2 * i][at + (e >> 1)];
              w[0][i] = __builtin_amdgcn_perm(odd, even, 0x05040100u), w[1][i] = __builtin_amdgcn_perm(odd, even, 0x07060302u);
            }
#pragma unroll
            for (int part = 0; part < 2; ++part)
#pragma unroll
              for (int b = 0; b < NT; ++b)
#pragma unroll
                for (int k = 0; k < 2; ++k)
                  acc[b][at_acc + e + k] = mfma16<C>(__builtin_bit_cast(C8, w[k]), part == 0 ? rest[b] : pf[b], acc[b][at_acc + e + k]);
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
                acc[b][at_acc + 4 * dw + e] =
                    mfma16<C>(__builtin_bit_cast(C8, w), pf[b], mfma16<C>(__builtin_bit_cast(C8, w), rest[b], acc[b][at_acc + 4 * dw + e]));
            }
          }
        }
      });
      if constexpr (!decltype(last)::value) {
        load_values(next_row);
        page = page_next, page_next = page_after;
      }
    };
    if (tile < end) {
      for (; tile + kAttnWaves < end; tile += kAttnWaves) take(std::false_type{});
      take(std::true_type{});
    }

    // ---- the waves' results, joined in their order -------------------------------------------------------------
#pragma unroll
    for (int b = 0; b < NT; ++b) {
      l[b] = sum_over_groups(l[b]);
      if constexpr (PACKED) l[b] += other_half(l[b]);
      if (g == 0) sm[wave][16 * b + n][0] = m[b], sm[wave][16 * b + n][1] = l[b], sm[wave][16 * b + n][2] = (kWide ? (m[b] == -INFINITY ? m[b] : 0.f) : o_exp[b]) - kLift;
    }
#pragma unroll
    for (int b = 0; b < NT; ++b) {
      if (b > 0) __syncthreads();
      for_each<VB::count()>([&](auto block) {
        constexpr int blk = decltype(block)::value, e_count = VB::e(blk), at_acc = VB::rows(blk), start = VB::start(blk), lanes = VB::lanes(blk);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (lanes < 16 && 4 * g + i >= lanes) continue;
#pragma unroll
          for (int e = 0; e < e_count; ++e) result(wave, n)[start + (4 * g + i) * e_count + e] = acc[b][at_acc + e][i];
        }
      });
      __syncthreads();
      // 16 lanes a head
      const int row = threadIdx.x >> 4, head_in_group = (head_block * NT + b) * 16 + row;
      if (head_in_group < group) {
        const int head = kv_head * group + head_in_group;
        float most = -INFINITY;
#pragma unroll
        for (int w = 0; w < kAttnWaves; ++w) most = fmaxf(most, sm[w][16 * b + row][0]);
        const float sink = complete ? sink_here[b] : -INFINITY;
        const float base = fmaxf(most, sink);
        float root[kAttnWaves], total_weight = weight(sink, base);
#pragma unroll
        for (int w = 0; w < kAttnWaves; ++w) {
          // (-inf: nothing summed up.  The root: a factor may lie below fp32's range where factor times sum does not)
          const float power = sm[w][16 * b + row][2];
          root[w] = power == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(0.5f * (sm[w][16 * b + row][0] - base + power));
          total_weight += weight(sm[w][16 * b + row][0], base) * sm[w][16 * b + row][1];
        }
        if (complete) {
          const size_t at = (size_t)sequence * a.heads + head;
          const float inv = total_weight > 0.f ? 1.f / total_weight : (total_weight == 0.f ? 0.f : total_weight);
          for (int d = threadIdx.x & 15; d < D; d += 16) {
            float x = 0.f;
#pragma unroll
            for (int w = 0; w < kAttnWaves; ++w) x += root[w] * result(w, row)[d] * root[w];
            reinterpret_cast<T*>(a.out)[at * D + d] = (T)(x * inv);
          }
          if (a.lse && (threadIdx.x & 15) == 0) a.lse[at] = log_of_sum(base, total_weight);
        } else {
          // the piece that a head begins with is a workgroup's second, any other its first
          const size_t part = ((size_t)blockIdx.x * 2 + (unit0 == 0)) * a.rows + 16 * b + row;
          for (int d = threadIdx.x & 15; d < D; d += 16) {
            float x = 0.f;
#pragma unroll
            for (int w = 0; w < kAttnWaves; ++w) x += root[w] * result(w, row)[d] * root[w];
            a.part_o[part * D + d] = x;
          }
          if ((threadIdx.x & 15) == 0) a.part_ml[2 * part] = most, a.part_ml[2 * part + 1] = total_weight;
        }
      }
    }
    if (unit0 == 0 && threadIdx.x == 0 && a.pieces) {
      int* const pieces = a.pieces + 2 * ((size_t)sequence * columns + column);
      pieces[0] = blockIdx.x, pieces[1] = complete ? blockIdx.x : shares.owner(column_begin + cost - 1);
    }
    __syncthreads();  // the LDS is free again
  }
}

template <class T, int FORMAT, int D, int NT, bool PACKED>
int launch_attention(const AttnArgs& a, hipStream_t stream) {
  constexpr int kLds = kAttnWaves * attention_wave_lds(D, FORMAT);
  if constexpr (kLds > 65536 - 4096) {
    static bool raised[kMaxDevices];
    if (raise_lds_limit<kLds>(attention_kernel<T, FORMAT, D, NT, PACKED>, raised) != 0) return -1;
  }
  attention_kernel<T, FORMAT, D, NT, PACKED><<<a.workgroups, 64 * kAttnWaves, kLds, stream>>>(a);
  DQ_CHECK_HIP(hipGetLastError());
  return 0;
}

template <class T, int FORMAT, int D>
int attention_of_width(const AttnArgs& a, hipStream_t stream) {
  const int group = a.heads / a.shape.kv_heads;
  if constexpr (attention_packs(1, D, FORMAT))
    if (attention_packs(group, D, FORMAT)) return launch_attention<T, FORMAT, D, 1, true>(a, stream);
  if (attention_row_blocks(group) == 2) return launch_attention<T, FORMAT, D, 2, false>(a, stream);
  return launch_attention<T, FORMAT, D, 1, false>(a, stream);
}

template <class T, int FORMAT>
int attention_of_type(const AttnArgs& a, hipStream_t stream) {
  switch (a.shape.head_dim) {
    case 64: return attention_of_width<T, FORMAT, 64>(a, stream);
    case 80: return attention_of_width<T, FORMAT, 80>(a, stream);
    case 96: return attention_of_width<T, FORMAT, 96>(a, stream);
    case 112: return attention_of_width<T, FORMAT, 112>(a, stream);
    case 128: return attention_of_width<T, FORMAT, 128>(a, stream);
    case 160: return attention_of_width<T, FORMAT, 160>(a, stream);
    case 192: return attention_of_width<T, FORMAT, 192>(a, stream);
    case 256: return attention_of_width<T, FORMAT, 256>(a, stream);
    default: DQ_FAIL("attention: no kernel for a head of %d", a.shape.head_dim);
  }
}

}  // namespace dq
