// The experts' products at a few rows an expert: a workgroup has 16 weight rows of the gate and the 16 of the up projection (or 32
// weight rows) of one expert and multiplies them with up to 16 of its rows at a time.
//
// What bounds it is the weights' way out of memory, every expert that has rows being read once, and the load unit of a CU, which
// takes two cycles for 64 bytes or a piece of a row, whichever is less.  So loads are whole cache lines of neighbouring lanes: a
// chunk of 256 k is 128 bytes of a weight row, eight rows a load, a step of 128 k is 256 bytes of an activation row, four rows a
// load, and of those rows only the expert's own.  K is cut over the workgroup's waves.  A wave is a pipeline of its own: what it loads,
// two chunks and two steps ahead, goes through LDS that it alone writes and reads into the order of the matrix instruction, whose
// k are labelled 32 g + 8 j + e for its lane group g and the j-th of the step's four instructions, for both operands; its LDS
// operations are carried out in their order, so there is no barrier.  The waves' sums meet in LDS at the end.
//
// Measured: one token, 8 of 128 experts, 1024 x 4096 uint4 "up" 10 us (3.4 TB/s; 17 with words straight into registers), 4096 x 1024 "down"
// 9; 64 tokens, 4 of 32 experts, 2880 x 2880 MXFP4 61 to 72 and 38 to 41 us (4.0 to 4.6 and 3.5 to 3.7 TB/s: rows end inside cache lines,
// where lines are whole it reaches 5.7).
#include "dq_experts.h"

#include <math.h>

#include <algorithm>
#include <type_traits>

namespace dq {

int experts_tiles(const experts::Args& a, int mxfp4, bool up, int tile_rows, hipStream_t stream);

namespace {

using experts::Args;

constexpr int kStep = 128;  // k of a step: 32 a lane group
constexpr int kWaves = 4;   // pipelines of a workgroup

// Work is counted in parts: up to `most` rows of an expert, the experts one behind the other.  Every wave counts and finds them for
// itself: a lane holds the rows of experts lane, 64 + lane, ... of the first 256, all asked for at once; beyond, they are asked for
// again.
struct Part {
  int expert, begin, end;  // rows begin .. end - 1
};
struct Parts {
  static constexpr int kHeld = 4;
  const Args& a;
  const int most;
  int begin[kHeld], end[kHeld];

  __device__ __forceinline__ Parts(const Args& args, int rows) : a(args), most(rows) {
    const int lane = threadIdx.x & 63;
    int raw[kHeld][2];
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
      const int e = min(64 * i + lane, a.experts - 1);
      raw[i][0] = a.Starts[e], raw[i][1] = a.Starts[e + 1];
    }
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
      begin[i] = min(max(raw[i][0], 0), a.pairs);
      end[i] = 64 * i + lane < a.experts ? min(max(raw[i][1], begin[i]), a.pairs) : begin[i];
    }
  }
  // f(first expert of 64, the lane's rows) until it is content
  template <class F>
  __device__ __forceinline__ void each(F f) const {
#pragma unroll
    for (int i = 0; i < kHeld; ++i)
      if (f(64 * i, begin[i], end[i])) return;
    for (int base = 64 * kHeld; base < a.experts; base += 64) {
      int b = 0, e = 0;
      if (base + (int)(threadIdx.x & 63) < a.experts) experts::rows_of(a, base + (threadIdx.x & 63), b, e);
      if (f(base, b, e)) return;
    }
  }
  // inclusive sum of the lanes' parts, bit by bit of them (most experts have one); `all`: of all lanes
  __device__ __forceinline__ int upto(int b, int e, int& all) const {
    const int n = (e - b + most - 1) / most;
    int sum = n;
    all = 0;
    for (int bit = 0;; ++bit) {
      if (__ballot(n >> bit != 0) == 0) return sum;
      const unsigned long long set = __ballot((n >> bit) & 1);
      sum += (int)__builtin_amdgcn_mbcnt_hi((unsigned)(set >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)set, 0)) << bit;
      all += __popcll(set) << bit;
    }
  }
  __device__ __forceinline__ int count() const {
    int all = 0;
    each([&](int, int b, int e) {
      int here;
      upto(b, e, here);
      all += here;
      return false;
    });
    return all;
  }
  __device__ __forceinline__ Part nth(int n) const {  // (n below count())
    Part found{0, 0, 0};
    each([&](int base, int b, int e) {
      int here;
      const int sum = upto(b, e, here);
      if (n >= here) {
        n -= here;
        return false;
      }
      const unsigned long long beyond = __ballot(sum > n);
      const int at = __builtin_ctzll(beyond);
      const int first = __builtin_amdgcn_readlane(b, at), last = __builtin_amdgcn_readlane(e, at);
      const int before = __builtin_amdgcn_readlane(sum, at) - (last - first + most - 1) / most;
      found.expert = base + at;
      found.begin = first + (n - before) * most;
      found.end = min(found.begin + most, last);
      return true;
    });
    return found;
  }
};

constexpr int kChunk = 256;       // k of a chunk: two steps, a cache line of a row
constexpr int kWordsArea = 4096;  // a wave's LDS: 32 weight rows of 128 bytes,
constexpr int kScalesArea = 512;  // and of up to 16 bytes of scales, and of zero points
constexpr int kSumsArea = 2048;   // 32 sums of 16 rows, twice
constexpr int kActsRoom = 120 * 1024;  // of a workgroup, at least
constexpr int kDescriptor = 0x00027000, kNontemporal = 2;

__device__ __forceinline__ __amdgpu_buffer_rsrc_t bytes_at(const void* p, unsigned bytes) {
  return __builtin_amdgcn_make_buffer_rsrc((void*)p, 0, bytes, kDescriptor);
}

// Where 16-byte piece `piece` of a row lies in the wave's LDS: the lanes of one row number each, or of one piece, are in different banks.
__device__ __forceinline__ int word_place(int row, int piece) { return row * 128 + ((piece ^ ((row >> 1) & 7)) << 4); }
__device__ __forceinline__ int act_place(int row, int piece, int stride) { return row * stride + ((piece ^ (row & 15)) << 4); }

constexpr unsigned kNowhere = 0xFFFFFF00u;  // an offset beyond the bytes of any descriptor

// What a lane's half of a chunk's scales is, a step's: bytes, and from where
template <class W>
__host__ __device__ constexpr int half_scales() {
  return (kStep >> W::kShift) * W::kScaleBytes;  // 2, 4 or 8
}

// Where a pipeline's two blocks of 16 weight rows come from, by their number in its sequence.
// Of one expert: tile after tile of its columns.
template <class W>
struct TilesOf {
  const uint8_t* words;
  size_t tile_bytes, second_bytes;  // of words; to the second block
  __amdgpu_buffer_rsrc_t scales, zeros;
  unsigned lane_scales, tile_scales;
  int end;

  __device__ __forceinline__ TilesOf(const Args& a, int expert, int rows, int columns, int second, int end_) : end(end_) {
    const int lane = threadIdx.x & 63;
    const unsigned row_bytes = (unsigned)a.K >> 1, row_scales = ((unsigned)a.K >> W::kShift) * W::kScaleBytes;
    const size_t first = (size_t)expert * rows;
    words = a.B + first * row_bytes;
    tile_bytes = (size_t)columns * row_bytes, second_bytes = (size_t)second * row_bytes;
    scales = bytes_at((const uint8_t*)a.S + first * row_scales, (unsigned)rows * row_scales);
    if constexpr (W::kZeros) zeros = bytes_at((const uint8_t*)a.Z + first * row_scales, (unsigned)rows * row_scales);
    lane_scales = (unsigned)((lane >> 1) + (lane < 32 ? 0 : second - 16)) * row_scales + (lane & 1) * half_scales<W>();
    tile_scales = columns * row_scales;
  }
  __device__ __forceinline__ const uint8_t* block(int tile, int t) const { return words + tile * tile_bytes + t * second_bytes; }
  __device__ __forceinline__ bool on(int tile, int) const { return tile < end; }
  __device__ __forceinline__ unsigned scale_at(int tile) const { return tile < end ? lane_scales + tile * tile_scales : kNowhere; }
};

// Of several experts the same 16 columns, two experts at a time.
template <class W>
struct ExpertsOf {
  const uint8_t* words;
  unsigned expert_scales, lane_scales;
  size_t expert_bytes;
  __amdgpu_buffer_rsrc_t scales, zeros;
  int experts, count;  // experts: lane i has the i-th

  __device__ __forceinline__ ExpertsOf(const Args& a, int n0, int experts_, int count_) : experts(experts_), count(count_) {
    const int lane = threadIdx.x & 63;
    const unsigned row_bytes = (unsigned)a.K >> 1, row_scales = ((unsigned)a.K >> W::kShift) * W::kScaleBytes;
    words = a.B + (size_t)n0 * row_bytes;
    expert_bytes = (size_t)a.N * row_bytes, expert_scales = (unsigned)a.N * row_scales;
    scales = bytes_at(a.S, (unsigned)a.experts * expert_scales);
    if constexpr (W::kZeros) zeros = bytes_at(a.Z, (unsigned)a.experts * expert_scales);
    lane_scales = (unsigned)(n0 + ((lane >> 1) & 15)) * row_scales + (lane & 1) * half_scales<W>();
  }
  __device__ __forceinline__ int expert(int q, int t) const { return __builtin_amdgcn_readlane(experts, min(2 * q + t, count - 1)); }
  __device__ __forceinline__ const uint8_t* block(int q, int t) const { return words + expert(q, t) * expert_bytes; }
  __device__ __forceinline__ bool on(int q, int t) const { return 2 * q + t < count; }
  __device__ __forceinline__ unsigned scale_at(int q) const {
    const int t = (threadIdx.x & 63) >> 5;
    return 2 * q + t < count ? lane_scales + (unsigned)(t ? expert(q, 1) : expert(q, 0)) * expert_scales : kNowhere;
  }
};

// A wave's part of the products of some rows, which lie in LDS, with pairs of blocks of 16 weight rows, one pair after the other: of
// each the chunks c0 .. c1 - 1.  The chunks of all pairs are one sequence, whose weights are asked for DEPTH chunks ahead.  A load that is
// of no use (behind the sequence, beyond K) names an offset beyond its descriptor's bytes, which reads zeros.
// LINES: rows are whole cache lines, which are read once (nontemporal); otherwise two chunks share a line, and the one that comes second
// is to find it in a cache.
template <class W, int DEPTH, bool LINES, class Source>
struct Pipeline {
  const Args& a;
  const Source& from;
  unsigned w_at[2];
  int c0, c1;
  int w_q, w_c;  // what is asked for next
  bool idle;
  unsigned char *words, *scales;
  const unsigned char* acts;
  int acts_stride, act_row;
  uint4_t w_reg[DEPTH][4];
  static constexpr int kHalf = half_scales<W>();
  static constexpr bool kPairs = W::kScaleBytes == 1 && !LINES;       // from where two bytes lie, not four
  static constexpr int kRegs = kHalf == 8 || kPairs ? 2 : 1;
  unsigned s_reg[DEPTH][kRegs], z_reg[DEPTH][kRegs];

  __device__ __forceinline__ void ask_scales(unsigned (&to)[kRegs], __amdgpu_buffer_rsrc_t rows, unsigned at) const {
    if constexpr (kPairs) {
      to[0] = (unsigned short)__builtin_amdgcn_raw_buffer_load_b16(rows, at, 0, 0);
      to[1] = (unsigned short)__builtin_amdgcn_raw_buffer_load_b16(rows, at + 2, 0, 0);
    } else if constexpr (kHalf == 2) {
      to[0] = (unsigned short)__builtin_amdgcn_raw_buffer_load_b16(rows, at, 0, 0);
    } else if constexpr (kHalf == 4) {
      to[0] = __builtin_amdgcn_raw_buffer_load_b32(rows, at, 0, 0);
    } else {
      const uint2_t both = __builtin_bit_cast(uint2_t, __builtin_amdgcn_raw_buffer_load_b64(rows, at, 0, 0));
      to[0] = both[0], to[1] = both[1];
    }
  }
  __device__ __forceinline__ void put_scales(const unsigned (&from)[kRegs], unsigned char* area) const {
    const int lane = threadIdx.x & 63;
    unsigned char* const at = area + (lane >> 1) * 16 + (lane & 1) * kHalf;
    if constexpr (kPairs) {
      ((unsigned short*)at)[0] = (unsigned short)from[0];
      ((unsigned short*)at)[1] = (unsigned short)from[1];
    } else if constexpr (kHalf == 2) {
      *(unsigned short*)at = (unsigned short)from[0];
    } else if constexpr (kHalf == 4) {
      *(unsigned*)at = from[0];
    } else {
      *(uint2_t*)at = uint2_t{from[0], from[1]};
    }
  }
  __device__ __forceinline__ unsigned scale_of(const unsigned char* area, int row, int k) const {  // k of the chunk
    const unsigned char* const at = area + row * 16 + (k >> W::kShift) * W::kScaleBytes;
    if constexpr (W::kScaleBytes == 1) return *at;
    else return *(const unsigned short*)at;
  }

  __device__ __forceinline__ Pipeline(const Args& args, const Source& source, int first, int begin, int end, bool nothing, unsigned char* area,
                                      const unsigned char* rows, int held, int stride)
      : a(args), from(source), c0(begin), c1(end), w_q(first), w_c(begin), idle(nothing), words(area), scales(area + kWordsArea), acts(rows), acts_stride(stride) {
    const int lane = threadIdx.x & 63;
    const unsigned row_bytes = (unsigned)a.K >> 1;
    act_row = min(lane & 15, held - 1);  // (of the rows beyond those that LDS has room for, the last)
#pragma unroll
    for (int i = 0; i < 2; ++i) w_at[i] = (unsigned)(8 * i + (lane >> 3)) * row_bytes + 16 * (lane & 7);
#pragma unroll
    for (int u = 0; u < DEPTH; ++u) ask(u);
  }

  // (no condition but by arithmetic: a branch around a load would leave the compiler without its count of those in flight)
  __device__ __forceinline__ void ask(int u) {
    const int lane = threadIdx.x & 63, left = a.K - w_c * kChunk;  // k
    const unsigned at = (from.scale_at(w_q) + ((unsigned)(w_c * kChunk) >> W::kShift) * W::kScaleBytes) | (!idle && (lane & 1) * kStep < left ? 0u : kNowhere);
    ask_scales(s_reg[u], from.scales, at);
    if constexpr (W::kZeros) ask_scales(z_reg[u], from.zeros, at);
    const unsigned beyond = (lane & 7) * 32 < left ? 0u : kNowhere, bytes = 8u * (unsigned)a.K;  // 16 rows
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const __amdgpu_buffer_rsrc_t rows = bytes_at(from.block(w_q, t), !idle && from.on(w_q, t) ? bytes : 0u);
#pragma unroll
      for (int i = 0; i < 2; ++i)
        w_reg[u][2 * t + i] = __builtin_bit_cast(uint4_t, __builtin_amdgcn_raw_buffer_load_b128(rows, (w_at[i] + w_c * (kChunk / 2)) | beyond, 0, LINES ? kNontemporal : 0));
    }
    asm volatile("" ::: "memory");  // (chunk by chunk: loads come back in the order that they go out in)
    const bool wraps = w_c + 1 == c1;
    w_q += wraps ? 1 : 0;
    w_c = wraps ? c0 : w_c + 1;
  }
  // a chunk, c of its pair of blocks, out of its registers
  __device__ __forceinline__ void chunk(int u, int c, float4_t (&acc)[2]) {
    const int lane = threadIdx.x & 63, g = lane >> 4, r = lane & 15;
#pragma unroll
    for (int i = 0; i < 4; ++i) *reinterpret_cast<uint4_t*>(words + word_place(8 * i + (lane >> 3), lane & 7)) = w_reg[u][i];
    put_scales(s_reg[u], scales);
    if constexpr (W::kZeros) put_scales(z_reg[u], scales + kScalesArea);
    asm volatile("" ::: "memory");  // (what is written here other lanes read)
    ask(u);
    if (!idle) {
      // a step's operands are asked for before the first of them is used
      uint4_t w[2][2];
      typename W::Scale scale[2][2];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          w[h][t] = *reinterpret_cast<const uint4_t*>(words + word_place(16 * t + r, 4 * h + g));
          const int k = h * kStep + 32 * g;
          scale[h][t] = W::scale(scale_of(scales, 16 * t + r, k), W::kZeros ? scale_of(scales + kScalesArea, 16 * t + r, k) : 0u);
        }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        typename W::frag x[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = *reinterpret_cast<const typename W::frag*>(acts + c * (2 * kChunk) + act_place(act_row, 16 * h + 4 * g + j, acts_stride));
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int t = 0; t < 2; ++t) acc[t] = W::mfma(x[j], W::decode(w[h][t][j], scale[h][t]), acc[t]);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    asm volatile("" ::: "memory");
  }
};

template <class W>
__host__ __device__ constexpr int wave_area() {
  return kWordsArea + kScalesArea * (W::kZeros ? 2 : 1);
}

// Bytes of a row in LDS: whole chunks
__host__ __device__ constexpr int acts_stride(int K) { return (K + kChunk - 1) / kChunk * (2 * kChunk); }

// A row of K activations into LDS, by one wave, zeros beyond K
template <class W>
__device__ __forceinline__ void put_row(const Args& a, size_t row, unsigned char* acts, int m, int stride) {
  const __amdgpu_buffer_rsrc_t x = bytes_at((const typename W::T*)a.A + row * a.K, (unsigned)a.K * 2);
  for (int piece = threadIdx.x & 63; piece < stride >> 4; piece += 512) {
    uint4_t v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = __builtin_bit_cast(uint4_t, __builtin_amdgcn_raw_buffer_load_b128(x, 16 * piece + 1024 * i, 0, 0));
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (piece + 64 * i < stride >> 4) *reinterpret_cast<uint4_t*>(acts + act_place(m, piece + 64 * i, stride)) = W::order(v[i]);
  }
}

// A wave's chunks of a pair of blocks.  Which run of them a wave has turns with the workgroup, so that not all ask the same stretch of
// every row at once; one that would have none has a chunk that is nothing.
struct Share {
  int c0, c1;
  bool idle;
  __device__ __forceinline__ Share(const Args& a, int wave) {
    const int turn = (wave + blockIdx.x) % kWaves, all = (a.K + kChunk - 1) / kChunk;
    c0 = turn * all / kWaves, c1 = (turn + 1) * all / kWaves;
    idle = c0 == c1;
    if (idle) ++c1;
  }
};

// All of a pipeline's sequence, `blocks` pairs of blocks: a pair ends where its last chunk does, with the wave's sums in one of two
// buffers and a barrier.  One turn is a chunk of each set of registers; the last turn's spare ones are nothing.
template <int DEPTH, class P>
__device__ __forceinline__ void run(P& p, int blocks, unsigned char* sums, int wave, int& done) {
  const int lane = threadIdx.x & 63;
  float4_t acc[2] = {};
  int c = p.c0, left = blocks;
  auto chunk = [&](int u) {
    p.chunk(u, c, acc);
    if (++c == p.c1) {
      c = p.c0;
      if (left > 0) {
        float4_t* const to = (float4_t*)(sums + ((done & 1) * kWaves + wave) * kSumsArea);  // [block][lane]
        to[lane] = acc[0];
        to[64 + lane] = acc[1];
        acc[0] = acc[1] = float4_t{};
        --left;
        ++done;
        __syncthreads();
      }
    }
  };
  const int turns = (blocks * (p.c1 - p.c0) + DEPTH - 1) / DEPTH;
  for (int i = 0; i < turns; ++i) {
#pragma unroll
    for (int u = 0; u < DEPTH; ++u) chunk(u);
  }
}

// The waves' sums of a pair of blocks: lane (g, c) has column c of either, rows 4 g .. 4 g + 3
__device__ __forceinline__ void add_up(const unsigned char* sums, int done, float4_t (&v)[2]) {
  const int lane = threadIdx.x & 63;
  const float4_t* const from = (const float4_t*)(sums + (done & 1) * kWaves * kSumsArea);
  float4_t part[kWaves][2];
#pragma unroll
  for (int w = 0; w < kWaves; ++w) part[w][0] = from[w * 128 + lane], part[w][1] = from[w * 128 + 64 + lane];
  __builtin_amdgcn_sched_barrier(0);
  v[0] = part[0][0], v[1] = part[0][1];
#pragma unroll
  for (int w = 1; w < kWaves; ++w) v[0] += part[w][0], v[1] += part[w][1];
}

// The workgroup's waves but the last are pipelines; the last adds their sums, a tile behind them, and is the only one that waits for
// anything else than weights while they run (loads come back in the order that they go out in).
template <class W, bool UP, int DEPTH, bool LINES>
__global__ __launch_bounds__((kWaves + 1) * 64, DEPTH == 1 ? 4 : 2) void rows_kernel(const Args a, int pass_rows) {
  using T = typename W::T;
  extern __shared__ __align__(16) unsigned char smem[];
  unsigned char* const sums = smem + kWaves * wave_area<W>();
  unsigned char* const acts = sums + 2 * kWaves * kSumsArea;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, c = lane & 15;
  constexpr int kColumns = UP ? 16 : 32;                       // of the output, in a tile
  const int rows = (UP ? 2 : 1) * a.N, second = UP ? a.N : 16;  // weight rows of an expert; from a tile's first block to its second
  const int tiles_n = a.N / kColumns, stride = acts_stride(a.K);
  const Parts parts(a, pass_rows);
  // (fewer than 2^31: the launch sees to it)
  const unsigned tiles = (unsigned)parts.count() * tiles_n, share = tiles / gridDim.x, more = tiles % gridDim.x;
  const unsigned t0 = blockIdx.x * share + min(blockIdx.x, more), t1 = t0 + share + (blockIdx.x < more ? 1 : 0);
  const Share chunks(a, wave);
  int done = 0;  // tiles, all waves alike: their sums go into two buffers in turn

  for (unsigned at = t0; at < t1;) {
    const Part part = parts.nth((int)(at / tiles_n));
    const int tile0 = (int)(at % tiles_n), tile1 = min(tiles_n, tile0 + (int)(t1 - at));
    const int r0 = part.begin, count = part.end - r0;
    at += tile1 - tile0;
    // lane m: row m's pair
    const unsigned pairs = (unsigned)a.Order[r0 + min(c, count - 1)];
    if (wave < kWaves) {
      const TilesOf<W> source(a, part.expert, rows, kColumns, second, tile1);
      Pipeline<W, DEPTH, LINES, TilesOf<W>> p(a, source, tile0, chunks.c0, chunks.c1, chunks.idle, smem + wave * wave_area<W>(), acts, pass_rows, stride);
      // a wave a row; places of rows that the part does not have keep what was there: theirs of the result are not stored
      for (int m = wave; m < count; m += kWaves) {
        size_t row = r0 + m;
        if constexpr (UP) row = min(__builtin_amdgcn_readlane(pairs, m) / (unsigned)a.top_k, (unsigned)a.tokens - 1);
        put_row<W>(a, row, acts, m, stride);
      }
      __syncthreads();
      run<DEPTH>(p, tile1 - tile0, sums, wave, done);
    } else {
      float weight[4];
      unsigned pair[4];
      if constexpr (!UP) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          pair[i] = __shfl(pairs, 4 * g + i, 64);
          weight[i] = a.Weights[min(pair[i], (unsigned)a.pairs - 1)];
        }
      }
      const T* const bias = a.Bias == nullptr ? nullptr : (const T*)a.Bias + (size_t)part.expert * rows + c;
      // (a tile's bias is asked for ahead of the stores of the tile before)
      T ahead[2] = {};
      if (bias != nullptr) ahead[0] = bias[tile0 * kColumns], ahead[1] = bias[tile0 * kColumns + second];
      __syncthreads();
      for (int tile = tile0; tile < tile1; ++tile) {
        const float b[2] = {(float)ahead[0], (float)ahead[1]};
        const int next = min(tile + 1, tile1 - 1) * kColumns;
        if (bias != nullptr) ahead[0] = bias[next], ahead[1] = bias[next + second];
        __syncthreads();
        float4_t v[2];
        add_up(sums, done++, v);
        const size_t n = (size_t)tile * kColumns + c;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (4 * g + i >= count) continue;
          if constexpr (UP) {
            ((T*)a.Out)[(size_t)(r0 + 4 * g + i) * a.N + n] = (T)(experts::activate(v[0][i] + b[0], a.gelu) * (v[1][i] + b[1]));
          } else if (pair[i] < (unsigned)a.pairs) {
            float* const to = a.Parts + (size_t)pair[i] * a.N + n;
            to[0] = (v[0][i] + b[0]) * weight[i];
            to[16] = (v[1][i] + b[1]) * weight[i];
          }
        }
      }
    }
  }
}

// "Down" for up to eight pairs, with nothing between the products and the tokens' sums: a workgroup has 16 columns of all experts that
// have rows, two experts at a time, and all rows as those of its matrix instructions.  An expert's sums of other experts' rows are
// left; every row's own are kept by the adding wave, and the tokens' sums, in the order of their choices, are its last step.
constexpr int kFewPairs = 8;

template <class W, bool LINES>
__global__ __launch_bounds__((kWaves + 1) * 64, 4) void few_pairs_kernel(const Args a) {
  using T = typename W::T;
  extern __shared__ __align__(16) unsigned char smem[];
  unsigned char* const sums = smem + kWaves * wave_area<W>();
  unsigned char* const acts = sums + 2 * kWaves * kSumsArea;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, c = lane & 15, n0 = blockIdx.x * 16, stride = acts_stride(a.K);
  // the experts that have rows, the i-th in lane i
  int experts = 0, begins = 0, ends = 0, count = 0;
  Parts(a, 16).each([&](int base, int b, int e) {
    const unsigned long long has = __ballot(e > b);
    if (has == 0) return false;
    const int rank = count + __builtin_amdgcn_mbcnt_hi((unsigned)(has >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)has, 0));
    const int here = __popcll(has), to = (e > b && rank < 16 ? rank : 63) * 4;  // (lane 63 takes what is nobody's)
    const int x = __builtin_amdgcn_ds_permute(to, base + lane), y = __builtin_amdgcn_ds_permute(to, b), z = __builtin_amdgcn_ds_permute(to, e);
    if (lane >= count && lane < min(count + here, 16)) experts = x, begins = y, ends = z;
    count = min(count + here, 16);
    return false;
  });
  const int rows = count > 0 ? __builtin_amdgcn_readlane(ends, count - 1) : 0;
  const int blocks = (count + 1) / 2;
  int done = 0;
  if (wave < kWaves) {
    const Share chunks(a, wave);
    const ExpertsOf<W> source(a, n0, experts, max(count, 1));
    Pipeline<W, 1, LINES, ExpertsOf<W>> p(a, source, 0, chunks.c0, chunks.c1, chunks.idle || count == 0, smem + wave * wave_area<W>(), acts, a.pairs, stride);
    for (int m = wave; m < rows; m += kWaves) put_row<W>(a, m, acts, m, stride);
    __syncthreads();
    run<1>(p, blocks, sums, wave, done);
  } else {
    // (asked for now, for the last step)
    float residual[4] = {0.f, 0.f, 0.f, 0.f};  // of tokens g, g + 4, ...
    if (a.Residual != nullptr)
#pragma unroll
      for (int i = 0; i < 4; ++i) residual[i] = (float)((const T*)a.Residual)[(size_t)min(g + 4 * i, a.tokens - 1) * a.N + n0 + c];
    const int pair = a.Order[min(c, a.pairs - 1)];
    const float weight = a.Weights[min((unsigned)pair, (unsigned)a.pairs - 1)];
    const T* const bias = a.Bias == nullptr ? nullptr : (const T*)a.Bias + n0 + c;
    auto bias_of = [&](int q, int t) { return bias[(size_t)__builtin_amdgcn_readlane(experts, min(2 * q + t, count - 1)) * a.N]; };
    T ahead[2] = {};
    if (bias != nullptr && count > 0) ahead[0] = bias_of(0, 0), ahead[1] = bias_of(0, 1);
    __syncthreads();
    float own[4] = {0.f, 0.f, 0.f, 0.f};  // row 4 g + i, column c
    for (int q = 0; q < blocks; ++q) {
      const float b[2] = {(float)ahead[0], (float)ahead[1]};
      if (bias != nullptr) ahead[0] = bias_of(q + 1, 0), ahead[1] = bias_of(q + 1, 1);
      __syncthreads();
      float4_t v[2];
      add_up(sums, done++, v);
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        if (2 * q + t >= count) break;
        const int first = __builtin_amdgcn_readlane(begins, 2 * q + t), last = __builtin_amdgcn_readlane(ends, 2 * q + t);
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (4 * g + i >= first && 4 * g + i < last) own[i] = v[t][i] + b[t];
      }
    }
    // rows to tokens, where the sums were: the last of them are read, and no pipeline writes more
    float* const values = (float*)sums;  // [pair][column]
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int i = 0; i < 4; ++i) values[(4 * g + i) * 16 + c] = 0.f;
    asm volatile("" ::: "memory");
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = 4 * g + i;
      const unsigned to = (unsigned)__shfl(pair, row, 64);
      const float w = __shfl(weight, row, 64);
      if (row < rows && to < (unsigned)a.pairs) values[to * 16 + c] = own[i] * w;
    }
    asm volatile("" ::: "memory");
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int token = g + 4 * i;
      if (token >= a.tokens) break;
      float sum = 0.f;
      for (int j = 0; j < a.top_k; ++j) sum += values[(token * a.top_k + j) * 16 + c];
      ((T*)a.Out)[(size_t)token * a.N + n0 + c] = (T)(sum + residual[i]);
    }
  }
}

// A token's pairs added, in the order of its choices and, of a choice's eight, of the slices, onto the residual: four columns a thread,
// eight choices asked for at once.  (A loop over one slice cost a third: 4096 tokens, two choices, 4096 columns 31 -> 43 us.)
template <class T, bool SLICES>
__global__ __launch_bounds__(256) void sum_kernel(const Args a) {
  typedef T vec4 __attribute__((ext_vector_type(4)));
  const size_t token = (size_t)blockIdx.z * gridDim.y + blockIdx.y;
  const int n = (blockIdx.x * blockDim.x + threadIdx.x) * 4;
  if (n >= a.N || token >= (size_t)a.tokens) return;
  const size_t at = token * a.N + n;
  vec4 r = {};
  if (a.Residual != nullptr) r = *reinterpret_cast<const vec4*>((const T*)a.Residual + at);
  float4_t v = {0.f, 0.f, 0.f, 0.f};
  for (int j0 = 0; j0 < a.top_k; j0 += 8) {
    for (int z = 0; z < (SLICES ? a.slices : 1); ++z) {
      float4_t part[8];
      unsigned id[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const size_t pair = token * a.top_k + min(j0 + j, a.top_k - 1);
        id[j] = (unsigned)a.Ids[pair] - (unsigned)a.first;
        part[j] = *reinterpret_cast<const float4_t*>(a.Parts + (SLICES ? (size_t)z * a.pairs * a.N : 0) + pair * a.N + n);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (j0 + j < a.top_k && id[j] < (unsigned)a.experts) v += part[j];  // (nobody has written another's)
    }
  }
  vec4 o;
#pragma unroll
  for (int i = 0; i < 4; ++i) o[i] = (T)(v[i] + (float)r[i]);
  *reinterpret_cast<vec4*>((T*)a.Out + at) = o;
}

template <class T>
int sum(const Args& a, hipStream_t stream) {
  const int threads = a.N >= 1024 ? 256 : 64, tokens = std::min(a.tokens, 65535);
  const auto kern = a.slices > 1 ? sum_kernel<T, true> : sum_kernel<T, false>;
  hipLaunchKernelGGL(kern, dim3((a.N / 4 + threads - 1) / threads, tokens, (a.tokens + tokens - 1) / tokens), dim3(threads), 0, stream, a);
  DQ_CHECK_HIP(hipGetLastError());
  return 0;
}

// The pairs that fall to these experts where choices are spread evenly, one at least
double expected(long pairs, int experts, int routed) { return std::max(1.0, (double)pairs * experts / std::max(experts, routed)); }

// Bytes of LDS of a workgroup beside the rows that it holds
template <class W>
constexpr int pipes_area() {
  return kWaves * (wave_area<W>() + 2 * kSumsArea);
}

template <class W, bool UP, int DEPTH, bool LINES>
int launch_rows(const Args& a, int pass_rows, int workgroups, hipStream_t stream) {
  constexpr int kMost = 160 * 1024 / (DEPTH == 1 ? 2 : 1);
  auto kern = rows_kernel<W, UP, DEPTH, LINES>;
  static bool raised[kMaxDevices];
  if (raise_lds_limit<kMost>(kern, raised)) return -1;
  hipLaunchKernelGGL(kern, dim3(workgroups), dim3((kWaves + 1) * 64), pipes_area<W>() + pass_rows * acts_stride(a.K), stream, a, pass_rows);
  DQ_CHECK_HIP(hipGetLastError());
  return 0;
}

template <class W, bool LINES>
int launch_few(const Args& a, hipStream_t stream) {
  constexpr int kMost = 160 * 1024;
  auto kern = few_pairs_kernel<W, LINES>;
  static bool raised[kMaxDevices];
  if (raise_lds_limit<kMost>(kern, raised)) return -1;
  hipLaunchKernelGGL(kern, dim3(a.N / 16), dim3((kWaves + 1) * 64), pipes_area<W>() + a.pairs * acts_stride(a.K), stream, a);
  DQ_CHECK_HIP(hipGetLastError());
  return 0;
}

// Two workgroups a CU, each a chunk ahead, where what an expert is likely to have of rows leaves room for that (us, against one
// workgroup that is two chunks ahead: one token, 8 of 128 experts, 1024 x 4096 10.5 and 11.7; 24 tokens, 4 of 64, 2048 x 1024 19.7 and
// 25.8); else one, with as many rows as it can hold (64 tokens, 4 of 32, 2880 x 2880 MXFP4: 69.6 and 74.5).
template <class W, bool UP>
int product(const Args& a, hipStream_t stream) {
  const int stride = acts_stride(a.K), mean = (int)std::max(1.0, expected(a.pairs, a.experts, a.routed) / std::min(a.experts, a.pairs));
  if constexpr (!UP) {
    const size_t scales = (size_t)a.experts * a.N * (a.K >> W::kShift) * W::kScaleBytes;
    // (us, against parts of every expert's rows and the sums behind them: 4096 x 1024, 8 pairs 9.0 and 13.1, 2048 x 768, 8 8.4 and 11.0,
    // 8192 x 4096 MXFP4, 2 10.6 and 12.2; 4096 x 1536, 16 pairs 19.7 and 18.7, 2048 x 1024, 16 12.1 and 9.3)
    if (a.pairs <= kFewPairs && pipes_area<W>() + a.pairs * stride <= 160 * 1024 && scales < kNowhere)
      return a.K % kChunk == 0 ? launch_few<W, true>(a, stream) : launch_few<W, false>(a, stream);
  }
  const int both = (80 * 1024 - pipes_area<W>()) / stride, alone = (160 * 1024 - pipes_area<W>()) / stride;
  const int likely = std::min(std::min(16, a.tokens), 3 * mean + 4);
  const bool two = likely <= both;
  const int pass_rows = std::min(std::min(16, a.tokens), two ? both : alone);
  // tiles that there can be
  const long most = (long)(a.pairs / pass_rows + std::min(a.experts, a.pairs)) * (a.N / (UP ? 16 : 32));
  if (most >= 1l << 31) DQ_FAIL("experts: %d rows of %d columns: more tiles than a call counts", a.pairs, a.N);
  const int workgroups = (int)std::min(most, two ? 512l : 256l);
  int rc;
  if (a.K % kChunk == 0) rc = two ? launch_rows<W, UP, 1, true>(a, pass_rows, workgroups, stream) : launch_rows<W, UP, 2, true>(a, pass_rows, workgroups, stream);
  else rc = two ? launch_rows<W, UP, 1, false>(a, pass_rows, workgroups, stream) : launch_rows<W, UP, 2, false>(a, pass_rows, workgroups, stream);
  if (rc != 0) return rc;
  if constexpr (!UP) return sum<typename W::T>(a, stream);
  return 0;
}

// Which kernel has a product: this file's, or that of tiles of 64 or 128 rows (dq_experts_tiles.hip), and "down" of the latter in how
// many slices of K.  What each would take is estimated from what bounds it, with experts that have the mean number of rows, and the
// least is taken; the number of an expert's parts is one up to 0.7 of what a part holds, beyond that half a part more than the mean's.
// * rows_kernel: the weights once a part, at 4.3 TB/s (uint4) and 5.2 (MXFP4, decoded with less);
// * tiles: 7.5 and 12.5 ns a k of a tile that has its CU for itself, and all of them 43 and 66 ps a k (MXFP4 40 and 54); slices, down
//   to 1024 k, while there are fewer than 256 workgroups, each with its results' way out and back (10 bytes at 5 TB/s a value).
// Measured, us, rows_kernel / tiles of 64 / of 128 [in 2, 4 slices]:
//   up uint4 8 experts of 4096 x 4096, 16 rows each: 48 / 47 / 64; 128 rows: 244 / 111 / 107; 128 of 1024 x 4096, 8 rows: 121 / - / 220;
//     4 of 2048 x 8192, 32 rows: 77 / 67 / 91, 256 rows: 499 / 88 / 107; 8 of 1024 x 4096, 32 rows: 28 / 38 / 51
//   down uint4 8 of 4096 x 14336, 2 rows: 64 / 121 / -; 32 rows: 391 / 132 [88, 84] / 176 [120, 118]; 128 rows: 1458 / 230 [208, 203] /
//     211 [199, 192]; 384 rows: - / 529 / 413 [430, 445]; 16 of 8192 x 4096, 32 rows: 180 / 100 [101, 119] / 138
//   down MXFP4 8 of 4096 x 14336, 4 rows: 64 / - [72, -]; 32 rows: 354 / 142 [84, 92] / 155; 96 rows: 980 / 164 [156, 160] / 185 [128, 130]
// Over 120 such products the choice is 3 % behind the best of these on average.  Tiles of 96 rows are between their neighbours
// everywhere, tiles of 256 ahead by 1 % at best (4096 tokens, two of 8 experts of 14336 x 4096: 1719 and 1740) and eight waves on a tile
// of 128 nowhere.
struct Plan {
  int rows, slices;  // of a tile, 0: rows_kernel
};
Plan plan(long all, int experts, int routed, int N, int K, int mxfp4, int group_shift, bool zeros, bool up) {
  const double pairs = expected(all, experts, routed), live = std::min((double)experts, pairs), mean = pairs / live;
  auto parts = [&](int rows) { return live * (mean <= 0.7 * rows ? 1.0 : mean / rows + 0.5); };
  const double weights = (up ? 2.0 : 1.0) * N * K;
  const int held = std::min(16, kActsRoom / acts_stride(K));  // rows of a part
  Plan best{0, 1};
  double least = INFINITY;
  if (held > 0) least = parts(held) * weights * (0.5 + (mxfp4 ? 1 : zeros ? 4 : 2) / (double)(1 << group_shift)) / (mxfp4 ? 5.2e6 : 4.3e6);
  if (K < 128) return best;  // (a tile takes two blocks of k)
  for (const bool tall : {false, true}) {
    const int rows = tall ? 128 : 64;
    const double tiles = parts(rows) * ((N + (up ? 127 : 255)) / (up ? 128 : 256));
    int slices = 1;
    if (!up && !experts::odd_rows(mxfp4, K, group_shift))
      while (slices < 4 && tiles * slices < 256 && K / (2 * slices) >= 1024) slices *= 2;
    const double pipe = tiles * (mxfp4 ? (tall ? 54e-6 : 40e-6) : (tall ? 66e-6 : 43e-6)), alone = (tall ? 12.5e-3 : 7.5e-3) / slices;
    const double us = K * std::max(pipe, alone) + (up ? 0.0 : slices * (double)all * N * 2e-6);
    if (us < least) least = us, best = {rows, slices};
  }
  return best;
}

template <bool UP>
int by_format(Args a, int mxfp4, hipStream_t stream) {
  const Plan by = plan(a.pairs, a.experts, a.routed, a.N, a.K, mxfp4, a.group_shift, a.Z != nullptr, UP);
  a.slices = by.slices;
  if (by.rows != 0) {
    if (const int rc = experts_tiles(a, mxfp4, UP, by.rows, stream)) return rc;
    if constexpr (!UP) return mxfp4 ? sum<bf16_t>(a, stream) : sum<half_t>(a, stream);
    return 0;
  }
  if (mxfp4) return product<experts::Mxfp4, UP>(a, stream);
#define DQ_UINT4(SHIFT_) (a.Z != nullptr ? product<experts::Uint4<true, SHIFT_>, UP>(a, stream) : product<experts::Uint4<false, SHIFT_>, UP>(a, stream))
  return a.group_shift == 5 ? DQ_UINT4(5) : a.group_shift == 6 ? DQ_UINT4(6) : DQ_UINT4(7);
#undef DQ_UINT4
}

}  // namespace

// (with zero points or without: the same)
size_t experts_down_workspace_bytes(int tokens, int experts, int routed, int top_k, int N, int K, int mxfp4, int group_shift) {
  const long pairs = (long)tokens * top_k;
  const int slices = std::max(plan(pairs, experts, routed, N, K, mxfp4, group_shift, false, false).slices, plan(pairs, experts, routed, N, K, mxfp4, group_shift, true, false).slices);
  return (size_t)slices * pairs * N * 4;
}

int experts_up(const Args& a, int mxfp4, hipStream_t stream) { return by_format<true>(a, mxfp4, stream); }
int experts_down(const Args& a, int mxfp4, hipStream_t stream) { return by_format<false>(a, mxfp4, stream); }

}  // namespace dq
