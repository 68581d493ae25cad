// Rotary positions, and the paged key-value cache as it is written and read back (layout: dq_kv.h).
//
// Rotation of a head x at position p, r = rotary_dim, h = r / 2, (c_i, s_i) = Table[p][i], Table[p][h + i]:
//   half layout:        y_i = x_i c_i - x_{i+h} s_i,      y_{i+h} = x_{i+h} c_i + x_i s_i        (i < h)
//   interleaved layout: y_{2i} = x_{2i} c_i - x_{2i+1} s_i, y_{2i+1} = x_{2i+1} c_i + x_{2i} s_i
// and y_j = x_j from r on; with s negated it is the transpose, which is the gradient.  The table is the caller's, in fp32
// from angles in 64 bits: position times frequency loses the angle in fp32 from some ten thousand positions on.
//
// Quantised: a = max_j |y_j| of a token's head, code_j = rne(y_j * (top / a)), scale = a / top (top 448 or 127); the
// rotated key is quantised from fp32, not from a rounded 16-bit key.  A head with an infinity or a NaN gets a NaN scale,
// so it reads back as NaN and not as plausible numbers.
//
// All three operators only move memory, and every byte once.
#include "dq_kv.h"

#include <algorithm>

namespace dq {

namespace {

enum RotaryLayout : int {
  ROTARY_NONE = 0,
  ROTARY_HALF = 1,         // rotary_dim % 16 == 0: a lane's eight elements have one partner piece
  ROTARY_INTERLEAVED = 2,  // rotary_dim % 8 == 0: pairs inside a lane's piece
  ROTARY_QUADS = 3,        // half layout, rotary_dim % 16 == 8: a piece has two partners of four elements
  ROTARY_ANY = 4,          // either layout, any even rotary_dim: element by element
};

struct RowArgs {
  const void* x;     // [tokens][row_stride]: heads (q, or q and k and v) of head_dim
  const void* v;     // values where they do not lie behind the keys in x; else null
  const float* table;
  const int* positions;
  const int* slots;
  void* out;         // rotated heads, [tokens][out_stride]
  void* cache[2];
  float* scale[2];
  long row_stride, out_stride;
  int tokens, q_heads, head_dim, rotary_dim, table_rows, interleaved, inverse;
  int row_end;       // elements of a row that are read and written: in place no more pieces than turn (64 of 128: 27.4 -> 13.2 us)
  CacheShape shape;
};

template <int LANES>
__device__ __forceinline__ uint32_t row_max(uint32_t v) {
  v = max(v, dpp_move<0xB1>(v));                              // xor 1
  v = max(v, dpp_move<0x4E>(v));                              // xor 2
  if constexpr (LANES >= 8) v = max(v, dpp_move<0x141>(v));   // mirror in eight lanes
  if constexpr (LANES >= 16) v = max(v, dpp_move<0x140>(v));  // mirror in sixteen
  return v;
}

template <class T>
__device__ __forceinline__ void load8(const T* p, float (&f)[8]) {
  const auto h = *reinterpret_cast<const typename Vec8<T>::type*>(p);
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = (float)h[i];
}

template <class T>
__device__ __forceinline__ typename Vec8<T>::type round8(const float (&f)[8]) {
  typename Vec8<T>::type h;
#pragma unroll
  for (int i = 0; i < 8; ++i) h[i] = (T)f[i];
  return h;
}

template <class T>
struct alignas(8) Quad {
  T at[4];
};

// A group of LANES lanes has a row (a head of a token), a lane two pieces of eight elements of it: in the half layout two that turn
// with each other, so that every element is read once.  One row a group: four of one token, with one look at the table,
// take as long on whole lines and longer where rows are none (7999 tokens of 64 heads of 80: 33 against 40 us); two and four
// rows side by side longer too (4000 tokens of 64 heads of 128: 24.9, 26.7, 28.9 us).  Nothing is
// streamed here: what comes in is fresh from the projection, what goes out is read next.  Bound by memory: 4096 tokens of 40
// heads of 128 in 15.3 us, 5.6 TB/s read and written of the 6.6 that a copy of that size reaches; one token is a launch.
template <class T, int LANES, int LAYOUT, int FORMAT>
__global__ __launch_bounds__(256) void rows_kernel(const RowArgs a) {
  // Every product and sum rounded by itself, as the formula stands in fp32.  Which of two products of a sum goes unrounded into a
  // fused one is the compiler's choice, another in each layout's kernel, and moves codes over ties; it would save no time here.
#pragma clang fp contract(off)
  const int lane = threadIdx.x % LANES;
  const int heads = a.q_heads + (FORMAT >= 0 ? 2 * a.shape.kv_heads : 0);
  const unsigned group = blockIdx.x * (256 / LANES) + threadIdx.x / LANES;
  const int token = group / heads, head = group - token * heads;
  if (token >= a.tokens) return;
  const int keys_end = a.q_heads + (FORMAT >= 0 ? a.shape.kv_heads : 0);  // rows that are rotated
  const int r = a.rotary_dim, h = r >> 1, pieces = a.row_end >> 3, half = (pieces + 1) >> 1;
  // this lane's pieces, as their first elements; one that lies behind the row is not there
  int d[2] = {lane < half ? 8 * lane : a.row_end, lane < half ? 8 * (lane + half) : a.row_end};
  if (LAYOUT == ROTARY_HALF) {
    const bool pair = lane < r >> 4;
    d[0] = pair ? 8 * lane : 16 * lane;  // (the pieces behind the rotated ones two by two: lane r / 16 begins at r)
    d[1] = pair ? 8 * lane + h : 16 * lane + 8;
  }
  const bool inside[2] = {d[0] < a.row_end, d[1] < a.row_end};
  const bool turns = LAYOUT != ROTARY_NONE && head < keys_end;

  const T* const row = FORMAT >= 0 && a.v && head >= keys_end
                           ? reinterpret_cast<const T*>(a.v) + ((size_t)token * a.shape.kv_heads + (head - keys_end)) * a.head_dim
                           : reinterpret_cast<const T*>(a.x) + (size_t)token * a.row_stride + (size_t)head * a.head_dim;
  float x[2][8], partner[2][8] = {};
#pragma unroll
  for (int k = 0; k < 2; ++k) load8(row + (inside[k] ? d[k] : 0), x[k]);
  if constexpr (LAYOUT == ROTARY_QUADS) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int j = d[q >> 1] + 4 * (q & 1);
      if (!(turns && j < r)) continue;
      const Quad<T> y = *reinterpret_cast<const Quad<T>*>(row + (j < h ? j + h : j - h));
#pragma unroll
      for (int i = 0; i < 4; ++i) partner[q >> 1][4 * (q & 1) + i] = (float)y.at[i];
    }
  } else if constexpr (LAYOUT == ROTARY_ANY) {
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int j = d[k] + i, p = a.interleaved ? j ^ 1 : (j < h ? j + h : j - h);
        partner[k][i] = j < r && turns ? (float)row[p] : 0.f;
      }
  }
  // in place: what other lanes of the row read is read before any lane of it writes
  __builtin_amdgcn_wave_barrier();
  asm volatile("" ::: "memory");

  if constexpr (LAYOUT != ROTARY_NONE) {
    const int position = turns ? a.positions[token] : 0;
    const bool known = (unsigned)position < (unsigned)a.table_rows;  // else NaN
    const float* const angle = a.table + (size_t)(known ? position : 0) * r;
    const float sign = a.inverse ? -1.f : 1.f;
    if constexpr (LAYOUT == ROTARY_HALF) {
      if (turns && lane < r >> 4) {
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const float4_t cq = *reinterpret_cast<const float4_t*>(angle + 8 * lane + 4 * q), sq = *reinterpret_cast<const float4_t*>(angle + h + 8 * lane + 4 * q);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float c = known ? cq[j] : __builtin_nanf(""), s = sq[j] * sign, lo = x[0][4 * q + j], hi = x[1][4 * q + j];
            x[0][4 * q + j] = lo * c - hi * s, x[1][4 * q + j] = hi * c + lo * s;
          }
        }
      }
    } else {
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        if (!(turns && d[k] < r)) continue;
        float c[8], s[8];
        if constexpr (LAYOUT == ROTARY_INTERLEAVED) {
          const float4_t cq = *reinterpret_cast<const float4_t*>(angle + (d[k] >> 1)), sq = *reinterpret_cast<const float4_t*>(angle + h + (d[k] >> 1));
#pragma unroll
          for (int j = 0; j < 8; ++j) c[j] = cq[j >> 1], s[j] = (j & 1) ? sq[j >> 1] : -sq[j >> 1], partner[k][j] = x[k][j ^ 1];
        } else if constexpr (LAYOUT == ROTARY_QUADS) {
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            const int j = d[k] + 4 * q;
            const float* const at = angle + (j < h ? j : j - h);  // (r % 8 == 0: a piece turns whole)
            const float4_t cq = *reinterpret_cast<const float4_t*>(at), sq = *reinterpret_cast<const float4_t*>(at + h);
#pragma unroll
            for (int i = 0; i < 4; ++i) c[4 * q + i] = cq[i], s[4 * q + i] = j < h ? -sq[i] : sq[i];
          }
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int j = d[k] + i, at = a.interleaved ? j >> 1 : (j < h ? j : j - h);
            const bool low = a.interleaved ? !(j & 1) : j < h;
            c[i] = j < r ? angle[at] : 1.f;
            s[i] = j < r ? (low ? -angle[h + at] : angle[h + at]) : 0.f;
          }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if (!known && (LAYOUT != ROTARY_ANY || d[k] + i < r)) c[i] = __builtin_nanf("");
          x[k][i] = x[k][i] * c[i] + partner[k][i] * (s[i] * sign);
        }
      }
    }
  }

  if (FORMAT < 0 || head < a.q_heads) {
    T* const out = reinterpret_cast<T*>(a.out) + (size_t)token * a.out_stride + (size_t)head * a.head_dim;
#pragma unroll
    for (int k = 0; k < 2; ++k)
      if (inside[k]) *reinterpret_cast<typename Vec8<T>::type*>(out + d[k]) = round8<T>(x[k]);
    return;
  }
  if constexpr (FORMAT >= 0) {
    const int slot = a.slots[token], page = slot >> a.shape.page_shift;  // negative: not written
    if ((unsigned)page >= (unsigned)a.shape.pages) return;
    const bool values = head >= keys_end;
    const size_t at = cache_row(a.shape, page, head - (values ? keys_end : a.q_heads), slot & ((1 << a.shape.page_shift) - 1));
    void* const cache = values ? a.cache[1] : a.cache[0];
    if constexpr (cache_is_16bit(FORMAT)) {
#pragma unroll
      for (int k = 0; k < 2; ++k)
        if (inside[k]) *reinterpret_cast<typename Vec8<T>::type*>(reinterpret_cast<T*>(cache) + at * a.head_dim + d[k]) = round8<T>(x[k]);
    } else {
      constexpr float kTop = FORMAT == CACHE_FP8 ? 448.f : 127.f;
      uint32_t most = 0;  // magnitudes order like their bits, infinities and NaN above every number
#pragma unroll
      for (int k = 0; k < 2; ++k)
        if (inside[k]) {
#pragma unroll
          for (int i = 0; i < 8; ++i) most = max(most, __builtin_bit_cast(uint32_t, x[k][i]) & 0x7FFFFFFFu);
        }
      most = row_max<LANES>(most);
      const float amax = __builtin_bit_cast(float, most);
      const bool finite = most < 0x7F800000u, some = finite && amax >= kSmallestHead;
      const float factor = some ? kTop / amax : 0.f;
#pragma unroll
      for (int k = 0; k < 2; ++k)
        if (inside[k]) {
          uint2_t codes = {0u, 0u};
          if (finite) {
            codes[0] = quantise4<FORMAT>(x[k][0] * factor, x[k][1] * factor, x[k][2] * factor, x[k][3] * factor);
            codes[1] = quantise4<FORMAT>(x[k][4] * factor, x[k][5] * factor, x[k][6] * factor, x[k][7] * factor);
          }
          *reinterpret_cast<uint2_t*>(reinterpret_cast<uint8_t*>(cache) + at * a.head_dim + d[k]) = codes;
        }
      if (lane == 0) (values ? a.scale[1] : a.scale[0])[at] = finite ? (some ? amax / kTop : 0.f) : __builtin_nanf("");
    }
  }
}

template <class T, int LANES, int LAYOUT, int FORMAT>
int launch_rows(const RowArgs& a, hipStream_t stream) {
  const long rows = (long)a.tokens * (a.q_heads + (FORMAT >= 0 ? 2 * a.shape.kv_heads : 0));
  rows_kernel<T, LANES, LAYOUT, FORMAT><<<(unsigned)((rows + 256 / LANES - 1) / (256 / LANES)), 256, 0, stream>>>(a);
  DQ_CHECK_HIP(hipGetLastError());
  return 0;
}

template <class T, int LANES, int FORMAT>
int launch_rows_layout(const RowArgs& a, hipStream_t stream) {
  if (a.rotary_dim == 0) return launch_rows<T, LANES, ROTARY_NONE, FORMAT>(a, stream);
  if (a.interleaved && a.rotary_dim % 8 == 0) return launch_rows<T, LANES, ROTARY_INTERLEAVED, FORMAT>(a, stream);
  if (!a.interleaved && a.rotary_dim % 16 == 0) return launch_rows<T, LANES, ROTARY_HALF, FORMAT>(a, stream);
  // (element by element, 4000 tokens of 64 heads of 80 with 40 turned took 38.8 us, so it takes 17.5; what is left there, halves of no
  // four elements and pairs that end inside a lane's piece, is rare: 20 turned 33 us, interleaved 37, where 32 turned take 16)
  if (!a.interleaved && a.rotary_dim % 8 == 0) return launch_rows<T, LANES, ROTARY_QUADS, FORMAT>(a, stream);
  return launch_rows<T, LANES, ROTARY_ANY, FORMAT>(a, stream);
}

template <class T, int FORMAT>
int launch_rows_lanes(const RowArgs& a, hipStream_t stream) {
  if (a.row_end <= 64) return launch_rows_layout<T, 4, FORMAT>(a, stream);
  if (a.row_end <= 128) return launch_rows_layout<T, 8, FORMAT>(a, stream);
  if (a.row_end <= 256) return launch_rows_layout<T, 16, FORMAT>(a, stream);
  if constexpr (FORMAT < 0) return launch_rows_layout<T, 32, FORMAT>(a, stream);
  DQ_FAIL("a head of %d is beyond the cache's %d", a.row_end, kMaxHeadDim);
}

// Reading back: a workgroup has some tokens of the packed result, 1024 pieces of eight elements or at most kReadTokens tokens.  It
// first finds each one's sequence, page and place, then its threads take the pieces in the order of the result, which is
// written as one run, 16 bytes a lane side by side.  Stores are streamed: such a result is larger than the caches.  Loads are not:
// what was just written still lies there, and a line of narrow heads or of scales is another workgroup's too (48 sequences of
// up to 1100 tokens, 12 heads of 96, int8: 21.2 us, streamed 29.7).  131071 tokens of 8 heads of 128, fp8: 138 us, 5.9 TB/s of
// the 6.7 that a large copy reaches (a row a lane group, nothing streamed: 197; 16 codes a lane, whose two stores lie 32
// bytes apart and fill no line at once: 290).
struct ReadArgs {
  const void* cache[2];
  const float* scale[2];
  const int* table;
  const int* starts;
  void* out;  // [2][tokens][kv_heads][head_dim]
  int sequences, tokens, max_pages;
  CacheShape shape;
  int tokens_each;             // of a workgroup, at most kReadTokens
  bool runs;                   // neighbouring workgroups by sixteens on one of the eight L2 caches
  int row_pieces, all_pieces;  // of a head, of a token
  unsigned row_magic, all_magic;  // ceil(2^32 / row_pieces), ceil(2^32 / all_pieces)
};
constexpr int kReadTokens = 64;
constexpr int kReadRun = 16;
constexpr int kReadStarts = 1024;  // starts of so many sequences are looked through in LDS

// i / n by its magic number: right for i < 2^16, as i * (magic * n - 2^32) < 2^32 there (n <= 2^16); n = 1 has none
__device__ __forceinline__ int divided(int i, int n, unsigned magic) { return n == 1 ? i : (int)__umulhi((unsigned)i, magic); }

template <class T, int FORMAT>
__global__ __launch_bounds__(256) void read_kernel(const ReadArgs a) {
  constexpr bool kWide = cache_is_16bit(FORMAT);
  constexpr int kElements = 8, PIECE = kWide ? 16 : 8;
  __shared__ int s_starts[kReadStarts + 1];
  __shared__ int s_page[kReadTokens], s_place[kReadTokens];
  int block = blockIdx.x;
  if (a.runs) {  // sixteen neighbours on one of the eight L2 caches, which share the lines between them (with the write 31.5 -> 29.4 us at 12 heads of 96)
    const int run = block / (8 * kReadRun) * (8 * kReadRun), in_run = block - run;
    block = run + (in_run & 7) * kReadRun + (in_run >> 3);
  }
  const int token0 = block * a.tokens_each, count = min(a.tokens_each, a.tokens - token0);
  if (count <= 0) return;
  const bool staged = a.sequences <= kReadStarts;
  if (staged) {
    for (int i = threadIdx.x; i <= a.sequences; i += 256) s_starts[i] = a.starts[i];
    __syncthreads();
  }
  if ((int)threadIdx.x < count) {
    const int token = token0 + threadIdx.x;
    auto start = [&](int b) { return staged ? s_starts[b] : a.starts[b]; };
    // the last sequence that starts at or before the token
    int lo = 0, hi = a.sequences;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (start(mid) <= token) lo = mid;
      else hi = mid;
    }
    const int position = token - start(lo), column = position >> a.shape.page_shift;
    int page = -1;
    if (position >= 0 && token < start(lo + 1) && column < a.max_pages) page = a.table[(size_t)lo * a.max_pages + column];
    s_page[threadIdx.x] = (unsigned)page < (unsigned)a.shape.pages ? page : -1;
    s_place[threadIdx.x] = position & ((1 << a.shape.page_shift) - 1);
  }
  __syncthreads();
  const int which = blockIdx.y;
  const char* const cache = reinterpret_cast<const char*>(which ? a.cache[1] : a.cache[0]);
  const float* const scale = which ? a.scale[1] : a.scale[0];
  T* const out = reinterpret_cast<T*>(a.out) + ((size_t)which * a.tokens + token0) * ((size_t)a.all_pieces * kElements);
  typedef uint32_t Raw __attribute__((ext_vector_type(PIECE / 4)));
  const int pieces = count * a.all_pieces;
  constexpr int U = 4;
  for (int i0 = threadIdx.x; i0 < pieces; i0 += 256 * U) {
    Raw raw[U];
    float s[U];
    bool there[U];
#pragma unroll
    for (int k = 0; k < U; ++k) {  // (without branches, so that the loads are in flight together)
      const int i = min(i0 + 256 * k, pieces - 1);
      const int token = divided(i, a.all_pieces, a.all_magic), piece = i - token * a.all_pieces;
      const int head = divided(piece, a.row_pieces, a.row_magic), in_row = piece - head * a.row_pieces;
      const int page = s_page[token];
      there[k] = page >= 0;
      const size_t row = cache_row(a.shape, max(page, 0), head, s_place[token]);
      raw[k] = *reinterpret_cast<const Raw*>(cache + (row * a.row_pieces + in_row) * PIECE);
      if constexpr (!kWide) s[k] = scale[row];
    }
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const int i = i0 + 256 * k;
      if (i >= pieces) break;
      if constexpr (kWide) {
        __builtin_nontemporal_store(there[k] ? raw[k] : Raw{}, reinterpret_cast<Raw*>(out + (size_t)i * kElements));
      } else {
        float x[8];
        codes8_to_float<FORMAT>(raw[k], x);
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = there[k] ? x[j] * s[k] : 0.f;
        __builtin_nontemporal_store(round8<T>(x), reinterpret_cast<typename Vec8<T>::type*>(out + (size_t)i * kElements));
      }
    }
  }
}

template <class T, int FORMAT>
int launch_read(ReadArgs a, hipStream_t stream) {
  a.row_pieces = a.shape.head_dim / 8, a.all_pieces = a.row_pieces * a.shape.kv_heads;
  auto magic = [](int n) { return (unsigned)(((1ull << 32) + n - 1) / n); };
  a.row_magic = magic(a.row_pieces), a.all_magic = magic(a.all_pieces);
  // four pieces a thread (two 144 us where four take 138, eight 140, sixteen 150), fewer where that leaves compute units idle
  int each = std::max(1, std::min(kReadTokens, 1024 / a.all_pieces));
  while (each > 1 && (long)(a.tokens + each - 1) / each * 2 < 4 * 256) each = (each + 1) / 2;
  a.tokens_each = each;
  unsigned blocks = (a.tokens + each - 1) / each;
  a.runs = blocks >= 16 * kReadRun;  // (of fewer the last, incomplete round of eight runs is too large a part)
  if (a.runs) blocks = (blocks + 8 * kReadRun - 1) / (8 * kReadRun) * (8 * kReadRun);
  read_kernel<T, FORMAT><<<dim3(blocks, 2), 256, 0, stream>>>(a);
  DQ_CHECK_HIP(hipGetLastError());
  return 0;
}

}  // namespace

int rotary(const void* X, const float* Table, const int* Positions, void* Out, int tokens, int heads, int head_dim, int rotary_dim,
           int positions, long row_stride, long out_stride, int interleaved, int inverse, int bf16, hipStream_t stream) {
  RowArgs a = {};
  a.x = X, a.table = Table, a.positions = Positions, a.out = Out, a.row_stride = row_stride, a.out_stride = out_stride;
  a.tokens = tokens, a.q_heads = heads, a.head_dim = head_dim, a.rotary_dim = rotary_dim, a.table_rows = positions;
  a.interleaved = interleaved, a.inverse = inverse;
  a.row_end = X == Out ? (rotary_dim + 7) & ~7 : head_dim;
  return bf16 ? launch_rows_lanes<bf16_t, -1>(a, stream) : launch_rows_lanes<half_t, -1>(a, stream);
}

int kv_cache_write(const void* X, const void* V, const float* Table, const int* Positions, const int* Slots, void* Q, void* KCache,
                   void* VCache, float* KScale, float* VScale, int tokens, int heads, int kv_heads, int head_dim, int rotary_dim,
                   int positions, int pages, int page_shift, int interleaved, int bf16, int format, hipStream_t stream) {
  RowArgs a = {};
  a.x = X, a.v = V, a.table = Table, a.positions = Positions, a.slots = Slots, a.out = Q;
  a.cache[0] = KCache, a.cache[1] = VCache, a.scale[0] = KScale, a.scale[1] = VScale;
  a.row_stride = (long)(heads + (V ? 1 : 2) * kv_heads) * head_dim, a.out_stride = (long)heads * head_dim;
  a.tokens = tokens, a.q_heads = heads, a.head_dim = head_dim, a.rotary_dim = rotary_dim, a.table_rows = positions;
  a.interleaved = interleaved, a.row_end = head_dim;
  a.shape = {pages, kv_heads, page_shift, head_dim};
  switch (format) {
    case CACHE_FP8: return bf16 ? launch_rows_lanes<bf16_t, CACHE_FP8>(a, stream) : launch_rows_lanes<half_t, CACHE_FP8>(a, stream);
    case CACHE_I8: return bf16 ? launch_rows_lanes<bf16_t, CACHE_I8>(a, stream) : launch_rows_lanes<half_t, CACHE_I8>(a, stream);
    default: return bf16 ? launch_rows_lanes<bf16_t, CACHE_BF16>(a, stream) : launch_rows_lanes<half_t, CACHE_F16>(a, stream);
  }
}

int kv_cache_read(const void* KCache, const void* VCache, const float* KScale, const float* VScale, const int* PageTable,
                  const int* Starts, void* KV, int sequences, int tokens, int kv_heads, int head_dim, int pages, int page_shift,
                  int max_pages, int bf16, int format, hipStream_t stream) {
  ReadArgs a = {};
  a.cache[0] = KCache, a.cache[1] = VCache, a.scale[0] = KScale, a.scale[1] = VScale;
  a.table = PageTable, a.starts = Starts, a.out = KV;
  a.sequences = sequences, a.tokens = tokens, a.max_pages = max_pages;
  a.shape = {pages, kv_heads, page_shift, head_dim};
  switch (format) {
    case CACHE_FP8: return bf16 ? launch_read<bf16_t, CACHE_FP8>(a, stream) : launch_read<half_t, CACHE_FP8>(a, stream);
    case CACHE_I8: return bf16 ? launch_read<bf16_t, CACHE_I8>(a, stream) : launch_read<half_t, CACHE_I8>(a, stream);
    default: return bf16 ? launch_read<bf16_t, CACHE_BF16>(a, stream) : launch_read<half_t, CACHE_F16>(a, stream);
  }
}

}  // namespace dq
