// Routing: scores of a token's experts, the best top_k of them by score and bias, their weights; and the pairs (token, choice)
// sorted by expert, for the experts' products.
//
// A wave has a token.  Its lane l holds experts l, l + 64, ...; a choice is the largest key left over the lanes, of equal ones the
// lowest index.  Without a bias a key is the logit itself: softmax and logistic function only rise, so their order is the logits',
// and nothing is lost where they saturate.  With a bias (and where groups count by the sum of their two best) keys are scores, and
// fp32 does not tell all of them apart as they are in exact arithmetic: a token whose choices (or groups) lie closer together than
// fp32's error is done again in 64 bits, so that who is chosen does not hang on how exp is rounded.
//
// The order is a counting sort that keeps the pairs' order within an expert: chunks of tokens are counted where they are routed,
// and with all chunks' counts every workgroup knows where its pairs of an expert begin.  Nothing depends on timing: the only
// atomics are counts in LDS.
//
// What bounds it is instructions, a choice after the other.  Measured: one token, 8 of 128 5.6 us in one launch; 1021 tokens, 4 of 60
// 5.8 us and 5.5 for the order; 8192 tokens, 8 of 256 in 4 of 8 groups with biases 23 to 24 and 7.9 (25 in all without biases, where nothing
// is done in 64 bits: one token that is adds 3, being the last).
#include "dq_kv.h"

#include <type_traits>

namespace dq {

namespace {

constexpr int kMaxChunks = 256;
constexpr int kWaves = 16;             // of a workgroup
constexpr int kPlaceWorkgroups = 64;   // at most
constexpr int kAlonePairs = 4096;      // up to here one workgroup sorts them all

struct RouteArgs {
  const void* Logits;
  const float* Bias;
  float* Weights;
  int* Ids;
  int tokens, experts, top_k, sigmoid, groups, top_groups, two, renormalize;
  float factor;
};

struct OrderArgs {
  const int* Ids;
  int* Order;
  int* Starts;
  uint16_t* Counts;  // [chunks][experts, rounded up to four]; nullptr: one workgroup has all pairs
  int pairs, experts, first, chunk_pairs, chunks;
};

// The largest of the lanes' values, in every lane; a NaN counts for nothing, and is what comes back where all are.  fp32 goes through
// the register file: neighbours, rows of 16, a row's last lane to the next row, lane 31 to the upper half.
template <int CTRL>
__device__ __forceinline__ float max_with(float v) {
  const int b = __builtin_bit_cast(int, v);
  return fmaxf(v, __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(b, b, CTRL, 0xF, 0xF, false)));
}
template <int CTRL>
__device__ __forceinline__ double max_with(double v) {
  const unsigned long long b = __builtin_bit_cast(unsigned long long, v);
  const int l = (int)b, h = (int)(b >> 32);
  const unsigned lo = (unsigned)__builtin_amdgcn_update_dpp(l, l, CTRL, 0xF, 0xF, false);
  const unsigned hi = (unsigned)__builtin_amdgcn_update_dpp(h, h, CTRL, 0xF, 0xF, false);
  return fmax(v, __builtin_bit_cast(double, (unsigned long long)hi << 32 | lo));
}
template <class F>
__device__ __forceinline__ F max_over_wave(F v) {
  v = max_with<0xB1>(v);   // lane ^ 1
  v = max_with<0x4E>(v);   // lane ^ 2
  v = max_with<0x124>(v);  // rotated by 4 in its row
  v = max_with<0x128>(v);  // by 8
  v = max_with<0x142>(v);
  v = max_with<0x143>(v);
  if constexpr (std::is_same<F, float>::value) {
    return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 63));
  } else {
    const unsigned long long b = __builtin_bit_cast(unsigned long long, v);
    const unsigned lo = (unsigned)__builtin_amdgcn_readlane((int)b, 63), hi = (unsigned)__builtin_amdgcn_readlane((int)(b >> 32), 63);
    return __builtin_bit_cast(double, (unsigned long long)hi << 32 | lo);
  }
}

template <class F>
__device__ __forceinline__ F sum_over_wave(F v) {
#pragma unroll
  for (int d = 1; d < 64; d *= 2) v += __shfl_xor(v, d, 64);
  return v;
}

// Whether two keys in fp32 may be the other way round in exact arithmetic.  `slack` is at least twice what the scores in both are off
// by, four scores where a key is a group's sum of two: a logistic score has three roundings and exp's, below 2^-22 together; a share
// is off by less than 2^-18.8 of the largest share (22 additions, exp's error and its argument's), nearly all of it by a factor that
// every share has.  The keys' own roundings are 2^-24 of each: of an expert's key, and where two are added, of both and of their sum,
// whose magnitudes can be far beyond the sum's (biases of either sign).
__device__ __forceinline__ bool too_close(float a, float b, float slack) { return a - b <= slack + 0x1p-21f * (fabsf(a) + fabsf(b)); }

template <class F>
__device__ __forceinline__ F exp_of(F x) {
  if constexpr (std::is_same<F, double>::value) return exp(x);
  else return expf(x);
}

// One token's choices: lane j < top_k gets the j-th one and its score.  In fp32 logits and keys are in registers, V a lane; in 64 bits
// logits come from memory and keys are made in LDS, one after the other, so that what few tokens need takes no registers from all
// others, and chosen among in registers where that is no more than V = 4 (0: in LDS).  `keys`: the wave's LDS, an F an expert.  Returns whether F is too narrow to tell (the same in every lane).  A NaN counts as the largest of all: it is
// chosen, and its weight shows it.
template <class T, int V, class F>
__device__ __forceinline__ bool choose(const RouteArgs& a, const T* logits, const float* held, F* keys, int& my_id, float& my_score) {
  const int lane = threadIdx.x & 63;
  constexpr F kNone = -(F)__builtin_inff(), kMost = (F)__builtin_inff(), kGone = (F)__builtin_nanf("");
  constexpr bool kNarrow = std::is_same<F, float>::value;
  static_assert(V > 0 || !kNarrow, "fp32 keys are in registers");
  constexpr int kUnroll = kNarrow ? V : 1, kRounds = V ? V : 1;
  const int n = kNarrow ? V : (a.experts + 63) / 64;  // experts a lane
  const bool by_score = a.Bias != nullptr;
  bool close = false;
  const auto x = [&](int i) -> float {
    if constexpr (kNarrow) return held[i];
    else return i * 64 + lane < a.experts ? (float)logits[i * 64 + lane] : 0.f;
  };

  F largest = 0, total = 1;
  if (!a.sigmoid) {
    float l = -__builtin_inff();
#pragma unroll kUnroll
    for (int i = 0; i < n; ++i)
      if (i * 64 + lane < a.experts) l = fmaxf(l, x(i));
    l = max_over_wave(l);
    largest = l == -__builtin_inff() ? (F)0 : (F)l;  // (every expert is masked)
    total = 0;
#pragma unroll kUnroll
    for (int i = 0; i < n; ++i) total += i * 64 + lane < a.experts ? exp_of<F>((F)x(i) - largest) : (F)0;
    total = sum_over_wave(total);
  }
  const auto score_of = [&](float v) -> F {
    if (a.sigmoid) {
      const F t = exp_of<F>(-fabs((F)v));
      return (v >= 0 ? (F)1 : t) / ((F)1 + t);
    }
    return total == 0 ? (F)0 : exp_of<F>((F)v - largest) / total;
  };
  const float slack = a.sigmoid ? 0x1p-19f : total == 0 ? 0.f : 0x1p-17f / (float)total;
  // what an expert is chosen by, and what its group counts by
  const auto bias = [&](int i) -> float { return by_score && i * 64 + lane < a.experts ? a.Bias[i * 64 + lane] : 0.f; };
  const auto key_from = [&](float v, float add) -> F {
    const F k = by_score ? score_of(v) + (F)add : (F)v;
    return k != k ? kMost : k;
  };
  const auto key_of = [&](int i) -> F { return key_from(x(i), bias(i)); };
  const auto group_key_of = [&](int i, F key) -> F {
    if (!a.two || by_score) return key;
    const F k = score_of(x(i));
    return k != k ? kMost : k;
  };
  // a key that is not to be chosen (any more) is NaN
  F key[kRounds];
  const auto at = [&](int i) -> F {
    if constexpr (kNarrow) return key[i];
    else return i * 64 + lane < a.experts ? keys[i * 64 + lane] : kGone;
  };
  const auto put = [&](int i, F k) {
    if constexpr (kNarrow) key[i] = k;
    else if (i * 64 + lane < a.experts) keys[i * 64 + lane] = k;
  };
  if constexpr (kNarrow) {
#pragma unroll
    for (int i = 0; i < n; ++i) put(i, i * 64 + lane < a.experts ? key_of(i) : kGone);
  } else {
    // (the next one's operands on their way)
    float v = x(0), add = bias(0);
    for (int i = 0; i < n; ++i) {
      const float next_v = x(i + 1), next_add = bias(i + 1);
      put(i, key_from(v, add));
      v = next_v, add = next_add;
    }
  }

  if (a.groups > 1) {
    const int size = a.experts / a.groups;
#pragma unroll kUnroll
    for (int i = 0; i < n; ++i)
      if (i * 64 + lane < a.experts) keys[i * 64 + lane] = group_key_of(i, at(i));
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup");
    // a group's two largest, by as many lanes as there are for it
    int each = 6;
    for (int g = 1; g < a.groups; g *= 2) --each;
    const int group = lane >> each, first = lane & ((1 << each) - 1);
    F mine = kNone, next = kNone;
    if (group < a.groups) {
#pragma unroll 4
      for (int i = first; i < size; i += 1 << each) {
        const F k = keys[group * size + i];
        next = fmax(next, fmin(k, mine));
        mine = fmax(mine, k);
      }
    }
    for (int d = 1; d < 1 << each; d *= 2) {
      const F o = __shfl_xor(mine, d, 64), p = __shfl_xor(next, d, 64);
      next = fmax(fmin(o, mine), fmax(next, p));
      mine = fmax(mine, o);
    }
    // (halves: of two finite keys it is finite)
    F size_of = fabs(mine) * (F)0.5;
    if (a.two && size > 1) size_of += fabs(next) * (F)0.5, mine += next;
    if (mine != mine) mine = kMost;
    if (group >= a.groups || first != 0) mine = kGone;
    const F group_key = mine;
    __builtin_amdgcn_wave_barrier();
    unsigned long long taken = 0;  // a bit a group
    for (int r = 0; r < a.top_groups; ++r) {
      const F best = max_over_wave(mine);
      const int l = __builtin_ctzll(__ballot(mine == best));  // (of equal groups the first)
      if (lane == l) mine = kGone;
      taken |= 1ull << (l >> each);
    }
    if (kNarrow && (by_score || a.two) && a.top_groups < a.groups) {
      // whether the least that a taken group may count by is above the most that another may; what each is off by goes with the
      // magnitudes of its own keys, so neighbours in the order alone would not tell
      const float off = size_of < (F)__builtin_inff() ? 0.5f * slack + 0x1p-20f * (float)size_of : 0.f;
      const bool in = (taken >> group) & 1;
      const float least = -max_over_wave(in ? off - (float)group_key : __builtin_nanf("")), most = max_over_wave(in ? __builtin_nanf("") : (float)group_key + off);
      close = least <= most;
    }
    // (exact: the quotient is off by less than 2^-12 / size, and no nearer than 1 / (2 size) to a whole number)
    const float inverse = 1.f / (float)size;
#pragma unroll kUnroll
    for (int i = 0; i < n; ++i) {
      const int g = (int)(((float)(i * 64 + lane) + 0.5f) * inverse);
      F k = kGone;
      if (i * 64 + lane < a.experts && ((taken >> (g & 63)) & 1)) k = kNarrow || by_score || !a.two ? at(i) : key_of(i);
      put(i, k);
    }
  }

  if constexpr (!kNarrow && V > 0) {
#pragma unroll
    for (int i = 0; i < V; ++i) key[i] = at(i);
  }

  F last = 0;
  for (int r = 0; r < a.top_k + (kNarrow && by_score ? 1 : 0); ++r) {
    F best = kGone;
    int own = 0;  // (V = 0 alone: which of the lane's experts that is, the first)
    if constexpr (V) {
#pragma unroll
      for (int i = 0; i < V; ++i) best = fmax(best, key[i]);
    } else {
      for (int i = 0; i < n; ++i) {
        const F k = at(i);
        if (k > best || !(best == best)) best = k, own = i;
      }
    }
    const F most = best;
    best = max_over_wave(best);
    if (kNarrow && by_score && r > 0 && too_close((float)last, (float)best, slack)) close = true;
    if (r == a.top_k) break;
    last = best;
    // the lowest index of those that have it: expert 64 i + lane
    int index = 0;
    if constexpr (V) {
#pragma unroll
      for (int i = V - 1; i >= 0; --i) {
        const unsigned long long has = __ballot(key[i] == best);
        index = has != 0 ? i * 64 + __builtin_ctzll(has) : index;
      }
      const bool mine = lane == (index & 63);
#pragma unroll
      for (int i = 0; i < V; ++i) key[i] = mine && i == index >> 6 ? kGone : key[i];
    } else {
      for (int i = 0; i < n; ++i) {
        const unsigned long long has = __ballot(most == best && own == i);
        if (has == 0) continue;
        index = i * 64 + __builtin_ctzll(has);
        break;
      }
      if (lane == (index & 63)) keys[index] = kGone;
    }
    if (lane == r) my_id = index;
  }
  my_score = lane < a.top_k ? (float)score_of((float)logits[my_id]) : 0.f;
  return close;
}

template <class T, int V>
__device__ __forceinline__ int route_token(const RouteArgs& a, long token, unsigned char* lds) {
  const int lane = threadIdx.x & 63;
  float x[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int e = i * 64 + lane;
    x[i] = e < a.experts ? (float)((const T*)a.Logits)[token * a.experts + e] : 0.f;
  }
  int id = 0;
  float score = 0.f;
  const T* const logits = (const T*)a.Logits + token * a.experts;
  if (choose<T, V, float>(a, logits, x, (float*)lds, id, score)) {
    choose<T, V <= 4 ? V : 0, double>(a, logits, nullptr, (double*)lds, id, score);
  }
  const bool mine = lane < a.top_k;
  if (a.renormalize) {
    const float sum = sum_over_wave(score);
    score = sum == 0.f ? 0.f : score / sum;
  }
  if (mine) {
    a.Weights[token * a.top_k + lane] = score * a.factor;
    a.Ids[token * a.top_k + lane] = id;
  }
  return id;
}

// ---- the order ------------------------------------------------------------------------------------------------------------

constexpr int kFewPairs = 64;

__host__ __device__ constexpr int counts_stride(int experts) { return (experts + 3) & ~3; }

// Up to 64 pairs, a lane each, by one wave: a pair's place is how many have a lower expert, or its own and come earlier.
__device__ void place_few(const OrderArgs& o, int id) {
  const int lane = threadIdx.x & 63;
  const unsigned e = lane < o.pairs ? (unsigned)id - (unsigned)o.first : ~0u, mine = e < (unsigned)o.experts ? e : (unsigned)o.experts;
  int at = 0;
  for (int p = 0; p < o.pairs; ++p) {
    const unsigned other = (unsigned)__builtin_amdgcn_readlane((int)mine, p);
    at += other < mine || (other == mine && p < lane) ? 1 : 0;
  }
  // (pairs of other experts come behind all others: their places hold -1)
  if (lane < o.pairs) o.Order[at] = mine < (unsigned)o.experts ? lane : -1;
  for (int first = 0; first <= o.experts; first += 64) {
    int start = 0;
    for (int p = 0; p < o.pairs; ++p) start += __builtin_amdgcn_readlane((int)mine, p) < first + lane ? 1 : 0;
    if (first + lane <= o.experts) o.Starts[first + lane] = start;
  }
}

// A chunk's pairs of every expert, counted by all threads of the workgroup.
__device__ void count_chunk(const OrderArgs& o, int chunk, int* count) {
  for (int e = threadIdx.x; e < o.experts; e += kWaves * 64) count[e] = 0;
  __syncthreads();
  const int p1 = min((chunk + 1) * o.chunk_pairs, o.pairs);
  for (int p = chunk * o.chunk_pairs + threadIdx.x; p < p1; p += kWaves * 64) {
    const int e = (int)((unsigned)o.Ids[p] - (unsigned)o.first);
    if ((unsigned)e < (unsigned)o.experts) atomicAdd(&count[e], 1);
  }
  __syncthreads();
  for (int e = threadIdx.x; e < o.experts; e += kWaves * 64) o.Counts[(size_t)chunk * counts_stride(o.experts) + e] = (uint16_t)count[e];
}

// The pairs of some chunks into their places.  `lds`: (kWaves + 2) experts + 64 ints.
__device__ void place(const OrderArgs& o, int workgroup, int workgroups, int* lds) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, E = o.experts;
  int* const mine = lds + wave * E;      // a wave's pairs of every expert; then where its next one goes
  int* const total = lds + kWaves * E;   // all pairs of every expert
  int* const sums = total + E;           // kWaves
  const int per = (o.chunks + workgroups - 1) / workgroups;
  const int c0 = min(workgroup * per, o.chunks), c1 = min(c0 + per, o.chunks);
  const int p0 = min((long)c0 * o.chunk_pairs, (long)o.pairs), p1 = min((long)c1 * o.chunk_pairs, (long)o.pairs);
  const int segment = ((p1 - p0 + kWaves * 64 - 1) / (kWaves * 64)) * 64;  // a wave's
  const int w0 = min(p0 + wave * segment, p1), w1 = min(w0 + segment, p1);

  for (int e = lane; e < E; e += 64) mine[e] = 0;
  for (int p = w0 + lane; p < w1; p += 64) {
    const int e = (int)((unsigned)o.Ids[p] - (unsigned)o.first);
    if ((unsigned)e < (unsigned)E) atomicAdd(&mine[e], 1);
  }
  __syncthreads();
  // one thread an expert: all pairs, those of earlier workgroups, and where every wave's begin among this one's
  int before = 0, all = 0;
  if (o.Counts != nullptr) {
    // the chunks' counts by as many threads to four experts as there are, their parts added where the totals go later
    int wide = 16;
    while (wide * 4 < E) wide *= 2;
    const int e = (tid & (wide - 1)) * 4, slices = kWaves * 64 / wide;
    int part[4] = {0, 0, 0, 0}, early[4] = {0, 0, 0, 0};
    if (e < E) {
      const uint16_t* const counts = o.Counts + e;
      auto add = [&](uint2_t four, int c) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int n = (int)((four[i >> 1] >> (16 * (i & 1))) & 0xFFFFu);
          part[i] += n;
          early[i] += c < c0 ? n : 0;
        }
      };
      int c = tid / wide;
      for (; c + 15 * slices < o.chunks; c += 16 * slices) {  // (all of them on their way at once)
        uint2_t four[16];
#pragma unroll
        for (int u = 0; u < 16; ++u) four[u] = *reinterpret_cast<const uint2_t*>(counts + (size_t)(c + u * slices) * counts_stride(E));
#pragma unroll
        for (int u = 0; u < 16; ++u) add(four[u], c + u * slices);
      }
      for (; c < o.chunks; c += slices) add(*reinterpret_cast<const uint2_t*>(counts + (size_t)c * counts_stride(E)), c);
    }
    if (tid < E) total[tid] = 0, sums[64 + tid] = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (e + i >= E) break;
      atomicAdd(&total[e + i], part[i]);
      atomicAdd(&sums[64 + e + i], early[i]);
    }
    __syncthreads();
    if (tid < E) all = total[tid], before = sums[64 + tid];
  }
  if (tid < E) {
    int run = before;
    for (int w = 0; w < kWaves; ++w) {
      const int n = lds[w * E + tid];
      lds[w * E + tid] = run;
      run += n;
    }
    if (o.Counts == nullptr) all = run;
  }
  // exclusive sum over the experts
  int upto = all;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const int n = __shfl_up(upto, d, 64);
    if (lane >= d) upto += n;
  }
  if (lane == 63) sums[wave] = upto;
  __syncthreads();
  int start = upto - all;
  for (int w = 0; w < wave; ++w) start += sums[w];
  int end = 0;
  for (int w = 0; w < kWaves; ++w) end += sums[w];
  if (tid < E) total[tid] = start;
  if (workgroup == 0) {
    if (tid < E) o.Starts[tid] = start;
    if (tid == 0) o.Starts[E] = end;
  }
  __syncthreads();
  // places that no pair has: pairs whose expert is not among these
  for (int p = end + workgroup * (kWaves * 64) + tid; p < o.pairs; p += workgroups * (kWaves * 64)) o.Order[p] = -1;
  const int bits = 32 - __builtin_clz(E);
  for (int p = w0; p < w1; p += 64) {
    const int e = p + lane < w1 ? (int)((unsigned)o.Ids[p + lane] - (unsigned)o.first) : -1;
    const bool valid = (unsigned)e < (unsigned)E;
    // the lanes that have the same expert
    unsigned long long same = __ballot(valid);
    for (int b = 0; b < bits; ++b) {
      const unsigned long long set = __ballot((e >> b) & 1);
      same &= ((e >> b) & 1) ? set : ~set;
    }
    if (valid) {
      const int rank = __popcll(same & ((1ull << lane) - 1));
      const int at = mine[e];
      o.Order[total[e] + at + rank] = p + lane;
      if (rank == 0) mine[e] = at + __popcll(same);
    }
    __builtin_amdgcn_wave_barrier();
  }
}

template <class T, int V>
__global__ __launch_bounds__(kWaves * 64) void route_kernel(const RouteArgs a, const OrderArgs o) {
  extern __shared__ __align__(16) unsigned char smem[];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, chunk = blockIdx.x;
  const int tokens = o.chunk_pairs / a.top_k;  // of a chunk
  const long t1 = min((long)(chunk + 1) * tokens, (long)a.tokens);
  unsigned char* const keys = smem + kFewPairs * 4 + (size_t)wave * a.experts * 8;
  for (long t = (long)chunk * tokens + wave; t < t1; t += kWaves) {
    const int id = route_token<T, V>(a, t, keys);
    if (o.pairs <= kFewPairs && lane < a.top_k) ((int*)smem)[t * a.top_k + lane] = id;
  }
  __syncthreads();  // (the pairs that other waves wrote, and the LDS, which changes its use)
  if (o.pairs <= kFewPairs) {
    if (wave == 0) place_few(o, ((const int*)smem)[min(lane, o.pairs - 1)]);
  } else if (o.Counts != nullptr) {
    count_chunk(o, chunk, (int*)smem);
  } else {
    place(o, 0, 1, (int*)smem);
  }
}

__global__ __launch_bounds__(kWaves * 64) void count_kernel(const OrderArgs o) {
  extern __shared__ __align__(16) unsigned char smem[];
  count_chunk(o, blockIdx.x, (int*)smem);
}

__global__ __launch_bounds__(kWaves * 64) void place_kernel(const OrderArgs o) {
  extern __shared__ __align__(16) unsigned char smem[];
  if (o.pairs <= kFewPairs) {
    if (threadIdx.x < 64) place_few(o, o.Ids[min((int)threadIdx.x, o.pairs - 1)]);
    return;
  }
  place(o, blockIdx.x, gridDim.x, (int*)smem);
}

int place_lds(int experts) { return ((kWaves + 2) * experts + 64) * 4; }

// Whole tokens a chunk, at least a wave's worth, at most kMaxChunks chunks; 16-bit counts
bool cut(OrderArgs& o, int tokens, int top_k) {
  const long pairs = tokens * (long)top_k;
  if (pairs <= kFewPairs || (pairs <= kAlonePairs && tokens <= 2 * kWaves)) {
    o.chunk_pairs = tokens * top_k, o.chunks = 1;
    return false;
  }
  const int per = ((tokens + kMaxChunks - 1) / kMaxChunks + kWaves - 1) / kWaves * kWaves;
  o.chunk_pairs = per * top_k, o.chunks = (tokens + per - 1) / per;
  return true;
}

template <class T, int V>
int launch_route(const RouteArgs& a, const OrderArgs& o, hipStream_t stream) {
  constexpr int kMost = kFewPairs * 4 + kWaves * 1024 * 8;
  const int keys = kFewPairs * 4 + kWaves * a.experts * 8, room = place_lds(a.experts);
  const int lds = keys > room ? keys : room;
  auto kern = route_kernel<T, V>;
  static bool raised[kMaxDevices];
  if (raise_lds_limit<kMost>(kern, raised)) return -1;
  hipLaunchKernelGGL(kern, dim3(o.chunks), dim3(kWaves * 64), lds, stream, a, o);
  DQ_CHECK_HIP(hipGetLastError());
  return 0;
}

template <class T>
int route_experts_of(const RouteArgs& a, const OrderArgs& o, hipStream_t stream) {
  if (a.experts <= 64) return launch_route<T, 1>(a, o, stream);
  if (a.experts <= 128) return launch_route<T, 2>(a, o, stream);
  if (a.experts <= 256) return launch_route<T, 4>(a, o, stream);
  if (a.experts <= 512) return launch_route<T, 8>(a, o, stream);
  return launch_route<T, 16>(a, o, stream);
}

int launch_place(const OrderArgs& o, hipStream_t stream) {
  constexpr int kMost = (18 * 1024 + 64) * 4;
  auto kern = place_kernel;
  static bool raised[kMaxDevices];
  if (raise_lds_limit<kMost>(kern, raised)) return -1;
  const int workgroups = o.chunks < kPlaceWorkgroups ? o.chunks : kPlaceWorkgroups;
  hipLaunchKernelGGL(kern, dim3(o.Counts ? workgroups : 1), dim3(kWaves * 64), place_lds(o.experts), stream, o);
  DQ_CHECK_HIP(hipGetLastError());
  return 0;
}

}  // namespace

size_t order_workspace_bytes(int tokens, int top_k, int experts) {
  OrderArgs o{};
  return cut(o, tokens, top_k) ? ((size_t)o.chunks * counts_stride(experts) * 2 + 15) / 16 * 16 : 0;
}

int route_experts(const void* Logits, const float* Bias, float* Weights, int* Ids, int* Order, int* Starts, void* Workspace, int tokens,
                  int experts, int top_k, int sigmoid, int groups, int top_groups, int two, int renormalize, int dtype, float factor,
                  hipStream_t stream) {
  const RouteArgs a{Logits, Bias, Weights, Ids, tokens, experts, top_k, sigmoid, groups, top_groups, two, renormalize, factor};
  OrderArgs o{Ids, Order, Starts, nullptr, tokens * top_k, experts, 0, 0, 0};
  const bool chunks = cut(o, tokens, top_k);
  if (chunks) o.Counts = (uint16_t*)Workspace;
  const int rc = dtype == 0 ? route_experts_of<half_t>(a, o, stream) : dtype == 1 ? route_experts_of<bf16_t>(a, o, stream) : route_experts_of<float>(a, o, stream);
  return rc != 0 || !chunks ? rc : launch_place(o, stream);
}

int experts_order(const int* Ids, int* Order, int* Starts, void* Workspace, int tokens, int top_k, int experts, int first, hipStream_t stream) {
  OrderArgs o{Ids, Order, Starts, nullptr, tokens * top_k, experts, first, 0, 0};
  if (cut(o, tokens, top_k)) {
    o.Counts = (uint16_t*)Workspace;
    hipLaunchKernelGGL(count_kernel, dim3(o.chunks), dim3(kWaves * 64), (size_t)experts * 4, stream, o);
    DQ_CHECK_HIP(hipGetLastError());
  }
  return launch_place(o, stream);
}

}  // namespace dq
