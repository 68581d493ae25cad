// extern "C" entry points of the norm, the routing and the experts' products (declared in include/dqgemm.h).  Every argument that
// the host can see is checked before any launch; what only the device sees (ids, order, starts) is bounded by the kernels.
#include "../../include/dqgemm.h"
#include "dq_experts.h"

#include <limits.h>
#include <math.h>

namespace dq {

int rms_norm(const void* X, const void* Residual, const void* Weight, void* Y, void* Sum, float* Scale, int rows, int dim, long row_stride,
             int int8, int bf16, float eps, hipStream_t stream);
int router_logits(const void* X, const void* W, const void* Bias, float* Logits, int tokens, int experts, int K, int bf16, hipStream_t stream);
size_t order_workspace_bytes(int tokens, int top_k, int experts);
int route_experts(const void* Logits, const float* Bias, float* Weights, int* Ids, int* Order, int* Starts, void* Workspace, int tokens,
                  int experts, int top_k, int sigmoid, int groups, int top_groups, int two, int renormalize, int dtype, float factor,
                  hipStream_t stream);
int experts_order(const int* Ids, int* Order, int* Starts, void* Workspace, int tokens, int top_k, int experts, int first, hipStream_t stream);
size_t experts_down_workspace_bytes(int tokens, int experts, int routed, int top_k, int N, int K, int mxfp4, int group_shift);
int experts_up(const experts::Args& a, int mxfp4, hipStream_t stream);
int experts_down(const experts::Args& a, int mxfp4, hipStream_t stream);

namespace {

bool on(const void* p, unsigned bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

constexpr int kMaxNormDim = 32768, kMaxExperts = 1024, kMaxTopK = 32;
constexpr long kMaxPairs = 1l << 23;  // counted in 16 bits a chunk, 256 chunks
constexpr long kMaxWeights = 1l << 31;  // of an expert and projection: byte offsets are 32-bit

// The sizes that check_pairs lets through: what a workspace is asked for of others is nothing
bool takes_pairs(int tokens, int experts, int top_k) {
  return tokens > 0 && experts > 0 && experts <= kMaxExperts && top_k > 0 && top_k <= kMaxTopK && (long)tokens * top_k <= kMaxPairs;
}

int check_pairs(const char* fn, int tokens, int experts, int top_k) {
  if (tokens <= 0) DQ_FAIL("%s: tokens must be positive (got %d)", fn, tokens);
  if (experts <= 0 || experts > kMaxExperts) DQ_FAIL("%s: experts must be from 1 to %d (got %d)", fn, kMaxExperts, experts);
  if (top_k <= 0 || top_k > kMaxTopK) DQ_FAIL("%s: top_k must be from 1 to %d (got %d)", fn, kMaxTopK, top_k);
  if ((long)tokens * top_k > kMaxPairs) DQ_FAIL("%s: %d choices of %d tokens: at most %ld pairs in a call", fn, top_k, tokens, kMaxPairs);
  return 0;
}

int check_workspace(const char* fn, const void* Workspace, size_t have, size_t need) {
  if (need && (!Workspace || !on(Workspace, 16) || have < need))
    DQ_FAIL("%s: needs a 16-byte aligned workspace of %zu bytes (got %zu)", fn, need, Workspace ? have : (size_t)0);
  return 0;
}

int check_product(const char* fn, const void* A, const void* B, const void* Scale, const void* Zeros, const void* Bias, const void* Order,
                  const void* Starts, const void* Out, int tokens, int experts, int top_k, int N, int K, int group_size, int format, int routed) {
  if (check_pairs(fn, tokens, experts, top_k) != 0) return -1;
  if (routed < experts) DQ_FAIL("%s: routed must be at least experts=%d (got %d)", fn, experts, routed);
  if (format != DQ_EXPERTS_UINT4 && format != DQ_EXPERTS_MXFP4) DQ_FAIL("%s: unknown weight format %d", fn, format);
  const int unit = format == DQ_EXPERTS_UINT4 ? 128 : 64;
  if (K <= 0 || K % unit != 0) DQ_FAIL("%s: K must be a positive multiple of %d (got %d)", fn, unit, K);
  if (N <= 0 || N % 32 != 0) DQ_FAIL("%s: N must be a positive multiple of 32 (got %d)", fn, N);
  if (format == DQ_EXPERTS_UINT4 ? group_size != 32 && group_size != 64 && group_size != 128 : group_size != 32)
    DQ_FAIL("%s: group_size must be 32, 64 or 128, with MXFP4 32 (got %d)", fn, group_size);
  if (format == DQ_EXPERTS_MXFP4 && Zeros) DQ_FAIL("%s: MXFP4 weights have no zero points", fn);
  // (byte offsets in an expert's weights and in the activations are 32-bit)
  if ((long)N * K > kMaxWeights || (long)tokens * K > 1l << 30 || (long)tokens * top_k * (N > K ? N : K) > 1l << 40)
    DQ_FAIL("%s: at most 2^31 weights an expert and projection, and 2^30 elements of %d tokens (got N=%d, K=%d)", fn, tokens, N, K);
  if (!A || !B || !Scale || !Order || !Starts || !Out) DQ_FAIL("%s: an operand is NULL that is expected to have a non-NULL data pointer", fn);
  if (!on(A, 16) || !on(B, 16) || !on(Out, 16) || !on(Bias, 16)) DQ_FAIL("%s: activations, weights, bias and output must be 16-byte aligned", fn);
  if (!on(Scale, 4) || !on(Zeros, 4) || !on(Order, 4) || !on(Starts, 4)) DQ_FAIL("%s: Scale, Zeros, Order and Starts must be 4-byte aligned", fn);
  return 0;
}

int log2_of(int n) { return n == 32 ? 5 : n == 64 ? 6 : 7; }

}  // namespace
}  // namespace dq

using namespace dq;

extern "C" int call_rms_norm(const void* X, const void* Residual, const void* Weight, void* Y, void* Sum, void* Scale, int rows, int dim,
                             int row_stride, int int8, int dtype, float eps, dq_stream_t stream) {
  const char* const fn = "call_rms_norm";
  if (dtype != DQ_DT_F16 && dtype != DQ_DT_BF16) DQ_FAIL("%s: dtype must be DQ_DT_F16 or DQ_DT_BF16 (got %d)", fn, dtype);
  if (rows <= 0) DQ_FAIL("%s: rows must be positive (got %d)", fn, rows);
  if (dim <= 0 || dim % 8 != 0 || dim > kMaxNormDim) DQ_FAIL("%s: dim must be a multiple of 8, at most %d (got %d)", fn, kMaxNormDim, dim);
  if (row_stride < dim || row_stride % 8 != 0) DQ_FAIL("%s: row_stride must be a multiple of 8 and at least dim=%d (got %d)", fn, dim, row_stride);
  if (!(eps > 0.f) || !isfinite(eps)) DQ_FAIL("%s: eps must be positive and finite", fn);
  if (!X || !Weight || !Y) DQ_FAIL("%s: X, Weight and Y are expected to have non-NULL data pointers", fn);
  if ((Residual != nullptr) != (Sum != nullptr)) DQ_FAIL("%s: Residual and Sum go together", fn);
  if ((int8 != 0) != (Scale != nullptr)) DQ_FAIL("%s: Scale goes with int8 codes", fn);
  if (!on(X, 16) || !on(Residual, 16) || !on(Weight, 16) || !on(Y, 16) || !on(Sum, 16) || !on(Scale, 4))
    DQ_FAIL("%s: X, Residual, Weight, Y and Sum must be 16-byte and Scale 4-byte aligned", fn);
  return rms_norm(X, Residual, Weight, Y, Sum, (float*)Scale, rows, dim, row_stride, int8 != 0, dtype == DQ_DT_BF16, eps, (hipStream_t)stream);
}

extern "C" int call_router_logits(const void* X, const void* W, const void* Bias, void* Logits, int tokens, int experts, int K, int dtype,
                                  dq_stream_t stream) {
  const char* const fn = "call_router_logits";
  if (check_pairs(fn, tokens, experts, 1) != 0) return -1;
  if (K <= 0 || K % 32 != 0) DQ_FAIL("%s: K must be a positive multiple of 32 (got %d)", fn, K);
  if (dtype != DQ_DT_F16 && dtype != DQ_DT_BF16) DQ_FAIL("%s: dtype must be DQ_DT_F16 or DQ_DT_BF16 (got %d)", fn, dtype);
  if (!X || !W || !Logits) DQ_FAIL("%s: X, W and Logits are expected to have non-NULL data pointers", fn);
  if (!on(X, 16) || !on(W, 16) || !on(Bias, 2) || !on(Logits, 4)) DQ_FAIL("%s: X and W must be 16-byte, Bias 2-byte and Logits 4-byte aligned", fn);
  return router_logits(X, W, Bias, (float*)Logits, tokens, experts, K, dtype == DQ_DT_BF16, (hipStream_t)stream);
}

extern "C" size_t dq_experts_order_workspace_bytes(int tokens, int top_k, int experts) {
  if (!takes_pairs(tokens, experts, top_k)) return 0;
  return order_workspace_bytes(tokens, top_k, experts);
}

extern "C" int call_route_experts(const void* Logits, const void* Bias, void* Weights, void* Ids, void* Order, void* Starts, void* Workspace,
                                  size_t workspace_bytes, int tokens, int experts, int top_k, int scores, int groups, int top_groups,
                                  int group_score, int renormalize, int dtype, float factor, dq_stream_t stream) {
  const char* const fn = "call_route_experts";
  if (check_pairs(fn, tokens, experts, top_k) != 0) return -1;
  if (dtype != DQ_DT_F16 && dtype != DQ_DT_BF16 && dtype != DQ_DT_F32) DQ_FAIL("%s: dtype must be DQ_DT_F16, DQ_DT_BF16 or DQ_DT_F32 (got %d)", fn, dtype);
  if (scores != DQ_SCORES_SOFTMAX && scores != DQ_SCORES_SIGMOID) DQ_FAIL("%s: unknown scores %d", fn, scores);
  if (group_score != DQ_GROUP_MAX && group_score != DQ_GROUP_SUM2) DQ_FAIL("%s: unknown group_score %d", fn, group_score);
  if (groups <= 0 || groups > 64 || experts % groups != 0) DQ_FAIL("%s: groups must be from 1 to 64 and divide experts=%d (got %d)", fn, experts, groups);
  if (top_groups <= 0 || top_groups > groups) DQ_FAIL("%s: top_groups must be from 1 to groups=%d (got %d)", fn, groups, top_groups);
  if (top_k > top_groups * (experts / groups))
    DQ_FAIL("%s: top_k=%d choices of the %d experts of %d groups", fn, top_k, top_groups * (experts / groups), top_groups);
  if (!isfinite(factor)) DQ_FAIL("%s: factor must be finite", fn);
  if (!Logits || !Weights || !Ids || !Order || !Starts) DQ_FAIL("%s: Logits, Weights, Ids, Order and Starts are expected to have non-NULL data pointers", fn);
  if (!on(Logits, 4) || !on(Bias, 4) || !on(Weights, 4) || !on(Ids, 4) || !on(Order, 4) || !on(Starts, 4))
    DQ_FAIL("%s: Logits, Bias, Weights, Ids, Order and Starts must be 4-byte aligned", fn);
  if (check_workspace(fn, Workspace, workspace_bytes, order_workspace_bytes(tokens, top_k, experts)) != 0) return -1;
  return route_experts(Logits, (const float*)Bias, (float*)Weights, (int*)Ids, (int*)Order, (int*)Starts, Workspace, tokens, experts, top_k,
                       scores == DQ_SCORES_SIGMOID, groups, top_groups, group_score == DQ_GROUP_SUM2, renormalize != 0,
                       dtype == DQ_DT_F32 ? 2 : dtype, factor, (hipStream_t)stream);
}

extern "C" int call_experts_order(const void* Ids, void* Order, void* Starts, void* Workspace, size_t workspace_bytes, int tokens, int top_k,
                                  int experts, int first, dq_stream_t stream) {
  const char* const fn = "call_experts_order";
  if (check_pairs(fn, tokens, experts, top_k) != 0) return -1;
  if (first < 0 || first > INT_MAX - experts) DQ_FAIL("%s: first must be from 0 to 2^31 - 1 - experts=%d (got %d)", fn, experts, first);
  if (!Ids || !Order || !Starts) DQ_FAIL("%s: Ids, Order and Starts are expected to have non-NULL data pointers", fn);
  if (!on(Ids, 4) || !on(Order, 4) || !on(Starts, 4)) DQ_FAIL("%s: Ids, Order and Starts must be 4-byte aligned", fn);
  if (check_workspace(fn, Workspace, workspace_bytes, order_workspace_bytes(tokens, top_k, experts)) != 0) return -1;
  return experts_order((const int*)Ids, (int*)Order, (int*)Starts, Workspace, tokens, top_k, experts, first, (hipStream_t)stream);
}

extern "C" int call_experts_up(const void* X, const void* B, const void* Scale, const void* Zeros, const void* Bias, const void* Order,
                               const void* Starts, void* H, int tokens, int experts, int top_k, int N, int K, int group_size, int format,
                               int activation, int routed, dq_stream_t stream) {
  const char* const fn = "call_experts_up";
  if (check_product(fn, X, B, Scale, Zeros, Bias, Order, Starts, H, tokens, experts, top_k, N, K, group_size, format, routed) != 0) return -1;
  if (activation != DQ_ACT_SILU && activation != DQ_ACT_GELU) DQ_FAIL("%s: unknown activation %d", fn, activation);
  experts::Args a{};
  a.A = X, a.B = (const uint8_t*)B, a.S = Scale, a.Z = Zeros, a.Bias = Bias, a.Order = (const int*)Order, a.Starts = (const int*)Starts, a.Out = H;
  a.tokens = tokens, a.experts = experts, a.top_k = top_k, a.pairs = tokens * top_k, a.N = N, a.K = K, a.group_shift = log2_of(group_size);
  a.gelu = activation == DQ_ACT_GELU, a.routed = routed;
  return experts_up(a, format == DQ_EXPERTS_MXFP4, (hipStream_t)stream);
}

extern "C" size_t dq_experts_down_workspace_bytes(int tokens, int experts, int top_k, int N, int K, int group_size, int format, int routed) {
  if (!takes_pairs(tokens, experts, top_k) || routed < experts || N <= 0 || K < 64 || (long)N * K > kMaxWeights) return 0;
  return experts_down_workspace_bytes(tokens, experts, routed, top_k, N, K, format == DQ_EXPERTS_MXFP4, log2_of(group_size));
}

extern "C" int call_experts_down(const void* H, const void* B, const void* Scale, const void* Zeros, const void* Bias, const void* Order,
                                 const void* Starts, const void* Ids, const void* Weights, const void* Residual, void* C, void* Workspace,
                                 size_t workspace_bytes, int tokens, int experts, int top_k, int N, int K, int group_size, int format, int first,
                                 int routed, dq_stream_t stream) {
  const char* const fn = "call_experts_down";
  if (check_product(fn, H, B, Scale, Zeros, Bias, Order, Starts, C, tokens, experts, top_k, N, K, group_size, format, routed) != 0) return -1;
  if (first < 0 || first > INT_MAX - experts) DQ_FAIL("%s: first must be from 0 to 2^31 - 1 - experts=%d (got %d)", fn, experts, first);
  // (and so they are in the rows of a tile of H: beyond tokens rows of an expert, where ids name it several times for a token)
  const long tile = (long)tokens * top_k < 128 ? (long)tokens * top_k : 128;
  if (tile * K > 1l << 31) DQ_FAIL("%s: at most 2^31 elements of 128 rows of H, or of all where they are fewer (got K=%d)", fn, K);
  if (!Ids || !Weights) DQ_FAIL("%s: Ids and Weights are expected to have non-NULL data pointers", fn);
  if (!on(Ids, 4) || !on(Weights, 4) || !on(Residual, 16)) DQ_FAIL("%s: Ids and Weights must be 4-byte and Residual 16-byte aligned", fn);
  if (check_workspace(fn, Workspace, workspace_bytes, dq_experts_down_workspace_bytes(tokens, experts, top_k, N, K, group_size, format, routed)) != 0) return -1;
  experts::Args a{};
  a.A = H, a.B = (const uint8_t*)B, a.S = Scale, a.Z = Zeros, a.Bias = Bias, a.Order = (const int*)Order, a.Starts = (const int*)Starts, a.Out = C;
  a.Ids = (const int*)Ids, a.Weights = (const float*)Weights, a.Residual = Residual, a.Parts = (float*)Workspace;
  a.tokens = tokens, a.experts = experts, a.top_k = top_k, a.pairs = tokens * top_k, a.N = N, a.K = K, a.group_shift = log2_of(group_size);
  a.first = first, a.routed = routed;
  return experts_down(a, format == DQ_EXPERTS_MXFP4, (hipStream_t)stream);
}
