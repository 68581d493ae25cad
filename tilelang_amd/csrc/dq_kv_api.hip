// extern "C" entry points of the rotation, the paged key-value cache and the attention over it (declared in
// include/dqgemm.h).  Every argument that the host can see is checked before any launch; what only the device sees
// (positions, slots, page ids, lengths) is bounded by the kernels themselves.
#include "../../include/dqgemm.h"
#include "dq_kv.h"

#include <math.h>

namespace dq {

int rotary(const void* X, const float* Table, const int* Positions, void* Out, int tokens, int heads, int head_dim, int rotary_dim,
           int positions, long row_stride, long out_stride, int interleaved, int inverse, int bf16, hipStream_t stream);
int kv_cache_write(const void* X, const void* V, const float* Table, const int* Positions, const int* Slots, void* Q, void* KCache,
                   void* VCache, float* KScale, float* VScale, int tokens, int heads, int kv_heads, int head_dim, int rotary_dim,
                   int positions, int pages, int page_shift, int interleaved, int bf16, int format, hipStream_t stream);
int kv_cache_read(const void* KCache, const void* VCache, const float* KScale, const float* VScale, const int* PageTable,
                  const int* Starts, void* KV, int sequences, int tokens, int kv_heads, int head_dim, int pages, int page_shift,
                  int max_pages, int bf16, int format, hipStream_t stream);
size_t attention_workspace_bytes(int sequences, int heads, int kv_heads, int head_dim, int format, long capacity, int window);
bool attention_fits(int sequences, int heads, int kv_heads, long capacity);
bool attention_head_dim(int d);
int attention_decode(const void* Q, const void* KCache, const void* VCache, const float* KScale, const float* VScale,
                     const int* PageTable, const int* Lengths, const float* Sinks, void* Out, float* Lse, void* Workspace,
                     float scale, int sequences, int heads, int kv_heads, int head_dim, int pages, int page_shift, int max_pages,
                     int window, int bf16, int format, hipStream_t stream);

namespace {

bool on_16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
bool on_4(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 3u) == 0; }

int log2_of(int n) {
  int s = 0;
  while (s < 30 && (1 << s) < n) ++s;
  return (1 << s) == n ? s : -1;
}

int check_dtype(const char* fn, int dtype) {
  if (dtype != DQ_DT_F16 && dtype != DQ_DT_BF16) DQ_FAIL("%s: dtype must be DQ_DT_F16 or DQ_DT_BF16 (got %d)", fn, dtype);
  return 0;
}

// heads of one launch: a lane group each, at most 64 lanes, thread numbers in 32 bits
int check_rows(const char* fn, long tokens, long heads) {
  if (tokens <= 0 || heads <= 0) DQ_FAIL("%s: tokens and heads must be positive (got %ld and %ld)", fn, tokens, heads);
  if (tokens * heads > (1l << 25)) DQ_FAIL("%s: %ld tokens of %ld heads: at most %ld heads in a call", fn, tokens, heads, 1l << 25);
  return 0;
}

int check_rotation(const char* fn, const void* Table, const void* Positions, int head_dim, int rotary_dim, int positions) {
  if (rotary_dim < 2 || rotary_dim % 2 != 0 || rotary_dim > head_dim)
    DQ_FAIL("%s: rotary_dim must be even and from 2 to head_dim=%d (got %d)", fn, head_dim, rotary_dim);
  if (positions <= 0) DQ_FAIL("%s: the table must have a row (got positions=%d)", fn, positions);
  if (!Table || !Positions) DQ_FAIL("%s: Table and Positions are expected to have non-NULL data pointers", fn);
  if (!on_16(Table) || !on_4(Positions)) DQ_FAIL("%s: Table must be 16-byte and Positions 4-byte aligned", fn);
  return 0;
}

// The pool: its geometry and buffers.  Sets the page size's shift.
int check_cache(const char* fn, const void* K, const void* V, const void* KS, const void* VS, int kv_heads, int head_dim, int pages,
                int page_size, int dtype, int format, int* shift) {
  if (check_dtype(fn, dtype) != 0) return -1;
  if (format < DQ_CACHE_F16 || format > DQ_CACHE_I8) DQ_FAIL("%s: unknown cache format %d", fn, format);
  if (format <= DQ_CACHE_BF16 && format != (dtype == DQ_DT_BF16 ? DQ_CACHE_BF16 : DQ_CACHE_F16))
    DQ_FAIL("%s: a 16-bit cache must be of the same type as dtype=%d (got format %d)", fn, dtype, format);
  if (kv_heads <= 0 || pages <= 0) DQ_FAIL("%s: kv_heads and pages must be positive (got %d and %d)", fn, kv_heads, pages);
  if (head_dim <= 0 || head_dim % 8 != 0 || head_dim > kMaxHeadDim)
    DQ_FAIL("%s: head_dim must be a multiple of 8, at most %d (got %d)", fn, kMaxHeadDim, head_dim);
  *shift = log2_of(page_size);
  if (page_size < 8 || page_size > 1024 || *shift < 0) DQ_FAIL("%s: page_size must be a power of two from 8 to 1024 (got %d)", fn, page_size);
  if ((long)pages * page_size > 0x7FFFFFFFl) DQ_FAIL("%s: %d pages of %d tokens: slots are 32-bit", fn, pages, page_size);
  if (!K || !V) DQ_FAIL("%s: KCache and VCache are expected to have non-NULL data pointers", fn);
  if (!on_16(K) || !on_16(V)) DQ_FAIL("%s: KCache and VCache must be 16-byte aligned", fn);
  if (format >= DQ_CACHE_FP8) {
    if (!KS || !VS) DQ_FAIL("%s: KScale and VScale are expected to have non-NULL data pointers for an 8-bit cache", fn);
    if (!on_16(KS) || !on_16(VS)) DQ_FAIL("%s: KScale and VScale must be 16-byte aligned", fn);
  }
  return 0;
}

int check_table(const char* fn, const void* PageTable, int sequences, int max_pages, int page_size) {
  if (sequences <= 0 || max_pages <= 0) DQ_FAIL("%s: sequences and max_pages must be positive (got %d and %d)", fn, sequences, max_pages);
  if (!PageTable || !on_4(PageTable)) DQ_FAIL("%s: PageTable must be a 4-byte aligned, non-NULL data pointer", fn);
  // (some tiles more than a sequence's tokens are counted ahead)
  if ((long)max_pages * page_size > 0x7FFFF000l) DQ_FAIL("%s: %d pages of %d tokens a sequence: lengths are 32-bit", fn, max_pages, page_size);
  return 0;
}

}  // namespace
}  // namespace dq

using namespace dq;

extern "C" int call_rotary(const void* X, const void* Table, const void* Positions, void* Out, int tokens, int heads, int head_dim,
                           int rotary_dim, int positions, int row_stride, int interleaved, int inverse, int dtype, dq_stream_t stream) {
  const char* const fn = "call_rotary";
  if (check_dtype(fn, dtype) != 0 || check_rows(fn, tokens, heads) != 0) return -1;
  if (head_dim <= 0 || head_dim % 8 != 0 || head_dim > kMaxRotaryHead)
    DQ_FAIL("%s: head_dim must be a multiple of 8, at most %d (got %d)", fn, kMaxRotaryHead, head_dim);
  if (check_rotation(fn, Table, Positions, head_dim, rotary_dim, positions) != 0) return -1;
  if (row_stride % 8 != 0 || row_stride < (long)heads * head_dim)
    DQ_FAIL("%s: row_stride must be a multiple of 8 and at least heads * head_dim = %ld (got %d)", fn, (long)heads * head_dim, row_stride);
  if (!X || !Out) DQ_FAIL("%s: X and Out are expected to have non-NULL data pointers", fn);
  if (!on_16(X) || !on_16(Out)) DQ_FAIL("%s: X and Out must be 16-byte aligned", fn);
  return rotary(X, (const float*)Table, (const int*)Positions, Out, tokens, heads, head_dim, rotary_dim, positions, row_stride,
                X == Out ? row_stride : (long)heads * head_dim, interleaved != 0, inverse != 0, dtype == DQ_DT_BF16, (hipStream_t)stream);
}

extern "C" int call_kv_cache_write(const void* K, const void* V, const void* Slots, void* KCache, void* VCache, void* KScale,
                                   void* VScale, int tokens, int kv_heads, int head_dim, int pages, int page_size, int dtype,
                                   int cache_format, dq_stream_t stream) {
  const char* const fn = "call_kv_cache_write";
  int shift;
  if (check_cache(fn, KCache, VCache, KScale, VScale, kv_heads, head_dim, pages, page_size, dtype, cache_format, &shift) != 0) return -1;
  if (check_rows(fn, tokens, 2l * kv_heads) != 0) return -1;
  if (!K || !V || !Slots) DQ_FAIL("%s: K, V and Slots are expected to have non-NULL data pointers", fn);
  if (!on_16(K) || !on_16(V) || !on_4(Slots)) DQ_FAIL("%s: K and V must be 16-byte and Slots 4-byte aligned", fn);
  return kv_cache_write(K, V, nullptr, nullptr, (const int*)Slots, nullptr, KCache, VCache, (float*)KScale, (float*)VScale, tokens, 0,
                        kv_heads, head_dim, 0, 0, pages, shift, 0, dtype == DQ_DT_BF16, cache_format, (hipStream_t)stream);
}

extern "C" int call_rotary_kv_cache_write(const void* QKV, const void* Table, const void* Positions, const void* Slots, void* Q,
                                          void* KCache, void* VCache, void* KScale, void* VScale, int tokens, int heads, int kv_heads,
                                          int head_dim, int rotary_dim, int positions, int pages, int page_size, int interleaved,
                                          int dtype, int cache_format, dq_stream_t stream) {
  const char* const fn = "call_rotary_kv_cache_write";
  int shift;
  if (check_cache(fn, KCache, VCache, KScale, VScale, kv_heads, head_dim, pages, page_size, dtype, cache_format, &shift) != 0) return -1;
  if (heads <= 0) DQ_FAIL("%s: heads must be positive (got %d)", fn, heads);
  if (check_rows(fn, tokens, heads + 2l * kv_heads) != 0) return -1;
  if (check_rotation(fn, Table, Positions, head_dim, rotary_dim, positions) != 0) return -1;
  if (!QKV || !Q || !Slots) DQ_FAIL("%s: QKV, Q and Slots are expected to have non-NULL data pointers", fn);
  if (!on_16(QKV) || !on_16(Q) || !on_4(Slots)) DQ_FAIL("%s: QKV and Q must be 16-byte and Slots 4-byte aligned", fn);
  return kv_cache_write(QKV, nullptr, (const float*)Table, (const int*)Positions, (const int*)Slots, Q, KCache, VCache, (float*)KScale,
                        (float*)VScale, tokens, heads, kv_heads, head_dim, rotary_dim, positions, pages, shift, interleaved != 0,
                        dtype == DQ_DT_BF16, cache_format, (hipStream_t)stream);
}

extern "C" int call_kv_cache_read(const void* KCache, const void* VCache, const void* KScale, const void* VScale, const void* PageTable,
                                  const void* Starts, void* KV, int sequences, int tokens, int kv_heads, int head_dim, int pages,
                                  int page_size, int max_pages, int dtype, int cache_format, dq_stream_t stream) {
  const char* const fn = "call_kv_cache_read";
  int shift;
  if (check_cache(fn, KCache, VCache, KScale, VScale, kv_heads, head_dim, pages, page_size, dtype, cache_format, &shift) != 0) return -1;
  if (check_rows(fn, tokens, kv_heads) != 0 || check_table(fn, PageTable, sequences, max_pages, page_size) != 0) return -1;
  if ((long)kv_heads * head_dim > 8 * 65535l) DQ_FAIL("%s: %d heads of %d: at most 524280 elements a token", fn, kv_heads, head_dim);
  if (!Starts || !KV) DQ_FAIL("%s: Starts and KV are expected to have non-NULL data pointers", fn);
  if (!on_4(Starts) || !on_16(KV)) DQ_FAIL("%s: Starts must be 4-byte and KV 16-byte aligned", fn);
  return kv_cache_read(KCache, VCache, (const float*)KScale, (const float*)VScale, (const int*)PageTable, (const int*)Starts, KV,
                       sequences, tokens, kv_heads, head_dim, pages, shift, max_pages, dtype == DQ_DT_BF16, cache_format,
                       (hipStream_t)stream);
}

extern "C" size_t dq_paged_attention_workspace_bytes(int sequences, int heads, int kv_heads, int head_dim, int page_size, int max_pages,
                                                     int window, int cache_format) {
  if (sequences <= 0 || heads <= 0 || kv_heads <= 0 || head_dim <= 0 || page_size <= 0 || max_pages <= 0 || window < 0 || heads % kv_heads != 0) return 0;
  return attention_workspace_bytes(sequences, heads, kv_heads, head_dim, cache_format, (long)max_pages * page_size, window);
}

extern "C" int call_paged_attention_decode(const void* Q, const void* KCache, const void* VCache, const void* KScale, const void* VScale,
                                           const void* PageTable, const void* Lengths, const void* Sinks, void* Out, void* Lse,
                                           void* Workspace, size_t workspace_bytes, int sequences, int heads, int kv_heads,
                                           int head_dim, int pages, int page_size, int max_pages, int window, int dtype,
                                           int cache_format, float scale, dq_stream_t stream) {
  const char* const fn = "call_paged_attention_decode";
  int shift;
  if (check_cache(fn, KCache, VCache, KScale, VScale, kv_heads, head_dim, pages, page_size, dtype, cache_format, &shift) != 0) return -1;
  if (check_table(fn, PageTable, sequences, max_pages, page_size) != 0) return -1;
  if (!attention_head_dim(head_dim)) DQ_FAIL("%s: head_dim must be 64, 80, 96, 112, 128, 160, 192 or 256 (got %d)", fn, head_dim);
  if (heads <= 0 || heads % kv_heads != 0) DQ_FAIL("%s: heads must be a multiple of kv_heads=%d (got %d)", fn, kv_heads, heads);
  if (sequences > 65535 || heads > 65535) DQ_FAIL("%s: at most 65535 sequences and heads (got %d and %d)", fn, sequences, heads);
  if (!attention_fits(sequences, heads, kv_heads, (long)max_pages * page_size))
    DQ_FAIL("%s: %d sequences of %d heads and up to %ld tokens: more than the work that a call counts", fn, sequences, heads, (long)max_pages * page_size);
  if (window < 0) DQ_FAIL("%s: window must be 0 (none) or positive (got %d)", fn, window);
  if (!isfinite(scale)) DQ_FAIL("%s: scale must be finite", fn);
  if (!Q || !Lengths || !Out) DQ_FAIL("%s: Q, Lengths and Out are expected to have non-NULL data pointers", fn);
  if (!on_16(Q) || !on_16(Out) || !on_4(Lengths) || !on_4(Sinks) || !on_4(Lse))
    DQ_FAIL("%s: Q and Out must be 16-byte, Lengths, Sinks and Lse 4-byte aligned", fn);
  const size_t need = dq_paged_attention_workspace_bytes(sequences, heads, kv_heads, head_dim, page_size, max_pages, window, cache_format);
  if (need && (!Workspace || !on_16(Workspace) || workspace_bytes < need))
    DQ_FAIL("%s: needs a 16-byte aligned workspace of %zu bytes (got %zu)", fn, need, Workspace ? workspace_bytes : (size_t)0);
  return attention_decode(Q, KCache, VCache, (const float*)KScale, (const float*)VScale, (const int*)PageTable, (const int*)Lengths,
                          (const float*)Sinks, Out, (float*)Lse, Workspace, scale, sequences, heads, kv_heads, head_dim, pages, shift,
                          max_pages, window, dtype == DQ_DT_BF16, cache_format, (hipStream_t)stream);
}
