// What the kernels on a paged cache share: how a sequence's tokens are found, and how the work of a ragged batch is dealt.
#pragma once

#include "w4a32_decoder.h"
#include "w4a32_internal.h"

namespace w4 {
namespace paged {

typedef float f32x4 __attribute__((ext_vector_type(4)));

struct Cache {
  void *k, *v;
  float* weight;
  const int* table;
  const int* len;
  int n_pages, shift, kv_heads, dim, n_seqs, table_ld;  // shift: log2 of the page's tokens
  int cap;                                              // table_ld pages in tokens
};

// Most workgroups of a launch of `threads` each: a launch has less than 2^32 threads. What would need more is refused.
constexpr long long most_groups(int threads) { return (1ll << 32) / threads - 1; }
constexpr int kMost = 1 << 30;  // rows of a step, tokens of a sequence, pairs of row and head

inline int log2_of(int page) { return __builtin_ctz((unsigned)page); }

// Host: whether the cache's sizes are what the kernels assume. W4A32_OK or the code to return.
int check_cache(const w4a32_paged_cache* c);
int check_rows(const w4a32_paged_cache* c, const w4a32_paged_rows* r);
Cache view(const w4a32_paged_cache* c);

// The rows of sequence b and the tokens in front of them, with everything a device array may say wrongly brought back
// into range. A length may pass the table: row j stands at len + j all the same, of which neither that nor a window's start is moved.
struct Span {
  int r0, n, len;  // first row, rows, tokens in front (kMost at most, so that no row's place passes 31 bits)
};
__device__ __forceinline__ Span span_of(const Cache& c, const int* row_start, int rows, int max_rows, int b) {
  Span s;
  const int lo = row_start[b], hi = row_start[b + 1];
  s.len = min(max(c.len[b], 0), kMost);
  s.r0 = min(max(lo, 0), rows);
  s.n = min(min(max(hi, s.r0), rows) - s.r0, max_rows);
  return s;
}

// Element offset of slot t's row in a pool, for a page that is there.
__device__ __forceinline__ size_t slot_row(const Cache& c, int page, int head, int t) {
  return ((((size_t)page * c.kv_heads + head) << c.shift) + (t & ((1 << c.shift) - 1)));
}
__device__ __forceinline__ bool page_there(const Cache& c, int page) { return (unsigned)page < (unsigned)c.n_pages; }

}  // namespace paged
}  // namespace w4
