// The paged cache: argument checks shared by its operators, the rows' append and the eviction of tokens.
#include "w4a32_paged.h"

namespace w4 {
namespace paged {

namespace {
inline bool aligned(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }
inline int from_hip(hipError_t e) { return e == hipSuccess ? W4A32_OK : W4A32_ELAUNCH; }
}  // namespace

int check_cache(const w4a32_paged_cache* c) {
  if (!c || !c->d_k || !c->d_v || !c->d_table || !c->d_len) return W4A32_EINVAL;
  if (c->dtype < W4A32_CACHE_F32 || c->dtype > W4A32_CACHE_BF16) return W4A32_EINVAL;
  if (c->n_pages < 1 || c->kv_heads < 1 || c->n_seqs < 1 || c->table_ld < 1 || c->dim < 1 || c->page < 1) return W4A32_EINVAL;
  if (!aligned(c->d_k, 16) || !aligned(c->d_v, 16) || !aligned(c->d_weight, 4) || !aligned(c->d_table, 4) || !aligned(c->d_len, 4))
    return W4A32_EINVAL;
  if (c->page < 16 || c->page > kMost || (c->page & (c->page - 1)) || c->dim % 8) return W4A32_ESHAPE;
  if (c->dim > W4A32_PAGED_MAX_DIM) return W4A32_ENOTSUP;
  if ((long long)c->table_ld * c->page >= kMost || c->n_seqs >= kMost || (long long)c->n_pages * c->kv_heads >= kMost * 2ll)
    return W4A32_ESHAPE;
  return W4A32_OK;
}

int check_rows(const w4a32_paged_cache* c, const w4a32_paged_rows* r) {
  if (int e = check_cache(c)) return e;
  if (!r || !r->d_row_start || r->rows < 1 || r->max_rows < 1 || r->heads < 1) return W4A32_EINVAL;
  if (!aligned(r->d_row_start, 4) || !aligned(r->d_q, 16) || !aligned(r->d_out, 16)) return W4A32_EINVAL;
  if (r->rows >= kMost || r->heads >= kMost / c->dim || (long long)r->rows * r->heads >= kMost) return W4A32_ESHAPE;
  if (r->heads % c->kv_heads) return W4A32_ESHAPE;
  if (r->act_bf16 && c->dtype != W4A32_CACHE_BF16) return W4A32_ENOTSUP;
  if (r->d_q && (!r->d_out || r->ldq < r->heads * c->dim || r->ldo < r->heads * c->dim || r->ldq % 8 || r->ldo % 8)) return W4A32_EINVAL;
  return W4A32_OK;
}

Cache view(const w4a32_paged_cache* c) {
  return {c->d_k, c->d_v, c->d_weight, c->d_table, c->d_len, c->n_pages, log2_of(c->page), c->kv_heads, c->dim, c->n_seqs, c->table_ld,
          c->table_ld * c->page};
}

// ---------------------------------------------------------------------------------------------
// Append. A thread takes eight elements of one head of one row: four pairs (i, i + rot / 2) to be turned, or eight
// elements that stay. Everything is read and written once; a step of few rows is bound by its chain of dependent loads
// (row starts, length, page number) and prompts by memory. 64 rows of 28 + 4 + 4 heads of 128 dims in bf16: 3.3 us; 3000 rows of
// 12 + 2 + 2 heads, f32 kept as f16 (75 MB): 13 us, 5.8 TB/s of the memory and the cache in front of it.
// ---------------------------------------------------------------------------------------------
struct Append {
  Cache c;
  const int* row_start;
  const int* pos;
  const void *q, *k, *v;
  void* q_out;
  const float *sin_t, *cos_t;
  int rows, max_rows, heads, ldq, ldo, ldk, ldv, rot, table_rows;
};

template <typename T>
struct Elem;
template <>
struct Elem<float> {
  static __device__ __forceinline__ void load4(const void* p, size_t at, float (&x)[4]) {
    const f32x4 v = load_global<f32x4>((const float*)p + at);
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = v[i];
  }
  static __device__ __forceinline__ void store4(void* p, size_t at, const float (&x)[4]) {
    *(W4_GLOBAL f32x4*)((float*)p + at) = f32x4{x[0], x[1], x[2], x[3]};
  }
};
template <>
struct Elem<__bf16> {
  static __device__ __forceinline__ void load4(const void* p, size_t at, float (&x)[4]) {
    const u32x2 v = load_global<u32x2>((const uint16_t*)p + at);
    x[0] = __uint_as_float(v[0] << 16);
    x[1] = __uint_as_float(v[0] & 0xffff0000u);
    x[2] = __uint_as_float(v[1] << 16);
    x[3] = __uint_as_float(v[1] & 0xffff0000u);
  }
  static __device__ __forceinline__ void store4(void* p, size_t at, const float (&x)[4]) {
    typedef __bf16 b4 __attribute__((ext_vector_type(4)));
    *(W4_GLOBAL b4*)((uint16_t*)p + at) = b4{(__bf16)x[0], (__bf16)x[1], (__bf16)x[2], (__bf16)x[3]};
  }
};
template <>
struct Elem<_Float16> {
  static __device__ __forceinline__ void store4(void* p, size_t at, const float (&x)[4]) {
    typedef _Float16 h4 __attribute__((ext_vector_type(4)));
    *(W4_GLOBAL h4*)((uint16_t*)p + at) = h4{(_Float16)x[0], (_Float16)x[1], (_Float16)x[2], (_Float16)x[3]};
  }
};

// The last sequence whose rows start at or in front of row r: 64 starts at a time, so that the search costs one load's
// latency and not the six of a binary search over 64.
__device__ __forceinline__ int owner_of(const int* row_start, int n_seqs, int r) {
  int before = 0;
  for (int b = 0; b < n_seqs; b += 64) {
    const int i = b + (int)(threadIdx.x & 63);
    before += __popcll(__ballot(i < n_seqs && row_start[i] <= r));
  }
  return before - 1;
}

template <typename Act, typename KV>
__global__ __launch_bounds__(256) void append_kernel(Append a, int blocks_per_row) {
  const int r = blockIdx.x / blocks_per_row;
  const int unit = (blockIdx.x % blocks_per_row) * 256 + threadIdx.x;
  const int per_head = a.c.dim / 8, q_heads = a.q ? a.heads : 0;
  const int b = owner_of(a.row_start, a.c.n_seqs, r);
  if (b < 0) return;
  const Span s = span_of(a.c, a.row_start, a.rows, a.max_rows, b);
  const int j = r - s.r0;
  const int head = unit / per_head, e = unit - head * per_head;
  if (j < 0 || j >= s.n || head >= q_heads + 2 * a.c.kv_heads) return;
  const int p = (int)((unsigned)(a.pos ? a.pos[b] : s.len) + (unsigned)j), slot = s.len + j;
  const bool is_q = head < q_heads, is_v = head >= q_heads + a.c.kv_heads;
  if (a.rot && (unsigned)p >= (unsigned)a.table_rows) return;

  const int half = a.rot / 2;
  const bool turned = !is_v && 8 * e < a.rot;
  const int d0 = turned ? 4 * e : 8 * e, d1 = turned ? 4 * e + half : 8 * e + 4;
  const int h = is_q ? head : is_v ? head - q_heads - a.c.kv_heads : head - q_heads;
  const void* src = is_q ? a.q : is_v ? a.v : a.k;
  const size_t row = (size_t)r * (is_q ? a.ldq : is_v ? a.ldv : a.ldk) + (size_t)h * a.c.dim;
  float x0[4], x1[4];
  Elem<Act>::load4(src, row + d0, x0);
  Elem<Act>::load4(src, row + d1, x1);
  if (turned) {
    float sn[4], cs[4];
    Elem<float>::load4(a.sin_t, (size_t)p * half + d0, sn);
    Elem<float>::load4(a.cos_t, (size_t)p * half + d0, cs);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float u = x0[i], w = x1[i];
      x0[i] = u * cs[i] - w * sn[i];
      x1[i] = w * cs[i] + u * sn[i];
    }
  }
  if (is_q) {
    const size_t to = (size_t)r * a.ldo + (size_t)h * a.c.dim;
    Elem<Act>::store4(a.q_out, to + d0, x0);
    Elem<Act>::store4(a.q_out, to + d1, x1);
    return;
  }
  if (slot >= a.c.cap) return;
  const int page = a.c.table[(size_t)b * a.c.table_ld + (slot >> a.c.shift)];
  if (!page_there(a.c, page)) return;
  const size_t at = slot_row(a.c, page, h, slot);
  void* dst = is_v ? a.c.v : a.c.k;
  Elem<KV>::store4(dst, at * a.c.dim + d0, x0);
  Elem<KV>::store4(dst, at * a.c.dim + d1, x1);
  if (!is_v && e == 0 && a.c.weight) a.c.weight[at] = 0.0f;
}

// ---------------------------------------------------------------------------------------------
// Eviction. One workgroup per (sequence, kv head) finds the weight of the last token that stays, 12, 10 and 10 bits of its
// order-preserving key at a time (a histogram in LDS each: 12 first, so that weights of similar size, which have few exponents,
// do not all count in the same place), and lists the slots that stay in order; a second launch copies. Up to kHeld keys lie in
// LDS; beyond them every pass has the weights from memory. The selection is all latency, the copy all memory: 32 sequences of 1500
// to 9000 tokens, 4 heads of 128 dims in bf16, to 2048 each: 17 and 50 us, the latter 268 MB at 5.4 TB/s; one of 4099, 2 heads in f32,
// to 1024: 9.9 and 4.4 us. (The first and the last tokens copied by other workgroups of the first launch took as much longer
// there as the second took less.)
// ---------------------------------------------------------------------------------------------
struct Evict {
  Cache c, to;
  int budget, first, recent;
  int* kept;  // [n_seqs][kv_heads][budget]
  int* to_len;
};

// Larger weights have larger keys; NaN is +infinity and -0 is 0.
__device__ __forceinline__ uint32_t key_of(float w) {
  if (!(w == w)) w = INFINITY;
  const uint32_t u = __float_as_uint(w + 0.0f);
  return u >> 31 ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float weight_at(const Cache& c, int b, int head, int t) {
  const int page = c.table[(size_t)b * c.table_ld + (t >> c.shift)];
  return page_there(c, page) ? c.weight[slot_row(c, page, head, t)] : 0.0f;
}

// Threads copy 16 bytes of a token's key and of its value each: token t of a sequence's head to slot i.
__device__ __forceinline__ void copy_token(const Evict& a, int b, int head, int t, int i, int units, int u) {
  const int from = a.c.table[(size_t)b * a.c.table_ld + (t >> a.c.shift)];
  const int dst = a.to.table[(size_t)b * a.to.table_ld + (i >> a.to.shift)];
  if (!page_there(a.to, dst)) return;
  const bool there = page_there(a.c, from);
  const size_t src = slot_row(a.c, there ? from : 0, head, t), out = slot_row(a.to, dst, head, i);
  const u32x4 zero = {0, 0, 0, 0};
  const u32x4 k = load_global<u32x4>((const u32x4*)a.c.k + src * units + u), v = load_global<u32x4>((const u32x4*)a.c.v + src * units + u);
  *(W4_GLOBAL u32x4*)((u32x4*)a.to.k + out * units + u) = there ? k : zero;
  *(W4_GLOBAL u32x4*)((u32x4*)a.to.v + out * units + u) = there ? v : zero;
  if (u == 0) a.to.weight[out] = there ? a.c.weight[src] : 0.0f;
}
constexpr int kCopies = 4;  // tokens of a thread

constexpr int kSelect = 1024;
constexpr int kHeld = 32 * 1024;

template <bool kInLds>
__global__ __launch_bounds__(kSelect) void select_kernel(Evict a) {
  extern __shared__ __attribute__((aligned(16))) unsigned keys[];
  __shared__ unsigned hist[4096], in_wave[kSelect / 64], state[2];
  const int b = blockIdx.x / a.c.kv_heads, head = blockIdx.x % a.c.kv_heads, tid = threadIdx.x;
  const int n = min(max(a.c.len[b], 0), a.c.cap), stay = min(n, a.budget);
  int* kept = a.kept + (size_t)blockIdx.x * a.budget;
  if (head == 0 && tid == 0) a.to_len[b] = stay;
  for (int i = stay + tid; i < a.budget; i += kSelect) kept[i] = -1;
  if (n <= a.budget) {
    for (int i = tid; i < n; i += kSelect) kept[i] = i;
    return;
  }
  const int lo = a.first, hi = n - a.recent;
  unsigned want = a.budget - a.first - a.recent;  // of those in [lo, hi), of which there are more
  uint32_t prefix = 0;
  auto key_at = [&](int t) { return kInLds ? keys[t] : key_of(weight_at(a.c, b, head, t)); };
  const bool any = want != 0;
  if (any) {
    if (kInLds) {
#pragma unroll 8
      for (int t = lo + tid; t < hi; t += kSelect) keys[t] = key_of(weight_at(a.c, b, head, t));
    }
    int shift = 20;
    uint32_t mask = 0;
    for (int bits = 12;; bits = 10, shift -= 10) {
      const int each = (1 << bits) / kSelect;  // digits of a thread: 4, then 1
      for (int i = 0; i < each; ++i) hist[tid * each + i] = 0;
      __syncthreads();
      for (int t = lo + tid; t < hi; t += kSelect) {
        const uint32_t k = key_at(t);
        if ((k & mask) == prefix) atomicAdd(&hist[k >> shift & ((1u << bits) - 1)], 1u);
      }
      __syncthreads();
      // thread i: the i-th `each` digits from the largest on
      const int top = (1 << bits) - 1 - tid * each;
      unsigned sum = 0, all;
      for (int i = 0; i < each; ++i) sum += hist[top - i];
      const unsigned upto = block_scan<kSelect>(sum, in_wave, all);
      unsigned above = upto - sum;
      if (above < want && upto >= want) {
        for (int i = 0; i < each; ++i) {
          const unsigned h = hist[top - i];
          if (above < want && above + h >= want) {
            state[0] = top - i;
            state[1] = want - above;
          }
          above += h;
        }
      }
      __syncthreads();
      prefix |= state[0] << shift;
      want = state[1];
      mask |= ((1u << bits) - 1) << shift;
      if (shift == 0) break;
    }
  }
  // Those above the key stay, and of those that have it the first `want`. A thread has tokens in a row.
  const int per = ((n + kSelect - 1) / kSelect) | 1;  // odd: the threads' keys lie in different banks
  const int t0 = min(tid * per, n), t1 = min(t0 + per, n);
  unsigned ties = 0, sure = 0, all;
  for (int t = t0; t < t1; ++t) {
    const bool inner = any && t >= lo && t < hi;
    const uint32_t k = inner ? key_at(t) : 0;
    ties += inner && k == prefix;
    sure += t < lo || t >= hi || (inner && k > prefix);
  }
  unsigned rank = block_scan<kSelect>(ties, in_wave, all) - ties;
  const unsigned stays = sure + min(ties, want - min(want, rank));
  unsigned to = block_scan<kSelect>(stays, in_wave, all) - stays;
  for (int t = t0; t < t1; ++t) {
    const bool inner = any && t >= lo && t < hi;
    const uint32_t k = inner ? key_at(t) : 0;
    const bool tie = inner && k == prefix;
    if (t < lo || t >= hi || (inner && k > prefix) || (tie && rank < want)) kept[to++] = t;
    rank += tie;
  }
}

__global__ __launch_bounds__(256) void copy_kernel(Evict a, int units, int blocks_per_head) {
  const int bh = blockIdx.x / blocks_per_head, b = bh / a.c.kv_heads, head = bh % a.c.kv_heads;
  const int per = 256 / units, u = threadIdx.x % units;
  if ((int)threadIdx.x >= per * units) return;
  const int first = (blockIdx.x % blocks_per_head) * per * kCopies + threadIdx.x / units;
  int t[kCopies];
#pragma unroll
  for (int x = 0; x < kCopies; ++x) {
    const int i = first + x * per;
    t[x] = i < a.budget ? a.kept[(size_t)bh * a.budget + i] : -1;
  }
#pragma unroll
  for (int x = 0; x < kCopies; ++x)
    if (t[x] >= 0) copy_token(a, b, head, t[x], first + x * per, units, u);
}

}  // namespace paged
}  // namespace w4

using namespace w4::paged;

extern "C" {

int w4a32_op_paged_append(const w4a32_paged_cache* cache, const w4a32_paged_rows* rows, const void* d_k, int ldk, const void* d_v,
                          int ldv, const int* d_pos, const float* d_sin, const float* d_cos, int rot_dims, int table_rows,
                          void* stream) {
  if (int e = check_rows(cache, rows)) return e;
  if (!d_k || !d_v || !aligned(d_k, 16) || !aligned(d_v, 16) || !aligned(d_pos, 4)) return W4A32_EINVAL;
  const int width = cache->kv_heads * cache->dim;
  if (cache->kv_heads >= kMost / cache->dim) return W4A32_ESHAPE;
  if (ldk < width || ldv < width || ldk % 8 || ldv % 8) return W4A32_EINVAL;
  if (rot_dims < 0 || rot_dims > cache->dim || rot_dims % 8) return W4A32_ESHAPE;
  if (rot_dims && (!d_sin || !d_cos || table_rows < 1 || !aligned(d_sin, 16) || !aligned(d_cos, 16))) return W4A32_EINVAL;
  const Append a{view(cache), rows->d_row_start, d_pos,       rows->d_q, d_k, d_v, rows->d_out, d_sin,      d_cos, rows->rows,
                 rows->max_rows, rows->heads,   rows->ldq, rows->ldo, ldk, ldv, rot_dims,    table_rows};
  const long long units = (long long)((rows->d_q ? rows->heads : 0) + 2 * cache->kv_heads) * (cache->dim / 8);
  const long long per_row = (units + 255) / 256;
  if (per_row * rows->rows > most_groups(256)) return W4A32_ESHAPE;
  const dim3 grid((unsigned)(per_row * rows->rows)), block(256);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (rows->act_bf16)
    hipLaunchKernelGGL((append_kernel<__bf16, __bf16>), grid, block, 0, s, a, (int)per_row);
  else if (cache->dtype == W4A32_CACHE_F32)
    hipLaunchKernelGGL((append_kernel<float, float>), grid, block, 0, s, a, (int)per_row);
  else if (cache->dtype == W4A32_CACHE_F16)
    hipLaunchKernelGGL((append_kernel<float, _Float16>), grid, block, 0, s, a, (int)per_row);
  else
    hipLaunchKernelGGL((append_kernel<float, __bf16>), grid, block, 0, s, a, (int)per_row);
  return from_hip(hipGetLastError());
}

size_t w4a32_op_paged_evict_scratch_bytes(const w4a32_paged_cache* cache, int budget) {
  if (check_cache(cache) || budget < 1 || budget >= kMost) return 0;
  return (size_t)cache->n_seqs * cache->kv_heads * budget * sizeof(int);
}

int w4a32_op_paged_evict(const w4a32_paged_cache* cache, const w4a32_paged_cache* to, int budget, int first, int recent, int* d_kept,
                         void* d_scratch, size_t scratch_bytes, void* stream) {
  if (int e = check_cache(cache)) return e;
  if (int e = check_cache(to)) return e;
  if (!cache->d_weight || !to->d_weight || budget < 1 || first < 0 || recent < 0 || !aligned(d_kept, 4)) return W4A32_EINVAL;
  if (cache->dtype != to->dtype || cache->dim != to->dim || cache->kv_heads != to->kv_heads || cache->n_seqs != to->n_seqs)
    return W4A32_ESHAPE;
  if ((long long)first + recent > budget || budget > (long long)to->table_ld * to->page) return W4A32_ESHAPE;
  if (cache->d_len == to->d_len) return W4A32_EINVAL;
  if (cache->d_table == to->d_table && (cache->d_k == to->d_k || cache->d_v == to->d_v || cache->d_weight == to->d_weight))
    return W4A32_EINVAL;  // the same pages
  const size_t need = w4a32_op_paged_evict_scratch_bytes(cache, budget);
  if (!d_kept && (!d_scratch || !aligned(d_scratch, 16) || scratch_bytes < need)) return W4A32_EINVAL;
  const Evict a{view(cache), view(to), budget, first, recent, d_kept ? d_kept : static_cast<int*>(d_scratch), to->d_len};
  const long long heads = (long long)cache->n_seqs * cache->kv_heads;
  const int units = cache->dim * (cache->dtype == W4A32_CACHE_F32 ? 4 : 2) / 16, per = kCopies * (256 / units);
  const long long blocks = ((long long)budget + per - 1) / per;
  if (heads > most_groups(kSelect) || heads * blocks > most_groups(256)) return W4A32_ESHAPE;
  hipStream_t s = static_cast<hipStream_t>(stream);
  // the table says how long a sequence can be
  const size_t held = (size_t)cache->table_ld * cache->page;
  if (held <= kHeld) {
    static w4::LdsLimitOnce limit;
    if (limit.raise((const void*)select_kernel<true>, kHeld * sizeof(unsigned)) != hipSuccess) return W4A32_ELAUNCH;
    hipLaunchKernelGGL((select_kernel<true>), dim3((unsigned)heads), dim3(kSelect), held * sizeof(unsigned), s, a);
  } else {
    hipLaunchKernelGGL((select_kernel<false>), dim3((unsigned)heads), dim3(kSelect), 0, s, a);
  }
  if (hipGetLastError() != hipSuccess) return W4A32_ELAUNCH;
  hipLaunchKernelGGL(copy_kernel, dim3((unsigned)(heads * blocks)), dim3(256), 0, s, a, units, (int)blocks);
  return from_hip(hipGetLastError());
}

}  // extern "C"
