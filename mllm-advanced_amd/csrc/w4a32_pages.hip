// The pages of a paged cache: which sequence has which (fork), their copies in all layers' pools, and their move to the pool's front.
#include "w4a32_paged.h"

namespace w4 {
namespace paged {

namespace {
inline bool aligned(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }
inline int from_hip(hipError_t e) { return e == hipSuccess ? W4A32_OK : W4A32_ELAUNCH; }
inline size_t up256(size_t v) { return (v + 255) / 256 * 256; }

constexpr int kSettle = 1024;         // threads of the one workgroup that hands pages out
constexpr int kMostPlaces = 1 << 26;  // places of a table: a place's number and two marks are an int
// A page with a negative count, which is someone else's: changes by all places there are leave it below kHeldBelow.
constexpr int kHeld = -0x7f000000, kHeldBelow = -(1 << 30);
constexpr int kShared = 1 << 30, kStays = 1 << 29, kPlace = kMostPlaces - 1;

// ---------------------------------------------------------------------------------------------
// Fork. What each sequence becomes follows from its parent's length alone, so places are gone through in parallel: a new table
// and the pages' new counts go to scratch memory, by atomic sums of whole numbers. The rows' places (one or two of a sequence
// that decodes) are then listed in order and settled by one workgroup: who has to leave a shared page, which pages are free. Where
// there are enough the last launch makes it all true; else nothing has changed.
// ---------------------------------------------------------------------------------------------
struct Seq {
  int parent, len;  // -1: none; tokens
  int kept, need;   // places with tokens; with those and the rows
  int first;        // the first that the rows write; `need` where there are none
};
struct Fork {
  int *table, *len, *refs;
  const int *parent, *keep, *row_start;
  int n_seqs, width, shift, n_pages, rows, max_rows, most;
  int *moves, *counts;
  Seq* seq;     // [n_seqs]
  int* left;    // [n_pages]: counts as they become
  int* next;    // [n_seqs][width]
  int* place;   // [most]: places that the rows write, in order
  int* was;     // [most]: pages there, or -1
  int* fresh;   // [most]: free pages
};

__device__ __forceinline__ bool named(const Fork& a, int page) { return (unsigned)page < (unsigned)a.n_pages; }

__device__ __forceinline__ Seq seq_of(const Fork& a, int b) {
  Seq s;
  s.parent = a.parent ? a.parent[b] : b;
  if ((unsigned)s.parent >= (unsigned)a.n_seqs) s.parent = -1;
  s.len = s.parent < 0 ? 0 : min(max(a.len[s.parent], 0), kMost);
  if (a.keep) s.len = min(s.len, max(a.keep[b], 0));
  int n = 0;
  if (a.row_start) {
    const int lo = min(max(a.row_start[b], 0), a.rows);
    n = min(min(max(a.row_start[b + 1], lo), a.rows) - lo, a.max_rows);
  }
  const int page = 1 << a.shift;
  s.kept = min((s.len + page - 1) >> a.shift, a.width);
  s.need = n ? max(s.kept, (int)min((unsigned)(s.len + n - 1) / (unsigned)page + 1, (unsigned)a.width)) : s.kept;
  s.first = n ? min(s.len >> a.shift, s.need) : s.need;
  return s;
}

__global__ __launch_bounds__(256) void fork_begin_kernel(Fork a) {
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (i < a.n_pages) {
    const int r = a.refs[i];
    a.left[i] = r < 0 ? kHeld : min(r, kMostPlaces);
  }
  if (i < a.n_seqs) a.seq[i] = seq_of(a, i);
}

__global__ __launch_bounds__(256) void fork_places_kernel(Fork a) {
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (i >= a.n_seqs * a.width) return;
  const int b = i / a.width, at = i - b * a.width;
  const Seq s = a.seq[b];
  const int old = a.table[i];
  int page = -1;
  if (at < s.kept)
    page = s.parent == b ? old : a.table[(size_t)s.parent * a.width + at];
  else if (at < s.need && s.parent == b)
    page = old;
  a.next[i] = page;
  if (page == old) return;
  if (named(a, old)) atomicSub(&a.left[old], 1);
  if (named(a, page)) atomicAdd(&a.left[page], 1);
}

__device__ __forceinline__ int count_of(const Fork& a, int page) {
  return __hip_atomic_load(&a.left[page], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

__global__ __launch_bounds__(kSettle) void fork_settle_kernel(Fork a) {
  __shared__ unsigned in_wave[kSettle / 64];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  // ---- the places that rows write ----
  unsigned total = 0;
  for (int b0 = 0; b0 < a.n_seqs; b0 += kSettle) {
    const int b = b0 + tid;
    Seq s = {};
    if (b < a.n_seqs) s = a.seq[b];
    const unsigned n = (unsigned)(s.need - s.first);
    unsigned all;
    const unsigned at = total + block_scan<kSettle>(n, in_wave, all) - n;
    for (unsigned i = 0; i < n; ++i) {
      if (at + i >= (unsigned)a.most) break;
      const int place = b * a.width + s.first + (int)i, page = a.next[place];
      a.place[at + i] = place;
      // a sequence's last tokens that are not there stay so, and the place with them
      a.was[at + i] = named(a, page) ? page : s.first + (int)i < s.kept ? -2 : -1;
    }
    total += all;
  }
  const int n = (int)min(total, (unsigned)a.most);
  __syncthreads();
  // ---- who has to leave a shared page: all that write it, or, where nobody else has it, all but the last ----
  for (int c = tid; c < n; c += kSettle)
    if (a.was[c] >= 0 && count_of(a, a.was[c]) != 1) a.place[c] |= kShared;
  __syncthreads();
  for (int c = tid; c < n; c += kSettle)
    if (a.place[c] & kShared && count_of(a, a.was[c]) >= kHeldBelow) atomicSub(&a.left[a.was[c]], 1);
  __syncthreads();
  for (int c = tid; c < n; c += kSettle)
    if (a.place[c] & kShared) {
      const int r = count_of(a, a.was[c]);
      if (r <= 0 && r >= kHeldBelow) atomicMin(&a.left[a.was[c]], -2 - (a.place[c] & kPlace));
    }
  __syncthreads();
  for (int c = tid; c < n; c += kSettle)
    if (a.place[c] & kShared && count_of(a, a.was[c]) == -2 - (a.place[c] & kPlace)) a.place[c] |= kStays;
  __syncthreads();
  unsigned wanted = 0;
  auto leaves = [&](int c) { return (a.place[c] & (kShared | kStays)) == kShared; };
  for (int c = tid; c < n; c += kSettle) {
    if (a.place[c] & kStays) __hip_atomic_store(&a.left[a.was[c]], 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    wanted += leaves(c) || a.was[c] == -1;
  }
  unsigned all;
  block_scan<kSettle>(wanted, in_wave, all);  // its barriers stand behind the stores
  wanted = all;
  // ---- free pages, the lowest first: a run of pages of each wavefront ----
  const int run = (a.n_pages / (kSettle / 64) + 64) & -64, p0 = min(wave * run, a.n_pages), p1 = min(p0 + run, a.n_pages);
  unsigned free = 0;
  for (int p = p0; p < p1; p += 64) free += __popcll(__ballot(p + lane < p1 && count_of(a, min(p + lane, p1 - 1)) == 0));
  unsigned nth = block_scan<kSettle>(lane == 0 ? free : 0, in_wave, all);
  nth = (unsigned)__builtin_amdgcn_readfirstlane((int)nth) - free;
  const bool ok = wanted <= all && total <= (unsigned)a.most;
  if (ok) {
    for (int p = p0; p < p1 && nth < wanted; p += 64) {
      const bool here = p + lane < p1 && count_of(a, min(p + lane, p1 - 1)) == 0;
      const unsigned long long who = __ballot(here);
      const unsigned mine = nth + __popcll(who & ((1ull << lane) - 1));
      if (here && mine < wanted) a.fresh[mine] = p + lane;
      nth += __popcll(who);
    }
  }
  __syncthreads();
  // ---- and who gets them ----
  unsigned given = 0, copied = 0;
  for (int c0 = 0; ok && c0 < n; c0 += kSettle) {
    const int c = c0 + tid;
    const bool leave = c < n && leaves(c), want = leave || (c < n && a.was[c] == -1);
    const int place = c < n ? a.place[c] & kPlace : 0, b = place / a.width;
    const bool copy = leave && place - b * a.width < a.seq[b].kept;
    const unsigned x = (unsigned)want | (unsigned)copy << 16, upto = block_scan<kSettle>(x, in_wave, all);
    if (want) {
      const int page = a.fresh[given + (upto & 0xffff) - 1];
      a.next[place] = page;
      __hip_atomic_store(&a.left[page], 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      if (copy) {
        int* to = a.moves + 2 * (size_t)(copied + (upto >> 16) - 1);
        to[0] = a.was[c];
        to[1] = page;
      }
    }
    given += all & 0xffff;
    copied += all >> 16;
  }
  for (unsigned i = copied + tid; i < (unsigned)a.n_seqs; i += kSettle) a.moves[2 * (size_t)i] = a.moves[2 * (size_t)i + 1] = -1;
  if (tid == 0) {
    a.counts[0] = (int)copied;
    a.counts[1] = ok ? 0 : max((int)(wanted - min(wanted, all)), 1);
  }
}

__global__ __launch_bounds__(256) void fork_end_kernel(Fork a) {
  if (a.counts[1] != 0) return;
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (i < a.n_seqs * a.width) a.table[i] = a.next[i];
  if (i < a.n_seqs) a.len[i] = a.seq[i].len;
  if (i < a.n_pages && a.left[i] >= kHeldBelow) a.refs[i] = max(a.left[i], 0);
}

// ---------------------------------------------------------------------------------------------
// Copies. A unit is kUnit bytes of one page's keys, values or weights in one cache; workgroups take every gridDim.x-th, so that a
// captured launch serves as many pairs as the list then has.
// ---------------------------------------------------------------------------------------------
constexpr int kUnit = 8192;
constexpr int kAtOnce = 32;  // caches of a launch
struct Copy {
  const int *moves, *count;
  int most, n_pages, n_caches;
  unsigned units, k_units;  // of a page in a cache; of its keys
  unsigned row_bytes, weight_bytes;
  void *k[kAtOnce], *v[kAtOnce];
  float* w[kAtOnce];
};

__global__ __launch_bounds__(256) void copy_pages_kernel(Copy a) {
  const unsigned pairs = (unsigned)min(max(*a.count, 0), a.most);
  const unsigned long long all = (unsigned long long)pairs * a.n_caches * a.units;
  for (unsigned long long u = blockIdx.x; u < all; u += gridDim.x) {
    const unsigned of_pair = (unsigned)a.n_caches * a.units;
    const unsigned pair = (unsigned)(u / of_pair), in = (unsigned)(u - (unsigned long long)pair * of_pair);
    const unsigned cache = in / a.units, unit = in - cache * a.units;
    const int from = a.moves[2 * (size_t)pair], to = a.moves[2 * (size_t)pair + 1];
    if ((unsigned)from >= (unsigned)a.n_pages || (unsigned)to >= (unsigned)a.n_pages) continue;
    if (unit < 2 * a.k_units) {
      const bool is_v = unit >= a.k_units;
      uint8_t* pool = (uint8_t*)(is_v ? a.v[cache] : a.k[cache]);
      const unsigned lo = (unit - (is_v ? a.k_units : 0)) * kUnit + 16 * threadIdx.x;
      const uint8_t* src = pool + (size_t)from * a.row_bytes;
      uint8_t* dst = pool + (size_t)to * a.row_bytes;
      u32x4 x[kUnit / 4096];
#pragma unroll
      for (int i = 0; i < kUnit / 4096; ++i)
        if (lo + 4096 * i < a.row_bytes) x[i] = load_global<u32x4>(src + lo + 4096 * i);
#pragma unroll
      for (int i = 0; i < kUnit / 4096; ++i)
        if (lo + 4096 * i < a.row_bytes) *(W4_GLOBAL u32x4*)(dst + lo + 4096 * i) = x[i];
    } else {
      const unsigned words = a.weight_bytes / 4, lo = (unit - 2 * a.k_units) * (kUnit / 4);
      const float* src = a.w[cache] + (size_t)from * words;
      float* dst = a.w[cache] + (size_t)to * words;
      for (unsigned i = lo + threadIdx.x; i < min(lo + kUnit / 4, words); i += 256) dst[i] = src[i];
    }
  }
}

// ---------------------------------------------------------------------------------------------
// Compaction. Which pages are used and which may move are bits, 64 of a word, and a page's place among the movers or the holes
// is the words' running sum and the bits below it. The i-th mover goes to the i-th hole.
// ---------------------------------------------------------------------------------------------
typedef unsigned long long Bits64;
struct Head {
  int used, pairs;
};
struct Compact {
  int *table, *refs;
  int n_seqs, width, n_pages, words;
  int *moves, *counts;
  Head* head;
  Bits64 *used, *mover;  // [words]; the latter of all pages that may move, then of those behind the last that stays
  int* before;           // [words]: movers in front of a word
};

__global__ __launch_bounds__(256) void compact_bits_kernel(Compact a) {
  const int p = blockIdx.x * 256 + threadIdx.x;
  const int r = p < a.n_pages ? a.refs[p] : 0;
  const Bits64 used = __ballot(r != 0), mover = __ballot(r > 0);
  if ((threadIdx.x & 63) == 0 && p < a.n_pages) {
    a.used[p >> 6] = used;
    a.mover[p >> 6] = mover;
  }
}

__global__ __launch_bounds__(kSettle) void compact_lists_kernel(Compact a) {
  __shared__ unsigned in_wave[kSettle / 64];
  __shared__ int last;
  const int tid = threadIdx.x;
  if (tid == 0) last = 0;
  unsigned mine = 0, all;
  for (int w = tid; w < a.words; w += kSettle) mine += __popcll(a.used[w]);
  block_scan<kSettle>(mine, in_wave, all);
  const int used = (int)all;
  auto below = [&](int w) { return used >= 64 * (w + 1) ? ~0ull : used <= 64 * w ? 0ull : (1ull << (used - 64 * w)) - 1; };
  auto movers_of = [&](int w) { return a.mover[w] & ~below(w); };
  mine = 0;
  for (int w = tid; w < a.words; w += kSettle) {
    mine += __popcll(movers_of(w));
    const Bits64 held = a.used[w] & ~a.mover[w] & ~below(w);
    if (held) atomicMax(&last, 64 * w + 64 - __builtin_clzll(held));
  }
  block_scan<kSettle>(mine, in_wave, all);
  const unsigned pairs = all;  // as many holes as movers or more
  unsigned movers = 0, holes = 0;
  for (int w0 = 0; w0 < a.words; w0 += kSettle) {
    const int w = w0 + tid;
    Bits64 from = w < a.words ? movers_of(w) : 0, to = w < a.words ? ~a.used[w] & below(w) : 0;
    unsigned i = movers + block_scan<kSettle>(__popcll(from), in_wave, all) - __popcll(from);
    movers += all;
    if (w < a.words) {
      a.before[w] = (int)i;
      a.mover[w] = from;
    }
    for (; from; from &= from - 1) a.moves[2 * (size_t)i++] = 64 * w + __builtin_ctzll(from);
    i = holes + block_scan<kSettle>(__popcll(to), in_wave, all) - __popcll(to);
    holes += all;
    for (; to && i < pairs; to &= to - 1) a.moves[2 * (size_t)i++ + 1] = 64 * w + __builtin_ctzll(to);
  }
  if (tid == 0) {
    a.head->used = used;
    a.head->pairs = (int)pairs;
    a.counts[0] = (int)pairs;
    a.counts[1] = max(last, used);
  }
}

__global__ __launch_bounds__(256) void compact_apply_kernel(Compact a) {
  const int i = blockIdx.x * 256 + threadIdx.x;
  const int pairs = a.head->pairs;
  if (i < a.n_seqs * a.width) {
    const int page = a.table[i];
    if ((unsigned)page < (unsigned)a.n_pages) {
      const Bits64 word = a.mover[page >> 6], bit = 1ull << (page & 63);
      if (word & bit) a.table[i] = a.moves[2 * (size_t)(a.before[page >> 6] + __popcll(word & (bit - 1))) + 1];
    }
  }
  if (i >= a.n_pages / 2) return;
  int* move = a.moves + 2 * (size_t)i;
  if (i < pairs) {
    a.refs[move[1]] = a.refs[move[0]];
    a.refs[move[0]] = 0;
  } else {
    move[0] = move[1] = -1;
  }
}

// ---- host ------------------------------------------------------------------------------------------------------------------
int check_table(const w4a32_paged_cache* c) {
  if (int e = check_cache(c)) return e;
  if ((long long)c->n_seqs * c->table_ld > kMostPlaces || c->n_pages > kMostPlaces) return W4A32_ESHAPE;
  return W4A32_OK;
}

// Places that so many rows write: each sequence has a page that they begin in and one that they end in
long long most_written(const w4a32_paged_cache* c, int rows) {
  const long long each = rows / c->page + 2ll * (rows < c->n_seqs ? rows : c->n_seqs), all = (long long)c->n_seqs * c->table_ld;
  return each < all ? each : all;
}

struct ForkRoom {
  size_t seq, left, next, place, was, fresh, total;
};
ForkRoom fork_room(const w4a32_paged_cache* c, int rows) {
  ForkRoom r;
  const size_t most = (size_t)most_written(c, rows);
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t here = at;
    at = up256(at + bytes);
    return here;
  };
  r.seq = take((size_t)c->n_seqs * sizeof(Seq));
  r.left = take((size_t)c->n_pages * 4);
  r.next = take((size_t)c->n_seqs * c->table_ld * 4);
  r.place = take(most * 4);
  r.was = take(most * 4);
  r.fresh = take(most * 4);
  r.total = at;
  return r;
}

struct CompactRoom {
  size_t used, mover, before, total;
  int words;
};
CompactRoom compact_room(const w4a32_paged_cache* c) {
  CompactRoom r;
  r.words = (c->n_pages + 63) / 64;
  r.used = 256;
  r.mover = r.used + up256((size_t)r.words * 8);
  r.before = r.mover + up256((size_t)r.words * 8);
  r.total = r.before + up256((size_t)r.words * 4);
  return r;
}
}  // namespace

}  // namespace paged
}  // namespace w4

using namespace w4::paged;

extern "C" {

size_t w4a32_op_paged_fork_scratch_bytes(const w4a32_paged_cache* cache, int rows) {
  if (check_table(cache) || rows < 0 || rows >= kMost) return 0;
  return fork_room(cache, rows).total;
}

int w4a32_op_paged_fork(const w4a32_paged_cache* cache, const w4a32_paged_fork_args* f, void* d_scratch, size_t scratch_bytes, void* stream) {
  if (int e = check_table(cache)) return e;
  if (!f || !f->d_refs || !f->d_moves || !f->d_counts || !d_scratch) return W4A32_EINVAL;
  if (!aligned(f->d_refs, 4) || !aligned(f->d_moves, 4) || !aligned(f->d_counts, 4) || !aligned(f->d_parent, 4) || !aligned(f->d_keep, 4) ||
      !aligned(f->d_row_start, 4) || !aligned(d_scratch, 16))
    return W4A32_EINVAL;
  if (f->d_row_start && (f->rows < 1 || f->max_rows < 1)) return W4A32_EINVAL;
  const int rows = f->d_row_start ? f->rows : 0;
  if (rows >= kMost) return W4A32_ESHAPE;
  const ForkRoom r = fork_room(cache, rows);
  if (scratch_bytes < r.total) return W4A32_EINVAL;
  uint8_t* s = static_cast<uint8_t*>(d_scratch);
  const Fork a{const_cast<int*>(cache->d_table), cache->d_len, f->d_refs, f->d_parent, f->d_keep, f->d_row_start, cache->n_seqs, cache->table_ld,
               log2_of(cache->page), cache->n_pages, rows, f->max_rows, (int)most_written(cache, rows), f->d_moves, f->d_counts, (Seq*)(s + r.seq),
               (int*)(s + r.left), (int*)(s + r.next), (int*)(s + r.place), (int*)(s + r.was), (int*)(s + r.fresh)};
  hipStream_t st = static_cast<hipStream_t>(stream);
  const unsigned places = (unsigned)cache->n_seqs * cache->table_ld, pages = (unsigned)cache->n_pages;
  const unsigned seqs = (unsigned)cache->n_seqs, begin = pages > seqs ? pages : seqs, end = places > pages ? places : pages;
  hipLaunchKernelGGL(fork_begin_kernel, dim3((begin + 255) / 256), dim3(256), 0, st, a);
  if (hipGetLastError() != hipSuccess) return W4A32_ELAUNCH;
  hipLaunchKernelGGL(fork_places_kernel, dim3((places + 255) / 256), dim3(256), 0, st, a);
  if (hipGetLastError() != hipSuccess) return W4A32_ELAUNCH;
  hipLaunchKernelGGL(fork_settle_kernel, dim3(1), dim3(kSettle), 0, st, a);
  if (hipGetLastError() != hipSuccess) return W4A32_ELAUNCH;
  hipLaunchKernelGGL(fork_end_kernel, dim3((end + 255) / 256), dim3(256), 0, st, a);
  return from_hip(hipGetLastError());
}

int w4a32_op_paged_copy(const w4a32_paged_cache* const* caches, int n_caches, const int* d_moves, const int* d_count, int most, void* stream) {
  if (!caches || n_caches < 1 || !d_moves || !d_count || most < 1 || !aligned(d_moves, 4) || !aligned(d_count, 4)) return W4A32_EINVAL;
  for (int i = 0; i < n_caches; ++i)
    if (int e = check_cache(caches[i])) return e;
  const w4a32_paged_cache& c = *caches[0];
  for (int i = 1; i < n_caches; ++i) {
    const w4a32_paged_cache& o = *caches[i];
    if (o.dtype != c.dtype || o.n_pages != c.n_pages || o.page != c.page || o.kv_heads != c.kv_heads || o.dim != c.dim || !o.d_weight != !c.d_weight)
      return W4A32_ESHAPE;
  }
  const unsigned long long tokens = (unsigned long long)c.kv_heads * c.page, bytes = tokens * c.dim * (c.dtype == W4A32_CACHE_F32 ? 4 : 2);
  if (bytes >= 1ull << 31) return W4A32_ESHAPE;
  Copy a;
  a.moves = d_moves;
  a.count = d_count;
  a.most = most;
  a.n_pages = c.n_pages;
  a.row_bytes = (unsigned)bytes;
  a.weight_bytes = c.d_weight ? (unsigned)tokens * 4 : 0;
  a.k_units = (a.row_bytes + kUnit - 1) / kUnit;
  a.units = 2 * a.k_units + (a.weight_bytes + kUnit - 1) / kUnit;
  for (int at = 0; at < n_caches; at += kAtOnce) {
    a.n_caches = n_caches - at < kAtOnce ? n_caches - at : kAtOnce;
    if ((unsigned long long)a.n_caches * a.units >= 1ull << 32) return W4A32_ESHAPE;
    for (int i = 0; i < a.n_caches; ++i) {
      a.k[i] = caches[at + i]->d_k;
      a.v[i] = caches[at + i]->d_v;
      a.w[i] = caches[at + i]->d_weight;
    }
    const unsigned long long units = (unsigned long long)most * a.n_caches * a.units;
    hipLaunchKernelGGL(copy_pages_kernel, dim3((unsigned)(units < 2048 ? units : 2048)), dim3(256), 0, static_cast<hipStream_t>(stream), a);
    if (hipGetLastError() != hipSuccess) return W4A32_ELAUNCH;
  }
  return W4A32_OK;
}

size_t w4a32_op_paged_compact_scratch_bytes(const w4a32_paged_cache* cache) {
  return check_table(cache) ? 0 : compact_room(cache).total;
}

int w4a32_op_paged_compact(const w4a32_paged_cache* cache, int* d_refs, int* d_moves, int* d_counts, void* d_scratch, size_t scratch_bytes,
                           void* stream) {
  if (int e = check_table(cache)) return e;
  if (!d_refs || (!d_moves && cache->n_pages > 1) || !d_counts || !d_scratch) return W4A32_EINVAL;
  if (!aligned(d_refs, 4) || !aligned(d_moves, 4) || !aligned(d_counts, 4) || !aligned(d_scratch, 16)) return W4A32_EINVAL;
  const CompactRoom r = compact_room(cache);
  if (scratch_bytes < r.total) return W4A32_EINVAL;
  uint8_t* s = static_cast<uint8_t*>(d_scratch);
  const Compact a{const_cast<int*>(cache->d_table), d_refs, cache->n_seqs, cache->table_ld, cache->n_pages, r.words, d_moves, d_counts, (Head*)s,
                  (Bits64*)(s + r.used), (Bits64*)(s + r.mover), (int*)(s + r.before)};
  hipStream_t st = static_cast<hipStream_t>(stream);
  const unsigned places = (unsigned)cache->n_seqs * cache->table_ld, pages = (unsigned)cache->n_pages, most = places > pages ? places : pages;
  hipLaunchKernelGGL(compact_bits_kernel, dim3((pages + 255) / 256), dim3(256), 0, st, a);
  if (hipGetLastError() != hipSuccess) return W4A32_ELAUNCH;
  hipLaunchKernelGGL(compact_lists_kernel, dim3(1), dim3(kSettle), 0, st, a);
  if (hipGetLastError() != hipSuccess) return W4A32_ELAUNCH;
  hipLaunchKernelGGL(compact_apply_kernel, dim3((most + 255) / 256), dim3(256), 0, st, a);
  return from_hip(hipGetLastError());
}

}  // extern "C"
