// The pages of a paged cache: which sequence has which (fork), their copies in all layers' pools, and their move to the pool's front.
#include <climits>

#include "w4a32_paged.h"

namespace w4 {
namespace paged {

namespace {
inline bool aligned(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }
inline int from_hip(hipError_t e) { return e == hipSuccess ? W4A32_OK : W4A32_ELAUNCH; }
inline size_t up256(size_t v) { return (v + 255) / 256 * 256; }

constexpr int kSettle = 1024;         // threads of the one workgroup that hands pages out
constexpr int kMostPlaces = 1 << 26;  // places of a table: a place's number and two marks are an int
// A page with a negative count, which is someone else's: changes by all places there are, up or down, leave it an int and below kHeldBelow; other counts
// stay above, with the marks of those that write such a page.
constexpr int kHeld = -(3 << 29), kHeldBelow = -(1 << 30);
static_assert((long long)kHeld - kMostPlaces >= INT_MIN && kHeld + kMostPlaces < kHeldBelow && -2 - 2 * kMostPlaces >= kHeldBelow, "counts of pages");
constexpr int kShared = 1 << 30, kStays = 1 << 29, kGiven = 1 << 28, kPlace = kMostPlaces - 1;

// ---------------------------------------------------------------------------------------------
// Fork. What each sequence becomes follows from its parent's length alone, so places are gone through in parallel, and the pages' new
// counts are atomic sums of whole numbers. The places that rows write (one or two of a sequence that decodes) are then listed in
// order and settled by one workgroup: who has to leave a shared page, which pages are free. Where there are enough it all becomes true;
// else nothing has changed.
// What is moved is small (4 bytes of a place and of a page); latency bounds all of it, waits for memory and barriers of 16 wavefronts one after the
// other. Where the counts fit into LDS: one launch of one workgroup. Else four launches, with the new table and the new counts in scratch memory (32
// prompts of up to 32000 tokens with eight children each, 2.9 MB: 2.6 + 8.2 + 11.9 + 4.0 us, of which the third is the one workgroup that settles).
// ---------------------------------------------------------------------------------------------
struct Seq {
  int parent, len;  // -1: none; tokens
  int kept, need;   // places with tokens; with those and the rows
  int first;        // the first that the rows write; `need` where there are none
  int end;          // places of its own in front of it stay, where it goes on from itself: end_of()
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
// Behind a sequence's tokens its pages follow each other: where one goes on from itself, with all places of its tokens, and the first place behind those that
// it needs names -1, that is the end of them, and what may stand behind it is not looked at. So all ways of a fork leave the same, of which the
// shortest has no time to look at all places.
__device__ __forceinline__ int end_of(const Fork& a, int b, const Seq& s) {
  if (s.parent != b || s.need >= a.width) return s.need;
  const int had = min((min(max(a.len[b], 0), kMost) + (1 << a.shift) - 1) >> a.shift, a.width);
  return s.need >= had && a.table[(size_t)b * a.width + s.need] == -1 ? a.width : s.need;
}
__device__ __forceinline__ int count_at_first(int refs) { return refs < 0 ? kHeld : min(refs, kMostPlaces); }
// The page that a place gets before rows are looked at; `old`: what is there
__device__ __forceinline__ int inherited(const Fork& a, const Seq& s, int b, int at, int old) {
  if (at < s.kept) return s.parent == b ? old : a.table[(size_t)s.parent * a.width + at];
  return at < s.end && s.parent == b ? old : -1;
}

// Counts in LDS, and in memory that several compute units have written: past the caches of this one.
struct NearCounts {
  static constexpr bool kNear = true;
  int* left;
  __device__ __forceinline__ int get(int p) const { return left[p]; }
  __device__ __forceinline__ void set(int p, int v) const { left[p] = v; }
};
struct FarCounts {
  static constexpr bool kNear = false;
  int* left;
  __device__ __forceinline__ int get(int p) const { return __hip_atomic_load(&left[p], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
  __device__ __forceinline__ void set(int p, int v) const { __hip_atomic_store(&left[p], v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
};

// Settles the places that rows write, by one workgroup. seq, page_at: what the sequences become, and the pages of their places; place, was, fresh:
// room for a.most of each, in LDS or not. Returns how many places there are, of which those with kGiven get page was[..]; -1: it cannot be done.
// leave(page): a page that a sequence leaves, its count being what it will be.
template <typename Counts, typename SeqAt, typename PageAt, typename Leave>
__device__ __forceinline__ int settle(const Fork& a, Counts left, SeqAt seq, PageAt page_at, int* place, int* was, int* fresh, Leave leave_page) {
  __shared__ unsigned in_wave[kSettle / 64];
  const int tid = threadIdx.x;
  unsigned total = 0;
  bool shared = false;
  for (int b0 = 0; b0 < a.n_seqs; b0 += kSettle) {
    const int b = b0 + tid;
    Seq s = {};
    if (b < a.n_seqs) s = seq(b);
    const unsigned n = (unsigned)(s.need - s.first);
    unsigned all;
    const unsigned at = total + block_scan<kSettle>(n, in_wave, all) - n;
    for (unsigned i = 0; i < n && at + i < (unsigned)a.most; ++i) {
      const int i_at = s.first + (int)i, page = page_at(s, b, i_at);
      // a sequence's last tokens that are not there stay so, and the place with them
      was[at + i] = named(a, page) ? page : i_at < s.kept ? -2 : -1;
      const bool more = named(a, page) && left.get(page) != 1;
      place[at + i] = b * a.width + i_at + (more ? kShared : 0);
      shared |= more;
    }
    total += all;
  }
  const int n = (int)min(total, (unsigned)a.most);
  // ---- who has to leave a shared page: all that write it, or, where nobody else has it, all but the last ----
  if (__syncthreads_or(shared)) {
    for (int c = tid; c < n; c += kSettle)
      if (place[c] & kShared && left.get(was[c]) >= kHeldBelow) atomicSub(&left.left[was[c]], 1);
    __syncthreads();
    for (int c = tid; c < n; c += kSettle)
      if (place[c] & kShared) {
        const int r = left.get(was[c]);
        if (r <= 0 && r >= kHeldBelow) atomicMin(&left.left[was[c]], -2 - (place[c] & kPlace));
      }
    __syncthreads();
    for (int c = tid; c < n; c += kSettle)
      if (place[c] & kShared && left.get(was[c]) == -2 - (place[c] & kPlace)) place[c] |= kStays;
    __syncthreads();
    for (int c = tid; c < n; c += kSettle)
      if (place[c] & kStays) left.set(was[c], 1);
  }
  auto leaves = [&](int c) { return (place[c] & (kShared | kStays)) == kShared; };
  unsigned wanted = 0, all;
  for (int c = tid; c < n; c += kSettle) wanted += leaves(c) || was[c] == -1;
  block_scan<kSettle>(wanted, in_wave, all);  // its barriers stand behind the stores
  wanted = all;
  // ---- free pages, the lowest first. In LDS a thread has the bits of up to 31 that follow each other, an odd number, so that its reads and those of the
  // other threads meet in different banks; else a wavefront has a run of 64s, a lane the bits of one of these, and the first 16384 pages are looked at
  // alone (67000 pages of which a half is free: 14.6 us with all of them) ----
  constexpr int kAhead = Counts::kNear ? 8 : 16;
  const int lane = tid & 63, wave = tid >> 6;
  unsigned found = 0;
  for (int p0 = 0, each; p0 < a.n_pages && found < wanted; p0 += each * kSettle) {
    unsigned long long bits = 0;
    int first;
    if constexpr (Counts::kNear) {
      each = min((a.n_pages - p0 + kSettle - 1) / kSettle | 1, 31);
      first = p0 + tid * each;
      for (int i0 = 0; i0 < each; i0 += kAhead) {
        int counts[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) counts[i] = left.get(min(first + i0 + i, a.n_pages - 1));
#pragma unroll
        for (int i = 0; i < kAhead; ++i) bits |= (counts[i] == 0 && i0 + i < each && first + i0 + i < a.n_pages ? 1u : 0u) << ((i0 + i) & 31);
      }
    } else {
      each = min((a.n_pages - p0 + kSettle - 1) / kSettle, p0 ? 64 : 16);
      first = p0 + wave * each * 64;
      for (int i0 = 0; i0 < each; i0 += kAhead) {
        int counts[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) counts[i] = left.get(min(first + 64 * (i0 + i) + lane, a.n_pages - 1));
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
          const unsigned long long b = __ballot(i0 + i < each && first + 64 * (i0 + i) + lane < a.n_pages && counts[i] == 0);
          if (lane == i0 + i) bits = b;
        }
      }
      first += 64 * lane;
    }
    const unsigned mine = __popcll(bits), upto = block_scan<kSettle>(mine, in_wave, all);
    for (unsigned at = found + upto - mine; bits && at < wanted; bits &= bits - 1) fresh[at++] = first + __builtin_ctzll(bits);
    found += all;
  }
  const bool ok = wanted <= found && total <= (unsigned)a.most;
  __syncthreads();
  // ---- and who gets them ----
  unsigned given = 0, copied = 0;
  for (int c0 = 0; ok && c0 < n; c0 += kSettle) {
    const int c = c0 + tid;
    const bool leave = c < n && leaves(c), want = leave || (c < n && was[c] == -1);
    const int at = c < n ? place[c] & kPlace : 0, b = at / a.width;
    const bool copy = leave && at - b * a.width < seq(b).kept;
    unsigned upto = 0;
    if (wanted) upto = block_scan<kSettle>((unsigned)want | (unsigned)copy << 16, in_wave, all);
    if (want) {
      const int page = fresh[given + (upto & 0xffff) - 1];
      left.set(page, 1);
      if (copy) {
        int* to = a.moves + 2 * (size_t)(copied + (upto >> 16) - 1);
        to[0] = was[c];
        to[1] = page;
      }
      if (leave) leave_page(was[c]);
      place[c] = at | kGiven;
      was[c] = page;
    }
    if (wanted) {
      given += all & 0xffff;
      copied += all >> 16;
    }
  }
  for (unsigned i = copied + tid; i < (unsigned)a.n_seqs; i += kSettle) a.moves[2 * (size_t)i] = a.moves[2 * (size_t)i + 1] = -1;
  if (tid == 0) {
    a.counts[0] = (int)copied;
    a.counts[1] = ok ? 0 : max((int)(wanted - min(wanted, found)), 1);
  }
  return ok ? n : -1;
}

// ---- one launch ----
// One workgroup and four launches, us of a pass among others with a table's copy of 2: rows for sequences that go on, 64 of up to 2000 tokens (8064
// places) 13 and 21, 500 of 1000 (31500 places) 13 and 23; with parents, eight children each, 64 of 1000 (4032 places) 13 and 24, 512 of 250 (8192) 18 and
// 30, 128 of 2000 (16128) 21 to 23 and 25, 500 of 1000 (31500) 35 and 28; with kept lengths, 64 of 1000 13 and 20, 128 of 2000 19 and 20, 256 of 2000
// (32256) 27 and 21. The rest is what there is room for. fork_nothing() is a part of the one launch, though it goes through no places: a decode step of 64
// sequences takes 8 us with tables of 512 places and 15 with 513 to 8192, or with pools of 100000 to 300000 pages.
constexpr int kNearPages = 32 * 1024, kNearSeqs = 512, kNearWritten = 1536, kNearPlaces = 32 * 1024, kNearChanged = 16 * 1024;

// A step that shares nothing and gives nothing back, as most are: rows' places that name no page get free ones, and that is all. Returns
// false where there is more to do, with nothing changed. A thread has a sequence; a wavefront a run of pages, 64 of each lane, whose counts are under
// way while the sequences' lengths are. Of the places behind those that a sequence needs only the first is looked at. (All of them instead, 128 KB by one
// workgroup: 11.9 us against 6.7.)
__device__ __forceinline__ bool fork_nothing(const Fork& a, int* fresh) {
  __shared__ unsigned in_wave[kSettle / 64];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  Seq s = {};
  if (tid < a.n_seqs) s = seq_of(a, tid);
  constexpr int kAhead = 16;
  const int run = (a.n_pages + 64 * (kSettle / 64) - 1) / (64 * (kSettle / 64)), first = wave * run * 64;  // at most 64 of 64
  unsigned long long bits = 0;
  for (int i0 = 0; i0 < run; i0 += kAhead) {
    int refs[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) refs[i] = load_global<int>(a.refs + min(first + 64 * (i0 + i) + lane, a.n_pages - 1));
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const unsigned long long b = __ballot(refs[i] == 0);
      if (lane == i0 + i && i0 + i < run) bits = b;
    }
  }
  const int left = a.n_pages - first - 64 * lane;  // the last page's count stands for those behind it
  bits &= left >= 64 ? ~0ull : left <= 0 ? 0ull : (1ull << left) - 1;
  const int* row = a.table + (size_t)tid * a.width;
  bool more = false;
  unsigned wants = 0;
  if (tid < a.n_seqs) {
    more = end_of(a, tid, s) < a.width;
    for (int at = s.first; at < s.need; ++at) {
      const int page = row[at];
      if (named(a, page))
        more |= a.refs[page] != 1;
      else
        wants += at >= s.kept;  // a sequence's last tokens that are not there stay so, and the place with them
    }
  }
  if (__syncthreads_or(more)) return false;
  unsigned wanted, found;
  const unsigned mine = __popcll(bits);
  unsigned nth = block_scan<kSettle>(wants, in_wave, wanted) - wants, at = block_scan<kSettle>(mine, in_wave, found) - mine;
  const bool ok = wanted <= found && wanted <= (unsigned)a.most;
  if (ok)
    for (; bits && at < wanted; bits &= bits - 1) fresh[at++] = first + 64 * lane + __builtin_ctzll(bits);
  __syncthreads();
  if (ok && tid < a.n_seqs) {
    for (int at = s.first; wants && at < s.need; ++at) {
      if (at < s.kept || named(a, row[at])) continue;
      const int page = fresh[nth++];
      a.table[(size_t)tid * a.width + at] = page;
      a.refs[page] = 1;
    }
    a.len[tid] = s.len;
  }
  for (int i = tid; i < 2 * a.n_seqs; i += kSettle) a.moves[i] = -1;
  if (tid == 0) {
    a.counts[0] = 0;
    a.counts[1] = ok ? 0 : max((int)(wanted - min(wanted, found)), 1);
  }
  return true;
}

// kForked: sequences have parents; else each goes on from itself, and only places from Seq::end on change here.
template <bool kForked>
__global__ __launch_bounds__(kSettle) void fork_kernel(Fork a) {
  extern __shared__ int lds[];
  int *left = lds, *place = left + a.n_pages, *was = place + a.most, *fresh = was + a.most;
  Seq* seqs = (Seq*)(fresh + a.most);
  if (!kForked && fork_nothing(a, fresh)) return;
  const int tid = threadIdx.x;
  constexpr int kAhead = 8;
  for (int p0 = tid; p0 < a.n_pages; p0 += kAhead * kSettle) {
    int refs[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) refs[i] = a.refs[min(p0 + i * kSettle, a.n_pages - 1)];
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
      if (p0 + i * kSettle < a.n_pages) left[p0 + i * kSettle] = count_at_first(refs[i]);
  }
  if (tid < a.n_seqs) {
    Seq s = seq_of(a, tid);
    s.end = end_of(a, tid, s);
    seqs[tid] = s;
  }
  __syncthreads();
  // A thread has every kSettle-th place, kFar of them at a time, and a bit for each that changes
  constexpr int kFar = 4;
  static_assert(kNearPlaces <= 32 * kSettle, "a thread's places are bits of a word");
  const int places = a.n_seqs * a.width;
  const unsigned per_width = 0xffffffffu / (unsigned)a.width + 1;  // quotients of less than 2^15 by no more than that are exact
  unsigned changed = 0;
  for (int i0 = tid, j0 = 0; i0 < places; i0 += kFar * kSettle, j0 += kFar) {
    int old[kFar], page[kFar];
    bool mine[kFar];
#pragma unroll
    for (int x = 0; x < kFar; ++x) {
      const int i = min(i0 + x * kSettle, places - 1), b = a.width == 1 ? i : (int)__umulhi((unsigned)i, per_width), at = i - b * a.width;
      const int parent = seqs[b].parent;
      mine[x] = i0 + x * kSettle < places && (parent != b || at >= seqs[b].end);
      old[x] = page[x] = -1;
      if (mine[x]) old[x] = a.table[i];
      if (kForked && mine[x] && parent != b && at < seqs[b].kept) page[x] = a.table[parent * a.width + at];
    }
#pragma unroll
    for (int x = 0; x < kFar; ++x) {
      if (kForked && mine[x]) a.next[i0 + x * kSettle] = page[x];
      if (old[x] == page[x]) continue;
      changed |= 1u << (j0 + x);
      if (named(a, old[x])) atomicSub(&left[old[x]], 1);
      if (named(a, page[x])) atomicAdd(&left[page[x]], 1);
    }
  }
  __syncthreads();
  auto count = [&](int p) {
    if (named(a, p) && left[p] >= kHeldBelow) a.refs[p] = max(left[p], 0);
  };
  const int n = settle(
      a, NearCounts{left}, [&](int b) { return seqs[b]; },
      [&](const Seq& s, int b, int at) { return inherited(a, s, b, at, s.parent == b ? a.table[b * a.width + at] : -1); }, place, was, fresh, count);
  if (n < 0) return;
  __syncthreads();  // the counts
  for (int i0 = tid; changed; i0 += kFar * kSettle, changed >>= kFar) {
    int old[kFar], page[kFar];
#pragma unroll
    for (int x = 0; x < kFar; ++x) {
      old[x] = page[x] = -1;
      if (!(changed >> x & 1)) continue;
      old[x] = a.table[i0 + x * kSettle];
      if (kForked) page[x] = a.next[i0 + x * kSettle];
    }
#pragma unroll
    for (int x = 0; x < kFar; ++x) {
      if (!(changed >> x & 1)) continue;
      a.table[i0 + x * kSettle] = page[x];
      count(old[x]);
      if (kForked) count(page[x]);
    }
  }
  if (tid < a.n_seqs) a.len[tid] = seqs[tid].len;
  __syncthreads();
  for (int c = tid; c < n; c += kSettle) {
    if (place[c] & kGiven) a.table[place[c] & kPlace] = was[c];
    count(was[c]);
  }
}

// ---- four launches ----
__global__ __launch_bounds__(256) void fork_begin_kernel(Fork a) {
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (i < a.n_pages) a.left[i] = count_at_first(a.refs[i]);
  if (i < a.n_seqs) {
    Seq s = seq_of(a, i);
    s.end = end_of(a, i, s);
    a.seq[i] = s;
  }
}

// A thread has the same place of kSide sequences that follow each other: children of one parent name one page there, and one atomic sum counts them
// (32 prompts of up to 32000 tokens with eight children each: 13.6 us one by one).
constexpr int kSide = 8;
__global__ __launch_bounds__(256) void fork_places_kernel(Fork a, int chunks) {
  const int b0 = blockIdx.x / chunks * kSide, at = (blockIdx.x % chunks) * 256 + threadIdx.x;
  if (at >= a.width) return;
  int old[kSide], page[kSide];
#pragma unroll
  for (int i = 0; i < kSide; ++i) {
    const int b = b0 + i;
    old[i] = page[i] = -1;
    if (b >= a.n_seqs) continue;
    old[i] = a.table[(size_t)b * a.width + at];
    page[i] = inherited(a, a.seq[b], b, at, old[i]);
    a.next[(size_t)b * a.width + at] = page[i];
  }
  int many = 0;
#pragma unroll
  for (int i = 0; i < kSide; ++i) {
    if (old[i] != page[i]) {
      if (named(a, old[i])) atomicSub(&a.left[old[i]], 1);
      many += named(a, page[i]);
    }
    // the last of a run of equal pages
    if (many && (i + 1 == kSide || page[i + 1] != page[i])) {
      atomicAdd(&a.left[page[i]], many);
      many = 0;
    }
  }
}

// kLists: the lists of places that rows write lie in LDS.
template <bool kLists>
__global__ __launch_bounds__(kSettle) void fork_settle_kernel(Fork a) {
  __shared__ int lists[kLists ? 3 * kNearWritten : 1];
  int *place = kLists ? lists : a.place, *was = kLists ? lists + kNearWritten : a.was, *fresh = kLists ? lists + 2 * kNearWritten : a.fresh;
  const int n = settle(
      a, FarCounts{a.left}, [&](int b) { return a.seq[b]; }, [&](const Seq&, int b, int at) { return a.next[(size_t)b * a.width + at]; }, place, was, fresh,
      [](int) {});
  __syncthreads();
  for (int c = threadIdx.x; c < n; c += kSettle)
    if (place[c] & kGiven) a.next[place[c] & kPlace] = was[c];
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
// captured launch serves as many pairs as the list then has. Memory bounds it: 64 pages of 64 KB and their weights in 28 caches, 237 MB read and
// written, take 47 us among other passes (5.0 TB/s, where a copy of 2 GiB reaches 4.9), and 37 where they are in the cache in front; eight pages of
// 32 KB in one cache 3 us, a launch. Copies are written past the caches, which keep what is read (52 us otherwise).
// ---------------------------------------------------------------------------------------------
constexpr int kUnit = 16384;
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
        if (lo + 4096 * i < a.row_bytes) __builtin_nontemporal_store(x[i], (W4_GLOBAL u32x4*)(dst + lo + 4096 * i));
    } else {
      const unsigned words = a.weight_bytes / 4, lo = (unit - 2 * a.k_units) * (kUnit / 4);
      const float* src = a.w[cache] + (size_t)from * words;
      float* dst = a.w[cache] + (size_t)to * words;
      for (unsigned i = lo + threadIdx.x; i < min(lo + kUnit / 4, words); i += 256) __builtin_nontemporal_store(src[i], (W4_GLOBAL float*)(dst + i));
    }
  }
}

// ---------------------------------------------------------------------------------------------
// Compaction. Which pages are used and which may move are bits, 64 of a word, and a page's place among the movers or the holes
// is the words' running sum and the bits below it. The i-th mover goes to the i-th hole: the last word whose sum does not pass i has it. One
// workgroup adds the words up; pages and places are then gone through by all. (Lists of movers and holes written by that one workgroup, a
// store of every bit, took 23 us for 65536 pages.) Latency bounds it: 2.6 + 8.1 us of two launches for 65536 pages, the second three
// scans, a search of ten dependent reads and the names; 2.5 + 4.4 + 6.7 of three for 65537; 6.6 us of one launch for 2000 pages.
// ---------------------------------------------------------------------------------------------
typedef unsigned long long Bits64;
struct Compact {
  int *table, *refs;
  int n_seqs, width, n_pages, words;
  int *moves, *counts;
  Bits64 *hole, *mover;             // [words]; at first the pages in use, and those that may move
  int *holes_before, *movers_before;  // [words]
};

// The lowest n bits, by halves as all that follows: a 64-bit shift by the last of a wavefront's registers is wrong now and then
__device__ __forceinline__ Bits64 first_bits(int n) {
  auto half = [](int n) { return n >= 32 ? ~0u : n <= 0 ? 0u : (1u << n) - 1; };
  return (Bits64)half(n - 32) << 32 | half(n);
}

__device__ __forceinline__ void compact_bits(const Compact& a, int p) {
  const int r = p < a.n_pages ? a.refs[p] : 0;
  const Bits64 used = __ballot(r != 0), mover = __ballot(r > 0);
  if ((threadIdx.x & 63) == 0 && p < a.n_pages) {
    a.hole[p >> 6] = used;
    a.mover[p >> 6] = mover;
  }
}

// By one workgroup; returns how many pages move, which is written where `writes`
__device__ __forceinline__ int compact_sums(const Compact& a, bool writes) {
  __shared__ unsigned in_wave[kSettle / 64];
  __shared__ int last;
  const int tid = threadIdx.x, each = (a.words + kSettle - 1) / kSettle, w0 = min(tid * each, a.words), w1 = min(w0 + each, a.words);
  if (tid == 0) last = 0;
  unsigned mine = 0, all;
  for (int w = w0; w < w1; ++w) mine += __popcll(a.hole[w]);
  block_scan<kSettle>(mine, in_wave, all);
  const int used = (int)all;
  auto below = [&](int w) { return first_bits(used - 64 * w); };
  unsigned movers = 0, holes = 0;
  int held = 0;
  for (int w = w0; w < w1; ++w) {
    const Bits64 in_use = a.hole[w], may = a.mover[w], from = may & ~below(w), to = ~in_use & below(w), stays = in_use & ~may & ~below(w);
    a.hole[w] = to;
    a.mover[w] = from;
    movers += __popcll(from);
    holes += __popcll(to);
    if (stays) held = 64 * w + 64 - __builtin_clzll(stays);
  }
  if (held) atomicMax(&last, held);
  unsigned h = block_scan<kSettle>(holes, in_wave, all) - holes;
  unsigned m = block_scan<kSettle>(movers, in_wave, all) - movers;
  for (int w = w0; w < w1; ++w) {
    a.holes_before[w] = (int)h;
    a.movers_before[w] = (int)m;
    h += __popcll(a.hole[w]);
    m += __popcll(a.mover[w]);
  }
  if (writes && tid == 0) {
    a.counts[0] = (int)all;  // as many holes as movers or more
    a.counts[1] = max(last, used);
  }
  return (int)all;
}

__device__ __forceinline__ int nth_hole(const Compact& a, int n) {
  int lo = 0, hi = a.words;  // holes_before[lo] <= n < holes_before[hi]
  while (hi - lo > 1) {
    const int mid = lo + (hi - lo) / 2;
    if (a.holes_before[mid] <= n)
      lo = mid;
    else
      hi = mid;
  }
  const Bits64 both = a.hole[lo];
  unsigned word = (unsigned)both;
  int in = n - a.holes_before[lo], at = 64 * lo;
  if (const int low = __popc(word); in >= low) {
    in -= low;
    at += 32;
    word = (unsigned)(both >> 32);
  }
#pragma unroll
  for (int half = 16; half; half /= 2) {
    const int low = __popc(word & ((1u << half) - 1));
    if (in >= low) {
      in -= low;
      at += half;
      word >>= half;
    }
  }
  return at;
}
// The number that a page gets; -1: it stays
__device__ __forceinline__ int mover_number(const Compact& a, int page) {
  const Bits64 both = a.mover[page >> 6];
  const unsigned low = (unsigned)both, bit = 1u << (page & 31), word = page & 32 ? (unsigned)(both >> 32) : low;
  return word & bit ? a.movers_before[page >> 6] + __popc(word & (bit - 1)) + (page & 32 ? __popc(low) : 0) : -1;
}

__device__ __forceinline__ void compact_apply(const Compact& a, int i, int pairs) {
  if (i < a.n_seqs * a.width) {
    const int page = a.table[i];
    if ((unsigned)page < (unsigned)a.n_pages) {
      const int n = mover_number(a, page);
      if (n >= 0) a.table[i] = nth_hole(a, n);
    }
  }
  if (i < a.n_pages) {
    const int n = mover_number(a, i);
    if (n >= 0) {
      const int to = nth_hole(a, n);
      a.moves[2 * (size_t)n] = i;
      a.moves[2 * (size_t)n + 1] = to;
      a.refs[to] = a.refs[i];
      a.refs[i] = 0;
    }
  }
  if (i < a.n_pages / 2 && i >= pairs) a.moves[2 * (size_t)i] = a.moves[2 * (size_t)i + 1] = -1;
}

__global__ __launch_bounds__(256) void compact_bits_kernel(Compact a) { compact_bits(a, blockIdx.x * 256 + threadIdx.x); }
__global__ __launch_bounds__(kSettle) void compact_sums_kernel(Compact a) { compact_sums(a, true); }
__global__ __launch_bounds__(256) void compact_apply_kernel(Compact a) { compact_apply(a, blockIdx.x * 256 + threadIdx.x, a.counts[0]); }

// The sums by every workgroup for itself, in LDS (65536 pages: 8.1 us where a launch of one workgroup and one of all with its searches in memory take 4.5
// and 6.7; 14.4 against 16.6 of a pass among others, 10000 pages 13.2 against 15.8, 131072 17.6 either way; with tables of some thousand places. There are as
// many workgroups as places by 1024, and where those are rounds of the chip so are the sums: 5000 pages and tables of 512 x 8192 places 29 us, 2048 x 8192 106)
constexpr int kWords = 1024;
__global__ __launch_bounds__(kSettle) void compact_both_kernel(Compact a) {
  __shared__ Bits64 hole[kWords], mover[kWords];
  __shared__ int holes_before[kWords], movers_before[kWords];
  for (int w = threadIdx.x; w < a.words; w += kSettle) {
    hole[w] = a.hole[w];
    mover[w] = a.mover[w];
  }
  a.hole = hole;
  a.mover = mover;
  a.holes_before = holes_before;
  a.movers_before = movers_before;
  __syncthreads();
  const int pairs = compact_sums(a, blockIdx.x == 0);
  __syncthreads();
  compact_apply(a, blockIdx.x * kSettle + threadIdx.x, pairs);
}

// All of it by one workgroup, where pages and places are few (2000 pages 12.2 us of a pass among others against 14.0 in two launches, 4096 12.3
// against 14.4, 5000 the same, 6000 16.0 against 14.3)
constexpr int kNearMoves = 4096;
__global__ __launch_bounds__(kSettle) void compact_kernel(Compact a) {
  __shared__ Bits64 hole[kNearMoves / 64], mover[kNearMoves / 64];
  __shared__ int holes_before[kNearMoves / 64], movers_before[kNearMoves / 64];
  a.hole = hole;
  a.mover = mover;
  a.holes_before = holes_before;
  a.movers_before = movers_before;
  for (int p = threadIdx.x; p < 64 * a.words; p += kSettle) compact_bits(a, p);
  __syncthreads();
  const int pairs = compact_sums(a, true);
  __syncthreads();
  for (int i = threadIdx.x; i < max(a.n_seqs * a.width, a.n_pages); i += kSettle) compact_apply(a, i, pairs);
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
  size_t mover, holes, movers, total;
  int words;
};
CompactRoom compact_room(const w4a32_paged_cache* c) {
  CompactRoom r;
  r.words = (c->n_pages + 63) / 64;
  r.mover = up256((size_t)r.words * 8);
  r.holes = r.mover + up256((size_t)r.words * 8);
  r.movers = r.holes + up256((size_t)r.words * 4);
  r.total = r.movers + up256((size_t)r.words * 4);
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
  if (cache->n_pages <= kNearPages && cache->n_seqs <= kNearSeqs && a.most <= kNearWritten &&
      places <= (unsigned)(a.parent || a.keep ? kNearChanged : kNearPlaces)) {
    static w4::LdsLimitOnce limit[2];
    auto kernel = a.parent ? fork_kernel<true> : fork_kernel<false>;
    if (limit[a.parent != nullptr].raise((const void*)kernel, 4 * (kNearPages + 3 * kNearWritten) + kNearSeqs * sizeof(Seq)) != hipSuccess) return W4A32_ELAUNCH;
    hipLaunchKernelGGL(kernel, dim3(1), dim3(kSettle), 4 * (size_t)(cache->n_pages + 3 * a.most) + cache->n_seqs * sizeof(Seq), st, a);
    return from_hip(hipGetLastError());
  }
  const unsigned seqs = (unsigned)cache->n_seqs, begin = pages > seqs ? pages : seqs, end = places > pages ? places : pages;
  hipLaunchKernelGGL(fork_begin_kernel, dim3((begin + 255) / 256), dim3(256), 0, st, a);
  if (hipGetLastError() != hipSuccess) return W4A32_ELAUNCH;
  const unsigned chunks = ((unsigned)cache->table_ld + 255) / 256;
  hipLaunchKernelGGL(fork_places_kernel, dim3((seqs + kSide - 1) / kSide * chunks), dim3(256), 0, st, a, (int)chunks);
  if (hipGetLastError() != hipSuccess) return W4A32_ELAUNCH;
  hipLaunchKernelGGL((a.most <= kNearWritten ? fork_settle_kernel<true> : fork_settle_kernel<false>), dim3(1), dim3(kSettle), 0, st, a);
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
    hipLaunchKernelGGL(copy_pages_kernel, dim3((unsigned)(units < 8192 ? units : 8192)), dim3(256), 0, static_cast<hipStream_t>(stream), a);
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
  const Compact a{const_cast<int*>(cache->d_table), d_refs, cache->n_seqs, cache->table_ld, cache->n_pages, r.words, d_moves, d_counts, (Bits64*)s,
                  (Bits64*)(s + r.mover), (int*)(s + r.holes), (int*)(s + r.movers)};
  hipStream_t st = static_cast<hipStream_t>(stream);
  const unsigned places = (unsigned)cache->n_seqs * cache->table_ld, pages = (unsigned)cache->n_pages, most = places > pages ? places : pages;
  if (most <= kNearMoves) {
    hipLaunchKernelGGL(compact_kernel, dim3(1), dim3(kSettle), 0, st, a);
    return from_hip(hipGetLastError());
  }
  hipLaunchKernelGGL(compact_bits_kernel, dim3((pages + 255) / 256), dim3(256), 0, st, a);
  if (hipGetLastError() != hipSuccess) return W4A32_ELAUNCH;
  if (r.words <= kWords) {
    hipLaunchKernelGGL(compact_both_kernel, dim3((most + kSettle - 1) / kSettle), dim3(kSettle), 0, st, a);
    return from_hip(hipGetLastError());
  }
  hipLaunchKernelGGL(compact_sums_kernel, dim3(1), dim3(kSettle), 0, st, a);
  if (hipGetLastError() != hipSuccess) return W4A32_ELAUNCH;
  hipLaunchKernelGGL(compact_apply_kernel, dim3((most + 255) / 256), dim3(256), 0, st, a);
  return from_hip(hipGetLastError());
}

}  // extern "C"
