// Log probabilities of given tokens, entropies and the most probable tokens of rows of logits.
//
// A wavefront takes kBlock logits of a row, 16 of each lane: their maximum m', with e = e^((z - m') / T) the sums of e and of
// e (m' - z), and how many of them come before the given token. The second launch joins a row's blocks,
//   S = sum S' e^((m' - m) / T),  W = sum (W' + S' (m - m')) e^((m' - m) / T),  log p = (z - m) / T - ln S,  H = ln S + W / (S T),
// all of whose terms are positive. Sums are f32 within a block and f64 over blocks. 1 / T goes into the exponents as two f32 terms: one
// alone is off by the same 2^-25 of every exponent, which would add up.
//
// The k most probable tokens: of the blocks' maxima the k-th largest bounds them from below, so only blocks whose maximum reaches it
// are read again, about k of them, and of their logits about k reach it; those are put in order by counting. Where many are alike and do
// not fit into LDS, the k-th largest itself is found by its bits, and of equal ones the first are taken.
//
// Memory bounds the first launch where rows are many (500 rows of 151936, f32, 304 MB: 52 us, 5.6 TB/s, read only; the second launch takes 5), latency where
// they are few: 64 rows of 152064 with their 20 largest, 11 us of the first launch, which finds the logits in the cache in front, and 9.8 of the second, a chain of
// the sums' join, the ranks of 149 maxima, 20 blocks read again and the order of some 25 logits.
#include <type_traits>

#include "w4a32_decoder.h"
#include "w4a32_internal.h"
#include "w4a32_paged.h"
#include "w4a32_wave.h"

namespace w4 {
namespace {
inline bool aligned(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

constexpr int kBlock = 1024;
constexpr int kThreads = 1024;   // of the launch that finds the most probable tokens
constexpr int kMaxima = 1024;    // blocks, or runs of them, whose maxima are compared
constexpr int kList = 2048;      // logits that are put in order by counting
constexpr int kMostTop = 1024;
// Rows from which on those of the two launches meet in an XCD's L2 (24 rows of 152064 with their 20 largest: the same, 48 18.5 us against 19.0, 200 32.3
// against 32.9)
constexpr int kXcds = 8, kApart = 32;

struct Part {
  float top, sum, weighted;  // sum is NaN where a logit is NaN or +infinity
  int before;
};
struct Logprobs {
  const void* logits;
  const int64_t* tokens;
  float* logprob;
  int* rank;
  float* entropy;
  int64_t* top_token;
  float* top_logprob;
  int rows, vocab, ldl, top, blocks;
  double inv_t;
  float scale, scale_low;  // log2(e) / T
  float far;               // a difference of logits that leaves nothing, and whose products with these are finite
  Part* part;  // [rows][blocks]
};

template <typename T>
__device__ __forceinline__ float value_of(const void* row, int i) {
  if constexpr (sizeof(T) == 4) return load_global<float>((const float*)row + i);
  const uint16_t h = load_global<uint16_t>((const uint16_t*)row + i);
  if constexpr (std::is_same<T, __bf16>::value) return __uint_as_float((uint32_t)h << 16);
  return (float)__builtin_bit_cast(_Float16, h);
}

// A lane's logits of kChunks chunks of 64 times 16 bytes that begin at base[c] (those from the row's end on: none), -infinity behind the row's end,
// and their places. Bases are the same for all lanes. Rows may lie off 16 bytes: one branch for all chunks, so that their loads
// are under way together.
template <typename T, int kN>
struct Chunks {
  static constexpr int kWide = 16 / (int)sizeof(T), kChunk = 64 * kWide;
  float v[kN][kWide];
  bool wide;
  __device__ __forceinline__ int place(int i) const {
    const int lane = threadIdx.x & 63;
    return wide ? lane * kWide + i : i * 64 + lane;
  }
  __device__ __forceinline__ void load(const T* row, const int (&base)[kN], int vocab) {
    const int lane = threadIdx.x & 63;
    wide = ((uintptr_t)row & 15) == 0;
#pragma unroll
    for (int c = 0; c < kN; ++c) wide = wide && (base[c] + kChunk <= vocab || base[c] >= vocab);
    if (wide) {
      u32x4 x[kN];
#pragma unroll
      for (int c = 0; c < kN; ++c) x[c] = load_global<u32x4>((const u32x4*)(row + (base[c] < vocab ? base[c] : 0)) + (base[c] < vocab ? lane : 0));
#pragma unroll
      for (int c = 0; c < kN; ++c)
#pragma unroll
        for (int e = 0; e < kWide; ++e) {
          float f;
          if constexpr (sizeof(T) == 4) {
            f = __uint_as_float(x[c][e]);
          } else {
            const uint32_t h = e & 1 ? x[c][e / 2] >> 16 : x[c][e / 2] & 0xffffu;
            if constexpr (std::is_same<T, __bf16>::value)
              f = __uint_as_float(h << 16);
            else
              f = (float)__builtin_bit_cast(_Float16, (uint16_t)h);
          }
          v[c][e] = base[c] < vocab ? f : -INFINITY;
        }
    } else {
#pragma unroll
      for (int c = 0; c < kN; ++c)
#pragma unroll
        for (int i = 0; i < kWide; ++i) {
          const int at = base[c] + i * 64 + lane;
          const float x = value_of<T>(row, min(at, vocab - 1));
          v[c][i] = at < vocab ? x : -INFINITY;
        }
    }
  }
};

// By moves within the register file, as wave_add(double): six shuffles through LDS take 600 clocks
template <int kCtrl, int kRowMask>
__device__ __forceinline__ int moved(int x) {
  return __builtin_amdgcn_update_dpp(0, x, kCtrl, kRowMask, 0xf, false);
}
template <int kCtrl, int kRowMask>
__device__ __forceinline__ float moved(float x) {
  return __int_as_float(moved<kCtrl, kRowMask>(__float_as_int(x)));
}
template <typename T>
__device__ __forceinline__ T wave_sum(T x) {
  x += moved<0x111, 0xf>(x);  // row_shr 1, 2, 4, 8
  x += moved<0x112, 0xf>(x);
  x += moved<0x114, 0xf>(x);
  x += moved<0x118, 0xf>(x);
  x += moved<0x142, 0xa>(x);  // row_bcast 15, 31
  x += moved<0x143, 0xc>(x);
  return __builtin_bit_cast(T, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), 63));
}

// A wavefront per block
template <typename T>
__global__ __launch_bounds__(256) void blocks_kernel(Logprobs a, int groups, bool apart) {
  // kXcds rows go on side by side where `apart`: workgroups of numbers kXcds apart are one XCD's, and so are a row's here and in the next launch
  const int unit = apart ? blockIdx.x / kXcds : blockIdx.x, of = unit / groups, r = apart ? of * kXcds + blockIdx.x % kXcds : of;
  const int block = (unit - of * groups) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (block >= a.blocks || r >= a.rows) return;
  const T* row = (const T*)a.logits + (size_t)r * a.ldl;
  const int64_t token = a.tokens ? a.tokens[r] : -1;
  const bool known = token >= 0 && token < a.vocab;
  constexpr int kChunk = Chunks<T, 1>::kChunk, kN = kBlock / kChunk, kWide = Chunks<T, 1>::kWide;
  int base[kN];
#pragma unroll
  for (int c = 0; c < kN; ++c) base[c] = block * kBlock + c * kChunk;
  Chunks<T, kN> x;
  x.load(row, base, a.vocab);
  const float mine = value_of<T>(row, known ? (int)token : 0);
  float top = -INFINITY;
  bool odd = false;
  int before = 0;
#pragma unroll
  for (int c = 0; c < kN; ++c)
#pragma unroll
    for (int i = 0; i < kWide; ++i) {
      const float v = x.v[c][i];
      top = fmaxf(top, v);
      odd |= !(v < INFINITY);
      before += v > mine || (v == mine && base[c] + x.place(i) < (int)token);
    }
  top = wave_max(top);
  // the difference first: products of large logits would be off by their own rounding
  const float from = top == -INFINITY ? 0.0f : top;
  float sum = 0.0f, weighted = 0.0f;
#pragma unroll
  for (int c = 0; c < kN; ++c)
#pragma unroll
    for (int i = 0; i < kWide; ++i) {
      const float d = fminf(from - x.v[c][i], a.far), e = __builtin_amdgcn_exp2f(-__fmaf_rn(d, a.scale_low, d * a.scale));
      sum += e;
      weighted += e > 0.0f ? e * d : 0.0f;
    }
  sum = wave_sum(sum);
  weighted = wave_sum(weighted);
  before = wave_sum(before);
  if (__any(odd)) sum = NAN;
  if ((threadIdx.x & 63) == 0) a.part[(size_t)r * a.blocks + block] = Part{top, sum, weighted, known ? before : -1};
}

// Larger logits have larger keys, -0 is 0; -infinity has kNone.
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t u = __float_as_uint(x + 0.0f);
  return u >> 31 ? ~u : u | 0x80000000u;
}
constexpr uint32_t kNone = 0x007fffffu;
__device__ __forceinline__ float of_key(uint32_t k) { return __uint_as_float(k >> 31 ? k & 0x7fffffffu : ~k); }

template <int kN>
struct Shared {
  double sum[kN / 64], weighted[kN / 64];
  float top[kN / 64];
  int before[kN / 64];
};
struct Row {
  double norm;  // ln S
  float top;
  float mine;   // maximum of this thread's first block
  bool none;    // no distribution
};
// A row's sums from its blocks', by all threads. The last wavefront writes what belongs to the given token, and the entropy.
template <typename T, int kN>
__device__ __forceinline__ Row join(const Logprobs& a, int r, Shared<kN>& sh) {
  const Part* parts = a.part + (size_t)r * a.blocks;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const Part mine = (int)threadIdx.x < a.blocks ? parts[threadIdx.x] : Part{-INFINITY, 0.0f, 0.0f, 0};  // all there is up to kN blocks
  const bool writes = threadIdx.x == kN - 64;
  const int64_t token = writes && a.tokens ? a.tokens[r] : -1;
  const bool known = token >= 0 && token < a.vocab;
  const float x = writes ? value_of<T>((const T*)a.logits + (size_t)r * a.ldl, known ? (int)token : 0) : 0.0f;
  float top = mine.top;
  for (int i = threadIdx.x + kN; i < a.blocks; i += kN) top = fmaxf(top, parts[i].top);
  top = wave_max(top);
  if constexpr (kN > 64) {
    if (lane == 0) sh.top[wave] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kN / 64; ++w) top = fmaxf(top, sh.top[w]);
  }
  double sum = 0.0, weighted = 0.0;
  int before = 0;
  auto add = [&](const Part& p) {
    before += p.before;
    if (p.top == -INFINITY && p.sum == p.sum) return;
    const double d = (double)top - p.top, e = exp(-d * a.inv_t);
    sum += p.sum * e;
    weighted += (p.weighted + p.sum * d) * e;
  };
  add(mine);
  for (int i = threadIdx.x + kN; i < a.blocks; i += kN) add(parts[i]);
  sum = wave_add(sum);
  weighted = wave_add(weighted);
  before = wave_sum(before);
  if constexpr (kN > 64) {
    if (lane == 0) {
      sh.sum[wave] = sum;
      sh.weighted[wave] = weighted;
      sh.before[wave] = before;
    }
    __syncthreads();
    sum = weighted = 0.0;
    before = 0;
#pragma unroll
    for (int w = 0; w < kN / 64; ++w) {
      sum += sh.sum[w];
      weighted += sh.weighted[w];
      before += sh.before[w];
    }
  }
  Row row;
  row.top = top;
  row.mine = mine.top;
  row.none = !(sum > 0.0);
  row.norm = log(sum);
  if (writes) {
    if (a.entropy) a.entropy[r] = row.none ? NAN : (float)(row.norm + weighted / sum * a.inv_t);
    if (a.logprob) a.logprob[r] = row.none ? NAN : known ? (float)(((double)x - top) * a.inv_t - row.norm) : -INFINITY;
    if (a.rank) a.rank[r] = row.none || !known ? -1 : before;
  }
  return row;
}

// A wavefront per row
template <typename T>
__global__ __launch_bounds__(64) void rows_kernel(Logprobs a) {
  Shared<64> sh;
  join<T, 64>(a, blockIdx.x, sh);
}

// A workgroup per row
template <typename T>
__global__ __launch_bounds__(kThreads) void top_kernel(Logprobs a) {
  __shared__ Shared<kThreads> sh;
  __shared__ uint32_t maxima[kMaxima];
  __shared__ unsigned list[2 * kList];  // keys, places; or 4096 counts
  __shared__ int runs[kMaxima], ranks[kMaxima];
  __shared__ unsigned n_runs, n_list, state[2], in_wave[kThreads / 64];
  __shared__ uint32_t bound;
  const int r = blockIdx.x, tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), top = min(a.top, a.vocab);
  const T* logits = (const T*)a.logits + (size_t)r * a.ldl;
  int64_t* out_token = a.top_token + (size_t)r * a.top;
  float* out_logprob = a.top_logprob + (size_t)r * a.top;
  const Row row = join<T, kThreads>(a, r, sh);
  if (row.none) {
    for (int i = tid; i < a.top; i += kThreads) {
      out_token[i] = -1;
      out_logprob[i] = NAN;
    }
    return;
  }
  auto put = [&](unsigned at, uint32_t key, unsigned place) {
    out_token[at] = place;
    out_logprob[at] = (float)(((double)of_key(key) - row.top) * a.inv_t - row.norm);
  };
  // ---- the bound: the top-th largest maximum ----
  const Part* parts = a.part + (size_t)r * a.blocks;
  const int run = (a.blocks + kMaxima - 1) / kMaxima, count = (a.blocks + run - 1) / run;
  float most = row.mine;
  if (run > 1 && tid < count) {
    most = -INFINITY;
    for (int i = tid * run; i < min((tid + 1) * run, a.blocks); ++i) most = fmaxf(most, parts[i].top);
  }
  maxima[tid] = key_of(most);
  if (tid == 0) {
    n_runs = n_list = 0;
    bound = kNone + 1;
  }
  ranks[tid] = 0;
  __syncthreads();
  // How many of n come before each, to ranks: n threads have the i-th of them, and what it is compared with is dealt to as many more as there are
  auto rank = [&](int n, auto before) {
    const int slices = max(kThreads / n, 1), each = (n + slices - 1) / slices;
    for (int x = tid; x < n * slices; x += kThreads) {
      const int slice = x / n, i = x - slice * n, end = min((slice + 1) * each, n);
      int count = 0;
#pragma unroll 8
      for (int j = slice * each; j < end; ++j) count += before(j, i);
      if (slices == 1)
        ranks[i] = count;
      else if (count)
        atomicAdd(&ranks[i], count);
    }
    __syncthreads();
  };
  rank(count, [&](int j, int i) { return maxima[j] > maxima[i] || (maxima[j] == maxima[i] && j < i); });
  if (tid < count && ranks[tid] == top - 1 && maxima[tid] > kNone) bound = maxima[tid];
  __syncthreads();
  const uint32_t least = bound;
  ranks[tid] = 0;
  if (tid < count && maxima[tid] >= least) runs[atomicAdd(&n_runs, 1u)] = tid;
  __syncthreads();
  // What of them is to be read again, by put_one(key, place): a wavefront has every 16th chunk, several of them at once
  constexpr int kChunk = Chunks<T, 1>::kChunk, kChunks = kBlock / kChunk, kAhead = sizeof(T) == 4 ? 8 : 4;
  const float floor = of_key(least);
  const int chunks = __builtin_amdgcn_readfirstlane((int)n_runs) * run * kChunks;
  auto each = [&](auto put_one) {
    for (int i0 = wave; i0 < chunks; i0 += kAhead * (kThreads / 64)) {
      int base[kAhead];
#pragma unroll
      for (int c = 0; c < kAhead; ++c) {
        const int i = i0 + c * (kThreads / 64), block = i / kChunks;
        base[c] = a.vocab;
        if (i < chunks) {
          const int at = run == 1 ? runs[block] : runs[block / run] * run + block % run;
          base[c] = min(__builtin_amdgcn_readfirstlane(at) * kBlock + i % kChunks * kChunk, a.vocab);
        }
      }
      Chunks<T, kAhead> x;
      x.load(logits, base, a.vocab);
#pragma unroll
      for (int c = 0; c < kAhead; ++c) {
        float most = x.v[c][0];
#pragma unroll
        for (int e = 1; e < Chunks<T, 1>::kWide; ++e) most = fmaxf(most, x.v[c][e]);
        if (!__any(most >= floor)) continue;  // most chunks
#pragma unroll
        for (int e = 0; e < Chunks<T, 1>::kWide; ++e) put_one(key_of(x.v[c][e]), (unsigned)(base[c] + x.place(e)));
      }
    }
  };
  each([&](uint32_t k, unsigned place) {
    if (k < least) return;
    const unsigned at = atomicAdd(&n_list, 1u);
    if (at < kList) {
      list[at] = k;
      list[kList + at] = place;
    }
  });
  __syncthreads();
  const unsigned found = n_list;
  auto order = [&](int n) {  // writes the first of the list's n
    if (n <= kMaxima) {
      rank(n, [&](int j, int i) { return list[j] > list[i] || (list[j] == list[i] && list[kList + j] < list[kList + i]); });
      if (tid < n && ranks[tid] < top) put((unsigned)ranks[tid], list[tid], list[kList + tid]);
      return;
    }
    for (int i = tid; i < n; i += kThreads) {
      const uint32_t k = list[i];
      const unsigned place = list[kList + i];
      int first = 0;
#pragma unroll 8
      for (int j = 0; j < n; ++j) first += list[j] > k || (list[j] == k && list[kList + j] < place);
      if (first < top) put((unsigned)first, k, place);
    }
  };
  for (unsigned i = min(found, (unsigned)top) + tid; i < (unsigned)a.top; i += kThreads) {
    out_token[i] = -1;
    out_logprob[i] = -INFINITY;
  }
  if (found <= kList) {
    order((int)found);
    return;
  }
  // ---- too many: the top-th largest key, 12, 10 and 10 bits at a time ----
  uint32_t prefix = 0, mask = 0;
  unsigned want = (unsigned)top;
  for (int bits = 12, shift = 20;; bits = 10, shift -= 10) {
    __syncthreads();
    for (int i = tid; i < 1 << bits; i += kThreads) list[i] = 0;
    __syncthreads();
    each([&](uint32_t k, unsigned) {
      if (k >= least && (k & mask) == prefix) atomicAdd(&list[k >> shift & ((1u << bits) - 1)], 1u);
    });
    __syncthreads();
    const int digits = (1 << bits) / kThreads, high = (1 << bits) - 1 - tid * digits;  // thread i: the i-th `digits` from the largest on
    unsigned sum = 0, all;
    for (int i = 0; i < digits; ++i) sum += list[high - i];
    const unsigned upto = paged::block_scan<kThreads>(sum, in_wave, all);
    unsigned above = upto - sum;
    if (above < want && upto >= want)
      for (int i = 0; i < digits; ++i) {
        const unsigned h = list[high - i];
        if (above < want && above + h >= want) {
          state[0] = (unsigned)(high - i);
          state[1] = want - above;
        }
        above += h;
      }
    __syncthreads();
    prefix |= state[0] << shift;
    want = state[1];
    mask |= ((1u << bits) - 1) << shift;
    if (shift == 0) break;
  }
  // the larger ones, fewer than top, and the first `want` of those that have this key, in the row's order
  if (tid == 0) n_list = 0;
  __syncthreads();
  each([&](uint32_t k, unsigned place) {
    if (k <= prefix) return;
    const unsigned at = atomicAdd(&n_list, 1u);
    list[at] = k;
    list[kList + at] = place;
  });
  __syncthreads();
  const unsigned larger = n_list;
  ranks[tid] = 0;
  __syncthreads();
  if (larger) order((int)larger);
  unsigned taken = 0;
  for (int block = 0; block < a.blocks && taken < want; ++block) {
    if (maxima[block / run] < prefix) continue;
    static_assert(kThreads == kBlock, "a thread per logit");
    const int at = block * kBlock + tid;
    const bool tie = at < a.vocab && key_of(value_of<T>(logits, min(at, a.vocab - 1))) == prefix;
    unsigned all;
    const unsigned upto = paged::block_scan<kThreads>(tie, in_wave, all);
    if (tie && taken + upto <= want) put(larger + taken + upto - 1, prefix, (unsigned)at);
    taken += all;
  }
}

bool layout_of(int rows, int vocab, int top, int& blocks, size_t& total) {
  if (rows < 1 || vocab < 1 || top < 0 || rows >= 1 << 24 || vocab >= 1 << 30 || top > kMostTop) return false;
  blocks = (vocab + kBlock - 1) / kBlock;
  // a launch has less than 2^32 threads: 256 of four blocks, 1024 of a row
  if (((long long)rows + kXcds) * ((blocks + 3) / 4) >= 1ll << 24 || (top && rows >= 1 << 22)) return false;
  total = (size_t)rows * blocks * sizeof(Part);
  return true;
}

template <typename T>
int launch(const Logprobs& a, hipStream_t s) {
  const int groups = (a.blocks + 3) / 4;
  const bool apart = a.top && a.rows >= kApart;
  const unsigned rows = apart ? (unsigned)(a.rows + kXcds - 1) / kXcds * kXcds : (unsigned)a.rows;
  hipLaunchKernelGGL((blocks_kernel<T>), dim3(rows * groups), dim3(256), 0, s, a, groups, apart);
  if (hipGetLastError() != hipSuccess) return W4A32_ELAUNCH;
  if (a.top)
    hipLaunchKernelGGL((top_kernel<T>), dim3((unsigned)a.rows), dim3(kThreads), 0, s, a);
  else
    hipLaunchKernelGGL((rows_kernel<T>), dim3((unsigned)a.rows), dim3(64), 0, s, a);
  return hipGetLastError() == hipSuccess ? W4A32_OK : W4A32_ELAUNCH;
}
}  // namespace
}  // namespace w4

using namespace w4;

extern "C" {

size_t w4a32_op_token_logprobs_scratch_bytes(int rows, int vocab, int top) {
  int blocks;
  size_t total;
  return layout_of(rows, vocab, top, blocks, total) ? total : 0;
}

int w4a32_op_token_logprobs(const w4a32_logprobs_args* v, void* d_scratch, size_t scratch_bytes, void* stream) {
  if (!v || !v->d_logits || !d_scratch || v->rows < 1 || v->vocab < 1 || v->top < 0 || v->ldl < v->vocab) return W4A32_EINVAL;
  if (v->dtype < W4A32_CACHE_F32 || v->dtype > W4A32_CACHE_BF16) return W4A32_EINVAL;
  if (!(v->temperature >= 1e-30) || v->temperature > 1e30) return W4A32_EINVAL;
  if ((v->d_logprob || v->d_rank) && !v->d_tokens) return W4A32_EINVAL;
  if (v->top && (!v->d_top_token || !v->d_top_logprob)) return W4A32_EINVAL;
  if (!aligned(v->d_logits, v->dtype == W4A32_CACHE_F32 ? 4 : 2) || !aligned(v->d_tokens, 8) || !aligned(v->d_logprob, 4) || !aligned(v->d_rank, 4) ||
      !aligned(v->d_entropy, 4) || !aligned(v->d_top_token, 8) || !aligned(v->d_top_logprob, 4) || !aligned(d_scratch, 16))
    return W4A32_EINVAL;
  int blocks;
  size_t total;
  if (!layout_of(v->rows, v->vocab, v->top, blocks, total)) return W4A32_ESHAPE;
  if (scratch_bytes < total) return W4A32_EINVAL;
  const double inv_t = 1.0 / v->temperature, scale = inv_t * 1.4426950408889634074;
  const Logprobs a{v->d_logits, v->d_tokens, v->d_logprob, v->d_rank, v->d_entropy, v->d_top_token, v->d_top_logprob, v->rows, v->vocab,
                   v->ldl, v->top, blocks, inv_t, (float)scale, (float)(scale - (double)(float)scale), (float)(300.0 / scale), static_cast<Part*>(d_scratch)};
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (v->dtype == W4A32_CACHE_F32) return launch<float>(a, s);
  if (v->dtype == W4A32_CACHE_F16) return launch<_Float16>(a, s);
  return launch<__bf16>(a, s);
}

}  // extern "C"
