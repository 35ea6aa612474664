// Log probabilities of given tokens, entropies and the most probable tokens of rows of logits.
//
// A wavefront takes kBlock logits of a row, 16 of each lane: their maximum m', with e = e^((z - m') / T) the sums of e and of
// e (m' - z), and how many of them come before the given token. The second launch joins a row's blocks,
//   S = sum S' e^((m' - m) / T),  W = sum (W' + S' (m - m')) e^((m' - m) / T),  log p = (z - m) / T - ln S,  H = ln S + W / (S T),
// all of whose terms are positive. Sums are f32 within a block and f64 over blocks. 1 / T goes into the exponents as two f32 terms: one
// alone is off by the same 2^-25 of every exponent, which would add up.
//
// The k most probable tokens: of the blocks' maxima the k-th largest bounds them from below, so only chunks (1 KB) of such blocks whose own maximum reaches
// it are read again, little more than k of them, and of their logits about k reach it; those are put in order by counting. Where more reach it than fit
// into LDS, the k-th largest itself is found by its bits, and of equal ones the first are taken. That holds while the blocks are a good deal more than k. With
// k blocks the bound is the least of their maxima, and with fewer there is none: then all chunks are read again, each logit that reaches the bound
// takes a place of the list by an atomic in LDS, and beyond 2048 of them the search by bits reads all of it four times more (64 rows of 32000: 16 us with the 31
// largest, 30 with 32, 61 with 50, of which the first launch is 5; of 65536 35 with 64 and 104 with 65; of 152064 18 with 20, 22 with 64 and 255 with 200).
//
// Memory bounds the first launch where rows are many (500 rows of 151936, f32, 304 MB: 48.5 us, 6.3 TB/s, read only, part of it from the cache in front; the
// second launch takes 5), instructions and latency where they are few: 64 rows of 152064 with their 20 largest, 9.4 us of the first launch, and 8.7 of
// the second, a chain of the ranks of 149 maxima (2 us), some 25 chunks read again (2.5), their logits' order (1.5) and barriers. Logits of 16 bits are half the
// bytes, but as many instructions: the same rows in bf16 42 and 9.0 us of the first launch, 45 and 18 of both.
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
  Part* part;        // [rows][blocks]
  float* chunk_max;  // [rows][blocks][chunks of one], where the most probable tokens are asked for
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
// are under way together; meanwhile() is done while they are. They pass the caches by: nobody reads all of the logits again (500 rows of 151936 in f32 50.3
// us against 55.4 of a pass among others, 64 rows with their 20 largest the same).
template <typename T, int kN>
struct Chunks {
  static constexpr int kWide = 16 / (int)sizeof(T), kChunk = 64 * kWide;
  float v[kN][kWide];
  bool wide;
  __device__ __forceinline__ int place(int i) const {
    const int lane = threadIdx.x & 63;
    return wide ? lane * kWide + i : i * 64 + lane;
  }
  template <typename Meanwhile>
  __device__ __forceinline__ void load(const T* row, const int (&base)[kN], int vocab, Meanwhile meanwhile) {
    const int lane = threadIdx.x & 63;
    wide = ((uintptr_t)row & 15) == 0 && vocab >= kWide;  // chunks that are not there read the row's first 16 bytes
#pragma unroll
    for (int c = 0; c < kN; ++c) wide = wide && (base[c] + kChunk <= vocab || base[c] >= vocab);
    if (wide) {
      u32x4 x[kN];
#pragma unroll
      for (int c = 0; c < kN; ++c) x[c] = __builtin_nontemporal_load((const W4_GLOBAL u32x4*)(row + (base[c] < vocab ? base[c] : 0)) + (base[c] < vocab ? lane : 0));
      meanwhile();
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
      meanwhile();
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

// Chunks' maxima from the lanes', to memory; returns their maximum. Lanes exchange what they have of the others' chunks, so that a lane has one chunk
// of a quad's, or a pair's, lanes, and only one value goes on from there.
template <int kCtrl>
__device__ __forceinline__ float from_lane(float x) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), kCtrl, 0xf, 0xf, true));
}
template <int kN>
__device__ __forceinline__ float of_all_chunks(const float (&tops)[kN], float* out) {
  static_assert(kN == 2 || kN == 4, "chunks of a block");
  const int lane = threadIdx.x & 63;
  auto half = [&](float even, float odd) {
    const bool is_odd = lane & 1;
    return fmaxf(is_odd ? odd : even, from_lane<0xb1>(is_odd ? even : odd));  // quad_perm 1, 0, 3, 2
  };
  float x = half(tops[0], tops[1]);
  if constexpr (kN == 4) {
    const float y = half(tops[2], tops[3]);
    const bool upper = lane & 2;
    x = fmaxf(upper ? y : x, from_lane<0x4e>(upper ? x : y));  // quad_perm 2, 3, 0, 1
  } else {
    x = fmaxf(x, from_lane<0x4e>(x));
  }
  x = fmaxf(x, from_lane<0x124>(x));  // row_ror 4, 8
  x = fmaxf(x, from_lane<0x128>(x));
  x = fmaxf(x, __shfl_xor(x, 16));
  x = fmaxf(x, __shfl_xor(x, 32));
  if (lane < kN) out[lane] = x;
  x = fmaxf(x, from_lane<0xb1>(x));
  if constexpr (kN == 4) x = fmaxf(x, from_lane<0x4e>(x));
  return __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(x)));
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
  x.load(row, base, a.vocab, [] {});
  const float mine = value_of<T>(row, known ? (int)token : 0);
  // Instructions bound this kernel where the logits are in the cache in front: one for the maximum of two values, one of each two for what is no number
  // (bits above those of infinity), and a comparison for the rank, whose sums are the scalar unit's.
  float tops[kN], top;
  int high = (int)0x80000000;
  unsigned low = 0;
#pragma unroll
  for (int c = 0; c < kN; ++c) {
    tops[c] = -INFINITY;
#pragma unroll
    for (int i = 0; i < kWide; ++i) {
      tops[c] = fmaxf(tops[c], x.v[c][i]);
      high = max(high, __float_as_int(x.v[c][i]));
      low = max(low, __float_as_uint(x.v[c][i]));
    }
  }
  const bool odd = high >= 0x7f800000 || low > 0xff800000u;
  int before = known ? 0 : -1;
  auto count = [&](auto comes_before) {
#pragma unroll
    for (int c = 0; c < kN; ++c)
#pragma unroll
      for (int i = 0; i < kWide; ++i) before += __popcll(__ballot(comes_before(x.v[c][i], base[c] + x.place(i))));
  };
  if (known) {
    if (token < base[0])
      count([&](float v, int) { return v > mine; });
    else if (token >= base[0] + kBlock)
      count([&](float v, int) { return v >= mine; });
    else
      count([&](float v, int at) { return v > mine || (v == mine && at < (int)token); });
  }
  if (a.top) {
    top = of_all_chunks(tops, a.chunk_max + ((size_t)r * a.blocks + block) * kN);
  } else {
    top = tops[0];
#pragma unroll
    for (int c = 1; c < kN; ++c) top = fmaxf(top, tops[c]);
    top = wave_max(top);
  }
  // the difference first: products of large logits would be off by their own rounding
  const float from = top == -INFINITY ? 0.0f : top;
  float sum = 0.0f, weighted = 0.0f;
#pragma unroll
  for (int c = 0; c < kN; ++c)
#pragma unroll
    for (int i = 0; i < kWide; ++i) {
      const float d = fminf(from - x.v[c][i], a.far), e = __builtin_amdgcn_exp2f(-__fmaf_rn(d, a.scale_low, d * a.scale));
      sum += e;
      weighted = __fmaf_rn(e, d, weighted);
    }
  sum = wave_sum(sum);
  weighted = wave_sum(weighted);
  if (__any(odd)) sum = NAN;
  if ((threadIdx.x & 63) == 0) a.part[(size_t)r * a.blocks + block] = Part{top, sum, weighted, before};
}

// Larger logits have larger keys, -0 is 0; -infinity has kNone.
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t u = __float_as_uint(x + 0.0f);
  return u >> 31 ? ~u : u | 0x80000000u;
}
constexpr uint32_t kNone = 0x007fffffu;
__device__ __forceinline__ float of_key(uint32_t k) { return __uint_as_float(k >> 31 ? k & 0x7fffffffu : ~k); }

// A row's sums from its blocks', relative to the row's maximum
struct Sums {
  double sum, weighted;
  int before;
  __device__ __forceinline__ void add(const Logprobs& a, float top, const Part& p) {
    before += p.before;
    if (p.top == -INFINITY) return;
    const double d = (double)top - p.top, e = exp(-d * a.inv_t);
    sum += p.sum * e;
    weighted += (p.weighted + p.sum * d) * e;
  }
  __device__ __forceinline__ void join_wave() {
    sum = wave_add(sum);
    weighted = wave_add(weighted);
    before = wave_sum(before);
  }
};
// What belongs to the given token, whose logit is x, and the entropy; none: no distribution
struct Given {
  bool known;
  float x;
};
template <typename T>
__device__ __forceinline__ Given given_of(const Logprobs& a, int r) {
  const int64_t token = a.tokens ? a.tokens[r] : -1;
  const bool known = token >= 0 && token < a.vocab;
  return {known, value_of<T>((const T*)a.logits + (size_t)r * a.ldl, known ? (int)token : 0)};
}
__device__ __forceinline__ void write(const Logprobs& a, int r, const Given& g, float top, const Sums& s, double norm, bool none) {
  if (a.entropy) a.entropy[r] = none ? NAN : (float)(norm + s.weighted / s.sum * a.inv_t);
  if (a.logprob) a.logprob[r] = none ? NAN : g.known ? (float)(((double)g.x - top) * a.inv_t - norm) : -INFINITY;
  if (a.rank) a.rank[r] = none || !g.known ? -1 : s.before;
}

// A wavefront per row
template <typename T>
__global__ __launch_bounds__(64) void rows_kernel(Logprobs a) {
  const int r = blockIdx.x, lane = threadIdx.x;
  const Part* parts = a.part + (size_t)r * a.blocks;
  const Part mine = lane < a.blocks ? parts[lane] : Part{-INFINITY, 0.0f, 0.0f, 0};  // all there is up to 64 blocks
  const Given given = given_of<T>(a, r);
  float top = mine.top;
  bool none = mine.sum != mine.sum;
  for (int i = lane + 64; i < a.blocks; i += 64) {
    top = fmaxf(top, parts[i].top);
    none |= parts[i].sum != parts[i].sum;
  }
  top = wave_max(top);
  none = __any(none) || top == -INFINITY;
  Sums s = {0.0, 0.0, 0};
  s.add(a, top, mine);
  for (int i = lane + 64; i < a.blocks; i += 64) s.add(a, top, parts[i]);
  s.join_wave();
  if (lane == 0) write(a, r, given, top, s, log(s.sum), none);
}

// How many of n larger ones each of n numbers at(i) has, none of which are alike, by all threads of the workgroup: done(i, how many) by one of them.
// A wavefront has a 16th of the numbers, one in each lane, and compares all with one after the other. ready(): by all threads, in front of the first done().
typedef unsigned long long Bits64;
__device__ __forceinline__ Bits64 of_two(uint32_t high, uint32_t low) { return __builtin_bit_cast(Bits64, u32x2{low, high}); }
template <typename At, typename Ready, typename Done>
__device__ __forceinline__ void rank_of_all(int n, At at, Ready ready, Done done) {
  constexpr int kWaves = kThreads / 64, kGroups = 4;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), per = (n + kWaves - 1) / kWaves;
  for (int j0 = 0; j0 < per; j0 += 64) {
    const int i = wave * per + j0 + lane, here = min(min(per, n - wave * per) - j0, 64);
    const Bits64 mine = lane < here ? at(i) : 0;
    const u32x2 halves = __builtin_bit_cast(u32x2, mine);
    int larger = 0;
    for (int g = 0; g < n; g += 64 * kGroups) {
      Bits64 with[kGroups];
#pragma unroll
      for (int x = 0; x < kGroups; ++x) with[x] = g + 64 * x + lane < n ? at(g + 64 * x + lane) : 0;
      for (int c = 0; c < here; ++c) {
        const Bits64 one = of_two((uint32_t)__builtin_amdgcn_readlane((int)halves[1], c), (uint32_t)__builtin_amdgcn_readlane((int)halves[0], c));
        int count = 0;
#pragma unroll
        for (int x = 0; x < kGroups; ++x) count += __popcll(__ballot(with[x] > one));
        if (lane == c) larger += count;
      }
    }
    if (j0 == 0) ready();
    if (lane < here) done(i, larger);
  }
}

// A workgroup per row. The sums' join, some f64 instructions long, is done while the blocks that are read again are under way, and its logarithm by one
// wavefront while the others put those in order.
template <typename T>
__global__ __launch_bounds__(kThreads) void top_kernel(Logprobs a) {
  __shared__ Sums sums[kThreads / 64];
  __shared__ float tops[kThreads / 64];
  __shared__ double norm;
  __shared__ uint32_t maxima[kMaxima];
  __shared__ unsigned list[2 * kList];  // keys, places; or 4096 counts
  __shared__ int runs[kMaxima];
  __shared__ float chunk_max[kThreads];
  __shared__ unsigned n_runs, n_list, state[2], in_wave[kThreads / 64];
  __shared__ uint32_t bound;
  const int r = blockIdx.x, tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), top = min(a.top, a.vocab);
  const T* logits = (const T*)a.logits + (size_t)r * a.ldl;
  int64_t* out_token = a.top_token + (size_t)r * a.top;
  float* out_logprob = a.top_logprob + (size_t)r * a.top;
  const Part* parts = a.part + (size_t)r * a.blocks;
  const Part mine = tid < a.blocks ? parts[tid] : Part{-INFINITY, 0.0f, 0.0f, 0};  // all there is up to kThreads blocks
  const bool last = wave == kThreads / 64 - 1;  // the wavefront that writes what is the row's
  Given given = {};
  if (last) given = given_of<T>(a, r);
  constexpr int kChunk = Chunks<T, 1>::kChunk, kChunks = kBlock / kChunk, kAhead = 4;
  const float* far_max = a.chunk_max + (size_t)r * a.blocks * kChunks;
  const bool near = a.blocks <= kThreads / kChunks;  // all of them have room
  if (near && tid < a.blocks * kChunks) chunk_max[tid] = far_max[tid];
  const int run = (a.blocks + kMaxima - 1) / kMaxima, count = (a.blocks + run - 1) / run;
  float most = mine.top;
  bool none = mine.sum != mine.sum;
  if (run > 1) {
    most = -INFINITY;
    for (int i = tid * run; i < min((tid + 1) * run, a.blocks); ++i) {
      most = fmaxf(most, parts[i].top);
      none |= parts[i].sum != parts[i].sum;
    }
  }
  maxima[tid] = key_of(most);
  const float in_wave_top = wave_max(most);
  if ((tid & 63) == 0) tops[wave] = in_wave_top;
  if (tid == 0) {
    n_runs = n_list = 0;
    bound = kNone + 1;
  }
  none = __syncthreads_or(none);
  float row_top = tops[0];
#pragma unroll
  for (int w = 1; w < kThreads / 64; ++w) row_top = fmaxf(row_top, tops[w]);
  if (none || row_top == -INFINITY) {
    if (tid == kThreads - 64) write(a, r, given, row_top, {0.0, 0.0, 0}, 0.0, true);
    for (int i = tid; i < a.top; i += kThreads) {
      out_token[i] = -1;
      out_logprob[i] = NAN;
    }
    return;
  }
  auto put = [&](unsigned at, uint32_t key, unsigned place) {
    out_token[at] = place;
    out_logprob[at] = (float)(((double)of_key(key) - row_top) * a.inv_t - norm);
  };
  // ---- the bound: the top-th largest maximum. Of maxima that are alike the first are taken, as of tokens ----
  rank_of_all(
      count, [&](int i) { return of_two(maxima[i], ~(unsigned)i); }, [] {},
      [&](int i, int at) {
        if (at >= top || maxima[i] <= kNone) return;
        runs[at] = i;
        atomicMax(&n_runs, (unsigned)at + 1);
        if (at == top - 1) bound = maxima[i];
      });
  __syncthreads();
  const uint32_t least = bound;
  // What of them is to be read again, by put_one(key, place): a wavefront has every 16th chunk, several of them at once. meanwhile(): once by each
  // wavefront
  const float floor = of_key(least);
  const int chunks = __builtin_amdgcn_readfirstlane((int)n_runs) * run * kChunks;
  auto each = [&](auto put_one, auto meanwhile) {
    bool again = false;
    for (int i0 = wave; i0 < chunks || !again; i0 += kThreads) {
      const int i = i0 + (kThreads / 64) * (tid & 63), block = i / kChunks;
      int chunk = -1;
      if (i < chunks) {
        const int at = run == 1 ? runs[block] : runs[block / run] * run + block % run;
        if (at < a.blocks) chunk = at * kChunks + i % kChunks;
      }
      if (chunk >= 0 && !((near ? chunk_max[chunk] : far_max[chunk]) >= floor)) chunk = -1;
      Bits64 left = __ballot(chunk >= 0);
      do {
        int base[kAhead];
#pragma unroll
        for (int c = 0; c < kAhead; ++c) {
          base[c] = left ? __builtin_amdgcn_readlane(chunk, __builtin_ctzll(left)) * kChunk : a.vocab;
          left &= left - 1;
        }
        Chunks<T, kAhead> x;
        x.load(logits, base, a.vocab, [&] {
          if (!again) meanwhile();
        });
        again = true;
#pragma unroll
        for (int c = 0; c < kAhead; ++c) {
          if (base[c] >= a.vocab) continue;
#pragma unroll
          for (int e = 0; e < Chunks<T, 1>::kWide; ++e) put_one(key_of(x.v[c][e]), (unsigned)(base[c] + x.place(e)));
        }
      } while (left);
    }
  };
  each(
      [&](uint32_t k, unsigned place) {
        if (k < least) return;
        const unsigned at = atomicAdd(&n_list, 1u);
        if (at < kList) {
          list[at] = k;
          list[kList + at] = place;
        }
      },
      [&] {
        Sums s = {0.0, 0.0, 0};
        s.add(a, row_top, mine);
        for (int i = tid + kThreads; i < a.blocks; i += kThreads) s.add(a, row_top, parts[i]);
        s.join_wave();
        if ((tid & 63) == 0) sums[wave] = s;
      });
  __syncthreads();
  const unsigned found = n_list;
  if (last) {
    Sums all = {0.0, 0.0, 0};
#pragma unroll
    for (int w = 0; w < kThreads / 64; ++w) {
      all.sum += sums[w].sum;
      all.weighted += sums[w].weighted;
      all.before += sums[w].before;
    }
    const double x = log(all.sum);
    if (tid == kThreads - 64) {
      norm = x;
      write(a, r, given, row_top, all, x, false);
    }
  }
  for (unsigned i = min(found, (unsigned)top) + tid; i < (unsigned)a.top; i += kThreads) {
    out_token[i] = -1;
    out_logprob[i] = -INFINITY;
  }
  auto order = [&](int n) {  // writes the first of the list's n
    rank_of_all(
        n, [&](int i) { return of_two(list[i], ~list[kList + i]); }, [] { __syncthreads(); },  // the norm
        [&](int i, int at) {
          if (at < top) put((unsigned)at, list[i], list[kList + i]);
        });
  };
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
    }, [] {});
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
  }, [] {});
  __syncthreads();
  const unsigned larger = n_list;
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
  total = (size_t)rows * blocks * (sizeof(Part) + (top ? kBlock / Chunks<float, 1>::kChunk * sizeof(float) : 0));
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
                   v->ldl, v->top, blocks, inv_t, (float)scale, (float)(scale - (double)(float)scale), (float)(300.0 / scale), static_cast<Part*>(d_scratch),
                   reinterpret_cast<float*>(static_cast<Part*>(d_scratch) + (size_t)v->rows * blocks)};
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (v->dtype == W4A32_CACHE_F32) return launch<float>(a, s);
  if (v->dtype == W4A32_CACHE_F16) return launch<_Float16>(a, s);
  return launch<__bf16>(a, s);
}

}  // extern "C"
