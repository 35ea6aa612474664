// Verification of drafted tokens against the target's logits and given random numbers.
//
// A row of logits is cut into segments of kSegment. The first launch takes every segment of every row once: its maximum and
// the sum of its exponentials, relative to that maximum. The second combines them per row, tests the drafted tokens of a
// sequence and, where one was refused, adds up max(p - q, 0) over the segments of its row; the third finds the segment and
// then the index that the given number falls on.
//
// Exponentials and sums are f64: an f64 sum or product takes as long as an f32 one here, an exponential 16 of them, and so the
// first launch stays near what memory gives: 48 sequences of 2 to 8 rows of 152064 logits, target and draft (270 MB): 57 us, 4.7 TB/s.
// The second, which reads the refused rows again, takes 22 there and the third 8; for one sequence of five rows the three
// take 4, 6 and 5 us, all of it latency. In f32 the sums' rounding would decide which token a number falls on whenever it
// lies within 1e-7 of a border, as one of 150000 tokens' borders often does.
#include "w4a32_internal.h"
#include "w4a32_decoder.h"

namespace w4 {
namespace {
inline bool aligned(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

constexpr int kSegment = 4096;  // logits of a segment: 16 of each thread, all requested at once
constexpr int kEach = kSegment / 256;
constexpr int kChoose = 1024;   // threads of the third launch: what takes time is their f64 arithmetic (with 256: 11 us for 48 sequences, not 8)
constexpr int kTestWaves = 8;   // wavefronts of the second launch: rows of a sequence that are tested at once

struct Part {
  double sum;
  float top;
  int at;  // greedy: index of the maximum
};
struct Found {  // what the second launch leaves for the third
  double rp, rq;  // one over the sums of the row's exponentials, target and draft
  float mp, mq;
  int count, refused, row;
};
struct Verify {
  const float *logits, *draft;
  const int* row_start;
  const int64_t* tokens;
  const float *uniform, *choice;
  int* count;
  int64_t* next;
  int* len;
  int rows, max_rows, n_seqs, vocab, ldl, ldd, segs;
  double inv_t;  // 0: greedy
  Part *p, *q;   // [rows][segs]
  double* left;  // [n_seqs][segs]: max(p - q, 0) of the row that refused
  Found* found;  // [n_seqs]
};

// e^x for x <= 0 (NaN stays NaN): 2^k times the Taylor polynomial of degree 10 on |r| <= ln 2 / 2, 3e-13 relative.
__device__ __forceinline__ double exp_neg(double x) {
  if (x < -700.0) return 0.0;
  const double k = __builtin_rint(x * 1.4426950408889634074);
  const double r = __builtin_fma(k, -0.69314718055994530942, x);
  double y = 1.0 / 3628800;
  y = __builtin_fma(y, r, 1.0 / 362880);
  y = __builtin_fma(y, r, 1.0 / 40320);
  y = __builtin_fma(y, r, 1.0 / 5040);
  y = __builtin_fma(y, r, 1.0 / 720);
  y = __builtin_fma(y, r, 1.0 / 120);
  y = __builtin_fma(y, r, 1.0 / 24);
  y = __builtin_fma(y, r, 1.0 / 6);
  y = __builtin_fma(y, r, 0.5);
  y = __builtin_fma(y, r, 1.0);
  y = __builtin_fma(y, r, 1.0);
  return __builtin_amdgcn_ldexp(y, (int)k);
}

// e^((l - top) / t) with c = log2(e) / t, for sums alone, 7e-12 relative: k from the low bits of a sum that has no bits behind the
// point, 2^f by the Taylor polynomial of degree 9 on |f| <= 1/2, and k added to the exponent. At least 2^-1000 where it is less
// (-infinity, NaN). The difference first: c l - c top would be off by the rounding of c top, which a low temperature makes large.
__device__ __forceinline__ double exp_sum(float l, double c, double top) {
  constexpr double kMagic = 6755399441055744.0;  // 1.5 * 2^52
  const double y = fmax(((double)l - top) * c, -1000.0);
  const double t = y + kMagic, f = y - (t - kMagic);
  constexpr double L = 0.69314718055994530942;
  constexpr double c1 = L, c2 = c1 * L / 2, c3 = c2 * L / 3, c4 = c3 * L / 4, c5 = c4 * L / 5, c6 = c5 * L / 6, c7 = c6 * L / 7,
                   c8 = c7 * L / 8, c9 = c8 * L / 9;
  double p = c9;
  p = __builtin_fma(p, f, c8);
  p = __builtin_fma(p, f, c7);
  p = __builtin_fma(p, f, c6);
  p = __builtin_fma(p, f, c5);
  p = __builtin_fma(p, f, c4);
  p = __builtin_fma(p, f, c3);
  p = __builtin_fma(p, f, c2);
  p = __builtin_fma(p, f, c1);
  p = __builtin_fma(p, f, 1.0);
  const unsigned long long bits = __builtin_bit_cast(unsigned long long, p);
  const unsigned k = (unsigned)__builtin_bit_cast(unsigned long long, t);
  return __builtin_bit_cast(double, (bits & 0xffffffffull) | (unsigned long long)((unsigned)(bits >> 32) + (k << 20)) << 32);
}

struct Rows {
  int r0, n;
};
__device__ __forceinline__ Rows rows_of(const Verify& a, int b) {
  Rows s;
  s.r0 = min(max(a.row_start[b], 0), a.rows);
  s.n = min(min(max(a.row_start[b + 1], s.r0), a.rows) - s.r0, a.max_rows);
  return s;
}

// Sums, maxima and minima over a wavefront by moves within the register file; scan: up to this lane.
template <int kCtrl, int kRowMask>
__device__ __forceinline__ double moved(double x) {  // 0 where no lane is
  const unsigned long long b = __builtin_bit_cast(unsigned long long, x);
  const unsigned lo = (unsigned)__builtin_amdgcn_update_dpp(0, (int)(unsigned)b, kCtrl, kRowMask, 0xf, false);
  const unsigned hi = (unsigned)__builtin_amdgcn_update_dpp(0, (int)(unsigned)(b >> 32), kCtrl, kRowMask, 0xf, false);
  return __builtin_bit_cast(double, (unsigned long long)hi << 32 | lo);
}
__device__ __forceinline__ double wave_scan(double x) {
  x += moved<0x111, 0xf>(x);  // row_shr 1, 2, 4, 8
  x += moved<0x112, 0xf>(x);
  x += moved<0x114, 0xf>(x);
  x += moved<0x118, 0xf>(x);
  x += moved<0x142, 0xa>(x);  // row_bcast 15, 31
  x += moved<0x143, 0xc>(x);
  return x;
}
__device__ __forceinline__ double of_lane(double x, int lane) {
  const unsigned long long b = __builtin_bit_cast(unsigned long long, x);
  const unsigned lo = (unsigned)__builtin_amdgcn_readlane((int)(unsigned)b, lane), hi = (unsigned)__builtin_amdgcn_readlane((int)(unsigned)(b >> 32), lane);
  return __builtin_bit_cast(double, (unsigned long long)hi << 32 | lo);
}
__device__ __forceinline__ double wave_add(double x) { return of_lane(wave_scan(x), 63); }
template <int kCtrl, int kRowMask>
__device__ __forceinline__ float most(float x) {
  const int y = __builtin_amdgcn_update_dpp((int)0xff800000, __float_as_int(x), kCtrl, kRowMask, 0xf, false);  // -infinity where no lane is
  return fmaxf(x, __int_as_float(y));
}
__device__ __forceinline__ float wave_max(float x) {
  x = most<0x111, 0xf>(x);
  x = most<0x112, 0xf>(x);
  x = most<0x114, 0xf>(x);
  x = most<0x118, 0xf>(x);
  x = most<0x142, 0xa>(x);
  x = most<0x143, 0xc>(x);
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), 63));
}

// blockIdx: segment, row, target or draft
template <bool kGreedy>
__global__ __launch_bounds__(256) void stats_kernel(Verify a) {
  __shared__ float tops[4];
  __shared__ double sums[4];
  __shared__ int ats[4];
  const int seg = blockIdx.x % a.segs, r = blockIdx.x / a.segs, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const bool of_draft = blockIdx.y != 0;
  int before = 0;
  for (int b = 0; b < a.n_seqs; b += 64) before += __popcll(__ballot(b + lane < a.n_seqs && a.row_start[b + lane] <= r));
  if (before == 0) return;
  const Rows s = rows_of(a, before - 1);
  if (r - s.r0 >= s.n - (of_draft ? 1 : 0)) return;
  const float* x = of_draft ? a.draft + (size_t)r * a.ldd : a.logits + (size_t)r * a.ldl;
  const int base = seg * kSegment;
  float v[kEach];
  // four values of a thread together, 1024 apart
  if (((uintptr_t)x & 15) == 0 && base + kSegment <= a.vocab) {
#pragma unroll
    for (int i = 0; i < kEach; i += 4) {
      typedef float f4 __attribute__((ext_vector_type(4)));
      const f4 w = load_global<f4>(x + base + i * 256 + 4 * (int)threadIdx.x);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[i + e] = w[e];
    }
  } else {
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const int at = base + (i & ~3) * 256 + 4 * (int)threadIdx.x + (i & 3);
      v[i] = at < a.vocab ? load_global<float>(x + at) : -INFINITY;
    }
  }
  float top = -INFINITY;
  int where = 0x7fffffff;
  bool nan = false;
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    if (kGreedy && v[i] > top) where = base + (i & ~3) * 256 + 4 * (int)threadIdx.x + (i & 3);
    top = fmaxf(top, v[i]);
    nan |= v[i] != v[i];
  }
  const float mine = top;
  top = wave_max(top);
  if (lane == 0) tops[wave] = top;
  if (kGreedy) {  // the least index of the wavefront's maximum
    where = mine == top ? where : 0x7fffffff;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) where = min(where, __shfl_xor(where, o));
    if (lane == 0) ats[wave] = where;
  }
  __syncthreads();
  Part* out = (of_draft ? a.q : a.p) + (size_t)r * a.segs + seg;
  const float all = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
  if (kGreedy) {
    if (threadIdx.x == 0) {
      int at = 0x7fffffff;
#pragma unroll
      for (int w = 0; w < 4; ++w) at = tops[w] == all ? min(at, ats[w]) : at;
      out->top = all;
      out->at = at;
    }
    return;
  }
  double sum = 0.0;
  const double c = a.inv_t * 1.4426950408889634074;
  const double from = all == -INFINITY ? 0.0 : (double)all;
#pragma unroll
  for (int i = 0; i < kEach; ++i) sum += exp_sum(v[i], c, from);
  // A NaN or +infinity leaves no distribution, and its sum stays NaN whatever else the segment has: its maximum may be -infinity.
  if (all == -INFINITY) sum = 0.0;
  if (nan || all == INFINITY) sum = (double)NAN;
  sum = wave_add(sum);
  if (lane == 0) sums[wave] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    out->top = all;
    out->sum = (sums[0] + sums[1]) + (sums[2] + sums[3]);
  }
}

// The maximum and sum of a row, or of two at once, from their segments', by one wavefront
template <int kRows>
__device__ __forceinline__ void combine(const Verify& a, const Part* const (&parts)[kRows], float (&m)[kRows], double (&z)[kRows]) {
  const int lane = threadIdx.x & 63;
  Part mine[kRows];
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    mine[r] = lane < a.segs ? parts[r][lane] : Part{0.0, -INFINITY, 0};
    m[r] = mine[r].top;
  }
  for (int i = lane + 64; i < a.segs; i += 64)
#pragma unroll
    for (int r = 0; r < kRows; ++r) m[r] = fmaxf(m[r], parts[r][i].top);
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    m[r] = wave_max(m[r]);
    const double base = m[r] == -INFINITY ? 0.0 : (double)m[r];
    z[r] = mine[r].sum * exp_neg(((double)mine[r].top - base) * a.inv_t);
    for (int i = lane + 64; i < a.segs; i += 64) z[r] += parts[r][i].sum * exp_neg(((double)parts[r][i].top - base) * a.inv_t);
    z[r] = wave_add(z[r]);
  }
}

// What is left for the next token at an index with these logits, in the row that refused
__device__ __forceinline__ double left_of(const Verify& a, const Found& f, float p, float q, bool draft, bool drafted) {
  const double x = exp_neg(((double)p - (double)f.mp) * a.inv_t) * f.rp;
  if (!draft) return drafted ? 0.0 : x;
  const double y = x - exp_neg(((double)q - (double)f.mq) * a.inv_t) * f.rq;
  return y < 0.0 ? 0.0 : y;
}

// blockIdx: segment, sequence. Every workgroup tests its sequence's tokens by itself, a row of each wavefront at a time.
__global__ __launch_bounds__(64 * kTestWaves) void test_kernel(Verify a) {
  __shared__ Found found[kTestWaves];
  __shared__ double sums[kTestWaves];
  __shared__ int stops[kTestWaves];
  const int seg = blockIdx.x % a.segs, b = blockIdx.x / a.segs, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const Rows s = rows_of(a, b);
  if (s.n == 0) {
    if (seg == 0 && threadIdx.x == 0) a.found[b] = Found{0.0, 0.0, 0.0f, 0.0f, 0, 0, 0};
    return;
  }
  int at = 0;  // the wavefront that had the first row behind which it ends
  for (int j0 = 0; j0 < s.n; j0 += kTestWaves) {
    const int j = j0 + wave, r = s.r0 + j;
    int stop = 0;
    if (j < s.n) {
      const bool judges = j < s.n - 1;  // the last row has no token behind it
      const int64_t t = judges ? a.tokens[r + 1] : 0;
      const float u = judges ? a.uniform[r] : 0.0f;
      const bool known = t >= 0 && t < a.vocab, both = judges && a.draft;
      const Part* const parts[2] = {a.p + (size_t)r * a.segs, (both ? a.q : a.p) + (size_t)r * a.segs};
      const float lt = a.logits[(size_t)r * a.ldl + (known ? t : 0)], dt = both ? a.draft[(size_t)r * a.ldd + (known ? t : 0)] : 0.0f;
      float m[2];
      double z[2];
      combine(a, parts, m, z);
      const double rp = 1.0 / z[0], rq = 1.0 / z[1];
      const double pt = exp_neg(((double)lt - (double)m[0]) * a.inv_t) * rp;
      const double qt = both ? exp_neg(((double)dt - (double)m[1]) * a.inv_t) * rq : 1.0;
      stop = !(judges && known && (double)u * qt < pt);
      if (lane == 0) found[wave] = Found{rp, both ? rq : 1.0, m[0], both ? m[1] : 0.0f, j + 1, judges, r};
    }
    if (lane == 0) stops[wave] = stop;
    __syncthreads();
    at = kTestWaves;
#pragma unroll
    for (int w = kTestWaves - 1; w >= 0; --w) at = stops[w] ? w : at;
    if (at < kTestWaves) break;  // the last row stops at the latest
    __syncthreads();
  }
  const Found f = found[at];
  if (seg == 0 && threadIdx.x == 0) a.found[b] = f;
  if (!f.refused) return;  // p itself: its segments' sums are there
  const float *p = a.logits + (size_t)f.row * a.ldl, *q = a.draft ? a.draft + (size_t)f.row * a.ldd : nullptr;
  const int64_t token = a.tokens[f.row + 1];
  constexpr int kMine = kSegment / (64 * kTestWaves);
  const int base = seg * kSegment + (int)threadIdx.x;
  float x[kMine], y[kMine];
#pragma unroll
  for (int i = 0; i < kMine; ++i) {
    const int k = min(base + i * 64 * kTestWaves, a.vocab - 1);
    x[i] = load_global<float>(p + k);
    y[i] = q ? load_global<float>(q + k) : 0.0f;
  }
  double sum = 0.0;
#pragma unroll
  for (int i = 0; i < kMine; ++i) {
    const int k = base + i * 64 * kTestWaves;
    if (k < a.vocab) sum += left_of(a, f, x[i], y[i], q != nullptr, k == token);
  }
  sum = wave_add(sum);
  if (lane == 0) sums[wave] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    sum = 0.0;
#pragma unroll
    for (int w = 0; w < kTestWaves; ++w) sum += sums[w];
    a.left[(size_t)b * a.segs + seg] = sum;
  }
}

// A workgroup per sequence
__global__ __launch_bounds__(kChoose) void choose_kernel(Verify a) {
  constexpr int kEach = kSegment / kChoose, kWaves = kChoose / 64;
  __shared__ double in_wave[kWaves], before, target;
  __shared__ int seg, refused, last[kWaves], hit[kWaves];
  const int b = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  Found f = a.found[b];
  const float choice = a.choice[b];
  if (f.count == 0) {  // no rows
    if (threadIdx.x == 0) {
      a.count[b] = 0;
      a.next[b] = -1;
    }
    return;
  }
  const int r = f.row;
  const Part* parts = a.p + (size_t)r * a.segs;
  auto sum_of = [&](int i) {
    return f.refused ? a.left[(size_t)b * a.segs + i]
                     : parts[i].sum * exp_neg(((double)parts[i].top - (f.mp == -INFINITY ? 0.0 : (double)f.mp)) * a.inv_t) * f.rp;
  };
  if (wave == 0) {
    double mine = lane < a.segs ? sum_of(lane) : 0.0;  // of the first 64 segments
    auto whole = [&]() {
      double sum = mine;
      for (int i = lane + 64; i < a.segs; i += 64) sum += sum_of(i);
      return wave_add(sum);
    };
    double total = whole();
    if (f.refused && total == 0.0) {  // p and q are the same: nothing is left over but p
      f.refused = 0;
      mine = lane < a.segs ? sum_of(lane) : 0.0;
      total = whole();
    }
    int at = -1;
    double in_front = 0.0;
    const double mark = (double)choice * total;
    if (total > 0.0 && total < (double)INFINITY) {
      double up = 0.0;
      for (int i0 = 0; i0 < a.segs; i0 += 64) {
        const double x = i0 == 0 ? mine : i0 + lane < a.segs ? sum_of(i0 + lane) : 0.0, upto = up + wave_scan(x);
        // the first whose sum passes the mark, and until there is one the last that has a share
        const unsigned long long past = __ballot(upto > mark && x > 0.0), some = __ballot(x > 0.0);
        if (some) {
          const int l = past ? __builtin_ctzll(past) : 63 - __builtin_clzll(some);
          at = i0 + l;
          in_front = of_lane(upto - x, l);
        }
        if (past) break;
        up = of_lane(upto, 63);
      }
    }
    if (lane == 0) {
      seg = at;
      before = in_front;
      target = mark;
      refused = f.refused;
    }
  }
  __syncthreads();
  f.refused = refused;
  int64_t token = -1;
  if (seg >= 0) {
    const float *p = a.logits + (size_t)r * a.ldl, *q = a.draft && f.refused ? a.draft + (size_t)r * a.ldd : nullptr;
    const int64_t not_this = f.refused ? a.tokens[r + 1] : -1;
    const int base = seg * kSegment + (int)threadIdx.x * kEach;
    float lp[kEach], lq[kEach];
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const int k = min(base + i, a.vocab - 1);
      lp[i] = load_global<float>(p + k);
      lq[i] = q ? load_global<float>(q + k) : 0.0f;
    }
    double x[kEach], sum = 0.0;
    int positive = -1;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      x[i] = base + i < a.vocab ? left_of(a, f, lp[i], lq[i], q != nullptr, base + i == not_this) : 0.0;
      sum += x[i];
      if (x[i] > 0.0) positive = base + i;
    }
    const double upto = wave_scan(sum);
    if (lane == 63) in_wave[wave] = upto;
    __syncthreads();
    double up = before + (upto - sum);
    for (int w = 0; w < wave; ++w) up += in_wave[w];
    int found = 0x7fffffff;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      up += x[i];
      if (x[i] > 0.0 && up > target) found = min(found, base + i);
    }
    // where rounding leaves none: the last one that has a share
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      found = min(found, __shfl_xor(found, o));
      positive = max(positive, __shfl_xor(positive, o));
    }
    if (lane == 0) {
      hit[wave] = found;
      last[wave] = positive;
    }
    __syncthreads();
    int first = 0x7fffffff, end = -1;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      first = min(first, hit[w]);
      end = max(end, last[w]);
    }
    token = first != 0x7fffffff ? first : end;
  }
  if (threadIdx.x == 0) {
    a.count[b] = f.count;
    a.next[b] = token;
    if (a.len) a.len[b] += f.count;
  }
}

// temperature 0: a wavefront per sequence
__global__ __launch_bounds__(64) void greedy_kernel(Verify a) {
  const int b = blockIdx.x, lane = threadIdx.x;
  const Rows s = rows_of(a, b);
  int64_t best = -1;
  int j = 0;
  for (; j < s.n; ++j) {
    const Part* parts = a.p + (size_t)(s.r0 + j) * a.segs;
    float top = -INFINITY;
    int at = 0x7fffffff;
    for (int i = lane; i < a.segs; i += 64) {
      const Part x = parts[i];
      if (x.top > top) {
        top = x.top;
        at = x.at;
      }
    }
    const float all = wave_max(top);
    at = top == all ? at : 0x7fffffff;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) at = min(at, __shfl_xor(at, o));
    best = at == 0x7fffffff ? -1 : at;
    if (j == s.n - 1 || a.tokens[s.r0 + j + 1] != best || best < 0) break;
  }
  if (lane == 0) {
    a.count[b] = s.n ? j + 1 : 0;
    a.next[b] = best;
    if (a.len && s.n) a.len[b] += j + 1;
  }
}

struct Layout {
  size_t q, left, found, total;
  int segs;
};
bool layout_of(int rows, int vocab, int n_seqs, Layout& l) {
  if (rows < 1 || vocab < 1 || n_seqs < 1 || rows >= 1 << 30 || vocab >= 1 << 30 || n_seqs >= 1 << 30) return false;
  l.segs = (vocab + kSegment - 1) / kSegment;
  // a launch has less than 2^32 threads: 256 of a row's segment, 512 of a sequence's, 1024 of a sequence
  if ((long long)rows * l.segs >= 1ll << 24 || (long long)n_seqs * l.segs >= 1ll << 23 || n_seqs >= 1 << 22) return false;
  l.q = (size_t)rows * l.segs * sizeof(Part);
  l.left = 2 * l.q;
  l.found = l.left + (size_t)n_seqs * l.segs * sizeof(double);
  l.total = l.found + (size_t)n_seqs * sizeof(Found);
  return true;
}
}  // namespace
}  // namespace w4

using namespace w4;

extern "C" {

size_t w4a32_op_verify_drafts_scratch_bytes(int rows, int vocab, int n_seqs) {
  Layout l;
  return layout_of(rows, vocab, n_seqs, l) ? l.total : 0;
}

int w4a32_op_verify_drafts(const w4a32_verify_args* v, void* d_scratch, size_t scratch_bytes, void* stream) {
  if (!v || !v->d_logits || !v->d_row_start || !v->d_tokens || !v->d_count || !v->d_next || !d_scratch) return W4A32_EINVAL;
  if (v->rows < 1 || v->max_rows < 1 || v->n_seqs < 1 || v->vocab < 1 || v->ldl < v->vocab) return W4A32_EINVAL;
  if (!(v->temperature >= 0.0f) || v->temperature > 3.0e38f) return W4A32_EINVAL;
  const bool greedy = v->temperature == 0.0f;
  if (!greedy && (!v->d_uniform || !v->d_choice || (v->d_draft && v->ldd < v->vocab))) return W4A32_EINVAL;
  if (!aligned(v->d_logits, 4) || !aligned(v->d_draft, 4) || !aligned(v->d_tokens, 8) || !aligned(v->d_next, 8) ||
      !aligned(v->d_uniform, 4) || !aligned(v->d_choice, 4) || !aligned(v->d_row_start, 4) || !aligned(v->d_count, 4) ||
      !aligned(v->d_len, 4) || !aligned(d_scratch, 16))
    return W4A32_EINVAL;
  Layout l;
  if (!layout_of(v->rows, v->vocab, v->n_seqs, l)) return W4A32_ESHAPE;
  if (scratch_bytes < l.total) return W4A32_EINVAL;
  uint8_t* scratch = static_cast<uint8_t*>(d_scratch);
  const Verify a{v->d_logits, greedy ? nullptr : v->d_draft, v->d_row_start, v->d_tokens, v->d_uniform, v->d_choice, v->d_count,
                 v->d_next, v->d_len, v->rows, v->max_rows, v->n_seqs, v->vocab, v->ldl, v->ldd, l.segs,
                 greedy ? 0.0 : 1.0 / (double)v->temperature, (Part*)scratch, (Part*)(scratch + l.q), (double*)(scratch + l.left),
                 (Found*)(scratch + l.found)};
  hipStream_t s = static_cast<hipStream_t>(stream);
  const dim3 stats((unsigned)(v->rows * (long long)l.segs), a.draft ? 2 : 1);
  if (greedy) {
    hipLaunchKernelGGL((stats_kernel<true>), stats, dim3(256), 0, s, a);
    if (hipGetLastError() != hipSuccess) return W4A32_ELAUNCH;
    hipLaunchKernelGGL(greedy_kernel, dim3((unsigned)v->n_seqs), dim3(64), 0, s, a);
  } else {
    hipLaunchKernelGGL((stats_kernel<false>), stats, dim3(256), 0, s, a);
    if (hipGetLastError() != hipSuccess) return W4A32_ELAUNCH;
    hipLaunchKernelGGL(test_kernel, dim3((unsigned)(v->n_seqs * (long long)l.segs)), dim3(64 * kTestWaves), 0, s, a);
    if (hipGetLastError() != hipSuccess) return W4A32_ELAUNCH;
    hipLaunchKernelGGL(choose_kernel, dim3((unsigned)v->n_seqs), dim3(kChoose), 0, s, a);
  }
  return hipGetLastError() == hipSuccess ? W4A32_OK : W4A32_ELAUNCH;
}

}  // extern "C"
