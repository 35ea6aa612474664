// Verification of drafted tokens against the target's logits and given random numbers.
//
// A row of logits is cut into segments of kSegment. The first launch takes every segment of every row once: its maximum and
// the sum of its exponentials, relative to that maximum. The second combines them per row, tests the drafted tokens of a
// sequence and, where one was refused, adds up max(p - q, 0) over the segments of its row; the third finds the segment and
// then the index that the given number falls on.
//
// Exponentials and sums are f64: an f64 instruction runs at the rate of an f32 one here, an exponential takes about 16 of
// them, and with two logits per 8 bytes read the launch stays bound by memory. In f32 the sums' rounding would decide which
// token a number falls on whenever it lies within 1e-7 of a border, as one of 150000 tokens' borders often does.
#include "w4a32_internal.h"
#include "w4a32_decoder.h"

namespace w4 {
namespace {
inline bool aligned(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

constexpr int kSegment = 4096;  // logits of a segment: 16 of each thread, all requested at once
constexpr int kEach = kSegment / 256;

struct Part {
  double sum;
  float top;
  int at;  // greedy: index of the maximum
};
struct Found {  // what the second launch leaves for the third
  double zp, zq;
  float mp, mq;
  int count, refused;
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

struct Rows {
  int r0, n;
};
__device__ __forceinline__ Rows rows_of(const Verify& a, int b) {
  Rows s;
  s.r0 = min(max(a.row_start[b], 0), a.rows);
  s.n = min(min(max(a.row_start[b + 1], s.r0), a.rows) - s.r0, a.max_rows);
  return s;
}

template <typename T>
__device__ __forceinline__ T wave_add(T x) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) x += __shfl_xor(x, o);
  return x;
}
__device__ __forceinline__ float wave_max(float x) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) x = fmaxf(x, __shfl_xor(x, o));
  return x;
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
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int at = base + i * 256 + (int)threadIdx.x;
    v[i] = at < a.vocab ? load_global<float>(x + at) : -INFINITY;
  }
  float top = -INFINITY;
  int where = 0x7fffffff;
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    if (kGreedy && v[i] > top) where = base + i * 256 + (int)threadIdx.x;
    top = fmaxf(top, v[i]);
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
  const double m = all == -INFINITY ? 0.0 : (double)all;
#pragma unroll
  for (int i = 0; i < kEach; ++i) sum += exp_neg(((double)v[i] - m) * a.inv_t);
  sum = wave_add(sum);
  if (lane == 0) sums[wave] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    out->top = all;
    out->sum = (sums[0] + sums[1]) + (sums[2] + sums[3]);
  }
}

// A row's maximum and sum from its segments', by one wavefront
__device__ __forceinline__ void combine(const Verify& a, const Part* parts, float& m, double& z) {
  const int lane = threadIdx.x & 63;
  m = -INFINITY;
  for (int i = lane; i < a.segs; i += 64) m = fmaxf(m, parts[i].top);
  m = wave_max(m);
  const double base = m == -INFINITY ? 0.0 : (double)m;
  z = 0.0;
  for (int i = lane; i < a.segs; i += 64) z += parts[i].sum * exp_neg(((double)parts[i].top - base) * a.inv_t);
  z = wave_add(z);
}

// What is left for the next token at index i of the row that refused
__device__ __forceinline__ double left_at(const Verify& a, const Found& f, const float* p, const float* q, int64_t token, int i) {
  const double x = exp_neg(((double)p[i] - (double)f.mp) * a.inv_t) / f.zp;
  if (!q) return i == token ? 0.0 : x;
  const double y = x - exp_neg(((double)q[i] - (double)f.mq) * a.inv_t) / f.zq;
  return y < 0.0 ? 0.0 : y;
}

// blockIdx: segment, sequence. Every workgroup tests its sequence's tokens by itself.
__global__ __launch_bounds__(256) void test_kernel(Verify a) {
  __shared__ Found f;
  __shared__ double sums[4];
  __shared__ int refused[4];
  const int seg = blockIdx.x % a.segs, b = blockIdx.x / a.segs, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const Rows s = rows_of(a, b);
  if (s.n == 0) {
    if (seg == 0 && threadIdx.x == 0) a.found[b] = Found{0.0, 0.0, 0.0f, 0.0f, 0, 0};
    return;
  }
  int stop = s.n - 1;  // tokens accepted
  for (int j0 = 0; j0 < s.n - 1; j0 += 4) {
    bool bad = false;
    const int r = s.r0 + j0 + wave;
    if (j0 + wave < s.n - 1) {
      float mp, mq = 0.0f;
      double zp, zq = 1.0, qt = 1.0;
      combine(a, a.p + (size_t)r * a.segs, mp, zp);
      const int64_t t = a.tokens[r + 1];
      const bool in = t >= 0 && t < a.vocab;
      if (a.draft && in) {
        combine(a, a.q + (size_t)r * a.segs, mq, zq);
        qt = exp_neg(((double)a.draft[(size_t)r * a.ldd + t] - (double)mq) * a.inv_t) / zq;
      }
      const double pt = in ? exp_neg(((double)a.logits[(size_t)r * a.ldl + t] - (double)mp) * a.inv_t) / zp : 0.0;
      bad = !((double)a.uniform[r] * qt < pt);
    }
    if (lane == 0) refused[wave] = bad;
    __syncthreads();
    int first = 4;
#pragma unroll
    for (int w = 3; w >= 0; --w) first = refused[w] ? w : first;
    __syncthreads();
    if (first < 4) {
      stop = j0 + first;
      break;
    }
  }
  const int r = s.r0 + stop;
  const bool no = stop < s.n - 1;
  if (wave == 0) {
    float m, mq = 0.0f;
    double z, zq = 1.0;
    combine(a, a.p + (size_t)r * a.segs, m, z);
    if (no && a.draft) combine(a, a.q + (size_t)r * a.segs, mq, zq);
    if (lane == 0) f = Found{z, zq, m, mq, stop + 1, no};
  }
  __syncthreads();
  if (seg == 0 && threadIdx.x == 0) a.found[b] = f;
  if (!no) return;  // p itself: its segments' sums are there
  const float *p = a.logits + (size_t)r * a.ldl, *q = a.draft ? a.draft + (size_t)r * a.ldd : nullptr;
  const int64_t token = a.tokens[r + 1];
  double sum = 0.0;
#pragma unroll 4
  for (int i = 0; i < kEach; ++i) {
    const int at = seg * kSegment + i * 256 + (int)threadIdx.x;
    if (at < a.vocab) sum += left_at(a, f, p, q, token, at);
  }
  sum = wave_add(sum);
  if (lane == 0) sums[wave] = sum;
  __syncthreads();
  if (threadIdx.x == 0) a.left[(size_t)b * a.segs + seg] = (sums[0] + sums[1]) + (sums[2] + sums[3]);
}

// A workgroup per sequence
__global__ __launch_bounds__(256) void choose_kernel(Verify a) {
  __shared__ double in_wave[4], before, target;
  __shared__ int seg, last[4], hit[4];
  const int b = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const Rows s = rows_of(a, b);
  if (s.n == 0) {
    if (threadIdx.x == 0) {
      a.count[b] = 0;
      a.next[b] = -1;
    }
    return;
  }
  Found f = a.found[b];
  const int r = s.r0 + f.count - 1;
  const Part* parts = a.p + (size_t)r * a.segs;
  auto sum_of = [&](int i) {
    return f.refused ? a.left[(size_t)b * a.segs + i]
                     : parts[i].sum * exp_neg(((double)parts[i].top - (f.mp == -INFINITY ? 0.0 : (double)f.mp)) * a.inv_t) / f.zp;
  };
  if (threadIdx.x == 0) {
    double total = 0.0;
    for (int i = 0; i < a.segs; ++i) total += sum_of(i);
    if (f.refused && total == 0.0) {  // p and q are the same: nothing is left over but p
      f.refused = 0;
      for (int i = 0; i < a.segs; ++i) total += sum_of(i);
    }
    seg = -1;
    if (total > 0.0 && total < INFINITY) {
      target = (double)a.choice[b] * total;
      double up = 0.0;
      for (int i = 0; i < a.segs; ++i) {
        const double x = sum_of(i);
        if (x > 0.0) {
          seg = i;
          before = up;
        }
        up += x;
        if (up > target) break;
      }
    }
    last[0] = f.refused;
  }
  __syncthreads();
  f.refused = last[0];
  __syncthreads();
  int64_t token = -1;
  if (seg >= 0) {
    const float *p = a.logits + (size_t)r * a.ldl, *q = a.draft && f.refused ? a.draft + (size_t)r * a.ldd : nullptr;
    const int64_t not_this = f.refused ? a.tokens[r + 1] : -1;
    const int base = seg * kSegment + (int)threadIdx.x * kEach;
    double x[kEach], sum = 0.0;
    int positive = -1;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      x[i] = base + i < a.vocab ? left_at(a, f, p, q, not_this, base + i) : 0.0;
      sum += x[i];
      if (x[i] > 0.0) positive = base + i;
    }
    double upto = sum;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const double y = __shfl_up(upto, o);
      if (lane >= o) upto += y;
    }
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
    const int first = min(min(hit[0], hit[1]), min(hit[2], hit[3]));
    token = first != 0x7fffffff ? first : max(max(last[0], last[1]), max(last[2], last[3]));
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
  if ((long long)rows * l.segs >= 1ll << 31 || (long long)n_seqs * l.segs >= 1ll << 31) return false;
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
    hipLaunchKernelGGL(test_kernel, dim3((unsigned)(v->n_seqs * (long long)l.segs)), dim3(256), 0, s, a);
    if (hipGetLastError() != hipSuccess) return W4A32_ELAUNCH;
    hipLaunchKernelGGL(choose_kernel, dim3((unsigned)v->n_seqs), dim3(256), 0, s, a);
  }
  return hipGetLastError() == hipSuccess ? W4A32_OK : W4A32_ELAUNCH;
}

}  // extern "C"
