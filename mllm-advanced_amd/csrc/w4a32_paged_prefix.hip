// Attention of a batch whose sequences share prefixes in groups: a prefix's keys and values are read once for all rows of the group.
//
// A row's softmax is joined from its sums over the prefix and those over its sequence's own tokens, each relative to its maximum:
//   m = max(m_P, m_own),  l = 2^(m_P - m) l_P + 2^(m_own - m) l_own,  o = 2^(m_P - m) o_P + 2^(m_own - m) o_own.
// The prefix is the prompts' kernel's with the rows of all of the group's sequences, which all see all of it, and its keys dealt to as many
// workgroups as the chip has; the own tokens are the rows' kernel's. Four launches: who has what (the lengths and the groups are
// device memory), the prefixes, the own tokens, the join.
#include "w4a32_paged_attention.h"

namespace w4 {
namespace paged {

namespace {
inline bool aligned(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }
inline int from_hip(hipError_t e) { return e == hipSuccess ? W4A32_OK : W4A32_ELAUNCH; }
inline size_t up256(size_t v) { return (v + 255) / 256 * 256; }

constexpr float kLog2e = 1.44269504088896340736f;
constexpr int kPlan = 1024;      // threads of the workgroup that deals
constexpr int kGrid = 256;       // workgroups that prefixes are dealt to: one per CU
constexpr int kJoins = 1 << 20;  // workgroups of the joining launch, beyond which they take several rows each
constexpr int kWideRows = 128;   // pairs of row and head of a group on average, from which on a workgroup has the most rows

struct Groups {
  const int *group_start, *tokens;
  int keys;   // of a tile
  int log2;   // of the rows of a workgroup
  int least;  // tiles of a share, where there are so many
  int grid;   // workgroups that the launch has
};

// Who has what. A wavefront per group finds how much of the prefix all of its sequences with rows have; a group with one such sequence
// has none.
__global__ __launch_bounds__(kPlan) void deal_kernel(Attend a, Groups d) {
  __shared__ unsigned in_wave[kPlan / 64];
  __shared__ unsigned long long tiles_of_wave[kPlan / 64];
  const Prefix& x = a.prefix;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n_seqs = a.c.n_seqs;
  for (int b = tid; b < n_seqs; b += kPlan) {
    x.from[b] = 0;
    x.group_of[b] = -1;
  }
  __syncthreads();
  unsigned long long tiles = 0;
  unsigned items = 0;
  auto bounds = [&](int g, int& b0, int& b1) {
    b0 = min(max(d.group_start[g], 0), n_seqs);
    b1 = min(max(d.group_start[g + 1], b0), n_seqs);
  };
  for (int g = wave; g < x.n_groups; g += kPlan / 64) {
    int b0, b1;
    bounds(g, b0, b1);
    int least = min(max(d.tokens[g], 0), a.c.cap), with_rows = 0;
    for (int b = b0 + lane; b - lane < b1; b += 64) {
      const bool here = b < b1;
      Span s = {};
      if (here) s = span_of(a.c, a.row_start, a.rows, a.max_rows, b);
      with_rows += __popcll(__ballot(s.n > 0));
      int len = s.n > 0 ? s.len : kMost;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) len = min(len, __shfl_xor(len, o));
      least = min(least, len);
    }
    if (with_rows < 2) least = 0;
    if (lane == 0) {
      PrefixGroup q = {b0, 0, 0, least, 0, 0, 0, 0};
      if (least) {
        q.r0 = min(max(a.row_start[b0], 0), a.rows);
        q.n = min(max(a.row_start[b1], q.r0), a.rows) - q.r0;
        q.blocks = (int)(((long long)q.n * a.group + (1 << d.log2) - 1) >> d.log2);
        items += (unsigned)(q.blocks * a.c.kv_heads);
        tiles += (unsigned long long)q.blocks * a.c.kv_heads * ((least + d.keys - 1) / d.keys);
      }
      x.group[g] = q;
    }
  }
  unsigned all;
  block_scan<kPlan>(lane == 0 ? items : 0, in_wave, all);
  items = all;
  if (lane == 0) tiles_of_wave[wave] = tiles;
  __syncthreads();  // the groups too
  tiles = 0;
#pragma unroll
  for (int w = 0; w < kPlan / 64; ++w) tiles += tiles_of_wave[w];
  // One item's share has tiles of that item only: with `more` workgroups beyond one per item, ceil(nt / per) shares of each are enough
  const unsigned more = (unsigned)kGrid - min((unsigned)kGrid, items);
  const unsigned per = more ? max((unsigned)((tiles + more - 1) / more), (unsigned)d.least) : 1u << 30;
  unsigned total = 0;
  for (int g0 = 0; g0 < x.n_groups; g0 += kPlan) {
    const int g = g0 + tid;
    unsigned n = 0;
    PrefixGroup q = {};
    if (g < x.n_groups) {
      q = x.group[g];
      const unsigned nt = (unsigned)(q.tokens + d.keys - 1) / d.keys;
      q.shares = (int)((nt + per - 1) / per);
      n = (unsigned)q.blocks * a.c.kv_heads * q.shares;
    }
    q.first = (int)(total + block_scan<kPlan>(n, in_wave, all) - n);
    if (g < x.n_groups) x.group[g] = q;
    total += all;
  }
  const bool fits = total <= (unsigned)d.grid;  // else (row or group starts that decrease) all read everything by themselves
  if (tid == 0) *x.total = fits ? (int)total : 0;
  if (!fits) return;
  __syncthreads();
  for (int g = wave; g < x.n_groups; g += kPlan / 64) {
    const int tokens = x.group[g].tokens;
    if (tokens == 0) continue;
    int b0, b1;
    bounds(g, b0, b1);
    for (int b = b0 + lane; b < b1; b += 64) {
      x.from[b] = tokens;
      x.group_of[b] = g;
    }
  }
}

// A row's shares, of the prefix and of its own tokens, as the join of shares of one item has them: a workgroup per row and kSlice of its
// values, its threads four values of every 256 / (kSlice / 4)th share each.
template <typename Act, int DT, int kSlice>
__device__ __forceinline__ void join(const Attend& a, unsigned unit, int log2) {
  constexpr int kPer = kSlice / 4, kAtOnce = 256 / kPer;
  __shared__ __attribute__((aligned(16))) float sums[4][kSlice];
  __shared__ float tops[4], totals[4];
  const int slice = unit % (DT / kSlice), r = unit / (DT / kSlice) % a.slot_rows;
  const unsigned item = unit / (DT / kSlice) / a.slot_rows;
  if (item >= *a.count) return;
  const Item it = a.item[item];
  if (r >= it.rows) return;
  const int g = a.prefix.group_of[a.prefix.item_seq[item]];
  int common = 0;
  size_t at0 = 0, step = 0;
  if (g >= 0) {
    const PrefixGroup q = a.prefix.group[g];
    const int of = it.row0 + r, j = by_group(a, of), row = it.r0 + j - q.r0;
    if ((unsigned)row < (unsigned)q.n) {  // always, where group starts do not decrease
      const int pair = row * a.group + of - j * a.group, block = pair >> log2;
      common = q.shares;
      at0 = ((size_t)(q.first + block * a.c.kv_heads + it.head) << log2) + (pair & ((1 << log2) - 1));
      step = (size_t)(q.blocks * a.c.kv_heads) << log2;
    }
  }
  const int d = slice * kSlice + threadIdx.x % kPer * 4, mine = threadIdx.x / kPer, count = common + it.shares;
  float top = -INFINITY, sum = 0.0f;
  f32x4 acc = {0, 0, 0, 0};
  for (int x0 = mine; x0 < count; x0 += 8 * kAtOnce) {
    float m[8], l[8];
    f32x4 v[8];
#pragma unroll
    for (int x = 0; x < 8; ++x) {
      const int i = x0 + x * kAtOnce, own = i - common;
      m[x] = -INFINITY;
      l[x] = 0.0f;
      v[x] = f32x4{0, 0, 0, 0};
      if (i < count) {
        const size_t at = own < 0 ? at0 + step * i
                                  : (size_t)(it.shares == 1 ? kOwnSlots + (int)item : 2 * (it.first + own) + (own == 0)) * a.slot_rows + r;
        const float *state = own < 0 ? a.prefix.state : a.state, *part = own < 0 ? a.prefix.part : a.part;
        m[x] = load_global<float>(state + 2 * at);
        l[x] = load_global<float>(state + 2 * at + 1);
        v[x] = load_global<f32x4>(part + at * DT + d);
      }
    }
    float most = top;
#pragma unroll
    for (int x = 0; x < 8; ++x) most = fmaxf(most, m[x]);
    const float base = most == -INFINITY ? 0.0f : most, down = pow2(top - base);
    sum *= down;
    acc *= fmaxf(down, kLeast);
    top = most;
#pragma unroll
    for (int x = 0; x < 8; ++x) {
      const float f = pow2(m[x] - base);
      sum += f * l[x];
      acc += fmaxf(f, kLeast) * v[x];
    }
  }
  float most = top;
#pragma unroll
  for (int x = kPer; x < 64; x <<= 1) most = fmaxf(most, __shfl_xor(most, x));
  const float in_wave = pow2(top - (most == -INFINITY ? 0.0f : most));
  sum *= in_wave;
  acc *= fmaxf(in_wave, kLeast);
#pragma unroll
  for (int x = kPer; x < 64; x <<= 1) {
    sum += __shfl_xor(sum, x);
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i] += __shfl_xor(acc[i], x);
  }
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if (lane < kPer) *(f32x4*)&sums[wave][4 * lane] = acc;
  if (lane == 0) {
    tops[wave] = most;
    totals[wave] = sum;
  }
  __syncthreads();
  if (threadIdx.x >= kPer) return;
  top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
  const float base = top == -INFINITY ? 0.0f : top;
  sum = 0.0f;
  acc = f32x4{0, 0, 0, 0};
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const float f = pow2(tops[w] - base);
    acc += fmaxf(f, kLeast) * *(const f32x4*)&sums[w][4 * lane];
    sum += f * totals[w];
  }
  finish<Act, false>(a, it.r0, it.row0 + r, it.head, 0, d, acc, base, sum);
}
template <typename Act, int DT, int kSlice>
__global__ __launch_bounds__(256) void join_kernel(Attend a, unsigned units, int log2) {
  for (unsigned u = blockIdx.x; u < units; u += gridDim.x) {
    join<Act, DT, kSlice>(a, u, log2);
    if (units > gridDim.x) __syncthreads();
  }
}

// ---- host ------------------------------------------------------------------------------------------------------------------
struct Plan {
  OwnPlan own;
  int log2, keys, least;
  unsigned grid;  // of the prefixes' launch
  size_t group_off, from_off, of_off, item_off, seq_off, part_off, state_off, pre_part_off, pre_state_off, total;
};

int plan_of(const w4a32_paged_cache* c, const w4a32_paged_rows* r, int n_groups, Plan& p) {
  if (int e = plan_own(c, r, p.own)) return e;
  const long long group = r->heads / c->kv_heads;
  const bool f32 = c->dtype == W4A32_CACHE_F32;
  const int dt = p.own.dt, wide = dt == 256 || f32 ? 7 : 8;
  p.log2 = f32 ? (dt == 64 ? 5 : wide) : r->rows * group >= (long long)kWideRows * n_groups ? wide : 5;
  p.keys = prefix_keys(c->dtype, dt, p.log2);
  p.least = p.log2 == 5 ? dt == 256 ? 2 : 4 : 1;  // a tile of each of its wavefronts
  const long long items = (((long long)r->rows * group >> p.log2) + n_groups) * c->kv_heads;
  const long long grid = items > kGrid ? items : kGrid;
  if (grid > most_groups(512)) return W4A32_ESHAPE;
  p.grid = (unsigned)grid;
  size_t at = 256;
  auto take = [&](size_t bytes) {
    const size_t here = at;
    at = up256(at + bytes);
    return here;
  };
  p.group_off = take((size_t)n_groups * sizeof(PrefixGroup));
  p.from_off = take((size_t)c->n_seqs * 4);
  p.of_off = take((size_t)c->n_seqs * 4);
  p.item_off = take((size_t)p.own.items * sizeof(Item));
  p.seq_off = take((size_t)p.own.items * 4);
  p.part_off = take((size_t)p.own.slots * p.own.slot_rows * dt * 4);
  p.state_off = take((size_t)p.own.slots * p.own.slot_rows * 8);
  p.pre_part_off = take(((size_t)p.grid << p.log2) * dt * 4);
  p.pre_state_off = take(((size_t)p.grid << p.log2) * 8);
  p.total = at;
  return W4A32_OK;
}

template <typename Act, int DT>
hipError_t launch_join(const Attend& a, const Plan& p, hipStream_t s) {
  const bool sliced = p.own.items * p.own.slot_rows <= 128;  // few rows: a row's values are dealt to several workgroups
  const long long units = p.own.items * p.own.slot_rows * (sliced ? DT / 32 : 1);
  auto kernel = sliced ? join_kernel<Act, DT, 32> : join_kernel<Act, DT, DT>;
  hipLaunchKernelGGL(kernel, dim3((unsigned)(units < kJoins ? units : kJoins)), dim3(256), 0, s, a, (unsigned)units, p.log2);
  return hipGetLastError();
}
template <typename Act>
hipError_t launch_join_dim(const Attend& a, const Plan& p, hipStream_t s) {
  if (p.own.dt == 64) return launch_join<Act, 64>(a, p, s);
  if (p.own.dt == 128) return launch_join<Act, 128>(a, p, s);
  return launch_join<Act, 256>(a, p, s);
}

int check(const w4a32_paged_cache* cache, const w4a32_paged_rows* rows, int n_groups) {
  if (int e = check_rows(cache, rows)) return e;
  if (!rows->d_q || !rows->d_out || n_groups < 1) return W4A32_EINVAL;
  if (n_groups > cache->n_seqs) return W4A32_ESHAPE;
  return W4A32_OK;
}
}  // namespace

}  // namespace paged
}  // namespace w4

using namespace w4::paged;

extern "C" {

size_t w4a32_op_paged_prefix_attention_scratch_bytes(const w4a32_paged_cache* cache, const w4a32_paged_rows* rows, int n_groups) {
  Plan p;
  return check(cache, rows, n_groups) || plan_of(cache, rows, n_groups, p) ? 0 : p.total;
}

int w4a32_op_paged_prefix_attention(const w4a32_paged_cache* cache, const w4a32_paged_rows* rows, float scale, const int* d_group_start,
                                    const int* d_prefix, int n_groups, void* d_scratch, size_t scratch_bytes, void* stream) {
  if (int e = check(cache, rows, n_groups)) return e;
  if (!(scale * kLog2e - scale * kLog2e == 0.0f) || !d_group_start || !d_prefix || !aligned(d_group_start, 4) || !aligned(d_prefix, 4) || !d_scratch ||
      !aligned(d_scratch, 16))
    return W4A32_EINVAL;
  Plan p;
  if (int e = plan_of(cache, rows, n_groups, p)) return e;
  if (scratch_bytes < p.total) return W4A32_EINVAL;
  uint8_t* scratch = static_cast<uint8_t*>(d_scratch);
  const Prefix x{(int*)(scratch + 128), (PrefixGroup*)(scratch + p.group_off), (int*)(scratch + p.from_off), (int*)(scratch + p.of_off),
                 (int*)(scratch + p.seq_off), (float*)(scratch + p.pre_part_off), (float*)(scratch + p.pre_state_off), n_groups};
  Attend a{view(cache), rows->d_q, rows->d_out, rows->d_row_start, rows->ldq, rows->ldo, rows->rows,
           rows->max_rows < rows->rows ? rows->max_rows : rows->rows, rows->heads, rows->heads / cache->kv_heads, 0, 0, 0, rows->rows, 0, 0, 0, p.log2,
           p.own.wide, p.own.slot_rows, (unsigned)p.own.items, (unsigned)p.own.tiles, scale * kLog2e, (Item*)(scratch + p.item_off),
           (unsigned*)scratch, (float*)(scratch + p.part_off), (float*)(scratch + p.state_off), nullptr, nullptr, x};
  set_group(a);
  hipStream_t s = static_cast<hipStream_t>(stream);
  const Groups d{d_group_start, d_prefix, p.keys, p.log2, p.least, (int)p.grid};
  hipLaunchKernelGGL(deal_kernel, dim3(1), dim3(kPlan), 0, s, a, d);
  if (hipGetLastError() != hipSuccess) return W4A32_ELAUNCH;
  if (launch_prefixes(a, cache->dtype, rows->act_bf16 != 0, p.own.dt, p.grid, s) != hipSuccess) return W4A32_ELAUNCH;
  if (launch_own(a, p.own, cache->dtype, rows->act_bf16 != 0, s) != hipSuccess) return W4A32_ELAUNCH;
  return from_hip(rows->act_bf16 ? launch_join_dim<__bf16>(a, p, s) : launch_join_dim<float>(a, p, s));
}

}  // extern "C"
