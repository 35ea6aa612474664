// Attention of a batch whose sequences share prefixes in groups: a prefix's keys and values are read once for all rows of the group.
//
// A row's softmax is joined from its sums over the prefix and those over its sequence's own tokens, each relative to its maximum:
//   m = max(m_P, m_own),  l = 2^(m_P - m) l_P + 2^(m_own - m) l_own,  o = 2^(m_P - m) o_P + 2^(m_own - m) o_own.
// The prefix is the prompts' kernel's with the rows of all of the group's sequences, which all see all of it, and its keys dealt to as many
// workgroups as the chip has; the own tokens are the rows' kernel's. Four launches: who has what (the lengths and the groups are
// device memory), the prefixes, the own tokens, the join.
#include "w4a32_paged_prompt.h"
#include "w4a32_paged_rows.h"

namespace w4 {
namespace paged {

namespace {
inline bool aligned(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }
inline int from_hip(hipError_t e) { return e == hipSuccess ? W4A32_OK : W4A32_ELAUNCH; }
inline size_t up256(size_t v) { return (v + 255) / 256 * 256; }

constexpr float kLog2e = 1.44269504088896340736f;
constexpr int kPlan = 1024;      // threads of the workgroup that deals
constexpr int kSlots = 512;      // workgroups that are there at once: two per CU
constexpr int kLog2 = 7;         // log2 of the rows of a workgroup of a prefix
constexpr int kManyRows = 8192;  // rows from which on a workgroup joins several of them
constexpr int kJoins = 1 << 20;  // workgroups of the joining launch, beyond which they take more

struct Groups {
  const int *group_start, *tokens;
  int keys, own_keys;  // of a tile of a prefix, and of one of own tokens
  int grid;            // most workgroups that prefixes get
};

__device__ __forceinline__ unsigned long long wave_sum(unsigned long long v) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) v += __shfl_xor(v, o);
  return v;
}
__device__ __forceinline__ unsigned wave_sum(unsigned v) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) v += __shfl_xor(v, o);
  return v;
}

// Who has what. A wavefront per group finds how much of the prefix all of its sequences with rows have (a group with one such sequence has
// none). The slots of the chip then go to the prefixes and to the own tokens as their work is estimated, and a prefix's tiles to as few
// workgroups per item as keep to that. kLds: everything that is read lies in LDS, asked for at once; else (many sequences) it is read
// where it is needed.
template <bool kLds>
__global__ __launch_bounds__(kPlan) void deal_kernel(Attend a, Groups d) {
  constexpr int kIn = kLds ? kPlan : 1;
  __shared__ int starts[kIn + 1], lens[kIn], group_starts[kIn + 1], wanted[kIn], froms[kIn];
  __shared__ PrefixGroup groups[kIn];
  __shared__ unsigned long long of_wave[kPlan / 64];
  const Prefix& x = a.prefix;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n_seqs = a.c.n_seqs, n_groups = x.n_groups;
  PrefixGroup* const group = kLds ? groups : x.group;
  int* const from = kLds ? froms : x.from;
  if constexpr (kLds) {
    if (tid <= n_seqs) starts[tid] = a.row_start[tid];
    if (tid == kPlan - 1 && n_seqs == kPlan) starts[kPlan] = a.row_start[kPlan];
    if (tid < n_seqs) lens[tid] = a.c.len[tid];
    if (tid <= n_groups) group_starts[tid] = d.group_start[tid];
    if (tid == kPlan - 1 && n_groups == kPlan) group_starts[kPlan] = d.group_start[kPlan];
    if (tid < n_groups) wanted[tid] = d.tokens[tid];
  }
  for (int b = tid; b < n_seqs; b += kPlan) {
    from[b] = 0;
    x.group_of[b] = -1;
  }
  __syncthreads();
  const int *row_start = kLds ? starts : a.row_start, *group_start = kLds ? group_starts : d.group_start, *tokens = kLds ? wanted : d.tokens;
  Cache c = a.c;
  if constexpr (kLds) c.len = lens;
  auto bounds = [&](int g, int& b0, int& b1) {
    b0 = min(max(group_start[g], 0), n_seqs);
    b1 = min(max(group_start[g + 1], b0), n_seqs);
  };
  for (int g = wave; g < n_groups; g += kPlan / 64) {
    int b0, b1;
    bounds(g, b0, b1);
    int least = min(max(tokens[g], 0), c.cap), with_rows = 0;
    for (int b = b0 + lane; b - lane < b1; b += 64) {
      Span s = {};
      if (b < b1) s = span_of(c, row_start, a.rows, a.max_rows, b);
      with_rows += __popcll(__ballot(s.n > 0));
      if (s.n > 0) least = min(least, s.len);
    }
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) least = min(least, __shfl_xor(least, o));
    if (with_rows < 2) least = 0;
    if (lane == 0) {
      PrefixGroup q = {b0, 0, 0, least, 0, 0, 0, 0};
      if (least) {
        q.r0 = min(max(row_start[b0], 0), a.rows);
        q.n = min(max(row_start[b1], q.r0), a.rows) - q.r0;
        q.blocks = (int)(((long long)q.n * a.group + (1 << kLog2) - 1) >> kLog2);
      }
      group[g] = q;
    }
    if (least)
      for (int b = b0 + lane; b < b1; b += 64) {
        from[b] = least;
        x.group_of[b] = g;
      }
  }
  __syncthreads();
  // ---- tiles of own tokens, of a wavefront each ----
  unsigned long long own = 0;
  for (int b = tid; b < n_seqs; b += kPlan) {
    const Span s = span_of(c, row_start, a.rows, a.max_rows, b);
    if (kLds) x.from[b] = from[b];
    if (s.n == 0) continue;
    const int keys = min(s.len + s.n, c.cap), first = min(from[b], c.cap - 1);
    own += (((unsigned long long)s.n * a.group + 15) / 16) * ((keys + d.own_keys - 1) / d.own_keys - first / d.own_keys);
  }
  own = wave_sum(own);
  if (lane == 0) of_wave[wave] = own;
  __syncthreads();
  if (wave != 0) return;
  own = 0;
#pragma unroll
  for (int w = 0; w < kPlan / 64; ++w) own += of_wave[w];
  // ---- and of prefixes ----
  auto tiles_of = [&](int g) { return (unsigned)(group[g].tokens + d.keys - 1) / (unsigned)d.keys; };
  unsigned long long tiles = 0;
  unsigned items = 0;
  for (int g = lane; g < n_groups; g += 64) {
    items += (unsigned)group[g].blocks * a.c.kv_heads;
    tiles += (unsigned long long)group[g].blocks * a.c.kv_heads * tiles_of(g);
  }
  items = wave_sum(items);
  tiles = wave_sum(tiles);
  // Times that a workgroup takes: 3 units for a tile of a prefix, 8 for kWaves tiles of own tokens
  const float work = (float)tiles * 3.0f, rest = (float)own * a.c.kv_heads * (8.0f / kWaves);
  unsigned most = min(max((unsigned)(kSlots * (work / (work + rest + 1.0f)) + 0.5f), (unsigned)kSlots / 4), (unsigned)kSlots * 7 / 8);
  if (2 * items > most) most *= 2;  // in two rounds, so that what one leaves over is small
  most = min(most, (unsigned)d.grid);
  // Shares of `per` tiles, the fewest that leave no more than `most` of them: ceil(tiles / (most - items)) are enough
  unsigned per = 1u << 30;
  if (most > items) {
    unsigned lo = (unsigned)max((tiles + most - 1) / most, 1ull);
    per = (unsigned)max((tiles + most - items - 1) / (most - items), 1ull);
    while (lo < per) {
      const unsigned mid = (lo + per) / 2;
      unsigned n = 0;
      for (int g = lane; g < n_groups; g += 64) n += (unsigned)group[g].blocks * a.c.kv_heads * ((tiles_of(g) + mid - 1) / mid);
      if (wave_sum(n) <= most)
        per = mid;
      else
        lo = mid + 1;
    }
  }
  unsigned total = 0;
  for (int g0 = 0; g0 < n_groups; g0 += 64) {
    const int g = g0 + lane;
    PrefixGroup q = {};
    unsigned n = 0;
    if (g < n_groups) {
      q = group[g];
      q.shares = (int)((tiles_of(g) + per - 1) / per);
      n = (unsigned)q.blocks * a.c.kv_heads * q.shares;
    }
    const unsigned upto = wave_scan(n);
    q.first = (int)(total + upto - n);
    if (g < n_groups) x.group[g] = q;
    total = add_sat(total, last_lane(upto));
  }
  const bool fits = total <= (unsigned)d.grid;  // else (row or group starts that decrease) all read everything by themselves
  if (!fits)
    for (int b = lane; b < n_seqs; b += 64) {
      x.from[b] = 0;
      x.group_of[b] = -1;
    }
  if (lane == 0) *x.total = fits ? (int)total : 0;
}

// A row's shares, those of the prefix first, and where they lie
struct Shares {
  int rows, common, count;  // rows of its item that are there
  size_t at0, step;         // places of the prefix's in its sums
  Item own;
};
__device__ __forceinline__ Shares shares_of(const Attend& a, unsigned item, int r) {
  const OwnItem it = a.prefix.item[min(item, a.most_items - 1)];
  Shares s;
  s.rows = item < *a.count ? it.own.rows : 0;
  s.common = it.shares;
  s.count = it.shares + it.own.shares;
  const int pair = it.pair + r;
  s.at0 = ((size_t)(it.from + (pair >> kLog2) * a.c.kv_heads) << kLog2) + (pair & ((1 << kLog2) - 1));
  s.step = (size_t)it.step << kLog2;
  s.own = it.own;
  return s;
}
// kAhead shares from i0 on, each kApart behind the last: brings top, sum and acc to their common maximum
template <int DT, int kAhead, int kApart>
__device__ __forceinline__ void add_shares(const Attend& a, const Shares& s, unsigned item, int r, int d, int i0, float& top, float& sum, f32x4& acc) {
  float m[kAhead], l[kAhead];
  f32x4 v[kAhead];
#pragma unroll
  for (int x = 0; x < kAhead; ++x) {
    const int i = i0 + x * kApart, own = i - s.common;
    m[x] = -INFINITY;
    l[x] = 0.0f;
    v[x] = f32x4{0, 0, 0, 0};
    if (i < s.count) {
      const size_t at = own < 0 ? s.at0 + s.step * i
                                : (size_t)(s.own.shares == 1 ? kOwnSlots + (int)item : 2 * (s.own.first + own) + (own == 0)) * a.slot_rows + r;
      const float *state = own < 0 ? a.prefix.state : a.state, *part = own < 0 ? a.prefix.part : a.part;
      m[x] = load_global<float>(state + 2 * at);
      l[x] = load_global<float>(state + 2 * at + 1);
      v[x] = load_global<f32x4>(part + at * DT + d);
    }
  }
  float most = top;
#pragma unroll
  for (int x = 0; x < kAhead; ++x) most = fmaxf(most, m[x]);
  const float base = most == -INFINITY ? 0.0f : most, down = pow2(top - base);
  sum *= down;
  acc *= fmaxf(down, kLeast);
  top = most;
#pragma unroll
  for (int x = 0; x < kAhead; ++x) {
    const float f = pow2(m[x] - base);
    sum += f * l[x];
    acc += fmaxf(f, kLeast) * v[x];
  }
}

// Both parts in one launch: the first workgroups have the prefixes
template <typename Act, typename KV, int DT>
__global__ __launch_bounds__(64 * kWaves, DT == 256 ? 1 : 2) void both_kernel(Attend a) {
  static_assert(Shape<Act, KV, DT, kHalfForm>::kThreads == 64 * kWaves, "workgroups of either kind");
  const unsigned prefixes = (unsigned)*a.prefix.total;
  if (blockIdx.x < prefixes)
    prompt_body<Act, KV, DT, kHalfForm, true>(a, blockIdx.x);
  else if (blockIdx.x - prefixes < kOwnGrid)
    rows_body<Act, KV, DT, false, kOwn>(a, blockIdx.x - prefixes, kOwnGrid);
}

// Where rows are few: a workgroup per row and kSlice of its values, its threads four values of every 256 / (kSlice / 4)th share each
template <typename Act, int DT, int kSlice>
__global__ __launch_bounds__(256) void join_kernel(Attend a) {
  constexpr int kPer = kSlice / 4, kAtOnce = 256 / kPer;
  __shared__ __attribute__((aligned(16))) float sums[4][kSlice];
  __shared__ float tops[4], totals[4];
  const int slice = blockIdx.x % (DT / kSlice), r = blockIdx.x / (DT / kSlice) % a.slot_rows;
  const unsigned item = blockIdx.x / (DT / kSlice) / a.slot_rows;
  const Shares s = shares_of(a, item, r);
  if (r >= s.rows) return;
  const int d = slice * kSlice + threadIdx.x % kPer * 4, mine = threadIdx.x / kPer;
  float top = -INFINITY, sum = 0.0f;
  f32x4 acc = {0, 0, 0, 0};
  for (int i0 = mine; i0 < s.count; i0 += 8 * kAtOnce) add_shares<DT, 8, kAtOnce>(a, s, item, r, d, i0, top, sum, acc);
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
  finish<Act, false>(a, s.own.r0, s.own.row0 + r, s.own.head, 0, d, acc, base, sum);
}

// Where they are many: DT / 4 threads per row
template <typename Act, int DT>
__global__ __launch_bounds__(256) void join_rows_kernel(Attend a, unsigned rows) {
  constexpr int kPer = DT / 4, kAtOnce = 256 / kPer;
  const int d = threadIdx.x % kPer * 4;
  for (unsigned u = blockIdx.x * kAtOnce + threadIdx.x / kPer; u < rows; u += gridDim.x * kAtOnce) {
    const unsigned item = u / (unsigned)a.slot_rows;
    const int r = (int)(u - item * a.slot_rows);
    const Shares s = shares_of(a, item, r);
    if (r >= s.rows) continue;
    float top = -INFINITY, sum = 0.0f;
    f32x4 acc = {0, 0, 0, 0};
    for (int i0 = 0; i0 < s.count; i0 += 4) add_shares<DT, 4, 1>(a, s, item, r, d, i0, top, sum, acc);
    finish<Act, false>(a, s.own.r0, s.own.row0 + r, s.own.head, 0, d, acc, top == -INFINITY ? 0.0f : top, sum);
  }
}

// ---- host ------------------------------------------------------------------------------------------------------------------
struct Plan {
  OwnPlan own;
  int keys;
  unsigned grid;  // workgroups of the prefixes
  size_t group_off, from_off, of_off, item_off, part_off, state_off, pre_part_off, pre_state_off, total;
};

int plan_of(const w4a32_paged_cache* c, const w4a32_paged_rows* r, int n_groups, Plan& p) {
  if (int e = plan_own(c, r, p.own)) return e;
  const long long group = r->heads / c->kv_heads;
  const int dt = p.own.dt;
  p.keys = prefix_keys(c->dtype, dt);
  const long long items = (((long long)r->rows * group >> kLog2) + n_groups) * c->kv_heads;
  const long long grid = items > 2 * kSlots ? items : 2 * kSlots;
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
  p.item_off = take((size_t)p.own.items * sizeof(OwnItem));
  p.part_off = take((size_t)p.own.slots * p.own.slot_rows * dt * 4);
  p.state_off = take((size_t)p.own.slots * p.own.slot_rows * 8);
  p.pre_part_off = take(((size_t)p.grid << kLog2) * dt * 4);
  p.pre_state_off = take(((size_t)p.grid << kLog2) * 8);
  p.total = at;
  return W4A32_OK;
}

template <typename Act, int DT>
hipError_t launch_join(const Attend& a, const Plan& p, hipStream_t s) {
  const long long rows = p.own.items * p.own.slot_rows;
  if (rows >= kManyRows) {
    constexpr int kAtOnce = 1024 / DT;
    const long long groups = (rows + kAtOnce - 1) / kAtOnce;
    hipLaunchKernelGGL((join_rows_kernel<Act, DT>), dim3((unsigned)(groups < kJoins ? groups : kJoins)), dim3(256), 0, s, a, (unsigned)rows);
  } else if (rows <= 128) {  // a row's values are dealt to several workgroups
    hipLaunchKernelGGL((join_kernel<Act, DT, 32>), dim3((unsigned)rows * (DT / 32)), dim3(256), 0, s, a);
  } else {
    hipLaunchKernelGGL((join_kernel<Act, DT, DT>), dim3((unsigned)rows), dim3(256), 0, s, a);
  }
  return hipGetLastError();
}
template <typename Act>
hipError_t launch_join_dim(const Attend& a, const Plan& p, hipStream_t s) {
  if (p.own.dt == 64) return launch_join<Act, 64>(a, p, s);
  if (p.own.dt == 128) return launch_join<Act, 128>(a, p, s);
  return launch_join<Act, 256>(a, p, s);
}

template <typename Act, typename KV, int DT>
hipError_t launch_both(const Attend& a, const Plan& p, hipStream_t s) {
  constexpr size_t one = Shape<Act, KV, DT, kHalfForm>::kLds, other = lds_bytes<KV, DT>(), lds = one > other ? one : other;
  if constexpr (lds > 64 * 1024) {
    static LdsLimitOnce limit;
    if (hipError_t e = limit.raise((const void*)both_kernel<Act, KV, DT>, lds); e != hipSuccess) return e;
  }
  hipLaunchKernelGGL((both_kernel<Act, KV, DT>), dim3(p.grid + kOwnGrid), dim3(64 * kWaves), lds, s, a);
  return hipGetLastError();
}
template <typename Act, typename KV>
hipError_t launch_both_dim(const Attend& a, const Plan& p, hipStream_t s) {
  if (p.own.dt == 64) return launch_both<Act, KV, 64>(a, p, s);
  if (p.own.dt == 128) return launch_both<Act, KV, 128>(a, p, s);
  return launch_both<Act, KV, 256>(a, p, s);
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
                 (OwnItem*)(scratch + p.item_off), (float*)(scratch + p.pre_part_off), (float*)(scratch + p.pre_state_off), n_groups};
  Attend a{view(cache), rows->d_q, rows->d_out, rows->d_row_start, rows->ldq, rows->ldo, rows->rows,
           rows->max_rows < rows->rows ? rows->max_rows : rows->rows, rows->heads, rows->heads / cache->kv_heads, 0, 0, 0, rows->rows, 0, 0, 0, kLog2,
           p.own.wide, p.own.slot_rows, (unsigned)p.own.items, (unsigned)p.own.tiles, scale * kLog2e, nullptr,
           (unsigned*)scratch, (float*)(scratch + p.part_off), (float*)(scratch + p.state_off), nullptr, nullptr, x};
  set_group(a);
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int dtype = cache->dtype;
  const bool bf16 = rows->act_bf16 != 0;
  const Groups d{d_group_start, d_prefix, p.keys, dtype == W4A32_CACHE_F32 ? 16 : 32, (int)p.grid};
  if (cache->n_seqs <= kPlan)
    hipLaunchKernelGGL((deal_kernel<true>), dim3(1), dim3(kPlan), 0, s, a, d);
  else
    hipLaunchKernelGGL((deal_kernel<false>), dim3(1), dim3(kPlan), 0, s, a, d);
  if (hipGetLastError() != hipSuccess) return W4A32_ELAUNCH;
  const hipError_t e = bf16                        ? launch_both_dim<__bf16, __bf16>(a, p, s)
                       : dtype == W4A32_CACHE_F32 ? launch_both_dim<float, float>(a, p, s)
                       : dtype == W4A32_CACHE_F16 ? launch_both_dim<float, _Float16>(a, p, s)
                                                  : launch_both_dim<float, __bf16>(a, p, s);
  if (e != hipSuccess) return W4A32_ELAUNCH;
  return from_hip(rows->act_bf16 ? launch_join_dim<__bf16>(a, p, s) : launch_join_dim<float>(a, p, s));
}

}  // extern "C"
