// Attention of a batch whose sequences share prefixes in groups: a prefix's keys and values are read once for all rows of the group.
//
// A row's softmax is joined from its sums over the prefix and those over its sequence's own tokens, each relative to its maximum:
//   m = max(m_P, m_own),  l = 2^(m_P - m) l_P + 2^(m_own - m) l_own,  o = 2^(m_P - m) o_P + 2^(m_own - m) o_own.
// The prefix is the prompts' kernel's with the rows of all of the group's sequences, which all see all of it, 128 rows of a workgroup, and its keys dealt to
// as many workgroups as the chip has room for; the own tokens are the rows' kernel's, and those of long prompts the prompts' kernel's again. All
// of these are workgroups of one launch, so that none waits for another kind, and each works out by itself what it has (the lengths and the
// groups are device memory; a launch in front does that for batches that a wavefront's lanes cannot hold); a second launch joins the sums, in a
// fixed order.
// What bounds it. 64 sequences behind 8003 tokens with 16 to 1200 of their own (28 heads on 4 of 128, bf16): 97 MB, 20 us of memory; 35 us and 5.4 of
// join. A workgroup of the own tokens takes 16 us, of which its loop over tiles is 8 (the deal 2, the first loads 4, its sums 2), and there are
// three rounds of them beside the prefix. 48 sequences of two to five rows in six groups behind 1000 to 6000 tokens, 12 heads on 2, f32 on f16: 30 and 6
// us, as an f32 operand is two f16 terms and a tile's product waits for its loads more than it takes. Eight prompts of 60 to 300 rows behind 4099
// tokens, 28 heads on 4, bf16: 97 GFLOP, 133 and 13 us, 865 TFLOP/s for each further token of the prefix: products and softmax of a wavefront
// take turns more than they overlap.
// 256 dims: one workgroup fits on a CU, and f32 rows on a bf16 cache do not fit into its registers (70 spilled; 4 with 128 dims). Prefixes go by this kernel all
// the same. 16 heads on 4 of 256, both launches against those of the rows on their own, us: the 64 sequences bf16 85 and 226, f32 on f16 99 and
// 240, f32 on bf16 120 and 272, f32 180 and 581; the 48 of two to five rows 83 and 187, 98 and 202, 141 and 223, 256 and 458; the prompts 243
// and 239, 360 and 372, 558 and 609, 1251 and 1309; four rows behind 200 tokens 16 and 15, 18 and 17, 18 and 17, 23 and 17.
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
// Workgroups that are there at once: two per CU. (256 dims: one, so that the deal's round is two there. What follows from it, here and in the rows' deal,
// was measured on 28 heads on 4 of 128 dims in bf16 and on 12 on 2 of 128, f32 on f16, and stands for all types and sizes.)
constexpr int kSlots = 512;
constexpr int kMostShares = kSlots * 7 / 8;  // of prefixes, where their items are not more
constexpr unsigned kUnits = 896;  // most workgroups where prefixes have kMostShares at most: those that find nothing take their time, too
constexpr int kLog2 = 7;         // log2 of the rows of a workgroup of a prefix
// Pairs of row and head from which on a sequence's own tokens go by blocks of 128 rows as well, and not by 16 of a wavefront (eight prompts of 60 to
// 300 rows, 28 heads on 4, bf16: behind 64 tokens 46 us against 68, behind 4099 141 against 148; 64, 256, 512: the same).
constexpr int kOwnPromptRows = 128;
constexpr int kManyRows = 1024;  // rows from which on a workgroup joins several of them
constexpr int kJoins = 1 << 20;  // workgroups of the joining launch, beyond which they take more

// Sequences up to which every wavefront deals the batch by itself, one in each lane, where there are few groups, which it goes through one by one (64
// sequences behind prefixes of 500 tokens, 28 heads on 4, bf16: one group 18 us against 24 with a launch in front, 4 groups 20 against 23, 8 the same, 16 31
// against 26; 12 heads on 2, f32 on f16, two to five rows each: 21 against 29, 22 against 29, 23 against 30, 24 against 29).
constexpr int kLanes = 64, kLaneGroups = 8;

__device__ __forceinline__ unsigned wave_sum(unsigned x) { return last_lane(wave_scan(x)); }  // sums that do not fit are the most
__device__ __forceinline__ int wave_min(int x) {
#define W4_MIN(ctrl, rows) x = min(x, __builtin_amdgcn_update_dpp(0x7fffffff, x, ctrl, rows, 0xf, false))
  W4_MIN(0x111, 0xf);  // row_shr 1, 2, 4, 8
  W4_MIN(0x112, 0xf);
  W4_MIN(0x114, 0xf);
  W4_MIN(0x118, 0xf);
  W4_MIN(0x142, 0xa);  // row_bcast 15, 31
  W4_MIN(0x143, 0xc);
#undef W4_MIN
  return __builtin_amdgcn_readlane(x, 63);
}

// A group whose sequences with rows, `with_rows` of them, have `least` tokens or more, rows from r0 to before r1: one such sequence alone has no
// prefix. Whose pages have it is for the caller to say: sequence b0's where they do, else those of the next that has so many tokens, as
// each with rows does (b0 may have ended, and have given its pages back).
__device__ __forceinline__ PrefixGroup group_of(const Attend& a, int b0, int with_rows, int least, int r0, int r1) {
  PrefixGroup q = {b0, 0, 0, 0, 0, 0, 0, 0};
  if (with_rows < 2 || least <= 0) return q;
  q.tokens = least;
  q.r0 = r0;
  q.n = max(r1 - r0, 0);
  q.blocks = (int)(((long long)q.n * a.group + (1 << kLog2) - 1) >> kLog2);
  return q;
}
// Tiles of a wavefront each, of the tokens behind `from`
template <int kKeys>
__device__ __forceinline__ unsigned own_tiles(const Attend& a, const Span& s, int from) {
  if (s.n == 0) return 0;
  const int keys = min(s.len + s.n, a.c.cap), first = min(from, a.c.cap - 1);
  const unsigned long long n = ((unsigned long long)s.n * a.group + 15) / 16 * (unsigned)((keys + kKeys - 1) / kKeys - first / kKeys);
  return (unsigned)min(n, 0xffffffffull);
}
// Numbers of shares and tiles, as sums of them: what does not fit is the most, so that a batch of too many is found to have too many
constexpr __host__ __device__ unsigned times(unsigned a, unsigned b) { return (u64)a * b > 0xffffffffu ? 0xffffffffu : a * b; }
constexpr __host__ __device__ unsigned parts(unsigned a, unsigned of) { return a / of + (a % of != 0); }  // of `of` each; a may be the most
static_assert(times(128, 1u << 25) == 0xffffffffu && times(896, times(1u << 16, 1u << 16)) == 0xffffffffu && times(3, 5) == 15 && times(0, 7) == 0, "");
static_assert(parts(0xffffffffu, 448) == 9586981 && parts(0, 3) == 0 && parts(6, 3) == 2 && parts(7, 3) == 3, "");
// Tiles of a prefix that a share of it has: the slots of the chip go to the prefixes and to the own tokens as their work is estimated (a workgroup
// takes 3 units of time for a tile of a prefix, 8 for kWaves tiles of own tokens), and an item gets as few shares as keep to that. But a share
// costs as well: its sums are written and read again, some 50 ns where all of a workgroup's rows are there, against 1 us for a tile (f32: 5), so
// that sqrt(tiles * 50 / 1000) tiles of a share take the least time together (six groups of eight, 12 heads on 2, f32 on f16, behind 1000
// tokens: 28 us against 36 with a tile of a share). count(per): shares of `per` tiles that all items have. Whole shares: ceil(tiles / (most - items))
// tiles always leave no more than `most`.
template <bool kF32, typename Count>
__device__ __forceinline__ unsigned share_of(const Attend& a, unsigned tiles, unsigned items, unsigned pairs, unsigned own, Count count) {
  const float work = (float)tiles * 3.0f, rest = (float)own * a.c.kv_heads * (8.0f / kWaves);
  unsigned most = min(max((unsigned)(kSlots * (work / (work + rest + 1.0f)) + 0.5f), (unsigned)kSlots / 4), (unsigned)kMostShares);
  if (2 * items > most) most *= 2;  // in two rounds, so that what one leaves over is small
  most = min(most, (unsigned)a.prefix.grid);
  if (most <= items) return 1u << 30;
  const float rows = (float)pairs / ((float)max(items, 1u) * (1 << kLog2));  // of those that a workgroup has room for
  const unsigned least = max((unsigned)(__builtin_sqrtf((float)tiles * rows * (kF32 ? 0.01f : 0.05f)) + 0.5f), 1u);
  unsigned lo = max(parts(tiles, most), least), per = max(parts(tiles, most - items), lo);
  while (lo < per) {
    const unsigned mid = (lo + per) / 2;
    if (count(mid) <= most)
      per = mid;
    else
      lo = mid + 1;
  }
  return per;
}
template <int kKeys>
__device__ __forceinline__ unsigned tiles_of(const PrefixGroup& q) { return (unsigned)(q.tokens + kKeys - 1) / kKeys; }

// What this lane's group and this lane's sequence have, by each wavefront
struct Mine {
  int total;      // workgroups that have a share of a prefix
  PrefixGroup q;  // of group `lane`
  int from, of;   // of sequence `lane`
};
__device__ __forceinline__ PrefixGroup of_lane(const PrefixGroup& q, int at) {
  auto from = [&](int x) { return __builtin_amdgcn_readlane(x, at); };
  return {from(q.b), from(q.r0), from(q.n), from(q.tokens), from(q.first), from(q.shares), from(q.blocks), 0};
}
template <int kKeys, int kOwnKeys, bool kF32>
__device__ __forceinline__ Mine deal_by_lanes(const Attend& a) {
  const Prefix& x = a.prefix;
  const int lane = threadIdx.x & 63, n_seqs = a.c.n_seqs;
  Mine m = {0, {}, 0, -1};
  Span s = {};
  int end = 0, b0 = 0, b1 = 0, want = 0;
  if (lane < n_seqs) {
    s = span_of(a.c, a.row_start, a.rows, a.max_rows, lane);
    end = min(a.row_start[lane + 1], a.rows);
  }
  if (lane < x.n_groups) {
    b0 = min(max(x.group_start[lane], 0), n_seqs);
    b1 = min(max(x.group_start[lane + 1], b0), n_seqs);
    want = min(x.tokens[lane], a.c.cap);
  }
  for (int g = 0; g < x.n_groups; ++g) {
    const int lo = __builtin_amdgcn_readlane(b0, g), hi = __builtin_amdgcn_readlane(b1, g);
    if (lo == hi) continue;
    const bool in = lane >= lo && lane < hi, has = in && s.n > 0;
    const int least = wave_min(has ? s.len : __builtin_amdgcn_readlane(want, g));
    PrefixGroup q = group_of(a, lo, __popcll(__ballot(has)), min(least, __builtin_amdgcn_readlane(want, g)), __builtin_amdgcn_readlane(s.r0, lo),
                             __builtin_amdgcn_readlane(end, hi - 1));
    if (q.tokens) q.b = __builtin_ctzll(__ballot(in && s.len >= q.tokens));
    if (lane == g) m.q = q;
    if (in && q.tokens) {
      m.from = q.tokens;
      m.of = g;
    }
  }
  const unsigned of_group = (unsigned)m.q.blocks * a.c.kv_heads, tiles = tiles_of<kKeys>(m.q);
  const unsigned pairs = (unsigned)(m.q.n * a.group) * a.c.kv_heads;
  const unsigned per = share_of<kF32>(a, wave_sum(times(of_group, tiles)), wave_sum(of_group), wave_sum(pairs), wave_sum(own_tiles<kOwnKeys>(a, s, m.from)),
                                      [&](unsigned n) { return wave_sum(times(of_group, (tiles + n - 1) / n)); });
  m.q.shares = (int)((tiles + per - 1) / per);
  const unsigned n = times(of_group, (unsigned)m.q.shares), upto = wave_scan(n);
  m.q.first = (int)(upto - n);
  m.total = (int)last_lane(upto);
  if ((unsigned)m.total > (unsigned)x.grid) m = {0, {}, 0, -1};  // row or group starts that decrease: all read everything by themselves
  return m;
}

// The same for many sequences, by a launch of its own: a wavefront per group, then one for all groups
template <int kKeys, int kOwnKeys, bool kF32>
__global__ __launch_bounds__(kPlan) void deal_kernel(Attend a) {
  __shared__ unsigned of_wave[kPlan / 64];
  const Prefix& x = a.prefix;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n_seqs = a.c.n_seqs;
  for (int b = tid; b < n_seqs; b += kPlan) {
    x.from[b] = 0;
    x.group_of[b] = -1;
  }
  __syncthreads();
  for (int g = wave; g < x.n_groups; g += kPlan / 64) {
    const int b0 = min(max(x.group_start[g], 0), n_seqs), b1 = min(max(x.group_start[g + 1], b0), n_seqs);
    int least = min(x.tokens[g], a.c.cap), with_rows = 0;
    for (int b = b0 + lane; b - lane < b1; b += 64) {
      Span s = {};
      if (b < b1) s = span_of(a.c, a.row_start, a.rows, a.max_rows, b);
      with_rows += __popcll(__ballot(s.n > 0));
      if (s.n > 0) least = min(least, s.len);
    }
    PrefixGroup q = group_of(a, b0, with_rows, wave_min(least), min(max(a.row_start[b0], 0), a.rows), min(a.row_start[b1], a.rows));
    for (u64 found = 0; q.tokens && !found && q.b < b1; q.b += found ? __builtin_ctzll(found) : 64)
      found = __ballot(q.b + lane < b1 && a.c.len[min(q.b + lane, b1 - 1)] >= q.tokens);
    if (lane == 0) x.group[g] = q;
    if (q.tokens)
      for (int b = b0 + lane; b < b1; b += 64) {
        x.from[b] = q.tokens;
        x.group_of[b] = g;
      }
  }
  __syncthreads();
  unsigned own = 0;
  for (int b = tid; b < n_seqs; b += kPlan) own = add_sat(own, own_tiles<kOwnKeys>(a, span_of(a.c, a.row_start, a.rows, a.max_rows, b), x.from[b]));
  own = wave_sum(own);
  if (lane == 0) of_wave[wave] = own;
  __syncthreads();
  if (wave != 0) return;
  own = 0;
#pragma unroll
  for (int w = 0; w < kPlan / 64; ++w) own = add_sat(own, of_wave[w]);
  auto all = [&](auto of) {  // of all groups together, per kv head
    unsigned sum = 0;
    for (int g = lane; g < x.n_groups; g += 64) sum = add_sat(sum, times(of(x.group[g]), (unsigned)a.c.kv_heads));
    return wave_sum(sum);
  };
  typedef const PrefixGroup& Q;
  const unsigned per = share_of<kF32>(a, all([](Q q) { return times((unsigned)q.blocks, tiles_of<kKeys>(q)); }), all([](Q q) { return (unsigned)q.blocks; }),
                                      all([&](Q q) { return (unsigned)(q.n * a.group); }), own,
                                      [&](unsigned n) { return all([&](Q q) { return times((unsigned)q.blocks, (tiles_of<kKeys>(q) + n - 1) / n); }); });
  unsigned total = 0;
  for (int g0 = 0; g0 < x.n_groups; g0 += 64) {
    const int g = g0 + lane;
    PrefixGroup q = {};
    if (g < x.n_groups) q = x.group[g];
    q.shares = (int)((tiles_of<kKeys>(q) + per - 1) / per);
    const unsigned n = times((unsigned)q.blocks * a.c.kv_heads, (unsigned)q.shares), upto = wave_scan(n);
    q.first = (int)(total + upto - n);
    if (g < x.n_groups) x.group[g] = q;
    total = add_sat(total, last_lane(upto));
  }
  const bool fits = total <= (unsigned)x.grid;
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
  using Sh = Shape<Act, KV, DT, kHalfForm>;
  static_assert(Sh::kThreads == 64 * kWaves && 32 * Sh::kMembers == 1 << kLog2, "workgroups of either kind");
  const Prefix& x = a.prefix;
  int unit = blockIdx.x;
  const int lane = threadIdx.x & 63;
  Mine m = {0, {}, 0, -1};
  if (x.from)
    m.total = *x.total;
  else
    m = deal_by_lanes<Sh::kKeys, tile_keys<KV>(), sizeof(KV) == 4>(a);
  if (unit < m.total) {
    // the last group whose first workgroup is this one or stands in front of it; groups without any are passed over
    PrefixGroup g;
    if (x.from) {
      int before = 0;
      for (int g0 = 0; g0 < x.n_groups; g0 += 64) before += __popcll(__ballot(g0 + lane < x.n_groups && x.group[g0 + lane].first <= unit));
      g = x.group[before - 1];
    } else {
      g = of_lane(m.q, __popcll(__ballot(lane < x.n_groups && m.q.first <= unit)) - 1);
    }
    const unsigned kv = a.c.kv_heads, in = (unsigned)(unit - g.first), in_kv = in / kv, share = in_kv / g.blocks;
    const unsigned tiles = tiles_of<Sh::kKeys>(g), each = tiles / g.shares, more = tiles - each * g.shares, first = each * share + min(share, more);
    const size_t row = (size_t)unit << kLog2;
    const Piece piece{g.b, {g.r0, g.n, g.tokens - 1}, (int)(in - in_kv * kv), (int)(in_kv - share * g.blocks), (int)first,
                      (int)(first + each + (share < more)), 0, x.part + row * DT, x.state + 2 * row};
    prompt_body<Act, KV, DT, kHalfForm, kPrefixTokens>(a, 0, piece);
    return;
  }
  unit -= m.total;
  auto group_at = [&](int b) {
    const int of = x.from ? x.group_of[b] : __builtin_amdgcn_readlane(m.of, b);
    return of < 0 ? PrefixGroup{} : x.from ? x.group[of] : of_lane(m.q, of);
  };
  if (a.prompt_rows) {
    Seqs<Sh::kKeys, kOwnPrompt> prompts;
    Seqs<tile_keys<KV>(), kOwn> seqs;
    prompts.own_from = seqs.own_from = m.from;
    unsigned blocks = 0, items = 0;
    for (int b0 = 0; b0 < a.c.n_seqs; b0 += 64) {
      prompts.load(a, b0);
      seqs.load(a, b0);
      blocks = add_sat(blocks, last_lane(wave_scan(prompts.items)));
      items = add_sat(items, last_lane(wave_scan(seqs.items)));
    }
    if (blocks > (unsigned)x.blocks || items > a.most_items) {  // row starts that overlap
      if (unit == 0 && threadIdx.x == 0) *a.count = 0;
      return;
    }
    if ((unsigned)unit < blocks) {
      const Place p = place_of(a, prompts, blocks - 1 - unit, kItems, 1);  // late rows first, which see most keys
      if (!p.there) return;
      // the items of the rows' kernel that this block is, by the sequences in front
      unsigned first = 0;
      for (int b0 = 0; b0 <= p.b; b0 += 64) {
        if (a.c.n_seqs > 64) seqs.load(a, b0);
        const unsigned upto = wave_scan(seqs.items);
        first += b0 + 64 <= p.b ? last_lane(upto) : (unsigned)__builtin_amdgcn_readlane((int)(upto - seqs.items), p.b - b0);
      }
      const int block = (int)(p.inner / (unsigned)a.c.kv_heads), hk = (int)p.inner - block * a.c.kv_heads, log2 = 4 + a.wide;
      const int all_rows = p.q.s.n * a.group, of_seq = (all_rows + (1 << log2) - 1) >> log2, of_block = 1 << (kLog2 - log2);
      first += (unsigned)(hk * of_seq + block * of_block);
      const PrefixGroup g = group_at(p.b);
      if ((int)threadIdx.x < min(of_block, of_seq - block * of_block)) {
        const int row0 = (block << kLog2) + ((int)threadIdx.x << log2);
        x.item[first + threadIdx.x] = own_item(a, {0, 1, p.q.s.r0, row0, min(all_rows - row0, 1 << log2), hk}, p.q.s.n, g);
      }
      const size_t row = (size_t)(kOwnSlots + first) * a.slot_rows;
      prompt_body<Act, KV, DT, kHalfForm, kOwnTokens>(a, 0, {p.b, p.q.s, hk, block, 0, 0, p.q.from, a.part + row * DT, a.state + 2 * row});
      return;
    }
    unit -= (int)blocks;
    m.total += (int)blocks;
  }
  // As many as there is room for beside the prefixes begin at once, if that leaves them short enough: shares are whole, and some four fifths of the
  // workgroups that they are dealt to get one (64 sequences with 16 to 1200 tokens of their own, 28 heads on 4, bf16: behind eight prefixes of 1000 tokens 33 us
  // against 38 with more and shorter ones; 48 behind six of 3000 32 against 36, of 6000 39 against 43).
  const unsigned one_round = (unsigned)max(kSlots - m.total, 0) * 5 / 4;
  const int own_grid = min(x.own_grid, (int)gridDim.x - m.total);
  if (unit < own_grid) rows_body<Act, KV, DT, false, kOwn>(a, (unsigned)unit, (unsigned)own_grid, one_round, m.from, group_at);
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
    for (int i0 = 0; i0 < s.count; i0 += 8) add_shares<DT, 8, 1>(a, s, item, r, d, i0, top, sum, acc);
    finish<Act, false>(a, s.own.r0, s.own.row0 + r, s.own.head, 0, d, acc, top == -INFINITY ? 0.0f : top, sum);
  }
}

// ---- host ------------------------------------------------------------------------------------------------------------------
struct Plan {
  OwnPlan own;
  bool dealt;       // by a launch in front
  int prompt_rows;  // pairs of a sequence from which on it goes by blocks of them, of which there are `blocks`; 0: none does
  unsigned blocks;
  unsigned grid, own_grid;  // workgroups of the prefixes, and of own tokens
  size_t group_off, from_off, of_off, item_off, part_off, state_off, pre_part_off, pre_state_off, total;
};

int plan_of(const w4a32_paged_cache* c, const w4a32_paged_rows* r, int n_groups, Plan& p) {
  if (int e = plan_own(c, r, p.own)) return e;
  const long long group = r->heads / c->kv_heads;
  const int dt = p.own.dt;
  p.dealt = c->n_seqs > kLanes || n_groups > kLaneGroups;
  const long long items = (((long long)r->rows * group >> kLog2) + n_groups) * c->kv_heads;
  // No more workgroups than can have something to do: each that has nothing finds that out by dealing the batch
  const long long grid = 2 * items <= kMostShares ? kMostShares : items > 2 * kMostShares ? items : 2 * kMostShares;
  // Own tokens: more than are there at once where items are many, so that most of them have a share of one item and no more (64 sequences of 16 to
  // 1200 tokens behind 8003, 4 kv heads: 47 us with 768, 51 with 512, 57 with 320, of which most have the end of one item and the start of the
  // next), else one per CU (11 sequences: 29 us with 512, 32 with 768)
  const long long own = 3 * p.own.items;
  p.own_grid = (unsigned)(own < kSlots / 2 ? kSlots / 2 : own > kOwnGrid ? kOwnGrid : own);
  const long long most = r->max_rows < r->rows ? r->max_rows : r->rows;
  p.prompt_rows = most * group >= kOwnPromptRows ? kOwnPromptRows : 0;
  const long long blocks = p.prompt_rows ? (((long long)r->rows * group >> kLog2) + c->n_seqs) * c->kv_heads : 0;
  if (grid + blocks + p.own_grid > most_groups(64 * kWaves)) return W4A32_ESHAPE;
  p.blocks = (unsigned)blocks;
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
  if (p.dealt) {
    hipLaunchKernelGGL((deal_kernel<Shape<Act, KV, DT, kHalfForm>::kKeys, tile_keys<KV>(), sizeof(KV) == 4>), dim3(1), dim3(kPlan), 0, s, a);
    if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  }
  const unsigned units = p.grid + p.own_grid, most = p.grid == kMostShares && units > kUnits ? kUnits : units;
  hipLaunchKernelGGL((both_kernel<Act, KV, DT>), dim3(most + p.blocks), dim3(64 * kWaves), lds, s, a);
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
  auto at = [&](size_t off) { return p.dealt ? (int*)(scratch + off) : nullptr; };
  const Prefix x{d_group_start, d_prefix, n_groups, (int)p.grid, (int)p.blocks, (int)p.own_grid, (OwnItem*)(scratch + p.item_off), (float*)(scratch + p.pre_part_off),
                 (float*)(scratch + p.pre_state_off), at(128), (PrefixGroup*)at(p.group_off), at(p.from_off), at(p.of_off)};
  Attend a{view(cache), rows->d_q, rows->d_out, rows->d_row_start, rows->ldq, rows->ldo, rows->rows,
           rows->max_rows < rows->rows ? rows->max_rows : rows->rows, rows->heads, rows->heads / cache->kv_heads, 0, 0, 0, rows->rows, 0, 0, p.prompt_rows, kLog2,
           p.own.wide, p.own.slot_rows, (unsigned)p.own.items, (unsigned)p.own.tiles, scale * kLog2e, nullptr,
           (unsigned*)scratch, (float*)(scratch + p.part_off), (float*)(scratch + p.state_off), nullptr, nullptr, x};
  set_group(a);
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int dtype = cache->dtype;
  const bool bf16 = rows->act_bf16 != 0;
  const hipError_t e = bf16                        ? launch_both_dim<__bf16, __bf16>(a, p, s)
                       : dtype == W4A32_CACHE_F32 ? launch_both_dim<float, float>(a, p, s)
                       : dtype == W4A32_CACHE_F16 ? launch_both_dim<float, _Float16>(a, p, s)
                                                  : launch_both_dim<float, __bf16>(a, p, s);
  if (e != hipSuccess) return W4A32_ELAUNCH;
  return from_hip(rows->act_bf16 ? launch_join_dim<__bf16>(a, p, s) : launch_join_dim<float>(a, p, s));
}

}  // extern "C"
