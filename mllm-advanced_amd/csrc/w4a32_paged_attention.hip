// Attention of a ragged batch over a paged cache: rows of one token, of a few drafted ones or of a prompt's portion.
//
// Work is cut into items of 16, 32 or 64 query rows that read the same kv head: of a sequence with n rows, the n * G pairs
// (token, head of the group of G) in that order. An item's keys are cut into tiles (32 keys of a 16-bit cache, 16 of an f32
// one), and the tiles of all items, in one row, are dealt to the workgroups in equal shares, whatever item they belong to. So a
// batch of short and long sequences is dealt evenly, one long sequence fills the chip, and a captured launch serves lengths
// that nobody knew when it was captured: every wavefront works the shares out from the lengths. Where an item is shared, its
// workgroups leave their sums in scratch memory and a second launch joins them. (The last workgroup to arrive can join them
// without it, but took longer: its stores, its count and its loads each go through to memory, and it is one workgroup of many.
// 40 us against 33 for 16 sequences of 2 to 5 rows, 15 against 13 for one row of 200 tokens.)
//
// A wavefront has 16 query rows and takes its item's tiles in turn with the others that have the same rows; those join their
// softmax states through LDS. Both products are transposed, so that a lane stands for one query row (lane % 16) and keeps its
// softmax state:
//   S^T = K Q^T     A = K: lane = key l % 16, 8 dims (16-bit) or 4 (f32) straight from the row in memory
//   O^T += V^T P^T  A = V^T: the tile goes through LDS, where ds_read_b64_tr_b16 turns it (f32: plain reads of 4 bytes);
//                   B = the softmaxed S^T as it lies in the registers: lane group g holds keys 4 g .. 4 g + 3 of a half
// The matrix instruction's 16 columns are what a group of 6 or 7 heads needs; a kv head with one query head uses one of 16,
// which costs no time: a 16-bit tile of head size 128 is 16 kilobytes for 16 to 48 instructions of 16 clocks.
//
// What bounds it: memory where contexts are long: one row each of 64 sequences of 500 to 8000 tokens, 28 heads on 4 of 128 dims in
// bf16 (559 MB): 109 us, 5.1 TB/s, and 5 for the join; one row on 131001 tokens, 12 heads on 2, f32 on f16 (134 MB): 25 us, 5.3 TB/s,
// and 6. Below that a chain of waits: one row on 60 tokens takes 7.3 us, of which 1.4 are the launch, 0.6 the deal, 1.6 the
// place and q, 0.6 the keys and values, 1.9 the tile and 1.5 the wavefronts' join and the store.
#include "w4a32_paged_rows.h"

namespace w4 {
namespace paged {

namespace {
inline bool aligned(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }
inline int from_hip(hipError_t e) { return e == hipSuccess ? W4A32_OK : W4A32_ELAUNCH; }

// The prompts' kernel takes sequences of at least kPromptRows pairs of token and head, where it has kPromptLeast workgroups of 32
// rows or more: it does not share a row's keys between workgroups, and few of them on a long context would leave the chip idle.
// From kPromptWide workgroups of eight times as many rows on it has those (28 heads on 4, bf16: 512 rows 22 us with either, 2048
// rows 72 us against 131); from kPromptWideSlow on with f32 rows, two or three terms of each operand (1024 rows 64 us against 76 in favour of
// 32, 2048 rows 164 against 147), and with 256 dims (16 heads on 4, bf16: 1024 rows 57 against 63, 2048 rows 167 against 115).
// With an f32 cache and 128 or 256 dims it takes none below that (12 heads on 2: 1000 rows 148 us against 116 of the rows' kernel and its
// join, 2000 rows 287 against 358). Nor does it with f32 rows on a bf16 cache of 256 dims where a row has over kPromptKeysSpilt keys more
// than its sequence has rows: three terms of q and 128 sums of a lane do not fit into its registers (97 are spilled with 32 rows of a
// workgroup, 92 with 128; two terms, on an f16 cache, spill 15 and none). 16 heads on 4, 32 rows of a workgroup against the rows'
// kernel: 512 rows alone 65 us against 82, behind 256 tokens 95 against 98, behind 4096 544 against 276, of those with a window of 500
// 68 against 114; 1024 rows alone 140 against 159, behind 256 tokens 179 against 186, behind 4096 1087 against 544. (On an f16
// cache behind 4096: 512 rows 209 against 250, 1024 421 against 486.)
constexpr int kPromptRows = 256, kPromptLeast = 128, kPromptWide = 64, kPromptWideSlow = 160;
// Sequences of fewer rows are its too where a row has at most kPromptKeys keys: it goes through 2560 of them in 33 us with 32 rows
// of a workgroup and in 50 with more (4096: 54 and 80), beside the others, where the rows' two launches take 9 us for nothing and 17
// for a row of 4096 (256 + 1 rows, the latter on 4096 keys: 48 us against 30; 1024 + 1: 88 against 56).
constexpr int kPromptKeys = 2560, kPromptKeysF32 = 512, kPromptKeysSpilt = 256;
constexpr float kLog2e = 1.44269504088896340736f;
constexpr int kJoins = 1 << 20;   // workgroups of the joining launch, beyond which they take several rows each
// Where weights are added up the scores of a pass lie in scratch memory, 4 bytes for each row of a head and each token that the table
// has room for: a step of more rows than fit into kMostScores is gone through in passes of kLeastPass rows or more (28 heads on 4 of
// 128 dims, bf16: 8192 rows 5.7 ms with 0.97 GB against 7.5 ms with 7.6 GB at once; 2048 rows on a table for 131072 tokens 1.13 ms with
// 1.9 GB against 1.00 with 30).
constexpr size_t kMostScores = (size_t)1 << 30;
constexpr int kLeastPass = 128;

template <typename Act, typename KV, int DT, bool kDump>
__global__ __launch_bounds__(64 * kWaves, DT == 256 ? 1 : 2) void rows_kernel(Attend a) {
  rows_body<Act, KV, DT, kDump, kRest>(a, blockIdx.x, gridDim.x, 0, 0, 0);
}

// Joins the shares of an item: a workgroup per query row and kSlice of its values, its threads four values of every 256 /
// (kSlice / 4)th share each.
template <typename Act, int DT, int kSlice, bool kDump>
__device__ __forceinline__ void join(const Attend& a, unsigned unit) {
  constexpr int kPer = kSlice / 4, kAtOnce = 256 / kPer;
  __shared__ __attribute__((aligned(16))) float sums[4][kSlice];
  __shared__ float tops[4], totals[4];
  const int slice = unit % (DT / kSlice), r = unit / (DT / kSlice) % a.slot_rows;
  const unsigned item = unit / (DT / kSlice) / a.slot_rows;
  const unsigned count = *a.count;
  const Item it = a.item[item];
  if (item >= count || it.shares == 1 || r >= it.rows) return;
  const int d = slice * kSlice + threadIdx.x % kPer * 4, mine = threadIdx.x / kPer;
  float top = -INFINITY, sum = 0.0f;
  f32x4 acc = {0, 0, 0, 0};
  for (int x0 = mine; x0 < it.shares; x0 += 8 * kAtOnce) {
    float m[8], l[8];
    f32x4 v[8];
#pragma unroll
    for (int x = 0; x < 8; ++x) {
      const int i = x0 + x * kAtOnce;
      m[x] = -INFINITY;
      l[x] = 0.0f;
      v[x] = f32x4{0, 0, 0, 0};
      if (i < it.shares) {
        const size_t at = (size_t)(2 * (it.first + i) + (i == 0)) * a.slot_rows + r;
        m[x] = load_global<float>(a.state + 2 * at);
        l[x] = load_global<float>(a.state + 2 * at + 1);
        v[x] = load_global<f32x4>(a.part + at * DT + d);
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
  // the threads of a wavefront that have the same values, by moves, then the wavefronts
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
  finish<Act, kDump>(a, it.r0, it.row0 + r, it.head, (size_t)item * a.slot_rows + r, d, acc, base, sum);
}
template <typename Act, int DT, int kSlice, bool kDump>
__global__ __launch_bounds__(256) void join_kernel(Attend a, unsigned units) {
  for (unsigned u = blockIdx.x; u < units; u += gridDim.x) {
    join<Act, DT, kSlice, kDump>(a, u);
    if (units > gridDim.x) __syncthreads();
  }
}

// Adds the weights of a tile's keys up: a wavefront per tile of a kv head, over its items in order. It reads the scores that the
// rows' kernel left, 64 bytes a key and 16 rows: an eighth of the key itself with 128 dims of 16 bits (16 sequences of 300 to
// 4100 tokens, 2 to 5 rows of 12 heads on 2: 7 us of 32).
template <typename KV>
__global__ __launch_bounds__(64 * kWaves) void weights_kernel(Attend a) {
  constexpr int KT = tile_keys<KV>(), kHalves = KT / 16;
  Seqs<KT> seqs;
  if (deal_of(a, seqs, (unsigned)kGrid, 0).per == 0) return;
  const Place p = place_of(a, seqs, blockIdx.x, kKeyTiles, 1);
  if (!p.there) return;
  const int per_head = (p.q.nt + kWaves - 1) / kWaves, hk = (int)p.inner / per_head;
  const int t = (int)p.inner % per_head * kWaves + (threadIdx.x >> 6);
  if (t >= p.q.nt) return;
  const int lane = threadIdx.x & 63, row = lane & 15, grp = lane >> 4;
  const int k0 = (t < p.q.ft ? t : t - p.q.ft + p.q.w0) * KT;
  float w[4 * kHalves] = {};
  for (int i = 0; i < p.q.items << a.wide; ++i) {
    const int item = hk * p.q.items + (i >> a.wide), rt = i & ((1 << a.wide) - 1), r = rt * kRows + row;
    const u64 tile = (u64)p.tile0 + (u64)item * p.q.nt + t;
    const int all_rows = p.q.s.n * a.group, row0 = i * kRows;
    if (row0 >= all_rows) break;
    auto slot_of = [&](int r) { return p.q.s.len + by_group(a, r); };
    const Sight sight = sight_of<KT>(a, p.q, slot_of(row0), slot_of(min(row0 + kRows, all_rows) - 1));
    if (t >= sight.to || sight.skips(t)) continue;
    const bool real = row0 + row < all_rows;
    const float lse = real ? a.lse[((size_t)p.item0 + item) * a.slot_rows + r] : INFINITY;
    const float* from = a.dump + (((tile << a.wide) + rt) * 64 + lane) * (4 * kHalves);
    f32x4 x[kHalves];
#pragma unroll
    for (int h = 0; h < kHalves; ++h) x[h] = load_global<f32x4>(from + 4 * h);
    if (__builtin_expect(__any(lse != lse), 0)) {  // a row of NaN: it has no weight, not NaN, for the keys that it does not see
      const int pos = slot_of(row0 + row);
#pragma unroll
      for (int h = 0; h < kHalves; ++h)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int key = k0 + 16 * h + 4 * grp + e;
          const bool sees = real & (key <= pos) & ((a.window == 0) | (key > pos - a.window) | (key < a.first));
          w[4 * h + e] += sees ? pow2(x[h][e] - lse) : 0.0f;
        }
      continue;
    }
#pragma unroll
    for (int h = 0; h < kHalves; ++h)
#pragma unroll
      for (int e = 0; e < 4; ++e) w[4 * h + e] += real ? pow2(x[h][e] - lse) : 0.0f;
  }
#pragma unroll
  for (int i = 0; i < 4 * kHalves; ++i)
#pragma unroll
    for (int x = 1; x < 16; x <<= 1) w[i] += __shfl_xor(w[i], x);
  if (row != 0) return;
#pragma unroll
  for (int h = 0; h < kHalves; ++h) {
    const int key = k0 + 16 * h + 4 * grp;
    if (key >= p.q.keys) continue;
    const int page = a.c.table[(size_t)p.b * a.c.table_ld + (key >> a.c.shift)];
    if (!page_there(a.c, page)) continue;
    float* to = a.c.weight + slot_row(a.c, page, hk, key);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (key + i < p.q.keys) to[i] += w[4 * h + i];
  }
}

// ---- host ------------------------------------------------------------------------------------------------------------------
struct Plan {
  long long items, tiles, grid, key_groups;
  int dt, wide, slot_rows;
  bool join, sliced, others;  // others: rows that are not the prompts' kernel's
  int pass_rows;              // rows of the step that are gone through at a time
  int prompt_rows, prompt_log2;
  long long prompts;          // its workgroups
  size_t item_off, part_off, state_off, lse_off, dump_off, total;
};

inline size_t up256(size_t v) { return (v + 255) / 256 * 256; }

// The rows' launches over `rows` rows of the step, `most` of a sequence at most
int plan_rows(const w4a32_paged_cache* c, long long group, long long rows, long long most, long long seqs, int window, int first, bool accumulate, Plan& p) {
  const int kt = c->dtype == W4A32_CACHE_F32 ? 16 : 32;
  // 32 or 64 rows of an item are two or four wavefronts' that ask for the same keys at about the same time: the caches serve
  // all but the first, where as items of their own each would have the keys from memory again. But then fewer of a workgroup's
  // wavefronts share its tiles, so not where there are too few tiles to give every workgroup kMinTiles (16 + 5 rows of 11 heads on
  // 160 tokens: 18 us with 64 rows of an item, 10 with 16).
  long long tiles = ((long long)c->table_ld * c->page + kt - 1) / kt;
  for (p.wide = most * group <= kRows ? 1 : most * group <= 2 * kRows ? 2 : 4;; p.wide /= 2) {
    const long long of_item = kRows * p.wide, by_seq = (most * group + of_item - 1) / of_item * seqs,
                    by_rows = rows * group / of_item + seqs;
    p.items = (by_seq < by_rows ? by_seq : by_rows) * c->kv_heads;
    p.slot_rows = (int)(most * group < of_item ? most * group : of_item);
    if (p.wide == 1 || p.items * tiles >= kGrid * kMinTiles) break;
  }
  if (window) {
    const long long near = ((long long)first + kt - 1) / kt + (window + most) / kt + 2;
    tiles = near < tiles ? near : tiles;
  }
  p.tiles = p.items * tiles;
  p.grid = p.tiles < kGrid ? p.tiles : kGrid;
  p.key_groups = (long long)c->n_seqs * c->kv_heads * ((tiles + kWaves - 1) / kWaves);
  if (p.tiles >= (1ll << 31) || p.items * p.slot_rows >= kMost) return W4A32_ESHAPE;
  if (accumulate && p.key_groups > most_groups(64 * kWaves)) return W4A32_ESHAPE;
  // Nothing is shared where every item is short. Where a join of one workgroup per row leaves most CUs
  // without work, a row's values are dealt to several.
  p.join = tiles > kAlone;
  p.sliced = p.items * p.slot_rows <= 128;
  size_t at = 256;
  p.item_off = at;
  at = up256(at + (size_t)p.items * sizeof(Item));
  p.part_off = at;
  if (p.join) at = up256(at + (size_t)2 * kGrid * p.slot_rows * p.dt * 4);
  p.state_off = at;
  if (p.join) at = up256(at + (size_t)2 * kGrid * p.slot_rows * 2 * 4);
  p.lse_off = at;
  if (accumulate) at = up256(at + (size_t)p.items * p.slot_rows * 4);
  p.dump_off = at;
  if (accumulate) at = up256(at + (size_t)p.tiles * p.wide * kRows * kt * 4);
  p.total = p.others ? at : 256;  // the prompts' kernel needs none
  return W4A32_OK;
}

// W4A32_OK and what a call takes at most, whatever the device arrays say; `room`: scratch memory that there is
int plan_of(const w4a32_paged_cache* c, const w4a32_paged_rows* r, int window, int first, bool accumulate, size_t room, Plan& p) {
  const long long group = r->heads / c->kv_heads, cap = (long long)c->table_ld * c->page;
  long long most = r->max_rows < r->rows ? r->max_rows : r->rows;
  p.dt = c->dim <= 64 ? 64 : c->dim <= 128 ? 128 : 256;
  auto blocks = [&](int log2) { return ((long long)r->rows * group / (1 << log2) + c->n_seqs) * c->kv_heads; };
  const bool f32 = c->dtype == W4A32_CACHE_F32;
  const int wide = p.dt == 256 || f32 ? 7 : 8;
  const int from = r->act_bf16 && p.dt <= 128 ? kPromptWide : kPromptWideSlow;
  p.prompt_log2 = (f32 ? p.dt != 64 : blocks(wide) >= from) ? wide : 5;
  p.prompts = blocks(p.prompt_log2);
  long long keys = cap;  // that a row can see
  if (window) {
    const long long near = (long long)first + window;
    keys = near < cap ? near : cap;
  }
  p.prompt_rows = 0;
  p.others = true;
  const bool spilt = !r->act_bf16 && c->dtype == W4A32_CACHE_BF16 && p.dt == 256 && keys > most + kPromptKeysSpilt;
  const bool wide_only = (f32 && p.dt != 64) || spilt;
  if (!accumulate && most * group >= kPromptRows && (wide_only ? blocks(wide) >= from : blocks(5) >= kPromptLeast)) {
    // Where every sequence can have max_rows rows they all do, or the batch is padded: one kernel for all then, as where few
    // keys are what a row has to go through. Else the rows' kernel has what is left, of so few rows.
    p.others = r->rows < (long long)r->max_rows * c->n_seqs && keys > (f32 ? kPromptKeysF32 : kPromptKeys) && (kPromptRows - 1) / group > 0;
    p.prompt_rows = p.others ? kPromptRows : 1;
    most = p.others ? (kPromptRows - 1) / group : 1;
    if (p.prompts > most_groups(512)) return W4A32_ESHAPE;
  }
  auto pass_of = [&](int rows) {
    const bool whole = rows == r->rows;
    p.pass_rows = rows;
    return plan_rows(c, group, rows, whole || most < rows ? most : rows, whole || c->n_seqs < rows ? c->n_seqs : rows, window, first, accumulate, p);
  };
  if (!accumulate || r->rows <= kLeastPass) return pass_of(r->rows);
  // The longest passes whose scores fit, or take no more than those of the shortest: many sequences' rows do not get fewer
  const int least = pass_of(kLeastPass);
  if (least) return least;
  const size_t scores = p.total - p.dump_off > kMostScores ? p.total - p.dump_off : kMostScores;
  for (int rows = r->rows; rows > kLeastPass; rows = rows > 2 * kLeastPass ? (rows / 2 + 63) & -64 : kLeastPass)
    if (pass_of(rows) == W4A32_OK && p.total - p.dump_off <= scores && p.total <= room) return W4A32_OK;
  return pass_of(kLeastPass);
}

template <typename Act, typename KV, int DT>
hipError_t launch(Attend a, const Plan& p, bool accumulate, hipStream_t s) {
  constexpr size_t lds = lds_bytes<KV, DT>();
  auto kernel = accumulate ? rows_kernel<Act, KV, DT, true> : rows_kernel<Act, KV, DT, false>;
  if constexpr (lds > 64 * 1024) {
    static LdsLimitOnce limit[2];
    if (hipError_t e = limit[accumulate].raise((const void*)kernel, lds); e != hipSuccess) return e;
  }
  if (!p.others) return hipSuccess;
  for (a.row_lo = 0; a.row_lo < a.rows; a.row_lo = a.row_hi) {
    a.row_hi = a.rows - a.row_lo > p.pass_rows ? a.row_lo + p.pass_rows : a.rows;
    hipLaunchKernelGGL(kernel, dim3((unsigned)p.grid), dim3(64 * kWaves), lds, s, a);
    if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
    if (p.join) {
      auto join = p.sliced ? (accumulate ? join_kernel<Act, DT, 32, true> : join_kernel<Act, DT, 32, false>)
                           : (accumulate ? join_kernel<Act, DT, DT, true> : join_kernel<Act, DT, DT, false>);
      const long long units = p.items * p.slot_rows * (p.sliced ? DT / 32 : 1);
      hipLaunchKernelGGL(join, dim3((unsigned)(units < kJoins ? units : kJoins)), dim3(256), 0, s, a, (unsigned)units);
      if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
    }
    if (!accumulate) continue;
    hipLaunchKernelGGL((weights_kernel<KV>), dim3((unsigned)p.key_groups), dim3(64 * kWaves), 0, s, a);
    if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  }
  return hipSuccess;
}
template <typename Act, typename KV>
hipError_t launch_dim(const Attend& a, const Plan& p, bool accumulate, hipStream_t s) {
  if (p.dt == 64) return launch<Act, KV, 64>(a, p, accumulate, s);
  if (p.dt == 128) return launch<Act, KV, 128>(a, p, accumulate, s);
  return launch<Act, KV, 256>(a, p, accumulate, s);
}

int check(const w4a32_paged_cache* cache, const w4a32_paged_rows* rows, int accumulate) {
  if (int e = check_rows(cache, rows)) return e;
  if (!rows->d_q || !rows->d_out) return W4A32_EINVAL;
  if (accumulate && !cache->d_weight) return W4A32_EINVAL;
  return W4A32_OK;
}
}  // namespace

int plan_own(const w4a32_paged_cache* c, const w4a32_paged_rows* r, OwnPlan& o) {
  Plan p;
  p.dt = c->dim <= 64 ? 64 : c->dim <= 128 ? 128 : 256;
  p.others = true;
  const long long most = r->max_rows < r->rows ? r->max_rows : r->rows;
  if (int e = plan_rows(c, r->heads / c->kv_heads, r->rows, most, c->n_seqs, 0, 0, false, p)) return e;
  o = {p.items, p.tiles, (unsigned)(kOwnSlots + p.items), p.wide == 4 ? 2 : p.wide - 1, p.slot_rows, p.dt};
  return W4A32_OK;
}

}  // namespace paged
}  // namespace w4

using namespace w4::paged;

extern "C" {

size_t w4a32_op_paged_attention_window_scratch_bytes(const w4a32_paged_cache* cache, const w4a32_paged_rows* rows, int window, int first,
                                                     int accumulate) {
  Plan p;
  if (check(cache, rows, accumulate) || window < 0 || first < 0) return 0;
  return plan_of(cache, rows, window, first, accumulate != 0, SIZE_MAX, p) ? 0 : p.total;
}

size_t w4a32_op_paged_attention_scratch_bytes(const w4a32_paged_cache* cache, const w4a32_paged_rows* rows, int accumulate) {
  return w4a32_op_paged_attention_window_scratch_bytes(cache, rows, 0, 0, accumulate);
}

int w4a32_op_paged_attention(const w4a32_paged_cache* cache, const w4a32_paged_rows* rows, float scale, int window, int first,
                             int accumulate, void* d_scratch, size_t scratch_bytes, void* stream) {
  if (int e = check(cache, rows, accumulate)) return e;
  if (window < 0 || first < 0 || !(scale * kLog2e - scale * kLog2e == 0.0f) || !d_scratch || !aligned(d_scratch, 16)) return W4A32_EINVAL;
  Plan p;
  if (int e = plan_of(cache, rows, window, first, accumulate != 0, scratch_bytes, p)) return e;
  if (scratch_bytes < p.total) return W4A32_EINVAL;
  uint8_t* scratch = static_cast<uint8_t*>(d_scratch);
  Attend a{view(cache), rows->d_q, rows->d_out, rows->d_row_start, rows->ldq, rows->ldo, rows->rows,
                 rows->max_rows < rows->rows ? rows->max_rows : rows->rows, rows->heads, rows->heads / cache->kv_heads, 0, 0, 0, rows->rows, window, first,
                 p.prompt_rows, p.prompt_log2, p.wide == 4 ? 2 : p.wide - 1, p.slot_rows, (unsigned)p.items, (unsigned)p.tiles, scale * kLog2e,
                 (Item*)(scratch + p.item_off), (unsigned*)scratch, (float*)(scratch + p.part_off),
                 (float*)(scratch + p.state_off), (float*)(scratch + p.lse_off), (float*)(scratch + p.dump_off)};
  set_group(a);
  hipStream_t s = static_cast<hipStream_t>(stream);
  const bool acc = accumulate != 0;
  if (p.prompt_rows)
    if (hipError_t e = launch_prompts(a, cache->dtype, rows->act_bf16 != 0, p.dt, (unsigned)p.prompts, s); e != hipSuccess)
      return W4A32_ELAUNCH;
  if (rows->act_bf16) return from_hip(launch_dim<__bf16, __bf16>(a, p, acc, s));
  if (cache->dtype == W4A32_CACHE_F32) return from_hip(launch_dim<float, float>(a, p, acc, s));
  if (cache->dtype == W4A32_CACHE_F16) return from_hip(launch_dim<float, _Float16>(a, p, acc, s));
  return from_hip(launch_dim<float, __bf16>(a, p, acc, s));
}

}  // extern "C"
