// Attention of prompts over a paged cache: the sequences of a batch that have so many rows that products bound them and not the
// cache.
//
// A workgroup has 256 query rows of one kv head (pairs of token and head of the group, 32 to a wavefront; 128 where a head has 256
// dims) and takes the keys that they can see through LDS, in tiles of 128 (64 of 256 dims): the next tile goes from memory
// straight to the other half of it (global_load_lds_dwordx4) while this one is multiplied. A tile's keys are worked through 64 at
// a time, or 32 where an f32 operand is two or three terms, so that a step's scores stay in registers. Against 128 rows and tiles
// of 64 a key is read half as often and waited for half as often (two prompts: 163 -> 154 us). Both products are transposed as in
// the rows' kernel, on v_mfma_f32_32x32x16: a lane stands for query row lane % 32, and lanes l and l + 32 share it.
//   S^T = K Q^T     A = K from LDS: lane = key l % 32, dims 16 c + 8 (l / 32) ..; B = Q in registers
//   O^T += V^T P^T  B = the softmaxed S^T registers: half h of the wavefront has keys 8 b + 4 h .. + 3 of a block of 32;
//                   A = V^T: ds_read_b64_tr_b16 of the same keys
// What bounds it: 64 keys and 128 dims cost a SIMD 32 x 32 = 1024 clocks of bf16 products per wavefront, and about as many of
// maxima, exponentials and sums, of which the other wavefront of the SIMD covers only a part: the matrix units are busy for 38% of
// the time (2048 + 1024 rows, 28 heads on 4 of 128 dims, bf16: 150 us, 765 TFLOP/s where all workgroups run). So the sums' reference
// follows a row's maximum only when that has grown by more than 2^kSlack: the 64 products that bring the sums to a new reference
// are then rare, and weights of up to 2^kSlack are as exact as those up to 1 (f16 has its weights' scale lowered for them).
// A wavefront's load fills 1024 bytes of LDS in lane order, so rows have no padding between them; instead the 16-byte pieces of a
// row of K lie exchanged by its number (a read of 16 rows then meets every bank once), and so do the 32-byte pieces of a row of V
// (the 8 rows of 64 bytes of a transposing read meet every bank twice, which is what they take): each lane asks for the piece that
// belongs where its 16 bytes go.
// Rows of one kv head lie together, so that a group of heads reads a key once; workgroups of consecutive numbers have
// consecutive kv heads, which the dispatcher deals to the XCDs in turn: an L2 sees few heads. Late rows, which see most keys,
// come first.
// Where there are few such workgroups, one has 32 rows instead, and each of its four wavefronts (two where the head has 256 dims)
// takes every fourth tile by itself, with no barrier; their softmax states are joined through LDS at the end.
// An f32 cache has tiles of 32 keys and v_mfma_f32_32x32x2, to which a lane gives one element of K or V: a tile of 128 dims
// costs a SIMD 128 x 64 = 8192 clocks per wavefront, beside which the rest is small (4096 rows, 28 heads on 4: 0.95 ms, 126 TFLOP/s, where
// the rows' kernel takes 3.15). 64 dims are always taken in the second way (2600 rows of 14 heads: 179 us against 237), 128 and 256, for
// which LDS has not the room, always in the first, with 128 rows of a workgroup.
#include "w4a32_paged_attention.h"

namespace w4 {
namespace paged {

namespace {
typedef float f32x16 __attribute__((ext_vector_type(16)));
constexpr int kSlack = 8;

__device__ __forceinline__ f32x16 mfma32(bf8 a, bf8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x16 mfma32(h8 a, h8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x16 mfma32(float a, float b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x2f32(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x16 mfma32(f8 a, f8 b, f32x16 c) {
#pragma unroll
  for (int i = 0; i < 8; ++i) c = mfma32(a[i], b[i], c);
  return c;
}

// A team of kMembers wavefronts shares tiles and has 32 rows of each; with kSplit a workgroup has several teams, of one wavefront
// each, on the same rows.
template <typename Act, typename KV, int DT, bool kSplit>
struct Shape {
  static constexpr int kTerms = Math<Act, KV>::kTerms;
  static constexpr bool k32 = sizeof(KV) == 4;
  static constexpr int kMembers = kSplit ? 1 : DT == 256 || k32 ? 4 : 8, kTeams = !kSplit ? 1 : DT == 256 ? 2 : 4;
  static constexpr int kThreads = 64 * kMembers * kTeams;
  static constexpr int kKeys = kSplit || k32 ? 32 : DT == 256 ? 64 : 128;              // of a tile
  static constexpr int kStep = !kSplit && !k32 && kTerms == 1 && DT <= 128 ? 64 : 32;  // of a step of the softmax
  static constexpr int kTile = kKeys * DT;                          // elements of a tile of K or V
  static constexpr size_t kTeam = (size_t)4 * kTile * sizeof(KV);   // bytes of a team's tiles: K and V, twice
  static constexpr int kSums = DT + 4;                    // floats of a row of sums, where teams are joined
  static constexpr int kStates = kSplit ? kTeams * 32 * 2 : 0;
  static constexpr size_t kLds = kTeams * kTeam + 8 * sizeof(int) + kStates * sizeof(float);
  static_assert(!kSplit || (size_t)32 * kSums * 4 <= kTeam, "a team's sums lie where its tiles were");
  // by which the pieces of row r are exchanged: 16 bytes of K, 32 bytes of V, 128 bytes of V in f32
  static __device__ __forceinline__ int k_turn(int r) { return DT == 64 && !k32 ? r >> 1 & 7 : r & 15; }
  static __device__ __forceinline__ int v_turn(int r) { return k32 ? r >> 2 & 1 : DT == 64 ? r >> 1 & 3 : r & 7; }
};

// 16 bytes of every lane, from `base` + `at` (or, second form, from `from`) to LDS from `to` on. The wait for it is the caller's:
// the compiler does not see these loads, whose arrival it would otherwise wait for at the next read of any LDS. Nor does it see to
// what has to lie in front of one: a wait state behind the scalar write of M0, which holds the place in LDS, and five between a
// vector instruction that writes a scalar register (a lane's value, a register brought back from its spill) and the load that
// reads it. The move of the base to scalar registers of the load's own is the first, and ends the second.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"  // M0 is a register that the compiler keeps to itself, and that is what is said here
__device__ __forceinline__ void load_lds(const void* base, unsigned at, unsigned to) {
  u64 own;
  asm volatile("s_mov_b32 m0, %3\n\ts_mov_b64 %0, %2\n\tglobal_load_lds_dwordx4 %1, %0" : "=&s"(own) : "v"(at), "s"(base), "s"(to) : "memory", "m0");
}
__device__ __forceinline__ void load_lds(const void* from, unsigned to) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(from), "s"(to) : "memory", "m0");
}
#pragma clang diagnostic pop
__device__ const u32x4 kZeros = {0, 0, 0, 0};

template <typename Act, typename KV, int DT, bool kSplit>
__global__ __launch_bounds__((Shape<Act, KV, DT, kSplit>::kThreads), DT == 256 || kSplit ? 1 : 2) void prompt_kernel(Attend a) {
  using M = Math<Act, KV>;
  using Sh = Shape<Act, KV, DT, kSplit>;
  constexpr int kTeams = Sh::kTeams, kTeamThreads = 64 * Sh::kMembers, kBlock = 32 * Sh::kMembers;
  constexpr int NT = Sh::kTerms, KB = Sh::kKeys, KS = Sh::kStep, kSub = KS / 32, kSteps = DT / 16, kDims = DT / 32;
  constexpr int kWeight = M::kScale ? M::kScale - kSlack : 0;  // exponent that weights carry
  constexpr bool k32 = Sh::k32;
  typedef typename std::conditional<k32, float, uint16_t>::type E;
  constexpr int kE = 16 / (int)sizeof(E);              // elements of a load
  constexpr int kPerKey = DT / kE;                     // 16-byte loads of a key
  constexpr unsigned kTileBytes = Sh::kTile * sizeof(E);
  constexpr int kLoads = KB * kPerKey / kTeamThreads;  // of a thread, for K and for V
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  int* odd_flags = (int*)(lds + kTeams * Sh::kTeam);
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, row = lane & 31, half = lane >> 5, dim = a.c.dim;
  const int team = wave / Sh::kMembers, member = wave % Sh::kMembers, team_tid = member * 64 + lane;

  // ---- which rows ----
  Seqs<KB, true> seqs;
  unsigned total = 0;
  for (int b0 = 0; b0 < a.c.n_seqs; b0 += 64) {
    seqs.load(a, b0);
    total = add_sat(total, last_lane(wave_scan(seqs.items)));
  }
  if (blockIdx.x >= total) return;
  const unsigned group = a.group, kv = a.c.kv_heads;
  const unsigned order = blockIdx.x / kv;
  const int hk = (int)(blockIdx.x - order * kv);
  Place p;
  int block;
  if (a.c.n_seqs > 1 && a.c.n_seqs <= 64) {
    // The blocks of all sequences by the last key that they see, most keys first: the position from which on `order` blocks
    // or fewer are left is searched for, all sequences counting at once.
    const Seq& q = seqs.q;
    const int len = min(q.s.len, a.c.cap);
    auto from = [&](int end) {  // this lane's blocks whose last row stands at `end` or behind
      if (!q.items || end > len + q.s.n - 1) return 0u;
      const long long need = (long long)(end - len) * a.group + 1;  // pairs up to the first that stands there
      return (unsigned)(q.items - (need <= 0 ? 0 : (int)((need + kBlock - 1) / kBlock) - 1));
    };
    int lo = 0, hi = a.c.cap + a.max_rows;  // from(lo) counts more than `order`, from(hi) does not
    while (hi - lo > 1) {
      const int mid = lo + (hi - lo) / 2;
      if (last_lane(wave_scan(from(mid))) > order)
        lo = mid;
      else
        hi = mid;
    }
    const unsigned more = from(hi), mine = from(lo) - more;
    const unsigned before = last_lane(wave_scan(more)), upto = wave_scan(mine);
    const u64 found = __ballot(before + upto > order);
    if (!found) return;
    const int at = __builtin_ctzll(found);
    auto of = [&](int x) { return __builtin_amdgcn_readlane(x, at); };
    p.b = at;
    p.q.s = {of(q.s.r0), of(q.s.n), of(q.s.len)};
    const unsigned nth = order - before - (unsigned)of((int)(upto - mine));
    block = of(q.items) - 1 - of((int)more) - (int)nth;
  } else {
    p = place_of(a, seqs, (total / kv - 1 - order) * kv + hk, kItems, 1);
    if (!p.there) return;
    block = (int)(p.inner / kv);
  }
  const Span s = p.q.s;
  const int all_rows = s.n * (int)group, of0 = block * kBlock, row0 = of0 + 32 * member, in_seq = row0 + row;
  const bool real = in_seq < all_rows;
  auto slot_of = [&](int r) { return s.len + by_group(a, min(r, all_rows - 1)); };
  const int j = by_group(a, min(in_seq, all_rows - 1)), head = hk * a.group + (real ? in_seq - j * a.group : 0);
  const int pos = s.len + j, pos_min = slot_of(row0), pos_max = slot_of(row0 + 31);
  const int block_min = slot_of(of0), block_max = slot_of(of0 + kBlock - 1);
  // tiles that the workgroup's rows can see: [0, ft) and [w0, ..), of those that the table has
  const int w0 = a.window ? max(0, min(block_min, a.c.cap - 1) - a.window + 1) / KB : 0;
  const int ft = a.window ? min((min(a.first, a.c.cap) + KB - 1) / KB, w0) : 0;
  const int nt = ft + min(block_max, a.c.cap - 1) / KB + 1 - w0;
  auto key_of = [&](int t) { return (t < ft ? t : t - ft + w0) * KB; };

  // ---- q ----
  float row_scale = fabsf(a.scale);
  typename M::V8 q[NT][kSteps];
  {
    const size_t at = (size_t)(s.r0 + j) * a.ldq + (size_t)head * dim;
    float x[kSteps][8], most = 0.0f;
#pragma unroll
    for (int c = 0; c < kSteps; ++c) {
      const int d = 16 * c + 8 * half;
      load8<Act>(a.q, at + (DT == dim || d < dim ? d : 0), x[c]);
    }
#pragma unroll
    for (int c = 0; c < kSteps; ++c) {
      const int d = 16 * c + 8 * half;
#pragma unroll
      for (int i = 0; i < 8; ++i) x[c][i] = DT == dim || d < dim ? x[c][i] : 0.0f;
#pragma unroll
      for (int i = 0; i < 8; ++i) most = fmaxf(most, fabsf(x[c][i]));
    }
    float up = a.scale < 0.0f ? -1.0f : 1.0f;  // the sign is q's, so that a larger product is a larger score
    if constexpr (M::kScale != 0) {
      most = fmaxf(most, __shfl_xor(most, 32));
      up *= M::row_scale(most, row_scale);
    }
    if (row_scale == 0.0f) {  // all alike (a scale of 0, or next to it): scores of 0, not infinity times 0 where a key is not seen
      up = 0.0f;
      row_scale = 1.0f;
    }
#pragma unroll
    for (int c = 0; c < kSteps; ++c) {
      typename M::V8 t[NT];
#pragma unroll
      for (int i = 0; i < 8; ++i) x[c][i] *= up;
      M::split(x[c], t);
#pragma unroll
      for (int k = 0; k < NT; ++k) q[k][c] = t[k];
    }
  }

  // ---- tiles ----
  const int* table = a.c.table + (size_t)p.b * a.c.table_ld;
  // Lane b has the page of the tile's b-th 16 keys. They are asked for a tile ahead of the loads that need them, and in front of
  // the loads of the tile between: loads return in order, so a page asked for behind these would be waited for as long as all.
  constexpr int kBlocks = KB / 16;
  int pages = -1;
  auto find = [&](int t) {
    const int at = (key_of(t) + 16 * min(lane, kBlocks - 1)) >> a.c.shift;
    pages = t < nt && at < a.c.table_ld ? table[at] : -1;
  };
  // Where this lane's 16 bytes of a wavefront's load come from, in a row of the load
  const int lane_row = lane / kPerKey, piece = lane % kPerKey, wave_row = 64 * member / kPerKey;
  // A load of the team has kRowsAtOnce rows. Load i's lie in the page of the tile's block block_of(i) of 16 keys, at place
  // i % kKinds * kRowsAtOnce + wave_row (mod 16) + lane_row of it; both turns repeat after 16 rows.
  constexpr int kRowsAtOnce = kTeamThreads / kPerKey, kKinds = kRowsAtOnce < 16 ? 16 / kRowsAtOnce : 1;
  unsigned k_at[kKinds], v_at[kKinds];
  bool k_in[kKinds], v_in[kKinds];
#pragma unroll
  for (int x = 0; x < kKinds; ++x) {
    const int r = (x * kRowsAtOnce + wave_row) % 16 + lane_row, from = piece ^ Sh::k_turn(r);
    k_in[x] = kE * from < dim;
    k_at[x] = (unsigned)((r * dim + kE * from) * sizeof(E));
    const int v_from = piece ^ Sh::v_turn(r) * (k32 ? 8 : 2);
    v_in[x] = kE * v_from < dim;
    v_at[x] = (unsigned)((r * dim + kE * v_from) * sizeof(E));
  }
  auto block_of = [&](int i) { return i * kRowsAtOnce / 16 + (kRowsAtOnce > 16 ? __builtin_amdgcn_readfirstlane(wave_row) / 16 : 0); };
  const unsigned lds0 = (unsigned)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)lds +
                        __builtin_amdgcn_readfirstlane(team) * (unsigned)Sh::kTeam;
  E* tiles = (E*)(lds + team * Sh::kTeam);
  // The team's n-th tile, t, to its buffer n & 1; returns the sixteens of keys whose page is not there.
  auto load = [&](int t, int n) {
    // every lane works its block's place in the pools out, and the loads take them from there
    const bool there = page_there(a.c, pages);
    const int gone = (int)(__ballot(!there) & ((1u << kBlocks) - 1));
    const u64 at = slot_row(a.c, there ? pages : 0, hk, key_of(t) + 16 * min(lane, kBlocks - 1)) * (unsigned)(sizeof(E) * dim);
    const unsigned at_lo = (unsigned)at, at_hi = (unsigned)(at >> 32);
    find(t + kTeams);
    const unsigned to = lds0 + (n & 1) * (2 * kTileBytes) + __builtin_amdgcn_readfirstlane(member) * 1024;
    constexpr int kStep = 1024 * Sh::kMembers;
    auto base_of = [&](int i) {
      const int b = block_of(i);
      return (u64)(unsigned)__builtin_amdgcn_readlane((int)at_hi, b) << 32 | (unsigned)__builtin_amdgcn_readlane((int)at_lo, b);
    };
    if (DT == dim) {
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        const u64 base = base_of(i);
        load_lds((const uint8_t*)a.c.k + base, k_at[i % kKinds], to + kStep * i);
        load_lds((const uint8_t*)a.c.v + base, v_at[i % kKinds], to + kStep * i + kTileBytes);
      }
    } else {  // zeros past the head's size
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        const u64 base = base_of(i);
        load_lds(k_in[i % kKinds] ? (const uint8_t*)a.c.k + base + k_at[i % kKinds] : (const uint8_t*)&kZeros, to + kStep * i);
        load_lds(v_in[i % kKinds] ? (const uint8_t*)a.c.v + base + v_at[i % kKinds] : (const uint8_t*)&kZeros, to + kStep * i + kTileBytes);
      }
    }
    return gone;
  };
  // Whether rows that stand from lo to hi all see all `keys` keys from k0 on
  auto seen_by = [&](int k0, int keys, int lo, int hi) {
    return k0 + keys - 1 <= lo && (a.window == 0 || k0 > hi - a.window || k0 + keys - 1 < a.first);
  };
  auto all_seen = [&](int k0, int lo, int hi) { return seen_by(k0, KB, lo, hi); };
  // The tile has arrived, for all wavefronts. Where not all rows see all of it: zeros for what no row sees, and for values that
  // are not finite; whether there were any of those is noted.
  if (lane == 0) odd_flags[wave] = 0;
  auto team_sync = [&]() {  // a team of one wavefront runs in step with itself
    if constexpr (kSplit)
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    else
      __syncthreads();
  };
  auto arrive = [&](int t, int n, int gone) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    team_sync();
    const int k0 = key_of(t);
    if (gone == 0 && all_seen(k0, block_min, block_max)) return;
    u32x4* vs = (u32x4*)(tiles + (n & 1) * (2 * Sh::kTile) + Sh::kTile);
    bool odd = false;
#pragma unroll 1
    for (int i = team_tid; i < KB * kPerKey; i += kTeamThreads) {
      const int key = i / kPerKey, at = k0 + key;
      const bool none = (gone >> key / 16 & 1) | (at > block_max) | ((a.window != 0) & (at <= block_min - a.window) & (at >= a.first));
      u32x4 x = vs[i];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t y = none ? 0u : M::finite(x[e]);
        odd = odd | (!none & (y != x[e]));
        x[e] = y;
      }
      vs[i] = x;
    }
    if (__any(odd) && lane == 0) odd_flags[wave] = 1;
    team_sync();
  };

  f32x16 o[kDims];
#pragma unroll
  for (int d = 0; d < kDims; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[d][i] = 0.0f;
  float m = -INFINITY, l = 0.0f;

  int t = __builtin_amdgcn_readfirstlane(team), n = 0, gone = 0;
  find(t);
  if (t < nt) {
    gone = load(t, 0);
    arrive(t, 0, gone);
  }
  for (; t < nt; t += kTeams, ++n) {
    const int next_gone = t + kTeams < nt ? load(t + kTeams, n + 1) : 0;
    const E* ks = tiles + (n & 1) * (2 * Sh::kTile);
    const E* vs = ks + Sh::kTile;
    const int tile0 = key_of(t);
#pragma unroll 1
    for (int k0 = tile0; k0 < tile0 + KB; k0 += KS, ks += KS * DT, vs += KS * DT) {
      const int gone_here = gone >> (k0 - tile0) / 16;
      const bool whole = gone == 0 && seen_by(k0, KS, pos_min, pos_max);
      if (row0 >= all_rows || k0 > pos_max) break;  // nothing for this wavefront
      // ---- scores ----
      const int k_turn = kE * Sh::k_turn(row);  // of rows 32 u + row
      f32x16 sc[kSub];
#pragma unroll
      for (int u = 0; u < kSub; ++u)
#pragma unroll
        for (int i = 0; i < 16; ++i) sc[u][i] = 0.0f;
#pragma unroll
      for (int c = 0; c < kSteps; ++c)
#pragma unroll
        for (int u = 0; u < kSub; ++u) {
          const E* at = ks + (32 * u + row) * DT;
          const int d = 8 * (2 * c + half);
          typename M::V8 kf;
          if constexpr (k32) {
            const f32x4 lo = *(const f32x4*)(at + (d ^ k_turn)), hi = *(const f32x4*)(at + ((d + 4) ^ k_turn));
            kf = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
          } else {
            kf = *(const typename M::V8*)(at + (d ^ k_turn));
          }
#pragma unroll
          for (int k = NT - 1; k >= 0; --k) sc[u] = mfma32(kf, q[k][c], sc[u]);
        }
      // four reads ahead of the products
      constexpr int kReads = k32 ? 2 : 1, kProducts = k32 ? 8 : NT;
      __builtin_amdgcn_sched_group_barrier(0x100, 4 * kReads, 0);
#pragma unroll
      for (int i = 0; i < kSteps * kSub - 4; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, kProducts, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, kReads, 0);
      }
      __builtin_amdgcn_sched_group_barrier(0x008, 4 * kProducts, 0);
      if (!whole) {
        int first_key = k0 + 4 * half;
        asm volatile("" : "+v"(first_key));  // here, not in front of the loop in a register for each key
#pragma unroll
        for (int u = 0; u < kSub; ++u)
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const int key = first_key + 32 * u + 8 * (i / 4) + i % 4;
            const bool gone_key = gone_here >> (2 * u + i / 8) & 1;
            const bool sees = real & (key <= pos) & ((a.window == 0) | (key > pos - a.window) | (key < a.first)) & !gone_key;
            sc[u][i] = sees ? sc[u][i] : -INFINITY;
          }
      }
      // ---- softmax: with c the scale of the row (times log2 e) and r its reference, 2^(c s - r) ----
      float mx = -INFINITY;
#pragma unroll
      for (int u = 0; u < kSub; ++u)
#pragma unroll
        for (int i = 0; i < 16; ++i) mx = fmaxf(mx, sc[u][i]);
      mx = fmaxf(mx, __shfl_xor(mx, 32)) * row_scale;
      if (__any(mx > m + (float)kSlack)) {
        const float m_new = fmaxf(m, mx), down = m == -INFINITY ? 0.0f : pow2(m - m_new);
        m = m_new;
        l *= down;
#pragma unroll
        for (int d = 0; d < kDims; ++d) o[d] *= down;
      }
      const float off = m == -INFINITY ? 0.0f : (float)kWeight - m;  // nothing seen yet: 2^-infinity is 0
      __builtin_amdgcn_s_setprio(1);  // over the other wavefront's scores, whose turn comes: 154 -> 150 us for two prompts
      float pr[kSub][16];
#pragma unroll
      for (int u = 0; u < kSub; ++u)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          pr[u][i] = pow2(__fmaf_rn(sc[u][i], row_scale, off));
          l += pr[u][i];
        }
#pragma unroll
      for (int c = 0; c < 2 * kSub; ++c) {  // 16 keys
        float p8[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) p8[i] = pr[c / 2][8 * (c % 2) + i];
        if constexpr (k32) {
#pragma unroll
          for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int d = 0; d < kDims; ++d)
              o[d] = mfma32(vs[(16 * c + 8 * (i / 4) + 4 * half + i % 4) * DT + 32 * (d ^ half) + row], p8[i], o[d]);
        } else {
          typename M::V8 pt[NT];
          M::split(p8, pt);
          const int r0 = 4 * half + ((lane & 15) >> 2);  // of rows 16 c + 8 x + r0
#pragma unroll
          for (int d = 0; d < kDims; ++d) {
            union {
              s4 part[2];
              typename M::V8 v8;
            } vt;
#pragma unroll
            for (int x = 0; x < 2; ++x)
              vt.part[x] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4*)(
                  vs + (16 * c + 8 * x + r0) * DT + ((2 * d + (lane >> 4 & 1)) ^ Sh::v_turn(8 * x + r0)) * 16 + 4 * (lane & 3)));
#pragma unroll
            for (int k = NT - 1; k >= 0; --k) o[d] = mfma32(vt.v8, pt[k], o[d]);
          }
        }
      }
      constexpr int kVReads = k32 ? 4 : 2, kVProducts = k32 ? 4 : NT;
      __builtin_amdgcn_sched_group_barrier(0x100, 4 * kVReads, 1);
#pragma unroll
      for (int i = 0; i < (k32 ? 4 : 2) * kSub * kDims - 4; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, kVProducts, 1);
        __builtin_amdgcn_sched_group_barrier(0x100, kVReads, 1);
      }
      __builtin_amdgcn_sched_group_barrier(0x008, 4 * kVProducts, 1);
      __builtin_amdgcn_s_setprio(0);
    }
    if (t + kTeams < nt) arrive(t + kTeams, n + 1, next_gone);
    gone = next_gone;
  }

  // ---- values that are not finite: as in the rows' kernel, where the results are ----
  l += __shfl_xor(l, 32);
  bool some_odd = odd_flags[wave] != 0;
  if constexpr (!kSplit)  // behind the last arrival's barrier
    for (int w = 0; w < Sh::kMembers; ++w) some_odd = some_odd || odd_flags[w] != 0;
  float probe[4] = {};
#pragma unroll
  for (int d = 0; d < kDims; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) probe[i % 4] = __fmaf_rn(o[d][i], 0.0f, probe[i % 4]);
  const float strange = (probe[0] + probe[1]) + (probe[2] + probe[3]);
  some_odd = some_odd || __any(real & (l == l) & (strange != strange));
  // ---- results: lane = row, four dims at a time ----
  if constexpr (kSplit) {
    float* sums = (float*)(lds + team * Sh::kTeam);
    float* states = (float*)(odd_flags + 8);
#pragma unroll
    for (int d = 0; d < kDims; ++d)
#pragma unroll
      for (int b = 0; b < 4; ++b)
        *(f32x4*)(sums + row * Sh::kSums + 32 * d + 8 * b + 4 * half) =
            f32x4{o[d][4 * b], o[d][4 * b + 1], o[d][4 * b + 2], o[d][4 * b + 3]};
    if (__builtin_expect(some_odd, 0)) {
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll 1
      for (int add = 0; add < 2; ++add)
#pragma unroll 1
        for (t = team; t < nt; t += kTeams)
          put_odd<M, KV, 32>(a, table, hk, key_of(t), KB, s.len, row0, all_rows, [&](int r, int d, float v) {
            float& sum = sums[r * Sh::kSums + d];
            sum = add ? sum + v : 0.0f;
          });
    }
    if (half == 0) {
      states[(team * 32 + row) * 2] = m;
      states[(team * 32 + row) * 2 + 1] = l;
    }
    __syncthreads();
    const int rows = min(all_rows - of0, 32);
    for (int i = tid; i < rows * (DT / 4); i += 64 * kTeams) {
      const int r = i / (DT / 4), d = i % (DT / 4) * 4;
      float top = -INFINITY, sum = 0.0f;
#pragma unroll
      for (int w = 0; w < kTeams; ++w) top = fmaxf(top, states[(w * 32 + r) * 2]);
      const float base = top == -INFINITY ? 0.0f : top;
      f32x4 acc = {0, 0, 0, 0};
#pragma unroll
      for (int w = 0; w < kTeams; ++w) {
        const float f = pow2(states[(w * 32 + r) * 2] - base);
        sum += f * states[(w * 32 + r) * 2 + 1];
        acc += fmaxf(f, kLeast) * *(const f32x4*)((const float*)(lds + w * Sh::kTeam) + r * Sh::kSums + d);
      }
      finish<Act, false>(a, s.r0, of0 + r, hk, 0, d, acc, base, sum);
    }
    return;
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  const size_t at = (size_t)(s.r0 + j) * a.ldo + (size_t)head * dim;
  if (real) {
#pragma unroll
    for (int d = 0; d < kDims; ++d)
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        const int to = 32 * d + 8 * b + 4 * half;
        if (DT == dim || to < dim) store4<Act>(a.out, at + to, f32x4{o[d][4 * b], o[d][4 * b + 1], o[d][4 * b + 2], o[d][4 * b + 3]} * inv);
      }
  }
  if (__builtin_expect(some_odd, 0)) {
    const u64 numbers = __ballot(l == l);  // the other rows are NaN
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");
#pragma unroll 1
    for (int add = 0; add < 2; ++add)
#pragma unroll 1
      for (t = team; t < nt; t += kTeams)
        put_odd<M, KV, 32>(a, table, hk, key_of(t), KB, s.len, row0, all_rows, [&](int r, int d, float v) {
          if (!(numbers >> r & 1)) return;
          const int of = row0 + r, token = by_group(a, of);
          Act* to = (Act*)a.out + (size_t)(s.r0 + token) * a.ldo + (size_t)(hk * (int)group + of - token * (int)group) * dim + d;
          *to = add ? (Act)((float)*to + v) : (Act)0.0f;
        });
  }
}

template <typename Act, typename KV, int DT, bool kSplit>
hipError_t launch(const Attend& a, unsigned items, hipStream_t s) {
  using Sh = Shape<Act, KV, DT, kSplit>;
  if constexpr (Sh::kLds > 64 * 1024) {
    static LdsLimitOnce limit;
    if (hipError_t e = limit.raise((const void*)prompt_kernel<Act, KV, DT, kSplit>, Sh::kLds); e != hipSuccess) return e;
  }
  hipLaunchKernelGGL((prompt_kernel<Act, KV, DT, kSplit>), dim3(items), dim3(Sh::kThreads), Sh::kLds, s, a);
  return hipGetLastError();
}
template <typename Act, typename KV, bool kSplit>
hipError_t launch_dim(const Attend& a, int dt, unsigned items, hipStream_t s) {
  if (dt == 64) return launch<Act, KV, 64, kSplit>(a, items, s);
  if (dt == 128) return launch<Act, KV, 128, kSplit>(a, items, s);
  return launch<Act, KV, 256, kSplit>(a, items, s);
}
template <typename Act, typename KV>
hipError_t launch_shape(const Attend& a, int dt, unsigned items, hipStream_t s) {
  return a.prompt_log2 == 5 ? launch_dim<Act, KV, true>(a, dt, items, s) : launch_dim<Act, KV, false>(a, dt, items, s);
}
}  // namespace

hipError_t launch_prompts(const Attend& a, int dtype, bool act_bf16, int dt, unsigned items, hipStream_t s) {
  if (dtype == W4A32_CACHE_F32) {
    if (dt == 64) return launch<float, float, 64, true>(a, items, s);
    return dt == 128 ? launch<float, float, 128, false>(a, items, s) : launch<float, float, 256, false>(a, items, s);
  }
  if (act_bf16) return launch_shape<__bf16, __bf16>(a, dt, items, s);
  if (dtype == W4A32_CACHE_F16) return launch_shape<float, _Float16>(a, dt, items, s);
  return launch_shape<float, __bf16>(a, dt, items, s);
}

}  // namespace paged
}  // namespace w4
