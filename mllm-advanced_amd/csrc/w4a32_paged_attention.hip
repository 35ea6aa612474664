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
#include "w4a32_paged_attention.h"

namespace w4 {
namespace paged {

namespace {
inline bool aligned(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }
inline int from_hip(hipError_t e) { return e == hipSuccess ? W4A32_OK : W4A32_ELAUNCH; }

// Workgroups that a batch is dealt to: two per CU, all there at once. (256 of eight wavefronts: one row on 200 tokens 14.2 us against
// 12.3, one on 131001 34.9 against 32.9, 64 sequences 116 against 114, 16 of drafted tokens 30.8 against 31.7.)
constexpr int kGrid = 512;
constexpr int kMinTiles = kWaves; // least tiles of a share, where items have so many
constexpr int kAlone = 8;         // tiles up to which items are not shared, where all are so short
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
constexpr int kFew = 16;          // tiles of a share up to which it has tiles of one item only
// Where weights are added up the scores of a pass lie in scratch memory, 4 bytes for each row of a head and each token that the table
// has room for: a step of more rows than fit into kMostScores is gone through in passes of kLeastPass rows or more (28 heads on 4 of
// 128 dims, bf16: 8192 rows 5.7 ms with 0.97 GB against 7.5 ms with 7.6 GB at once; 2048 rows on a table for 131072 tokens 1.13 ms with
// 1.9 GB against 1.00 with 30).
constexpr size_t kMostScores = (size_t)1 << 30;
constexpr int kLeastPass = 128;

template <int KT>
__device__ __forceinline__ Deal deal_of(const Attend& a, Seqs<KT>& s) {
  Deal d = {0, 0, 0, false};
  bool all_short = true;
  if (a.c.n_seqs == 1) {  // nothing to add up: a decode step of one sequence is all latency
    s.load(a, 0);
    d.total = (unsigned)__builtin_amdgcn_readfirstlane((int)s.tiles);
    d.items = (unsigned)__builtin_amdgcn_readfirstlane((int)s.items);
    all_short = __builtin_amdgcn_readfirstlane(s.q.nt) <= kAlone;
  } else for (int b0 = 0; b0 < a.c.n_seqs; b0 += 64) {
    s.load(a, b0);
    d.total = add_sat(d.total, last_lane(wave_scan(s.tiles)));
    d.items = add_sat(d.items, last_lane(wave_scan(s.items)));
    all_short = all_short && !__any(s.q.nt > kAlone);
  }
  if (d.total == 0 || d.total > a.most_tiles || d.items > a.most_items) return d;
  d.per = max((d.total + kGrid - 1) / kGrid, (unsigned)kMinTiles);
  const unsigned more = gridDim.x - min(gridDim.x, d.items);  // workgroups beyond one per item
  if (all_short) {  // a workgroup takes every gridDim.x-th
    d.per = kAlone;
    d.apart = true;
  } else if (more && (d.total + more - 1) / more <= kFew) {
    d.per = max((d.total + more - 1) / more, (unsigned)kMinTiles);
    d.apart = true;
  }
  return d;
}


// Of a sequence's tiles those that a wavefront's rows, which stand from lo to hi, can see: [0, firsts), which have the first tokens, and
// [from, to). The others are dealt like these but passed over (256 dims in f32, 850 rows that see 94 tokens each: 101 us against 253
// with all of them gone through).
struct Sight {
  int firsts, from, to;
  __device__ __forceinline__ bool skips(int t) const { return t >= firsts && t < from; }
};
template <int KT>
__device__ __forceinline__ Sight sight_of(const Attend& a, const Seq& q, int lo, int hi) {
  if (a.window == 0) return {0, 0, hi / KT + 1};
  return {(min(a.first, a.c.cap) + KT - 1) / KT, q.ft + max(0, lo - a.window + 1) / KT - q.w0, q.ft + hi / KT - q.w0 + 1};
}

template <typename KV>
constexpr int tile_keys() { return sizeof(KV) == 2 ? 32 : 16; }
template <typename KV, int DT>
constexpr int v_stride() { return sizeof(KV) == 2 ? DT + 16 : DT + 4; }  // elements of an LDS row: its reads meet no bank twice
template <typename KV, int DT>
constexpr size_t wave_lds() {  // a wavefront's tile of V; at the end its 16 rows of sums
  constexpr size_t v = (size_t)tile_keys<KV>() * v_stride<KV, DT>() * sizeof(KV), o = (size_t)kRows * (DT + 4) * 4;
  return v > o ? v : o;
}
template <typename KV, int DT>
constexpr size_t lds_bytes() { return kWaves * (wave_lds<KV, DT>() + kRows * 2 * sizeof(float)); }

// DT: the head size rounded up to 64, 128 or 256. kDump: leave the scores for the launch that adds the weights up.
template <typename Act, typename KV, int DT, bool kDump>
__global__ __launch_bounds__(64 * kWaves, DT == 256 ? 1 : 2) void rows_kernel(Attend a) {
  using M = Math<Act, KV>;
  constexpr int KT = tile_keys<KV>(), NT = M::kTerms, kHalves = KT / 16;
  constexpr bool k16 = sizeof(KV) == 2;
  constexpr int kSteps = k16 ? DT / 32 : DT / 16;         // 16-byte loads of a lane per 16 keys of K
  constexpr int kVLoads = KT * DT * (int)sizeof(KV) / 1024;  // 16-byte loads of a lane per tile of V
  constexpr int kVS = v_stride<KV, DT>();
  constexpr int kE = 16 / (int)sizeof(KV);                // elements of a load
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  float* states = (float*)(lds + kWaves * wave_lds<KV, DT>());
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, row = lane & 15, grp = lane >> 4, dim = a.c.dim;
  // wavefronts that share rows, and which of them this one is
  const int streams = kWaves >> a.wide, stream = wave >> a.wide, wide = 1 << a.wide;

  Seqs<KT> seqs;
  const Deal deal = deal_of<KT>(a, seqs);
  if (blockIdx.x == 0 && threadIdx.x == 0) *a.count = deal.per ? deal.items : 0;
  if (deal.per == 0) return;
  unsigned u = blockIdx.x, u_end = max(deal.items, gridDim.x);
  if (!deal.apart) {
    u *= deal.per;
    u_end = min(deal.total, u + deal.per);
  }
  while (u < u_end) {
    const Place p = place_of(a, seqs, u, deal.apart ? kShares : kTiles, deal.per);
    if (!p.there) return;
    const Span s = p.q.s;
    // the item (of the sequence), the tiles of this share, the workgroups that share the item
    int item, t_lo, t_hi, w_first, shares;
    if (deal.apart && p.q.nt <= (int)deal.per) {
      shares = 1;
      item = (int)p.inner;
      t_lo = 0;
      t_hi = p.q.nt;
      w_first = (int)blockIdx.x;
    } else if (deal.apart) {
      shares = (int)((p.q.nt + deal.per - 1) / deal.per);
      item = (int)(p.inner / (unsigned)shares);
      const int mine = (int)p.inner - item * shares;
      t_lo = (int)((unsigned)(p.q.nt * mine) / (unsigned)shares);  // at most kFew kGrid tiles
      t_hi = (int)((unsigned)(p.q.nt * (mine + 1)) / (unsigned)shares);
      w_first = (int)blockIdx.x - mine;
    } else {
      item = (int)(p.inner / p.q.nt);
      t_lo = (int)(p.inner - (unsigned)item * p.q.nt);
      t_hi = (int)min((unsigned)p.q.nt, t_lo + (u_end - u));
      const unsigned begin = p.tile0 + (unsigned)item * p.q.nt;
      w_first = (int)(begin / deal.per);
      shares = (int)((begin + p.q.nt - 1) / deal.per) - w_first + 1;
    }
    const int hk = p.q.items == 1 ? item : (int)((unsigned)item / (unsigned)p.q.items), of0 = (item - hk * p.q.items) * (kRows << a.wide);
    // this lane's query row, and the rows of its wavefront
    const int all_rows = s.n * a.group, row0 = of0 + (wave & (wide - 1)) * kRows;
    const int in_seq = row0 + row;
    const bool real = in_seq < all_rows, busy = row0 < all_rows;
    const int j = by_group(a, min(in_seq, all_rows - 1)), head = hk * a.group + (real ? in_seq - j * a.group : 0);
    const int j_min = by_group(a, min(row0, all_rows - 1)), j_max = by_group(a, min(row0 + kRows - 1, all_rows - 1));
    const int pos = s.len + j, pos_min = s.len + j_min, pos_max = s.len + j_max;

    // The page numbers of the first tile are asked for, then q, then its keys and values: q is made ready while those are on their way.
    typedef typename std::conditional<k16, u32x4, f32x4>::type Raw;
    const int* table = a.c.table + (size_t)p.b * a.c.table_ld;
    auto key_of = [&](int t) { return (t < p.q.ft ? t : t - p.q.ft + p.q.w0) * KT; };
    // Lane h has the page of half h of a tile (-1: not there). It is asked for a tile ahead of the loads that need it, and in front
    // of the loads of the tile between: loads return in order, and behind these it would take as long as all of them.
    int pages = -1;
    const Sight sight = sight_of<KT>(a, p.q, pos_min, pos_max);
    const int t_end = busy ? min(t_hi, sight.to) : 0;
    auto seen_from = [&](int t) { return sight.skips(t) ? t + ((sight.from - t + streams - 1) & -streams) : t; };
    auto find = [&](int t) {
      const int i = (key_of(t) + 16 * min(lane, kHalves - 1)) >> a.c.shift;
      pages = t < t_end && i < a.c.table_ld ? table[i] : -1;
    };

    Raw kr[kHalves][kSteps], vr[kVLoads];
    int page[kHalves];
    auto turn = [&](int t) {  // to the pages of tile t, and asks for those of the next
#pragma unroll
      for (int h = 0; h < kHalves; ++h) {
        const int pg = __builtin_amdgcn_readlane(pages, h);
        page[h] = page_there(a.c, pg) ? pg : -1;
      }
      find(seen_from(t + streams));
    };
    auto load_k = [&](int t) {
#pragma unroll
      for (int h = 0; h < kHalves; ++h) {
        const KV* base = (const KV*)a.c.k + slot_row(a.c, max(page[h], 0), hk, key_of(t) + 16 * h) * dim;
#pragma unroll
        for (int c = 0; c < kSteps; ++c) {
          const int d = (k16 ? 32 : 16) * c + kE * grp;
          kr[h][c] = DT == dim || d < dim ? load_global<Raw>(base + row * dim + d) : Raw{0, 0, 0, 0};
        }
      }
    };
    auto load_v = [&](int t) {
      constexpr int kPerKey = DT / kE;
#pragma unroll
      for (int i = 0; i < kVLoads; ++i) {
        const int key = (64 * i + lane) / kPerKey, d = (64 * i + lane) % kPerKey * kE;
        const int h = kHalves == 1 ? 0 : (64 * i) / (16 * kPerKey);
        const KV* base = (const KV*)a.c.v + slot_row(a.c, max(page[h], 0), hk, key_of(t) + 16 * h) * dim;
        vr[i] = DT == dim || d < dim ? load_global<Raw>(base + (key - 16 * h) * dim + d) : Raw{0, 0, 0, 0};
      }
    };
    int t = seen_from(t_lo + stream);
    find(t);

    // ---- q ----
    constexpr int kQ = k16 && sizeof(Act) == 4 ? 2 : 1;  // 16-byte loads of a step
    float row_scale = a.scale;
    u32x4 qr[kSteps][kQ], qt[k16 ? NT : 1][k16 ? kSteps : 1];
    f32x4 qf[k16 ? 1 : kSteps];
    const int q_step = k16 ? 32 : 16, q_first = (k16 ? 8 : 4) * grp;
    {
      const Act* from = (const Act*)a.q + (size_t)(s.r0 + j) * a.ldq + (size_t)head * dim;
#pragma unroll
      for (int c = 0; c < kSteps; ++c) {
        const int d = q_step * c + q_first;
#pragma unroll
        for (int h = 0; h < kQ; ++h) qr[c][h] = load_global<u32x4>(from + (DT == dim || d < dim ? d : 0) + 4 * h);
      }
    }
    if (t < t_end) {
      turn(t);
      load_k(t);
      load_v(t);
    }
    if constexpr (k16) {
      float x[kSteps][8], most = 0.0f;
#pragma unroll
      for (int c = 0; c < kSteps; ++c)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const uint32_t w = qr[c][kQ == 2 ? i / 4 : 0][kQ == 2 ? i % 4 : i / 2];
          const float f = __uint_as_float(kQ == 2 ? w : i & 1 ? w & 0xffff0000u : w << 16);
          x[c][i] = DT == dim || 32 * c + 8 * grp < dim ? f : 0.0f;
          most = fmaxf(most, fabsf(x[c][i]));
        }
      if constexpr (M::kScale != 0) {
        const float up = M::row_scale(group_max(most), row_scale);
#pragma unroll
        for (int c = 0; c < kSteps; ++c)
#pragma unroll
          for (int i = 0; i < 8; ++i) x[c][i] *= up;
      }
#pragma unroll
      for (int c = 0; c < kSteps; ++c) {
        typename M::V8 terms[NT];
        M::split(x[c], terms);
#pragma unroll
        for (int k = 0; k < NT; ++k) qt[k][c] = __builtin_bit_cast(u32x4, terms[k]);
      }
    } else {
#pragma unroll
      for (int c = 0; c < kSteps; ++c)
        qf[c] = DT == dim || q_step * c + q_first < dim ? __builtin_bit_cast(f32x4, qr[c][0]) : f32x4{0, 0, 0, 0};
    }

    KV* vs = (KV*)(lds + wave * wave_lds<KV, DT>());
    f32x4 o[DT / 16];
#pragma unroll
    for (int d = 0; d < DT / 16; ++d) o[d] = f32x4{0, 0, 0, 0};
    float m = -INFINITY, l = 0.0f;
    bool odd = false;  // values that are not finite, in a tile that not every row sees whole
    for (int next; t < t_end; t = next) {
      next = seen_from(t + streams);
      const int k0 = key_of(t);
      bool there = true;
      int cur[kHalves];
#pragma unroll
      for (int h = 0; h < kHalves; ++h) {
        cur[h] = page[h];
        there = there && cur[h] >= 0;
      }
      // every key seen by every row, or each looked at
      const bool whole = there && k0 + KT - 1 <= pos_min && (a.window == 0 || k0 > pos_max - a.window || k0 + KT - 1 < a.first);
      if (!whole) {
        asm volatile("");
        uint32_t top = 0;  // the signs' places: whether a value is not finite
        constexpr int kPerKey = DT / kE;
#pragma unroll
        for (int i = 0; i < kVLoads; ++i) {
          const int in = (64 * i + lane) / kPerKey, key = k0 + in;
          const bool none = ((kHalves == 1 ? cur[0] : in < 16 ? cur[0] : cur[kHalves - 1]) < 0) | (key > pos_max) |
                            ((a.window != 0) & (key <= pos_min - a.window) & (key >= a.first));
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            const uint32_t x = none ? 0u : __builtin_bit_cast(u32x4, vr[i])[w];
            top |= ((x & M::kSize) + M::kStep) & ~M::kSize;
            vr[i][w] = __builtin_bit_cast(Raw, u32x4{x, x, x, x})[0];
          }
        }
        if (__any(top != 0)) {
          odd = true;
#pragma unroll
          for (int i = 0; i < kVLoads; ++i)
#pragma unroll
            for (int w = 0; w < 4; ++w) {
              const uint32_t x = M::finite(__builtin_bit_cast(u32x4, vr[i])[w]);
              vr[i][w] = __builtin_bit_cast(Raw, u32x4{x, x, x, x})[0];
            }
        }
      }
      {
        constexpr int kPerKey = DT / kE;
#pragma unroll
        for (int i = 0; i < kVLoads; ++i)
          *(Raw*)(vs + (64 * i + lane) / kPerKey * kVS + (64 * i + lane) % kPerKey * kE) = vr[i];
      }
      // ---- scores ----
      f32x4 sc[kHalves];
#pragma unroll
      for (int h = 0; h < kHalves; ++h) {
        sc[h] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int c = 0; c < kSteps; ++c) {
          if constexpr (k16) {
#pragma unroll
            for (int k = NT - 1; k >= 0; --k)  // small terms first
              sc[h] = M::mfma(__builtin_bit_cast(typename M::V8, kr[h][c]), __builtin_bit_cast(typename M::V8, qt[k][c]), sc[h]);
          } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) sc[h] = M::mfma(kr[h][c][i], qf[c][i], sc[h]);
          }
        }
      }
      if (next < t_end) {
        turn(next);
        load_k(next);
        load_v(next);
      }
      uint32_t seen = 0xff;  // bit 4 h + i: key 16 h + 4 grp + i
      if (!whole) {
        asm volatile("");  // a branch: the compiler would rather do this for every tile
        seen = 0;
#pragma unroll
        for (int h = 0; h < kHalves; ++h)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int key = k0 + 16 * h + 4 * grp + i;
            const bool sees = real & (cur[h] >= 0) & (key <= pos) & ((a.window == 0) | (key > pos - a.window) | (key < a.first));
            seen |= sees ? 1u << (4 * h + i) : 0u;
          }
      }
      float mx = -INFINITY;
#pragma unroll
      for (int h = 0; h < kHalves; ++h)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float x = sc[h][i] * row_scale;
          sc[h][i] = seen >> (4 * h + i) & 1 ? x : -INFINITY;
          mx = fmaxf(mx, sc[h][i]);
        }
      if constexpr (kDump) {
        const u64 at = ((u64)p.tile0 + (u64)item * p.q.nt + t) * wide + (wave & (wide - 1));
#pragma unroll
        for (int h = 0; h < kHalves; ++h) *(W4_GLOBAL f32x4*)(a.dump + (at * 64 + lane) * (4 * kHalves) + 4 * h) = sc[h];
      }
      const float m_new = fmaxf(m, group_max(mx));
      const float base = m_new == -INFINITY ? 0.0f : m_new;  // nothing seen yet: exp2(-inf) is 0
      if (__any(m_new > m)) {
        const float down = pow2(m - base);
        l *= down;
#pragma unroll
        for (int d = 0; d < DT / 16; ++d) o[d] *= down;
      }
      m = m_new;
      float pr[8] = {};
#pragma unroll
      for (int h = 0; h < kHalves; ++h)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          pr[4 * h + i] = pow2(sc[h][i] - base + (float)M::kScale);
          l += pr[4 * h + i];
        }
      // ---- values ----
      if constexpr (k16) {
        typename M::V8 pt[NT];
        M::split(pr, pt);
        const KV* v = vs + (4 * grp + (row >> 2)) * kVS + 4 * (row & 3);
#pragma unroll
        for (int d = 0; d < DT / 16; ++d) {
          union {
            s4 half[2];
            typename M::V8 v8;
          } vt;
#pragma unroll
          for (int h = 0; h < 2; ++h)
            vt.half[h] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4*)(v + 16 * h * kVS + 16 * d));
#pragma unroll
          for (int k = NT - 1; k >= 0; --k) o[d] = M::mfma(vt.v8, pt[k], o[d]);
        }
      } else {
#pragma unroll
        for (int d = 0; d < DT / 16; ++d)
#pragma unroll
          for (int i = 0; i < 4; ++i) o[d] = M::mfma(vs[(4 * grp + i) * kVS + 16 * d + row], pr[i], o[d]);
      }
    }

    // ---- join the wavefronts ----
    l = group_sum(l) * ldexpf(1.0f, -M::kScale);
    float* sums = (float*)(lds + wave * wave_lds<KV, DT>());
    float probe[4] = {};
#pragma unroll
    for (int d = 0; d < DT / 16; ++d) {
      *(f32x4*)(sums + row * (DT + 4) + 16 * d + 4 * grp) = o[d] * ldexpf(1.0f, -M::kScale);
#pragma unroll
      for (int e = 0; e < 4; ++e) probe[e] = __fmaf_rn(o[d][e], 0.0f, probe[e]);
    }
    // Values that are not finite were zeros in the tiles that not every row sees whole; in the others they met weights of several
    // terms, of which one may be 0 or negative and make them NaN. So a row whose sums are not finite, though its weights are
    // numbers, has those values added up instead: first zeros in their place, then the values.
    const float strange = (probe[0] + probe[1]) + (probe[2] + probe[3]);
    if (__builtin_expect(odd || __any(real & (l == l) & (strange != strange)), 0)) {
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll 1
      for (int add = 0; add < 2; ++add)
#pragma unroll 1
        for (t = seen_from(t_lo + stream); t < t_end; t = seen_from(t + streams))
          put_odd<M, KV, kRows>(a, table, hk, key_of(t), KT, s.len, row0, all_rows, [&](int r, int d, float v) {
            float& sum = sums[r * (DT + 4) + d];
            sum = add ? sum + v : 0.0f;
          });
    }
    if (grp == 0) {
      states[(wave * kRows + row) * 2] = m;
      states[(wave * kRows + row) * 2 + 1] = l;
    }
    __syncthreads();
    // ---- and the shares of the item, where it is not this workgroup's alone ----
    // The share that has an item's first tile lies in slot 2 w + 1 and the others in 2 w: of two items that meet in a
    // workgroup one begins there and the other does not.
    const int rows = min(all_rows - of0, kRows << a.wide);
    const int slot = 2 * (int)blockIdx.x + (t_lo == 0);
    if (t_lo == 0 && threadIdx.x == 0) a.item[p.item0 + item] = Item{w_first, shares, s.r0, of0, rows, hk};
    constexpr int kPer = DT / 4;  // threads of a row
    for (int i = threadIdx.x; i < rows * kPer; i += 64 * kWaves) {
      const int r = i / kPer, d = i % kPer * 4, w0 = r / kRows;
      float top = -INFINITY, sum = 0.0f;
      f32x4 acc = {0, 0, 0, 0};
      for (int w = w0; w < kWaves; w += wide) top = fmaxf(top, states[(w * kRows + r % kRows) * 2]);
      const float base = top == -INFINITY ? 0.0f : top;
      for (int w = w0; w < kWaves; w += wide) {
        const float f = pow2(states[(w * kRows + r % kRows) * 2] - base);
        sum += f * states[(w * kRows + r % kRows) * 2 + 1];
        acc += fmaxf(f, kLeast) * *(const f32x4*)((const float*)(lds + w * wave_lds<KV, DT>()) + (r % kRows) * (DT + 4) + d);
      }
      if (shares > 1) {
        const size_t at = (size_t)slot * a.slot_rows + r;
        *(W4_GLOBAL f32x4*)(a.part + at * DT + d) = acc;
        if (d == 0) {
          a.state[2 * at] = top;
          a.state[2 * at + 1] = sum;
        }
      } else {
        finish<Act, kDump>(a, s.r0, of0 + r, hk, (size_t)(p.item0 + item) * a.slot_rows + r, d, acc, base, sum);
      }
    }
    u += deal.apart ? gridDim.x : t_hi - t_lo;
    if (u < u_end) __syncthreads();  // the next item's tiles go where these sums were read
  }
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
  if (deal_of<KT>(a, seqs).per == 0) return;
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
