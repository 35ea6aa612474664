// The rows' kernel of attention on a paged cache: what one workgroup does. (How and why stands in front of its launches.)
#pragma once

#include "w4a32_paged_attention.h"

namespace w4 {
namespace paged {

// Workgroups that a batch is dealt to: two per CU, all there at once. (256 of eight wavefronts: one row on 200 tokens 14.2 us against
// 12.3, one on 131001 34.9 against 32.9, 64 sequences 116 against 114, 16 of drafted tokens 30.8 against 31.7.)
constexpr int kGrid = 512;
constexpr int kMinTiles = kWaves; // least tiles of a share, where items have so many
constexpr int kAlone = 8;         // tiles up to which items are not shared, where all are so short
constexpr int kFew = 16;          // tiles of a share up to which it has tiles of one item only
constexpr unsigned kRound = 24;

// one_round (kOwn): to how many the shares are dealt so that all begin at once, if none has kRound tiles then
template <int KT, Which kWhich>
__device__ __forceinline__ Deal deal_of(const Attend& a, Seqs<KT, kWhich>& s, unsigned grid, unsigned one_round) {
  Deal d = {0, 0, 0, true, false};
  unsigned others = 0;  // items without tiles
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
    if constexpr (kWhich == kOwn) others = add_sat(others, last_lane(wave_scan(s.tiles ? 0 : s.items)));
  }
  d.fits = d.total <= a.most_tiles && d.items <= a.most_items;
  if (d.total == 0 || !d.fits) return d;
  if (kWhich == kOwn && one_round < grid && one_round > d.items - others && d.total / (one_round - (d.items - others)) < kRound) grid = one_round;
  d.per = max((d.total + grid - 1) / grid, (unsigned)kMinTiles);
  const unsigned more = grid - min(grid, d.items - others);  // workgroups beyond one per item
  if (all_short) {  // a workgroup takes every grid-th
    d.per = kAlone;
    d.apart = true;
  } else if (more && (kWhich == kOwn || (d.total + more - 1) / more <= kFew)) {
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
  if (a.window == 0) return {0, 0, hi / KT + 1 - q.w0};
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

// DT: the head size rounded up to 64, 128 or 256. kDump: leave the scores for the launch that adds the weights up. kWhich == kOwn: the tokens
// behind a prefix, whose sums another launch joins with the prefix's.
// An item of a sequence with n rows, in its group (without rows, where it has none)
__device__ __forceinline__ OwnItem own_item(const Attend& a, const Item& it, int n, const PrefixGroup& q) {
  const int row = it.r0 - q.r0;
  if (row < 0 || row + n > q.n) return {it, 0, 0, 0, 0};
  return {it, row * a.group + it.row0, q.first + it.head, q.shares, q.blocks * a.c.kv_heads};
}

// own_from: where this lane's sequence's own tokens begin; group_at: the group of a sequence, without rows where it has none.
template <typename Act, typename KV, int DT, bool kDump, Which kWhich, typename GroupAt>
__device__ __forceinline__ void rows_body(const Attend& a, unsigned block, unsigned grid, unsigned one_round, int own_from, GroupAt group_at) {
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

  Seqs<KT, kWhich> seqs;
  seqs.own_from = own_from;
  const Deal deal = deal_of(a, seqs, grid, one_round);
  if (block == 0 && threadIdx.x == 0) *a.count = deal.fits ? deal.items : 0;
  if (deal.per == 0) return;
  unsigned u = block, u_end = max(deal.items, grid);
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
      w_first = (int)block;
    } else if (deal.apart) {
      shares = (int)((p.q.nt + deal.per - 1) / deal.per);
      item = (int)(p.inner / (unsigned)shares);
      const int mine = (int)p.inner - item * shares;
      if constexpr (kWhich == kOwn) {
        const int each = (int)((unsigned)p.q.nt / (unsigned)shares), more = p.q.nt - each * shares;
        t_lo = each * mine + min(mine, more);
        t_hi = t_lo + each + (mine < more);
      } else {
        t_lo = (int)((unsigned)(p.q.nt * mine) / (unsigned)shares);  // at most kFew kGrid tiles
        t_hi = (int)((unsigned)(p.q.nt * (mine + 1)) / (unsigned)shares);
      }
      w_first = (int)block - mine;
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
      auto in_front = [&](int key) { return kWhich == kOwn && key < p.q.from; };  // in the prefix
      const bool whole = there && k0 + KT - 1 <= pos_min && !in_front(k0) && (a.window == 0 || k0 > pos_max - a.window || k0 + KT - 1 < a.first);
      if (!whole) {
        asm volatile("");
        uint32_t top = 0;  // the signs' places: whether a value is not finite
        constexpr int kPerKey = DT / kE;
#pragma unroll
        for (int i = 0; i < kVLoads; ++i) {
          const int in = (64 * i + lane) / kPerKey, key = k0 + in;
          const bool none = ((kHalves == 1 ? cur[0] : in < 16 ? cur[0] : cur[kHalves - 1]) < 0) | (key > pos_max) | in_front(key) |
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
            const bool sees = real & (cur[h] >= 0) & (key <= pos) & !in_front(key) & ((a.window == 0) | (key > pos - a.window) | (key < a.first));
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
        for (t = seen_from(t_lo + stream); t < t_end; t = seen_from(t + streams)) {
          const int before = kWhich == kOwn ? max(p.q.from - key_of(t), 0) : 0;
          put_odd<M, KV, kRows>(a, table, hk, key_of(t) + before, KT - before, s.len, row0, all_rows, [&](int r, int d, float v) {
            float& sum = sums[r * (DT + 4) + d];
            sum = add ? sum + v : 0.0f;
          });
        }
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
    const int slot = 2 * (int)block + (t_lo == 0);
    if constexpr (kWhich == kOwn) {
      if (t_lo == 0 && wave == 0) {
        const OwnItem o = own_item(a, {w_first, shares, s.r0, of0, rows, hk}, s.n, group_at(p.b));
        if (lane == 0) a.prefix.item[p.item0 + item] = o;
      }
    } else {
      if (t_lo == 0 && threadIdx.x == 0) a.item[p.item0 + item] = Item{w_first, shares, s.r0, of0, rows, hk};
    }
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
      if (kWhich == kOwn || shares > 1) {
        const size_t at = (size_t)(kWhich == kOwn && shares == 1 ? kOwnSlots + (int)(p.item0 + item) : slot) * a.slot_rows + r;
        *(W4_GLOBAL f32x4*)(a.part + at * DT + d) = acc;
        if (d == 0) {
          a.state[2 * at] = top;
          a.state[2 * at + 1] = sum;
        }
      } else {
        finish<Act, kDump>(a, s.r0, of0 + r, hk, (size_t)(p.item0 + item) * a.slot_rows + r, d, acc, base, sum);
      }
    }
    u += deal.apart ? grid : t_hi - t_lo;
    if (u < u_end) __syncthreads();  // the next item's tiles go where these sums were read
  }
}

}  // namespace paged
}  // namespace w4
