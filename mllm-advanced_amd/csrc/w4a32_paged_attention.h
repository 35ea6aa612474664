// What the two kernels of attention on a paged cache share: how rows are found and dealt, and the arithmetic of each element type.
#pragma once

#include <type_traits>

#include "w4a32_paged.h"

namespace w4 {
namespace paged {

constexpr int kRows = 16;         // query rows of a wavefront
constexpr int kWaves = 4;         // wavefronts of a workgroup
typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef float f8 __attribute__((ext_vector_type(8)));
typedef short s4 __attribute__((ext_vector_type(4)));
typedef unsigned long long u64;

// What the second launch has to know of an item
struct Item {
  int first, shares;  // workgroup that has its first tile, and how many have a part of it
  int r0, row0, rows, head;  // first row of the sequence, first of the item among (token, head of the group), their number, kv head
};

struct Attend {
  Cache c;
  const void* q;
  void* out;
  const int* row_start;
  int ldq, ldo, rows, max_rows, heads, group;
  unsigned group_mul;   // by_group()
  int group_shift;
  int row_lo, row_hi;   // of the step's rows those that the launch is about
  int window, first;
  int prompt_rows;      // (token, head of the group) pairs from which on a sequence is the prompts' kernel's; 0: none is
  int prompt_log2;      // log2 of the rows of a workgroup of that kernel: 8 (7 with 256 dims or in f32), or 5
  int wide;             // log2 of the wavefronts with rows of their own (1, 2 or 4): an item has 16 << wide rows
  int slot_rows;        // rows of an item that can be there: what a slot of scratch memory holds
  unsigned most_items, most_tiles;  // what the scratch memory holds: row starts that overlap could ask for more, and get nothing
  float scale;          // of the scores, times log2 e
  struct Item* item;    // [most_items]
  unsigned* count;      // how many there are
  float* part;          // [2 grid][slot_rows][dt]: sums of a share, relative to its maxima
  float* state;         // [2 grid][slot_rows][2]: maxima (log2) and sums of weights
  float* lse;           // [item][slot_rows] (accumulate)
  float* dump;          // [tile of an item][wide][lane][keys of the tile / 4]: scores (accumulate)
};

// x / group for x below 2^30, as x m / 2^(30 + l) with 2^l >= group > 2^(l - 1) and m the next whole number from 2^(30 + l) / group:
// m is off by less than 1, the quotient by less than 2^-l, and group is at most 2^l. A division takes the compiler 30 instructions.
inline void set_group(Attend& a) {
  int l = 0;
  while ((1ll << l) < a.group) ++l;
  a.group_shift = 30 + l;
  a.group_mul = (unsigned)(((1ull << (30 + l)) + a.group - 1) / a.group);
}
__device__ __forceinline__ int by_group(const Attend& a, int x) { return (int)((u64)(unsigned)x * a.group_mul >> a.group_shift); }

// The keys that a sequence's rows can see, in tiles: [0, ft) of the first tokens, then [w0, w0 + nt - ft).
struct Seq {
  Span s;
  int keys;        // tokens there are once the rows are appended
  int ft, w0, nt;  // tiles; at least one where there are rows
  int items;       // per kv head
};

// kPrompt: the sequences of the prompts' kernel, in items of 1 << prompt_log2 rows; else the others
template <int KT, bool kPrompt>
__device__ __forceinline__ Seq seq_of(const Attend& a, int b) {
  Seq q;
  q.s = span_of(a.c, a.row_start, a.rows, a.max_rows, b);
  const int before = max(a.row_lo - q.s.r0, 0);  // rows of an earlier launch: tokens to these
  q.s.n = max(min(q.s.n, a.row_hi - q.s.r0) - before, 0);
  q.s.r0 += before;
  q.s.len += before;
  const long long pairs = (long long)q.s.n * a.group;
  if ((a.prompt_rows && pairs >= a.prompt_rows) != kPrompt) q.s.n = 0;
  q.keys = min(q.s.len + q.s.n, a.c.cap);
  const int log2 = kPrompt ? a.prompt_log2 : 4 + a.wide;
  q.items = q.s.n ? (int)((pairs + (1 << log2) - 1) >> log2) : 0;
  q.w0 = 0;
  q.ft = 0;
  if (a.window) {
    q.w0 = max(0, min(q.s.len, a.c.cap - 1) - a.window + 1) / KT;
    q.ft = min((min(a.first, a.c.cap) + KT - 1) / KT, q.w0);
  }
  q.nt = q.s.n ? q.ft + (q.keys + KT - 1) / KT - q.w0 : 0;
  return q;
}

// Sums over the wavefront's lanes up to this one, by moves within the register file; sums that do not fit stay at the most.
__device__ __forceinline__ unsigned add_sat(unsigned a, unsigned b) { return __builtin_elementwise_add_sat(a, b); }
__device__ __forceinline__ unsigned wave_scan(unsigned x) {
  x = add_sat(x, (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, 0x111, 0xf, 0xf, false));  // row_shr 1, 2, 4, 8
  x = add_sat(x, (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, 0x112, 0xf, 0xf, false));
  x = add_sat(x, (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, 0x114, 0xf, 0xf, false));
  x = add_sat(x, (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, 0x118, 0xf, 0xf, false));
  x = add_sat(x, (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, 0x142, 0xa, 0xf, false));  // row_bcast 15, 31
  x = add_sat(x, (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, 0x143, 0xc, 0xf, false));
  return x;
}
__device__ __forceinline__ unsigned last_lane(unsigned x) { return (unsigned)__builtin_amdgcn_readlane((int)x, 63); }

// How a batch is dealt, and what is counted: tiles of items, shares of one item, tiles of a kv head, one for each wavefront (for
// the launch that adds weights up), or items.
enum Unit { kTiles, kShares, kKeyTiles, kItems };
struct Deal {
  unsigned total, items, per;  // tiles, items, tiles of a share; per = 0: nothing can be done
  bool apart;                  // a share has tiles of one item only: ceil(nt / per) of them per item
};
struct Place {
  bool there;
  int b;
  unsigned inner;   // which one of the sequence
  unsigned tile0;   // tiles of items in front of the sequence
  unsigned item0;   // items in front of the sequence
  Seq q;
};

// The sequences of a block of 64, one of each lane: kept where there is one block only.
template <int KT, bool kPrompt = false>
struct Seqs {
  Seq q;
  unsigned tiles, items;
  __device__ __forceinline__ void load(const Attend& a, int b0) {
    const int b = b0 + (int)(threadIdx.x & 63);
    q = {};
    tiles = items = 0;
    if (b < a.c.n_seqs) {
      q = seq_of<KT, kPrompt>(a, b);
      const u64 n = (u64)q.items * a.c.kv_heads;
      items = (unsigned)min(n, (u64)0xffffffffu);
      tiles = (unsigned)min(n * q.nt, (u64)0xffffffffu);
    }
  }
};

template <int KT, bool kPrompt>
__device__ __forceinline__ Place place_of(const Attend& a, Seqs<KT, kPrompt>& s, unsigned u, Unit unit, unsigned per) {
  Place p;
  p.there = false;
  p.tile0 = p.item0 = 0;
  if (a.c.n_seqs == 1) {
    auto from = [&](int x) { return __builtin_amdgcn_readfirstlane(x); };
    p.b = 0;
    p.inner = u;
    p.q = {{from(s.q.s.r0), from(s.q.s.n), from(s.q.s.len)}, from(s.q.keys), from(s.q.ft), from(s.q.w0), from(s.q.nt), from(s.q.items)};
    const unsigned each = unit == kTiles ? p.q.nt : unit == kShares ? (p.q.nt + per - 1) / per : unit == kItems ? 1 : (p.q.nt + kWaves - 1) / kWaves;
    p.there = u < each * (unsigned)a.c.kv_heads * (unit == kKeyTiles ? 1 : p.q.items);
    return p;
  }
  unsigned before = 0;
  for (int b0 = 0; b0 < a.c.n_seqs; b0 += 64) {
    if (a.c.n_seqs > 64) s.load(a, b0);
    const unsigned keys = (unsigned)a.c.kv_heads * ((s.q.nt + kWaves - 1) / kWaves);
    const unsigned items = wave_scan(s.items), tiles = wave_scan(s.tiles);
    const unsigned count = unit == kTiles ? s.tiles : unit == kShares ? s.items * ((s.q.nt + per - 1) / per) : unit == kItems ? s.items : keys;
    const unsigned upto = unit == kTiles ? tiles : unit == kItems ? items : wave_scan(count);
    const u64 found = __ballot(add_sat(before, upto) > u);
    if (found) {
      const int at = __builtin_ctzll(found);
      auto from = [&](unsigned x) { return __builtin_amdgcn_readlane((int)x, at); };
      p.there = true;
      p.b = b0 + at;
      p.inner = u - before - (unsigned)from(upto - count);
      p.tile0 += (unsigned)from(tiles - s.tiles);
      p.item0 += (unsigned)from(items - s.items);
      p.q.s.r0 = from(s.q.s.r0);
      p.q.s.n = from(s.q.s.n);
      p.q.s.len = from(s.q.s.len);
      p.q.keys = from(s.q.keys);
      p.q.ft = from(s.q.ft);
      p.q.w0 = from(s.q.w0);
      p.q.nt = from(s.q.nt);
      p.q.items = from(s.q.items);
      return p;
    }
    before = add_sat(before, last_lane(upto));
    p.tile0 = add_sat(p.tile0, last_lane(tiles));
    p.item0 = add_sat(p.item0, last_lane(items));
  }
  return p;
}

__device__ __forceinline__ float group_max(float x) {  // over the four lane groups: all lanes of one query row
  x = fmaxf(x, __shfl_xor(x, 16));
  return fmaxf(x, __shfl_xor(x, 32));
}
__device__ __forceinline__ float group_sum(float x) {
  x += __shfl_xor(x, 16);
  return x + __shfl_xor(x, 32);
}
__device__ __forceinline__ float pow2(float x) { return __builtin_amdgcn_exp2f(x); }

// ---- element types ---------------------------------------------------------------------------------------------------------
// Values that are not finite must reach only rows that see their key, and 0 times one would reach all. In a tile that not every
// row sees whole they are zeros to the product; where there were some, or where a row's sums are not finite, they are added behind
// the last tile, key by key.

// What brings a share's sums to a common reference is at least this for the values: an infinity stays one where the share's
// weight underflows, and finite ones add next to nothing.
constexpr float kLeast = 0x1p-126f;
template <typename KV>
using Bits = typename std::conditional<sizeof(KV) == 2, uint16_t, uint32_t>::type;  // an element as it lies in the pools

// kTerms operands stand for one f32 operand of the 16-bit matrix instruction. kScale: exponent that the softmaxed scores
// carry until the sums are divided (they cancel there).
template <typename Act, typename KV>
struct Math;

// bf16: three truncations hold the 24 bits of an f32 whatever its exponent. Rows of bf16 are operands as they are, and their weights,
// whose sum is f32, are rounded to one bf16 (half a step, 2^-8 at most, of signs that cancel): less than the rounding of the result, which is
// bf16 too (against 64 bits 1.8e-3 for one row on a long context and 2.3e-3 for a prompt, 1.7e-3 with exact weights), for a third of the products.
template <typename Act>
struct Math<Act, __bf16> {
  static constexpr int kTerms = sizeof(Act) == 4 ? 3 : 1;
  static constexpr int kScale = 0;
  typedef bf8 V8;
  static __device__ __forceinline__ f32x4 mfma(V8 a, V8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
  static __device__ __forceinline__ void split(const float (&x)[8], V8 (&t)[kTerms]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if constexpr (kTerms == 1) {
        t[0][i] = (__bf16)x[i];
      } else {
        float r = x[i];
#pragma unroll
        for (int k = 0; k < kTerms; ++k) {
          const uint32_t top = __float_as_uint(r) & 0xffff0000u;
          t[k][i] = __builtin_bit_cast(__bf16, (uint16_t)(top >> 16));
          r -= __uint_as_float(top);
        }
      }
    }
  }
  static constexpr uint32_t kSize = 0x7fff7fffu, kStep = 0x00800080u;  // a largest exponent and kStep give the sign's bit
  static __device__ __forceinline__ uint32_t finite(uint32_t w) {  // two elements, those that are not finite as 0
    return ((w & 0x7f80u) == 0x7f80u ? 0u : w & 0xffffu) | ((w & 0x7f800000u) == 0x7f800000u ? 0u : w & 0xffff0000u);
  }
  static __device__ __forceinline__ float widen(uint16_t h) { return __uint_as_float((uint32_t)h << 16); }
};
// f16: two roundings hold 22 to 24 bits of a number that is scaled near the type's largest, and of a smaller one whatever
// lies above 2^-40 of the row's largest
template <typename Act>
struct Math<Act, _Float16> {
  static constexpr int kTerms = 2;
  static constexpr int kScale = 15;
  typedef h8 V8;
  // the power of two (2^127 at most) that brings a row of q, of which `most` is the largest, to 2^14 .. 2^15; its inverse joins the
  // row's scale, which stays finite: what it is the scale of may be 0
  static __device__ __forceinline__ float row_scale(float most, float& scale) {
    int e = 0;
    if (most > 0.0f && most < INFINITY) e = min(14 - ilogbf(most), 127);
    scale = __builtin_amdgcn_fmed3f(scale * ldexpf(1.0f, -e), -3.40282347e38f, 3.40282347e38f);
    return ldexpf(1.0f, e);
  }
  static __device__ __forceinline__ f32x4 mfma(V8 a, V8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
  static __device__ __forceinline__ void split(const float (&x)[8], V8 (&t)[kTerms]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      t[0][i] = (_Float16)x[i];
      t[1][i] = (_Float16)(x[i] - (float)t[0][i]);
    }
  }
  static constexpr uint32_t kSize = 0x7fff7fffu, kStep = 0x04000400u;
  static __device__ __forceinline__ uint32_t finite(uint32_t w) {
    return ((w & 0x7c00u) == 0x7c00u ? 0u : w & 0xffffu) | ((w & 0x7c000000u) == 0x7c000000u ? 0u : w & 0xffff0000u);
  }
  static __device__ __forceinline__ float widen(uint16_t h) { return (float)__builtin_bit_cast(_Float16, h); }
};
// f32: the f32 matrix instruction, operands as they are
template <>
struct Math<float, float> {
  static constexpr int kTerms = 1;
  static constexpr int kScale = 0;
  typedef f8 V8;
  static __device__ __forceinline__ void split(const float (&x)[8], V8 (&t)[kTerms]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) t[0][i] = x[i];
  }
  static __device__ __forceinline__ f32x4 mfma(float a, float b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }
  static constexpr uint32_t kSize = 0x7fffffffu, kStep = 0x00800000u;
  static __device__ __forceinline__ uint32_t finite(uint32_t w) { return (w & 0x7f800000u) == 0x7f800000u ? 0u : w; }
  static __device__ __forceinline__ float widen(uint32_t x) { return __uint_as_float(x); }
};

template <typename Act>
__device__ __forceinline__ void load8(const void* p, size_t at, float (&x)[8]) {
  if constexpr (sizeof(Act) == 4) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const f32x4 v = load_global<f32x4>((const float*)p + at + 4 * h);
#pragma unroll
      for (int i = 0; i < 4; ++i) x[4 * h + i] = v[i];
    }
  } else {
    const u32x4 v = load_global<u32x4>((const uint16_t*)p + at);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = __uint_as_float(i & 1 ? v[i / 2] & 0xffff0000u : v[i / 2] << 16);
  }
}
template <typename Act>
__device__ __forceinline__ void store4(void* p, size_t at, f32x4 x) {
  if constexpr (sizeof(Act) == 4) {
    *(W4_GLOBAL f32x4*)((float*)p + at) = x;
  } else {
    typedef __bf16 b4 __attribute__((ext_vector_type(4)));
    *(W4_GLOBAL b4*)((uint16_t*)p + at) = b4{(__bf16)x[0], (__bf16)x[1], (__bf16)x[2], (__bf16)x[3]};
  }
}

// Of the keys [k0, k0 + keys), the values that are not finite to a wavefront's kRows rows that see them, by put(row, dim, value); the
// first is row0 of the sequence's all_rows, whose tokens follow len cached ones. Lanes have dims; all is rare and short but the look
// at every value.
template <typename M, typename KV, int kRows, typename Put>
__device__ __forceinline__ void put_odd(const Attend& a, const int* table, int hk, int k0, int keys, int len, int row0, int all_rows, Put put) {
#pragma unroll 1
  for (int key = k0; key < k0 + keys; ++key) {
    const int at = key >> a.c.shift, page = at < a.c.table_ld ? table[at] : -1;
    if (!page_there(a.c, page)) continue;
    const Bits<KV>* v = (const Bits<KV>*)a.c.v + slot_row(a.c, page, hk, key) * a.c.dim;
#pragma unroll 1
    for (int d = threadIdx.x & 63; d - (int)(threadIdx.x & 63) < a.c.dim; d += 64) {
      const uint32_t bits = d < a.c.dim ? v[d] : 0u;
      const bool odd = M::finite(bits) != bits;
      if (!__any(odd)) continue;
#pragma unroll 1
      for (int r = 0; r < min(kRows, all_rows - row0); ++r) {
        const int pos = len + by_group(a, row0 + r);
        if (key > pos || !(a.window == 0 || key > pos - a.window || key < a.first)) continue;
        if (odd) put(r, d, M::widen((Bits<KV>)bits));
      }
    }
  }
}

// A row's result, from its sums and the sum of its weights
template <typename Act, bool kDump>
__device__ __forceinline__ void finish(const Attend& a, int r0, int of, int hk, size_t lse_at, int d, f32x4 acc, float base, float sum) {
  if (d < a.c.dim) {
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    const int j = by_group(a, of);
    const size_t at = (size_t)(r0 + j) * a.ldo + (size_t)(hk * a.group + of - j * a.group) * a.c.dim;
    store4<Act>(a.out, at + d, acc * inv);
  }
  if (kDump && d == 0) a.lse[lse_at] = sum == 0.0f ? INFINITY : base + __log2f(sum);
}

// The prompts' kernel over the sequences of at least a.prompt_rows pairs (w4a32_paged_prompt.hip); items: its most workgroups
hipError_t launch_prompts(const Attend& a, int dtype, bool act_bf16, int dt, unsigned items, hipStream_t s);

}  // namespace paged
}  // namespace w4
