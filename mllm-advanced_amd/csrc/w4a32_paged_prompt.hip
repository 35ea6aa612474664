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
#include "w4a32_paged_prompt.h"

namespace w4 {
namespace paged {

namespace {
template <typename Act, typename KV, int DT, Form kForm>
__global__ __launch_bounds__((Shape<Act, KV, DT, kForm>::kThreads), DT == 256 || kForm == kTeamsForm ? 1 : 2) void prompt_kernel(Attend a) {
  prompt_body<Act, KV, DT, kForm, kAllTokens>(a, blockIdx.x, {});
}

template <typename Act, typename KV, int DT, Form kForm>
hipError_t launch(const Attend& a, unsigned items, hipStream_t s) {
  using Sh = Shape<Act, KV, DT, kForm>;
  if constexpr (Sh::kLds > 64 * 1024) {
    static LdsLimitOnce limit;
    if (hipError_t e = limit.raise((const void*)prompt_kernel<Act, KV, DT, kForm>, Sh::kLds); e != hipSuccess) return e;
  }
  hipLaunchKernelGGL((prompt_kernel<Act, KV, DT, kForm>), dim3(items), dim3(Sh::kThreads), Sh::kLds, s, a);
  return hipGetLastError();
}
template <typename Act, typename KV, Form kForm>
hipError_t launch_dim(const Attend& a, int dt, unsigned items, hipStream_t s) {
  if (dt == 64) return launch<Act, KV, 64, kForm>(a, items, s);
  if (dt == 128) return launch<Act, KV, 128, kForm>(a, items, s);
  return launch<Act, KV, 256, kForm>(a, items, s);
}
template <typename Act, typename KV>
hipError_t launch_form(const Attend& a, int dt, unsigned items, hipStream_t s) {
  return a.prompt_log2 == 5 ? launch_dim<Act, KV, kTeamsForm>(a, dt, items, s) : launch_dim<Act, KV, kWideForm>(a, dt, items, s);
}
}  // namespace

hipError_t launch_prompts(const Attend& a, int dtype, bool act_bf16, int dt, unsigned items, hipStream_t s) {
  if (dtype == W4A32_CACHE_F32) {
    if (dt == 64) return launch<float, float, 64, kTeamsForm>(a, items, s);
    return dt == 128 ? launch<float, float, 128, kWideForm>(a, items, s) : launch<float, float, 256, kWideForm>(a, items, s);
  }
  if (act_bf16) return launch_form<__bf16, __bf16>(a, dt, items, s);
  if (dtype == W4A32_CACHE_F16) return launch_form<float, _Float16>(a, dt, items, s);
  return launch_form<float, __bf16>(a, dt, items, s);
}

}  // namespace paged
}  // namespace w4
