// Sums and maxima over a wavefront.
#pragma once

#include <hip/hip_runtime.h>

namespace w4 {

// Sums, maxima and minima over a wavefront by moves within the register file; scan: up to this lane.
template <int kCtrl, int kRowMask>
__device__ __forceinline__ double moved(double x) {  // 0 where no lane is
  const unsigned long long b = __builtin_bit_cast(unsigned long long, x);
  const unsigned lo = (unsigned)__builtin_amdgcn_update_dpp(0, (int)(unsigned)b, kCtrl, kRowMask, 0xf, false);
  const unsigned hi = (unsigned)__builtin_amdgcn_update_dpp(0, (int)(unsigned)(b >> 32), kCtrl, kRowMask, 0xf, false);
  return __builtin_bit_cast(double, (unsigned long long)hi << 32 | lo);
}
__device__ __forceinline__ double wave_scan(double x) {
  x += moved<0x111, 0xf>(x);  // row_shr 1, 2, 4, 8
  x += moved<0x112, 0xf>(x);
  x += moved<0x114, 0xf>(x);
  x += moved<0x118, 0xf>(x);
  x += moved<0x142, 0xa>(x);  // row_bcast 15, 31
  x += moved<0x143, 0xc>(x);
  return x;
}
__device__ __forceinline__ double of_lane(double x, int lane) {
  const unsigned long long b = __builtin_bit_cast(unsigned long long, x);
  const unsigned lo = (unsigned)__builtin_amdgcn_readlane((int)(unsigned)b, lane), hi = (unsigned)__builtin_amdgcn_readlane((int)(unsigned)(b >> 32), lane);
  return __builtin_bit_cast(double, (unsigned long long)hi << 32 | lo);
}
__device__ __forceinline__ double wave_add(double x) { return of_lane(wave_scan(x), 63); }
template <int kCtrl, int kRowMask>
__device__ __forceinline__ float most(float x) {
  const int y = __builtin_amdgcn_update_dpp((int)0xff800000, __float_as_int(x), kCtrl, kRowMask, 0xf, false);  // -infinity where no lane is
  return fmaxf(x, __int_as_float(y));
}
__device__ __forceinline__ float wave_max(float x) {
  x = most<0x111, 0xf>(x);
  x = most<0x112, 0xf>(x);
  x = most<0x114, 0xf>(x);
  x = most<0x118, 0xf>(x);
  x = most<0x142, 0xa>(x);
  x = most<0x143, 0xc>(x);
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), 63));
}

}  // namespace w4
