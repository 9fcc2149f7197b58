// Operations over the 64 lanes of a wave without going through LDS: rotations
// within rows of 16 lanes (DPP), exchanges of rows and halves
// (v_permlane16_swap, v_permlane32_swap).  Operands are 32 bits wide, or 64 in
// two.
#pragma once
#include "hip_common.h"

namespace ane {

// the value of the lane N further on in the row of 16
template <int N>
__device__ __forceinline__ int row_ror(int v) {
  return __builtin_amdgcn_update_dpp(0, v, 0x120 + N, 0xf, 0xf, false);
}
template <int N>
__device__ __forceinline__ float row_ror(float v) {
  return __int_as_float(row_ror<N>(__float_as_int(v)));
}
template <int N>
__device__ __forceinline__ double row_ror(double v) {
  return __hiloint2double(row_ror<N>(__double2hiint(v)), row_ror<N>(__double2loint(v)));
}
// a's odd rows of 16 lanes with b's even ones
template <typename T>
__device__ __forceinline__ void swap16(T& a, T& b) {
  const auto r =
      __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b), false, false);
  const uint32_t x = r[0], y = r[1];
  a = __builtin_bit_cast(T, x);
  b = __builtin_bit_cast(T, y);
}
// a's upper half with b's lower half
template <typename T>
__device__ __forceinline__ void swap32(T& a, T& b) {
  const auto r =
      __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b), false, false);
  const uint32_t x = r[0], y = r[1];
  a = __builtin_bit_cast(T, x);
  b = __builtin_bit_cast(T, y);
}

struct Max {
  __device__ float operator()(float a, float b) const { return fmaxf(a, b); }
};
struct Sum {
  template <typename T>
  __device__ T operator()(T a, T b) const { return a + b; }
};
// In every lane, over N lanes (a power of two) that lie together; or, where
// what the lanes hold repeats every N <= 16 lanes, over one such stretch.
template <int N, typename T, typename Op>
__device__ __forceinline__ T over_lanes(T v, Op op) {
  if constexpr (N >= 2) v = op(v, row_ror<1>(v));
  if constexpr (N >= 4) v = op(v, row_ror<2>(v));
  if constexpr (N >= 8) v = op(v, row_ror<4>(v));
  if constexpr (N >= 16) v = op(v, row_ror<8>(v));
  if constexpr (N >= 32) {
    T w = v;
    swap16(v, w);
    v = op(v, w);
  }
  if constexpr (N >= 64) {
    T w = v;
    swap32(v, w);
    v = op(v, w);
  }
  return v;
}
// 64 bits wide: the rows one after the other
__device__ __forceinline__ double sum_over_lanes(double v) {
  v = over_lanes<16>(v, Sum());
  double s = 0.0;
#pragma unroll
  for (int r = 0; r < 4; r++)
    s += __hiloint2double(__builtin_amdgcn_readlane(__double2hiint(v), 16 * r),
                          __builtin_amdgcn_readlane(__double2loint(v), 16 * r));
  return s;
}

// The sum over the lanes up to this one: within rows of 16, then the last lane
// of a row to the row behind it, and of the lower half to the upper one.
template <int CTRL, int ROWS>
__device__ __forceinline__ int shifted(int v) {
  return __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xf, false);
}
__device__ __forceinline__ int sum_up_to(int v) {
  v += shifted<0x111, 0xf>(v);
  v += shifted<0x112, 0xf>(v);
  v += shifted<0x114, 0xf>(v);
  v += shifted<0x118, 0xf>(v);
  v += shifted<0x142, 0xa>(v);
  v += shifted<0x143, 0xc>(v);
  return v;
}

}  // namespace ane
