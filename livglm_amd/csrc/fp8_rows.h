// Rows and weights in E4M3 with f32 scales: a group of 128 channels of a row,
// or a 128 x 128 block of a weight, holds amax / 448 as its scale and
// e4m3(value * (448 / amax)) as its codes; both quotients are rounded once, in
// f32, so that every kernel here gives the same codes for the same values.
#pragma once

#include "glm_common.h"

namespace glm {

constexpr int kFp8Group = 128;
constexpr float kFp8Max = 448.0f;
// the smallest amax that is told apart: its scale is 2^-126, the smallest
// normal number, so that neither quotient leaves f32's normal range
constexpr float kFp8Tiny = 448.0f * 0x1p-126f;

__host__ __device__ constexpr int fp8_groups(int n) { return (n + kFp8Group - 1) / kFp8Group; }

// Eight values from 16 bytes of bf16 or 32 of f32.
__device__ __forceinline__ void unpack8(const glm_u32x4 &u, float v[8]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    v[2 * j] = __uint_as_float(u[j] << 16);
    v[2 * j + 1] = __uint_as_float(u[j] & 0xffff0000u);
  }
}
template <bool F32>
__device__ __forceinline__ void load8(const void *row, long long c, float v[8]) {
  if constexpr (F32) {
    const glm_f32x4 *p = reinterpret_cast<const glm_f32x4 *>((const float *)row + c);
    const glm_f32x4 a = p[0], b = p[1];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      v[j] = a[j];
      v[4 + j] = b[j];
    }
  } else {
    unpack8(*reinterpret_cast<const glm_u32x4 *>((const uint16_t *)row + c), v);
  }
}

// Largest magnitude of N values; a NaN is passed over, an infinity is not.
template <int N>
__device__ __forceinline__ float abs_max(const float (&v)[N]) {
  float m = 0.f;
#pragma unroll
  for (int j = 0; j < N; ++j) m = fmaxf(m, fabsf(v[j]));
  return m;
}
// The same without infinities, which become NaN (their codes are E4M3's NaN).
template <int N>
__device__ __forceinline__ float finite_abs_max(float (&v)[N]) {
  float m = 0.f;
#pragma unroll
  for (int j = 0; j < N; ++j) {
    if (isinf(v[j])) v[j] = __uint_as_float(0x7fc00000u);
    m = fmaxf(m, fabsf(v[j]));
  }
  return m;
}

// Maximum over the 16 lanes of a DPP row (rotations by 8, 4, 2, 1).
__device__ __forceinline__ float row16_max(float m) {
  m = fmaxf(m, __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(m), 0x128, 0xf, 0xf, true)));
  m = fmaxf(m, __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(m), 0x124, 0xf, 0xf, true)));
  m = fmaxf(m, __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(m), 0x122, 0xf, 0xf, true)));
  m = fmaxf(m, __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(m), 0x121, 0xf, 0xf, true)));
  return m;
}

// Largest finite magnitude of a group whose 128 values lie 8 a lane over the
// 16 lanes of a DPP row; infinities in v become NaN.
__device__ __forceinline__ float group_amax(float (&v)[8]) {
  float m = row16_max(abs_max(v));
  if (__builtin_expect(isinf(m), 0)) m = row16_max(finite_abs_max(v));  // (one answer in the row)
  return fmaxf(m, kFp8Tiny);
}

// Four values times `up` as codes, round to nearest even; |v * up| is 448 or
// less by at most a last place, which rounds to 448, or NaN.
__device__ __forceinline__ uint32_t fp8_codes4(float a, float b, float c, float d, float up) {
  typedef short s16x2 __attribute__((ext_vector_type(2)));
  s16x2 o = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(s16x2{0, 0}, a * up, b * up, 1.0f, false);
  o = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(o, c * up, d * up, 1.0f, true);
  return __builtin_bit_cast(uint32_t, o);
}

}  // namespace glm
