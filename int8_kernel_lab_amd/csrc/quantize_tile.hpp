// Eight values of a row at a time: loads, the largest magnitude, int8 codes.
// Shared by the quantizing kernel and the linear layers that quantize the few
// rows they read themselves.
#pragma once

#include "linear_common.hpp"

namespace i8conv {

#if defined(__HIPCC__)

// x[i .. i + 7] as floats.  kVec: 16-byte loads, all of them aligned.
template <int TYPE, bool kVec>
__device__ __forceinline__ void load8(const void *x, int64_t i, float (&v)[8]) {
  if constexpr (TYPE == I8CONV_FP32) {
    const float *const p = static_cast<const float *>(x) + i;
    if constexpr (kVec) {
      const v4f a = *reinterpret_cast<const v4f *>(p), b = *reinterpret_cast<const v4f *>(p + 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = a[e], v[4 + e] = b[e];
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = p[e];
    }
  } else {
    const uint16_t *const p = static_cast<const uint16_t *>(x) + i;
    if constexpr (kVec) {
      const v4u a = *reinterpret_cast<const v4u *>(p);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = from_half(a[e / 2] >> (16 * (e & 1)) & 0xffffu, TYPE);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = from_half(p[e], TYPE);
    }
  }
}

// The largest magnitude, as bits: whole-number order is the order of the
// magnitudes, with infinity above every number and NaN above infinity.
__device__ __forceinline__ uint32_t top8(const float (&v)[8]) {
  uint32_t t = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) t = max(t, f32_bits(v[e]) & 0x7fffffffu);
  return t;
}

// The largest of the wave's values, in every lane.
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
#pragma unroll
  for (int d = 1; d < 64; d *= 2) v = max(v, uint32_t(__shfl_xor(int(v), d)));
  return v;
}

// A row's step: its scale, and what its codes are computed with.  Rows beyond
// 2^100 are brought down by 2^-60 first: 127 times their values or the
// reciprocal of their largest would leave the range of normal numbers.
struct RowStep {
  float top, inverse, times, scale;
};
__device__ __forceinline__ RowStep row_step(uint32_t top_bits) {
  RowStep s;
  const float top = bits_f32(top_bits);
  const bool sound = top_bits < 0x7f800000u, live = sound && top >= 0x1p-100f;
  const float down = top > 0x1p100f ? 0x1p-60f : 1.0f;
  s.top = live ? top * down : 1.0f;
  s.times = 127.0f * down;
  s.inverse = live ? 1.0f / s.top : 0.0f;  // 0: every code is 0
  s.scale = live ? top / 127.0f : sound ? 0.0f : bits_f32(0x7fc00000u);
  return s;
}

// rint(127 v / top): the quotient by the reciprocal, and one correction step
// by its remainder, which is exact in a fused multiply-add.  (127 v by the
// rounded 127 / top alone is off by an ulp at times, and at the half steps
// that is another code; they are frequent where values have few bits.)
__device__ __forceinline__ int code1(float v, const RowStep &s) {
  const float n = s.times * v, q = n * s.inverse;
  return int(rintf(fmaf(fmaf(-q, s.top, n), s.inverse, q)));
}
__device__ __forceinline__ v2u codes8(const float (&v)[8], const RowStep &s) {
  // a dead row's values may be infinite or NaN: 0 times them is not 0
  const bool dead = s.inverse == 0.0f;
  uint32_t c[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) c[e] = uint32_t(code1(v[e], s));
  v2u r;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const uint32_t lo = __builtin_amdgcn_perm(c[4 * h + 1], c[4 * h], 0x0c0c0400u);
    const uint32_t hi = __builtin_amdgcn_perm(c[4 * h + 3], c[4 * h + 2], 0x0c0c0400u);
    r[h] = dead ? 0u : __builtin_amdgcn_perm(hi, lo, 0x05040100u);
  }
  return r;
}

#endif  // __HIPCC__

}  // namespace i8conv
