// A cache of e4m3 codes with a power-of-two scale for each page and head: its
// exponents, conversions and pieces of elements.
#pragma once

#include "common.h"

namespace nk {

template <int N> struct Count {  // a number as a type
  static constexpr int value = N;
};

// exponents outside this range count as the nearest end: 2^e and 2^-e are normal
// fp32 numbers, and 448 2^120 is past fp32's largest
#define C8_MIN -120
#define C8_MAX 120
NK_DEVICE int c8_clip(int e) { return min(max(e, C8_MIN), C8_MAX); }
NK_DEVICE float c8_power(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }  // 2^e, e of -126 to 127
// the least exponent under which a finite magnitude is at most 448 = 1.75 2^8
NK_DEVICE int c8_exponent(float top) {
  const uint32_t u = __float_as_uint(top);
  const int e = (int)(u >> 23) - 127 - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
  return max(e, C8_MIN);  // (0 and subnormal numbers: far below)
}

// Two values as codes, nearest, ties to even (v_cvt_pk_fp8_f32); what is not finite
// as NaN.  Finite values are at most 448 here.
NK_DEVICE int c8_pair(float a, float b, int into, bool high) {
  a = __builtin_isfinite(a) ? a : __uint_as_float(0x7fc00000u);
  b = __builtin_isfinite(b) ? b : __uint_as_float(0x7fc00000u);
  return high ? __builtin_amdgcn_cvt_pk_fp8_f32(a, b, into, true) : __builtin_amdgcn_cvt_pk_fp8_f32(a, b, into, false);
}
template <int E>
NK_DEVICE void c8_store(uint8_t *p, const float (&x)[E], float scale) {
  if constexpr (E == 8) {
    uint2 w;
    w.x = c8_pair(x[2] * scale, x[3] * scale, c8_pair(x[0] * scale, x[1] * scale, 0, false), true);
    w.y = c8_pair(x[6] * scale, x[7] * scale, c8_pair(x[4] * scale, x[5] * scale, 0, false), true);
    *reinterpret_cast<uint2 *>(p) = w;
  } else {
#pragma unroll
    for (int e = 0; e < E; ++e) p[e] = (uint8_t)c8_pair(x[e] * scale, 0.f, 0, false);
  }
}
template <int E>
NK_DEVICE void c8_load(const uint8_t *p, float (&x)[E]) {
  if constexpr (E == 8) {
    const uint2 w = *reinterpret_cast<const uint2 *>(p);
    x[0] = __builtin_amdgcn_cvt_f32_fp8((int)w.x, 0), x[1] = __builtin_amdgcn_cvt_f32_fp8((int)w.x, 1);
    x[2] = __builtin_amdgcn_cvt_f32_fp8((int)w.x, 2), x[3] = __builtin_amdgcn_cvt_f32_fp8((int)w.x, 3);
    x[4] = __builtin_amdgcn_cvt_f32_fp8((int)w.y, 0), x[5] = __builtin_amdgcn_cvt_f32_fp8((int)w.y, 1);
    x[6] = __builtin_amdgcn_cvt_f32_fp8((int)w.y, 2), x[7] = __builtin_amdgcn_cvt_f32_fp8((int)w.y, 3);
  } else {
#pragma unroll
    for (int e = 0; e < E; ++e) x[e] = __builtin_amdgcn_cvt_f32_fp8((int)p[e], 0);
  }
}

}  // namespace nk
