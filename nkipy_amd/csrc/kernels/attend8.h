// Attention over a paged cache of e4m3 codes: its arguments and one query row by
// one wave.
#pragma once

#include "attend.h"
#include "cache8.h"

namespace nk {

struct Attend8Args : AttendArgs {  // k, v: codes; strides in bytes
  const int32_t *ke, *ve;          // (pages, Hkv) exponents
};

// One query row by one wave, over blocks j0 .. j1-1 of its tile's span: eight lanes
// share a key's product, 64 keys a step; then the lanes share the head's elements,
// d = lane + 64 e.  Only the keys that the row sees are read; 32-bit weights of at
// most 1.  A code is finite or NaN, and NaN reaches the sum under any weight, 0
// included: no rule for values that are infinite, as those over 16-bit caches need.
// DIM: the head dim where it is known, which saves registers.
template <typename T, int DIM = 0>
NK_DEVICE void att8_row(const Attend8Args &a, const AttSeq &sq, const AttSpan &sp, int b, int i, int h, int j0, int j1,
                        float &m, float &l, float (&acc)[DIM ? (DIM + 63) / 64 : 4]) {
  const int lane = threadIdx.x & 63, c = lane & 7;
  const int g = h / (a.Hq / a.Hkv), p = sq.p0 + i, D = DIM ? DIM : a.D, per = (D + 7) / 8;
  constexpr int C = DIM ? (DIM + 7) / 8 : 32, V = DIM ? (DIM + 63) / 64 : 4;
  const T *q = (const T *)a.q + (int64_t)(sq.lo + i) * a.q_ss + (int64_t)h * a.q_sh;
  const uint8_t *k = (const uint8_t *)a.k + (int64_t)g * a.k_sh, *v = (const uint8_t *)a.v + (int64_t)g * a.v_sh;
  float qc[C];
#pragma unroll
  for (int e = 0; e < C; ++e) {
    const int d = c * per + e;
    qc[e] = e < per && d < D ? Elt<T>::load(q, d) * a.scale : 0.f;
  }
  m = -INFINITY, l = 0.f;
#pragma unroll
  for (int e = 0; e < V; ++e) acc[e] = 0.f;
  for (int x0 = j0 * ATT_KEYS; x0 < j1 * ATT_KEYS; x0 += 64) {
    const int x = x0 + lane;
    const int key = sp.kb(x / ATT_KEYS) * ATT_KEYS + x % ATT_KEYS;
    int row = -1;
    float ks = 0.f, vs = 0.f;
    if (x < j1 * ATT_KEYS && att_sees(a, sq, p, key)) {
      const int pg = a.tables[(int64_t)b * a.width + key / a.page];
      if (pg >= 0 && pg < a.pages) {
        row = pg * a.pitch + key % a.page;
        ks = c8_power(c8_clip(a.ke[(int64_t)pg * a.Hkv + g]));
        vs = c8_power(c8_clip(a.ve[(int64_t)pg * a.Hkv + g]));
      }
    }
    uint64_t todo = __ballot(row >= 0);
    if (!todo) continue;
    float s = -INFINITY;
    for (int n = 0; n < 8; ++n) {
      const int r = __shfl(row, (lane & 56) + n, 64);
      float d = 0.f;
      if (r >= 0) {
        const uint8_t *kr = k + (int64_t)r * a.k_ss;
#pragma unroll
        for (int e = 0; e < C; ++e)
          if (e < per && c * per + e < D) d = fmaf(qc[e], __builtin_amdgcn_cvt_f32_fp8((int)kr[c * per + e], 0), d);
      }
      d += __shfl_xor(d, 1, 64);
      d += __shfl_xor(d, 2, 64);
      d += __shfl_xor(d, 4, 64);
      if (c == n && row >= 0) s = d * ks;
    }
    const float mn = fmaxf(m, wave_max(s));
    const float w = s == -INFINITY ? 0.f : exp_acc(s - mn);
    const float alpha = m == mn ? 1.f : exp_acc(m - mn);
    m = mn;
    l = l * alpha + wave_sum(w);
#pragma unroll
    for (int e = 0; e < V; ++e) acc[e] *= alpha;
    while (todo) {
      const int n = __builtin_ctzll(todo);
      todo &= todo - 1;
      const float wn = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(w), n));
      const float vn = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(vs), n));
      const uint8_t *vr = v + (int64_t)__builtin_amdgcn_readlane(row, n) * a.v_ss;
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (lane + 64 * e < D) acc[e] = fmaf(wn, __builtin_amdgcn_cvt_f32_fp8((int)vr[lane + 64 * e], 0) * vn, acc[e]);
    }
  }
}

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 B8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
NK_DEVICE f32x4 mul16(B8 a, B8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
NK_DEVICE f32x16 mul32(B8 a, B8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }

// Codes enter the products as bf16: code 2^e is exact there (4 significant bits,
// fp32's exponents).  fp16 queries and the weights over them, which bf16 does not hold,
// enter as two bf16 numbers each, x = RN(x) + RN(x - RN(x)): exact for a query's 11 bits,
// a weight keeps 16.  (Weights of single tokens do so always.)
template <typename T> struct Parts;
template <> struct Parts<bf16> { static constexpr int N = 1; };
template <> struct Parts<f16> { static constexpr int N = 2; };
#define ATT8_LIMIT 65536.f
#define ATT8_LOWEST -3.40282347e38f  // the least finite offset
#define LOG2E 1.44269504088896340736f

template <typename T, int NP>
NK_DEVICE void load_q(const T *q, B8 (&f)[NP]) {
  if constexpr (NP == 1) {
    f[0] = *reinterpret_cast<const B8 *>(q);
  } else {
    float x[8];
    Vec8<T>::load(q, x);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      f[0][e] = (__bf16)x[e];
      f[1][e] = (__bf16)(x[e] - (float)f[0][e]);
    }
  }
}
template <int NP>
NK_DEVICE void put_weight(B8 *f, int e, float x) {
  f[0][e] = (__bf16)x;
  if constexpr (NP == 2) f[1][e] = (__bf16)(x - (float)f[0][e]);
}
// eight codes times a power of two
NK_DEVICE B8 codes8(uint32_t lo, uint32_t hi, float scale) {
  u32x4_t w;
  w[0] = bf16x2_bits(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false));
  w[1] = bf16x2_bits(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true));
  w[2] = bf16x2_bits(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false));
  w[3] = bf16x2_bits(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true));
  return __builtin_bit_cast(B8, w);
}

}  // namespace nk
