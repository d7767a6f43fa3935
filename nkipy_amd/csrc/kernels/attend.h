// Attention of queries at known positions to keys in a paged cache or in plain
// tensors: the wave's search for a sequence and one query row by one wave (the
// definition and the layout of the work stand in attend_index.h).
#pragma once

#include "common.h"

namespace nk {

// the last b with f(b) <= x, -1 for none; f does not decrease.  Every lane of
// the wave looks at sequences of its own: one load deep for 64 of them.
template <typename F>
NK_DEVICE int att_find(int n, int x, F f) {
  const int lane = threadIdx.x & 63;
  int c = 0;
  for (int b0 = 0; b0 < n; b0 += 64) {
    const int b = b0 + lane;
    c += __popcll(__ballot(b < n && f(min(b, n - 1)) <= x));
  }
  return c - 1;
}

}  // namespace nk

#include "attend_index.h"

namespace nk {

// Sums of weighted values: one that is not finite counts whole, also under a weight
// or a rescaling that rounds to 0.
NK_DEVICE float att_add(float w, float v, float acc) { return fmaf(__builtin_isfinite(v) ? w : 1.f, v, acc); }
NK_DEVICE float att_rescale(float acc, float alpha) { return __builtin_isfinite(acc) ? acc * alpha : acc; }

// One query row by one wave, over blocks j0 .. j1-1 of its tile's span: eight
// lanes share a key's product, 64 keys a step; then the lanes share the head's
// elements, d = lane + 64 e.  Only the keys that the row sees are read.  DIM: the head
// dim where it is known, which saves registers; WHOLE: sums by att_add (1000 tokens of
// 32 / 8 heads of 80: 2489 us with, 2231 without).
template <typename T, bool WHOLE, int DIM = 0>
NK_DEVICE void att_row(const AttendArgs &a, const AttSeq &sq, const AttSpan &sp, int b, int i, int h, int j0, int j1,
                       float &m, float &l, float (&acc)[DIM ? (DIM + 63) / 64 : 4]) {
  const int lane = threadIdx.x & 63, c = lane & 7;
  const int g = h / (a.Hq / a.Hkv), p = sq.p0 + i, D = DIM ? DIM : a.D, per = (D + 7) / 8;
  constexpr int C = DIM ? (DIM + 7) / 8 : 32, V = DIM ? (DIM + 63) / 64 : 4;
  const int64_t qrow = a.tables ? (int64_t)(sq.lo + i) * a.q_ss : (int64_t)b * a.q_sb + (int64_t)i * a.q_ss;
  const T *q = (const T *)a.q + qrow + (int64_t)h * a.q_sh;
  const T *k = (const T *)a.k + (a.tables ? 0 : (int64_t)b * a.k_sb) + (int64_t)g * a.k_sh;
  const T *v = (const T *)a.v + (a.tables ? 0 : (int64_t)b * a.v_sb) + (int64_t)g * a.v_sh;
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
    if (x < j1 * ATT_KEYS && att_sees(a, sq, p, key)) row = att_place(a, b, key);
    uint64_t todo = __ballot(row >= 0);
    if (!todo) continue;
    float s = -INFINITY;
    for (int n = 0; n < 8; ++n) {
      const int r = __shfl(row, (lane & 56) + n, 64);
      float d = 0.f;
      if (r >= 0) {
        const T *kr = k + (int64_t)r * a.k_ss;
#pragma unroll
        for (int e = 0; e < C; ++e)
          if (e < per && c * per + e < D) d = fmaf(qc[e], Elt<T>::load(kr, c * per + e), d);
      }
      d += __shfl_xor(d, 1, 64);
      d += __shfl_xor(d, 2, 64);
      d += __shfl_xor(d, 4, 64);
      if (c == n && row >= 0) s = d;
    }
    const float mn = fmaxf(m, wave_max(s));
    const float w = s == -INFINITY ? 0.f : exp_acc(s - mn);
    const float alpha = m == mn ? 1.f : exp_acc(m - mn);
    m = mn;
    l = l * alpha + wave_sum(w);
#pragma unroll
    for (int e = 0; e < V; ++e) acc[e] = WHOLE ? att_rescale(acc[e], alpha) : acc[e] * alpha;
    const uint64_t weighs = __ballot(s != -INFINITY);
    while (todo) {
      const int n = __builtin_ctzll(todo);
      const bool none = !(weighs >> n & 1);
      todo &= todo - 1;
      const float wn = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(w), n));
      const T *vr = v + (int64_t)__builtin_amdgcn_readlane(row, n) * a.v_ss;
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (lane + 64 * e < D) {
          const float y = Elt<T>::load(vr, lane + 64 * e);
          acc[e] = !WHOLE || none ? fmaf(wn, y, acc[e]) : att_add(wn, y, acc[e]);  // (0 x inf is NaN there)
        }
    }
  }
}

}  // namespace nk
