// Attention over a paged cache of e4m3 codes with a scale for each page and head
// (attend_index.h holds what a query sees and the layout of the work).

#include "attend8.h"

using namespace nk;

// ---------------------------------------------------------------------------
// Any head dim to 256, any strides and addresses, fp32 queries: one wave per query
// row, 32-bit weights, no matrix instructions.
// ---------------------------------------------------------------------------
template <typename T>
__device__ __forceinline__ void attend8_rows_body(const Attend8Args &a) {
  const int lane = threadIdx.x & 63;
  const int64_t r = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (r >= (int64_t)a.N * a.Hq) return;
  const int t = (int)(r / a.Hq), h = (int)(r % a.Hq);
  int b, i;
  AttSeq sq;
  float m, l = 0.f, acc[4];
  if (att_query(a, t, b, sq, i)) {
    const AttSpan sp = att_span(a, sq, (i * (a.Hq / a.Hkv) + h % (a.Hq / a.Hkv)) / ATT_ROWS);
    att8_row<T>(a, sq, sp, b, i, h, 0, sp.nb, m, l, acc);
  }
  T *o = (T *)a.o + r * a.D;
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (lane + 64 * e < a.D) Elt<T>::store(o, lane + 64 * e, l == 0.f ? 0.f : acc[e] / l);
}
extern "C" __global__ __launch_bounds__(256) void nk_attend8_rows_bf16(Attend8Args a) { attend8_rows_body<bf16>(a); }
extern "C" __global__ __launch_bounds__(256) void nk_attend8_rows_f16(Attend8Args a) { attend8_rows_body<f16>(a); }
extern "C" __global__ __launch_bounds__(256) void nk_attend8_rows_f32(Attend8Args a) { attend8_rows_body<float>(a); }

// ---------------------------------------------------------------------------
// One new token per sequence (16-bit queries, head dim 64 or 128): bound by the read
// of the codes.  A wave takes one piece of one sequence's blocks of 32 keys for one
// KV head, by itself: no LDS and no barrier.  Waves that run side by side take
// neighbouring heads of the same keys, whose rows lie next to each other in memory
// (64 contexts of up to 8192, 8 heads of 128, without the sums of what was read: 145 us
// where the four waves of a workgroup take blocks of one head, 120 so).
//
// A wave has up to 16 heads of the group as the columns of 16x16x32 products,
// S^T = K Q^T and O^T = V^T P^T.  Everything stays in registers: which element of
// a head, and which key of a block, has which place in a product's sum is free as
// long as both factors agree.  So a lane takes 16 bytes of a key as they lie in
// memory; and of the values it takes D / 16 columns of the eight keys whose weights
// it holds, pairs of which v_perm puts side by side after conversion.  A weight is two
// bf16 numbers, so that it keeps 2^-16 of itself: the products are not what bounds this
// (118 us a call with one number and with two; results off by 2.33e-3 and by 1.66e-3 of
// their norm, the latter their own rounding).  The next block's keys are read as soon as
// this one's scores stand, its values behind this one's products.  (Those 64 contexts:
// 113 us for 556 MB, 4.9 TB/s; one of 1500 keys: 5.6 us.)
// ---------------------------------------------------------------------------
template <typename T, int D>
__device__ __forceinline__ void attend8_step_body(const Attend8Args &a) {
  constexpr int NP = Parts<T>::N, WP = 2, VW = D / 64;
  const int lane = threadIdx.x & 63;
  const int l16 = lane & 15, grp = lane >> 4;
  const int rep = a.Hq / a.Hkv, per = (rep + 15) / 16, units = a.Hkv * per;
  int w = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = w % units / per, h0 = w % units % per * 16;  // (h0: first head of the group's)
  w /= units;
  // (nsplit is a multiple of eight: the first pieces, which all sequences have, come
  // to all XCDs by turns)
  const int b = w / a.nsplit, split = (w % a.nsplit + b) % a.nsplit;
  if (b >= a.B) return;
  const AttSeq sq = att_seq(a, b);
  const AttSpan sp = att_span(a, sq, 0);
  int j0, j1;
  const int pieces = att_split(a, sp.nb, split, j0, j1);
  if (split >= pieces) return;
  const int p = sq.p0, klim = min(p, sq.cap - 1);

  // element e of product kk of this lane: 64 (kk / 2) + 16 grp + 8 (kk % 2) + e
  B8 qf[D / 32][NP];
  {
    const T *q = (const T *)a.q + (int64_t)b * a.q_ss + (int64_t)(g * rep + min(h0 + l16, rep - 1)) * a.q_sh;
#pragma unroll
    for (int kk = 0; kk < D / 32; ++kk) load_q<T, NP>(q + (kk >> 1) * 64 + grp * 16 + (kk & 1) * 8, qf[kk]);
  }
  const uint8_t *kp = (const uint8_t *)a.k + (int64_t)g * a.k_sh + grp * 16;
  const uint8_t *vp = (const uint8_t *)a.v + (int64_t)g * a.v_sh + l16 * (D / 16);
  const int32_t *const ex = (lane < 32 ? a.ke : a.ve) + g;

  f32x4 acc[D / 16];
#pragma unroll
  for (int t = 0; t < D / 16; ++t) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m_run = ATT8_LOWEST, l_run = 0.f;
  const float sl2 = a.scale * LOG2E;

  // lane l looks up key l % 32 of a block: its page, -1 where it is not seen
  auto page_of = [&](int j, int &in) __attribute__((always_inline)) {
    const int key = sp.kb(j) * ATT_KEYS + (lane & 31);
    in = 0;
    if (!(j < j1 && key <= klim && (key > p - a.window || key < a.sinks))) return -1;
    const int x = key / a.page, pg = a.tables[(int64_t)b * a.width + x];
    in = key - x * a.page;
    return pg >= 0 && pg < a.pages ? pg : -1;
  };
  int at;                  // the next block's rows: this lane's key's, some row (unused) where it is not seen
  uint32_t seen, seen_next;
  float scale, scale_next;  // of key lane % 32: lanes below 32 keys', above values'
  uint4 kr[2][D / 64];
  uint32_t vr[8][VW];
  auto fetch_k = [&](int pg, int in) __attribute__((always_inline)) {
    at = max(pg, 0) * a.pitch + in;
    seen_next = (uint32_t)__ballot(pg >= 0);
    scale_next = c8_power(c8_clip(ex[(int64_t)max(pg, 0) * a.Hkv]));
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) {
      const uint8_t *k = kp + (int64_t)__shfl(at, kt * 16 + l16, 64) * a.k_ss;
#pragma unroll
      for (int i = 0; i < D / 64; ++i) kr[kt][i] = *reinterpret_cast<const uint4 *>(k + i * 64);
    }
  };
  auto fetch_v = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      const uint8_t *v = vp + (int64_t)__shfl(at, (r >> 2) * 16 + 4 * grp + (r & 3), 64) * a.v_ss;
      if constexpr (VW == 2) {
        const uint2 y = *reinterpret_cast<const uint2 *>(v);
        vr[r][0] = y.x, vr[r][1] = y.y;
      } else {
        vr[r][0] = *reinterpret_cast<const uint32_t *>(v);
      }
    }
  };

  int in, pg = page_of(j0, in);
  if (j0 < j1) {
    fetch_k(pg, in);
    fetch_v();
    pg = page_of(j0 + 1, in);
  }
  for (int j = j0; j < j1; ++j) {
    seen = seen_next, scale = scale_next;
    f32x4 s[2];
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) {
      const float ks = __shfl(scale, kt * 16 + l16, 64);
      s[kt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < D / 64; ++i) {
        const uint4 k = kr[kt][i];
        const B8 f0 = codes8(k.x, k.y, ks), f1 = codes8(k.z, k.w, ks);
#pragma unroll
        for (int n = 0; n < NP; ++n) {
          s[kt] = mul16(f0, qf[2 * i][n], s[kt]);
          s[kt] = mul16(f1, qf[2 * i + 1][n], s[kt]);
        }
      }
    }
    const bool more = j + 1 < j1;
    if (more) fetch_k(pg, in);
    // element r of tile kt is key 16 kt + 4 grp + r
    if (seen != 0xffffffffu) {
      const uint32_t mine = seen >> (grp * 4);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const bool is = mine >> ((e >> 2) * 16 + (e & 3)) & 1;
        s[e >> 2][e & 3] = is ? s[e >> 2][e & 3] : -INFINITY;
#pragma unroll
        for (int i = 0; i < VW; ++i) vr[e][i] = is ? vr[e][i] : 0;
      }
    }
    B8 pf[WP];
    auto weigh = [&]() __attribute__((always_inline)) {
      float sum = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float y = __builtin_amdgcn_exp2f((s[e >> 2][e & 3] - m_run) * sl2);
        sum += y;
        put_weight<WP>(pf, e, y);
      }
      return sum;
    };
    float ls = weigh();
    if (__builtin_amdgcn_ballot_w64(!(ls <= ATT8_LIMIT)) != 0) {
      float bm = s[0][0];
#pragma unroll
      for (int e = 1; e < 8; ++e) bm = fmaxf(bm, s[e >> 2][e & 3]);
      bm = fmaxf(bm, __shfl_xor(bm, 16, 64));
      bm = fmaxf(bm, __shfl_xor(bm, 32, 64));
      const float m_new = fmaxf(m_run, bm);
      const float alpha = __builtin_amdgcn_exp2f((m_run - m_new) * sl2);
      m_run = m_new;
#pragma unroll
      for (int t = 0; t < D / 16; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[t][r] *= alpha;
      l_run *= alpha;
      ls = weigh();
    }
    l_run += ls;
    float vs[8];
#pragma unroll
    for (int r = 0; r < 8; ++r) vs[r] = __shfl(scale, 32 + (r >> 2) * 16 + 4 * grp + (r & 3), 64);
#pragma unroll
    for (int i = 0; i < VW; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t c[8];  // columns 4 i + 2 h and the next, of each key
#pragma unroll
        for (int r = 0; r < 8; ++r)
          c[r] = bf16x2_bits(h ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(vr[r][i], vs[r], true)
                               : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(vr[r][i], vs[r], false));
        u32x4_t lo, hi;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          lo[r] = __builtin_amdgcn_perm(c[2 * r + 1], c[2 * r], 0x05040100);
          hi[r] = __builtin_amdgcn_perm(c[2 * r + 1], c[2 * r], 0x07060302);
        }
        const int t = 4 * i + 2 * h;
#pragma unroll
        for (int n = 0; n < WP; ++n) {
          acc[t] = mul16(__builtin_bit_cast(B8, lo), pf[n], acc[t]);
          acc[t + 1] = mul16(__builtin_bit_cast(B8, hi), pf[n], acc[t + 1]);
        }
      }
    if (more) {
      fetch_v();
      pg = page_of(j + 2, in);
    }
  }

  // acc[t][r] is column (4 grp + r) D / 16 + t of row l16
  l_run += __shfl_xor(l_run, 16, 64);
  l_run += __shfl_xor(l_run, 32, 64);
  float z = 0.f;
#pragma unroll
  for (int t = 0; t < D / 16; ++t)
#pragma unroll
    for (int r = 0; r < 4; ++r) z = __builtin_fmaf(acc[t][r], 0.f, z);
  // a bit for each row with a sum that is not finite under weights that are
  uint64_t bits = __ballot(z != 0.f && l_run == l_run && h0 + l16 < rep);
  bits |= bits >> 32;
  uint32_t again = (uint32_t)(bits | bits >> 16) & 0xffffu;
  const int64_t nr = (int64_t)a.N * a.Hq, r0 = (int64_t)b * a.Hq + g * rep + h0;
  float *const wo = a.ws + (split * nr + r0) * D, *const wm = a.ws + (int64_t)a.nsplit * nr * D + (split * nr + r0) * 2;
  if (h0 + l16 < rep && !(again >> l16 & 1)) {
    if (pieces == 1) {
      const float inv = l_run == 0.f ? 0.f : 1.f / l_run;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        float y[8];
        T *o = (T *)a.o + (r0 + l16) * D + (4 * grp + r) * (D / 16);
#pragma unroll
        for (int t = 0; t < D / 16; ++t) y[t] = l_run == 0.f ? 0.f : acc[t][r] * inv;
        if constexpr (D == 128) {
          Vec8<T>::store(o, y);
        } else {
#pragma unroll
          for (int t = 0; t < D / 16; ++t) Elt<T>::store(o, t, y[t]);
        }
      }
    } else {
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int t = 0; t < D / 16; t += 4)
          *reinterpret_cast<float4 *>(wo + l16 * D + (4 * grp + r) * (D / 16) + t) =
              make_float4(acc[t][r], acc[t + 1][r], acc[t + 2][r], acc[t + 3][r]);
      if (grp == 0) wm[2 * l16] = fmaxf(m_run * sl2, ATT8_LOWEST), wm[2 * l16 + 1] = l_run;
    }
  }
  // Sums that are not finite (NaN values, or large ones under weights past 1): those
  // rows again.
  for (; again; again &= again - 1) {
    const int r = __builtin_ctz(again);
    float mr, lr, y[D / 64];
    att8_row<T, D>(a, sq, sp, b, 0, g * rep + h0 + r, j0, j1, mr, lr, y);
#pragma unroll
    for (int e = 0; e < D / 64; ++e) {
      if (pieces == 1) {
        Elt<T>::store((T *)a.o + (r0 + r) * D, lane + 64 * e, lr == 0.f ? 0.f : y[e] / lr);
      } else {
        wo[r * D + lane + 64 * e] = y[e];
      }
    }
    if (pieces > 1 && lane == 0) wm[2 * r] = fmaxf(mr * LOG2E, ATT8_LOWEST), wm[2 * r + 1] = lr;
  }
}
#define NK_STEP8(T, name, D, OCC)                                                                          \
  extern "C" __global__ __launch_bounds__(256, OCC) void nk_attend8_step_##name##_d##D(Attend8Args a) {    \
    attend8_step_body<T, D>(a);                                                                            \
  }
NK_STEP8(bf16, bf16, 128, 3)
NK_STEP8(f16, f16, 128, 3)
NK_STEP8(bf16, bf16, 64, 4)
NK_STEP8(f16, f16, 64, 4)

// ---------------------------------------------------------------------------
// The pieces of a step's row joined: o = sum 2^(m_s - M) o_s / sum 2^(m_s - M) l_s,
// over the pieces with any weight, up to JOIN of them.  One workgroup per row: D / 4
// threads side by side for a piece's sums, the pieces shared out over the rest and
// added in a fixed order.  Bound by the latency of its two dependent reads (32 rows: 3.6
// us, 2048 rows of up to 10 pieces: 6.0).
// ---------------------------------------------------------------------------
#define ATT8_JOIN 256
template <typename T, int D>
__device__ __forceinline__ void attend8_join_body(const Attend8Args &a) {
  constexpr int DL = D / 4, PL = 256 / DL;  // threads of a piece, pieces side by side
  __shared__ float weight[ATT8_JOIN];
  __shared__ __attribute__((aligned(16))) float part[PL][D];
  __shared__ float total;
  const int tid = threadIdx.x, lane = tid & 63, d = tid % DL * 4, s0 = tid / DL;
  const int64_t r = blockIdx.x, nr = (int64_t)a.N * a.Hq;
  const int b = (int)(r / a.Hq);
  const AttSeq sq = att_seq(a, b);
  int j0, j1;
  const int pieces = att_split(a, att_span(a, sq, 0).nb, 0, j0, j1);
  if (pieces == 1) return;
  const float *ws = a.ws + r * D + d, *wm = a.ws + (int64_t)a.nsplit * nr * D;
  constexpr int U = 8;
  float4 x[U];
  auto fetch = [&](int s) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < U; ++u)  // (past the last piece: the last again, unused)
      x[u] = *reinterpret_cast<const float4 *>(ws + (int64_t)min(s + u * PL, pieces - 1) * nr * D);
  };
  fetch(s0);
  if (tid < 64) {
    float m[ATT8_JOIN / 64], l[ATT8_JOIN / 64], top = -INFINITY, sum = 0.f;
#pragma unroll
    for (int i = 0; i < ATT8_JOIN / 64; ++i) {
      m[i] = -INFINITY, l[i] = 0.f;
      if (lane + 64 * i < pieces) {
        const float2 v = *reinterpret_cast<const float2 *>(wm + ((lane + 64 * i) * nr + r) * 2);
        l[i] = v.y;
        if (l[i] != 0.f) m[i] = v.x;
      }
      top = fmaxf(top, m[i]);
    }
    top = wave_max(top);
#pragma unroll
    for (int i = 0; i < ATT8_JOIN / 64; ++i) {
      const float w = l[i] != 0.f ? __builtin_amdgcn_exp2f(m[i] - top) : 0.f;
      if (lane + 64 * i < pieces) weight[lane + 64 * i] = w;
      sum += w * l[i];
    }
    sum = wave_sum(sum);
    if (lane == 0) total = sum;
  }
  __syncthreads();
  float acc[4] = {};
  for (int s = s0; s < pieces; s += U * PL) {
    if (s != s0) fetch(s);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (s + u * PL >= pieces) break;
      const float w = weight[s + u * PL];
      acc[0] = fmaf(w, x[u].x, acc[0]), acc[1] = fmaf(w, x[u].y, acc[1]);
      acc[2] = fmaf(w, x[u].z, acc[2]), acc[3] = fmaf(w, x[u].w, acc[3]);
    }
  }
  *reinterpret_cast<float4 *>(&part[s0][d]) = make_float4(acc[0], acc[1], acc[2], acc[3]);
  __syncthreads();
  if (tid >= D) return;
  float y = 0.f;
#pragma unroll
  for (int i = 0; i < PL; ++i) y += part[i][tid];
  Elt<T>::store((T *)a.o + r * D, tid, total == 0.f ? 0.f : y / total);
}
#define NK_JOIN8(T, name, D)                                                                          \
  extern "C" __global__ __launch_bounds__(256) void nk_attend8_join_##name##_d##D(Attend8Args a) {    \
    attend8_join_body<T, D>(a);                                                                       \
  }
NK_JOIN8(bf16, bf16, 128)
NK_JOIN8(f16, f16, 128)
NK_JOIN8(bf16, bf16, 64)
NK_JOIN8(f16, f16, 64)
