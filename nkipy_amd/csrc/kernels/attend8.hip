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
// fp32's exponents).  fp16 queries and weights, which bf16 does not hold, enter as
// two bf16 numbers each, x = RN(x) + RN(x - RN(x)): exact for a query's 11 bits, a
// weight keeps 16.
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

// ---------------------------------------------------------------------------
// One new token per sequence (16-bit queries, head dim 64 or 128): bound by the read
// of the codes.  A wave takes one piece of one sequence's blocks of 32 keys for one
// KV head, by itself: no LDS and no barrier.  Waves that run side by side take
// neighbouring heads of the same keys, whose rows lie next to each other in memory
// (64 contexts of up to 8192, 8 heads of 128: 142 us where the four waves of a
// workgroup take blocks of one head, XXX so).
//
// A wave has up to 16 heads of the group as the columns of 16x16x32 products,
// S^T = K Q^T and O^T = V^T P^T.  Everything stays in registers: which element of
// a head, and which key of a block, has which place in a product's sum is free as
// long as both factors agree.  So a lane takes 16 bytes of a key as they lie in
// memory; and of the values it takes D / 16 columns of the eight keys whose weights
// it holds, pairs of which v_perm puts side by side after conversion.  The next
// block's keys are read as soon as this one's scores stand, its values behind this
// one's products.
// ---------------------------------------------------------------------------
template <typename T, int D>
__device__ __forceinline__ void attend8_step_body(const Attend8Args &a) {
  constexpr int NP = Parts<T>::N, VW = D / 64;
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
    B8 pf[NP];
    auto weigh = [&]() __attribute__((always_inline)) {
      float sum = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float y = __builtin_amdgcn_exp2f((s[e >> 2][e & 3] - m_run) * sl2);
        sum += y;
        put_weight<NP>(pf, e, y);
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
        for (int n = 0; n < NP; ++n) {
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
// added in a fixed order.  Bound by the latency of its two dependent reads.
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

// ---------------------------------------------------------------------------
// Packed queries (16-bit, head dim 64 or 128): the tiles of attend.hip.  One
// workgroup of four waves per (tile of 128 rows, KV head, split); a wave owns 32
// rows.  S^T = K Q^T and O^T = V^T P^T by 32x32x16 products, so that a lane owns one
// row and the weights leave the first product in the order the second one takes
// them.
//
// The codes of a block of 32 keys go through registers, where a thread converts the
// 16 it read into bf16 values once for all four waves, into two LDS slots each for K
// and V: iteration j has the scores of block j + 1, the values of block j - 1 and
// the softmax of block j, then stores K of block j + 2 and V of block j, read an
// iteration ago, and reads the next: one barrier per block.  A key's row and its
// scales are looked up once per workgroup, 32 blocks ahead.
//
// Softmax, masks and what is computed again at the end are those of attend.hip: the
// offset of a row is raised when a lane's 16 weights of a block exceed LIMIT, masks
// are applied only to blocks that some row does not see whole, and rows whose sums
// are not finite (a NaN value that other rows of the tile see), or whose offset is
// too large to cancel, are computed again, a wave each.
// ---------------------------------------------------------------------------
#define ATT8_AHEAD 32  // blocks whose rows are looked up at once
// rows outside every sequence: zeros, shared out over the grid
template <typename T>
NK_DEVICE void att8_zero_rest(const Attend8Args &a, int wg, int nwg) {
  const int s0 = min(max(a.starts[0], 0), a.N), s1 = min(max(a.starts[a.B], s0), a.N);
  const int n = a.Hq * a.D;
  for (int x = wg; x < s0 + a.N - s1; x += nwg) {
    T *o = (T *)a.o + (int64_t)(x < s0 ? x : x - s0 + s1) * n;
    for (int e = threadIdx.x; e < n; e += 256) o[e] = T{};
  }
}

template <typename T, int D>
__device__ __forceinline__ void attend8_tile_body(const Attend8Args &a) {
  constexpr int NP = Parts<T>::N;
  constexpr int RB = D * 2, TB = ATT_KEYS * RB;      // bytes of a row, of a block, as bf16
  constexpr int LPR = D / 16;                        // threads that read a key's codes
  constexpr bool BOTH = ATT_KEYS * LPR == 256;       // every thread reads keys and values (else half of them each)
  __shared__ __attribute__((aligned(1024))) uint8_t KR[2 * TB];
  __shared__ __attribute__((aligned(1024))) uint8_t VR[2 * TB];
  __shared__ __attribute__((aligned(16))) int32_t ent[2 * ATT8_AHEAD * ATT_KEYS];   // rows, -1: none
  __shared__ uint16_t exps[2 * ATT8_AHEAD * ATT_KEYS];  // exponents + 127, keys' below values'
  __shared__ int32_t lost[8];  // per half of ent and wave: some key has no page

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l32 = lane & 31, lhi = lane >> 5;
  const int rep = a.Hq / a.Hkv;

  if (a.starts) att8_zero_rest<T>(a, blockIdx.x, a.tiles * a.Hkv * a.nsplit);
  AttWork wk;
  AttSeq sq;
  if (!att_tile<true>(a, blockIdx.x, wk, sq)) return;
  const int g = wk.g, split = wk.split, b = wk.b, tile = wk.tile;
  const AttSpan sp = att_span(a, sq, tile);
  int j0, j1;
  const int pieces = att_split(a, sp.nb, split, j0, j1);
  if (split >= pieces) return;
  const int n = j1 - j0;  // blocks of this workgroup

  // this lane's row
  const int row0 = tile * ATT_ROWS + wave * 32, rows = sq.n * rep;
  const bool active = row0 < rows;
  B8 qf[D / 16][NP];
  int p, klim;  // its position and last key
  {
    const int rld = min(row0 + l32, rows - 1), qi = rld / rep, h = g * rep + rld % rep;
    p = sq.p0 + qi;
    klim = row0 + l32 < rows && p >= 0 && p < sq.len ? min(p, sq.cap - 1) : -1;
    const T *q = (const T *)a.q + (int64_t)(sq.lo + qi) * a.q_ss + (int64_t)h * a.q_sh;
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk) load_q<T, NP>(q + kk * 16 + lhi * 8, qf[kk]);
  }

  f32x16 acc[D / 32];
#pragma unroll
  for (int t2 = 0; t2 < D / 32; ++t2)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[t2][r] = 0.f;
  float m_run = -1e30f, l_run = 0.f;  // (finite: a masked score gives p = 0; scores below it: see `sees`)
  const float sl2 = a.scale * LOG2E;

  // swizzles: 16-byte chunk c of row r stands at chunk c ^ kswz / vswz, so that
  // 16 rows of a K fragment, and the four rows of a transposing V read, cover
  // all banks
  auto kswz = [](int r) __attribute__((always_inline)) { return D == 128 ? r & 15 : (r >> 1) & 7; };
  auto vswz = [](int r) __attribute__((always_inline)) { return D == 128 ? (r & 3) << 2 : ((r >> 1) & 1) << 2; };

  // look up the rows of blocks 32 c .. 32 c + 31 of this workgroup
  auto look_up = [&](int c) __attribute__((always_inline)) {
    bool miss = false;
#pragma unroll 1
    for (int x = tid; x < ATT8_AHEAD * ATT_KEYS; x += 256) {
      const int j = j0 + c * ATT8_AHEAD + x / ATT_KEYS;
      const int key = sp.kb(j) * ATT_KEYS + x % ATT_KEYS;
      int at = -1, ex = 0;
      if (j < j1 && key < sp.hi && (key >= sp.lo || key < a.sinks)) {
        const int pg = a.tables[(int64_t)b * a.width + key / a.page];
        if (pg >= 0 && pg < a.pages) {
          at = pg * a.pitch + key % a.page;
          ex = (c8_clip(a.ke[(int64_t)pg * a.Hkv + g]) + 127) | (c8_clip(a.ve[(int64_t)pg * a.Hkv + g]) + 127) << 8;
        }
        miss |= at < 0;
      }
      ent[(c & 1) * ATT8_AHEAD * ATT_KEYS + x] = at;
      exps[(c & 1) * ATT8_AHEAD * ATT_KEYS + x] = (uint16_t)ex;
    }
    const bool any = __ballot(miss) != 0;
    if (lane == 0) lost[(c & 1) * 4 + wave] = any;
  };

  // a thread's codes of a block: row rr, elements 16 cc ... ; `mine`: whether it reads this array
  const int rr = (BOTH ? tid : tid & 127) / LPR, cc = tid % LPR;
  const uint8_t *kp = (const uint8_t *)a.k + (int64_t)g * a.k_sh + cc * 16;
  const uint8_t *vp = (const uint8_t *)a.v + (int64_t)g * a.v_sh + cc * 16;
  struct Codes {
    uint4 w;
    float scale;
  };
  Codes ck, cv;
  auto load = [&](Codes &x, const uint8_t *base, int64_t ss, int jr, bool mine, int shift) __attribute__((always_inline)) {
    const int at = jr >= 0 && jr < n && mine ? ent[(jr & (2 * ATT8_AHEAD - 1)) * ATT_KEYS + rr] : -1;
    const int ex = at >= 0 ? exps[(jr & (2 * ATT8_AHEAD - 1)) * ATT_KEYS + rr] : 0;
    x.scale = __uint_as_float((uint32_t)(ex >> shift & 0xff) << 23);
    x.w = make_uint4(0, 0, 0, 0);
    if (at >= 0) x.w = *reinterpret_cast<const uint4 *>(base + at * ss);
  };
  const bool kmine = BOTH || tid < 128, vmine = BOTH || tid >= 128;
  auto load_k = [&](int jr) __attribute__((always_inline)) { load(ck, kp, a.k_ss, jr, kmine, 0); };
  auto load_v = [&](int jr) __attribute__((always_inline)) { load(cv, vp, a.v_ss, jr, vmine, 8); };
  auto store = [&](const Codes &x, uint8_t *to, int swz) __attribute__((always_inline)) {
    *reinterpret_cast<B8 *>(to + rr * RB + (((2 * cc) ^ swz) << 4)) = codes8(x.w.x, x.w.y, x.scale);
    *reinterpret_cast<B8 *>(to + rr * RB + (((2 * cc + 1) ^ swz) << 4)) = codes8(x.w.z, x.w.w, x.scale);
  };
  auto store_k = [&](int jr) __attribute__((always_inline)) { if (kmine) store(ck, KR + (jr & 1) * TB, kswz(rr)); };
  auto store_v = [&](int jr) __attribute__((always_inline)) { if (vmine) store(cv, VR + (jr & 1) * TB, vswz(rr)); };

  // K fragment kk: row l32, chunk 2 kk + lhi
  const int kbase = l32 * RB + ((lhi ^ (kswz(l32) & 1)) << 4), kx = (kswz(l32) & ~1) << 4;
  // transposing V read (group lane / 16, i = lane % 16): row 16 j + 8 si + 4 (group / 2) + i / 4,
  // columns 32 dt + 16 (group % 2) + 4 (i % 4)
  int vbase, vx;
  {
    const int grp = lane >> 4, gi = lane & 15, r = 4 * (grp >> 1) + (gi >> 2);
    vbase = r * RB + (((grp & 1) * 2 + ((gi & 3) >> 1)) << 4) + (gi & 1) * 8;
    vx = vswz(r) << 4;
  }
  auto qk1 = [&](const uint8_t *K, f32x16 &s, int kk) __attribute__((always_inline)) {
    const B8 f = *reinterpret_cast<const B8 *>(K + kbase + ((kk << 5) ^ kx));
#pragma unroll
    for (int i = 0; i < NP; ++i) s = mul32(f, qf[kk][i], s);
  };
  auto pv1 = [&](const uint8_t *Vt, const B8 (&pf)[2][NP], int j, int dt) __attribute__((always_inline)) {
    s16x4 v[2];
#pragma unroll
    for (int si = 0; si < 2; ++si)
      v[si] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          (lds_s16x4 *)(Vt + (16 * j + 8 * si) * RB + vbase + ((dt << 6) ^ vx)));
    const s16x8 vf = __builtin_shufflevector(v[0], v[1], 0, 1, 2, 3, 4, 5, 6, 7);
#pragma unroll
    for (int i = 0; i < NP; ++i) acc[dt] = mul32(__builtin_bit_cast(B8, vf), pf[j][i], acc[dt]);
  };
  // The scores of one block and the values of another, in turns: each product of
  // the scores waits for the one before it, the values' are apart.
  auto qk_pv = [&](const uint8_t *K, f32x16 &s, const uint8_t *Vt, const B8 (&pf)[2][NP]) __attribute__((always_inline)) {
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = 0.f;
#pragma unroll
    for (int i = 0; i < D / 16; ++i) {
      qk1(K, s, i);
      pv1(Vt, pf, i / (D / 32), i % (D / 32));
    }
  };
  auto expblock = [&](const f32x16 &s, B8 (&pf)[2][NP]) __attribute__((always_inline)) {
    float s0 = 0.f, s1 = 0.f;
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(s[8 * j + e], sl2, -m_run));
        if (e & 1) s1 += x; else s0 += x;
        put_weight<NP>(pf[j], e, x);
      }
    return s0 + s1;
  };
  int missing = 0;  // the blocks being worked on have keys without a page
  // What no row sees of block jr out of its scores; past the last block, all of it.
  // Element r of a lane is key 32 kb + 8 (r / 4) + 4 lhi + r % 4.
  auto mask = [&](f32x16 &s, int jr) __attribute__((always_inline)) {
    const int k0 = sp.kb(j0 + jr) * ATT_KEYS + lhi * 4;
    const int t0 = jr < n ? klim - k0 : -1, w0 = p - a.window - k0, s0 = a.sinks - k0;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int x = (r >> 2) * 8 + (r & 3);
      s[r] = x > t0 || (x <= w0 && x >= s0) ? -INFINITY : s[r];
    }
    if (missing) {
      const int32_t *en = ent + (jr & (2 * ATT8_AHEAD - 1)) * ATT_KEYS + lhi * 4;
#pragma unroll
      for (int r = 0; r < 16; r += 4) {
        const int4 e = *reinterpret_cast<const int4 *>(en + r * 2);
        s[r] = e.x < 0 ? -INFINITY : s[r];
        s[r + 1] = e.y < 0 ? -INFINITY : s[r + 1];
        s[r + 2] = e.z < 0 ? -INFINITY : s[r + 2];
        s[r + 3] = e.w < 0 ? -INFINITY : s[r + 3];
      }
    }
  };
  auto raise = [&](f32x16 &s, B8 (&pf)[2][NP], float ls) __attribute__((always_inline)) {
    if (__builtin_expect(__builtin_amdgcn_ballot_w64(!(ls <= ATT8_LIMIT)) != 0, 0)) {
      float bm = s[0];
#pragma unroll
      for (int r = 1; r < 16; ++r) bm = fmaxf(bm, s[r]);
      bm = fmaxf(bm, __shfl_xor(bm, 32, 64));
      const float m_new = fmaxf(m_run, bm * sl2);
      const float alpha = __builtin_amdgcn_exp2f(m_run - m_new);
      m_run = m_new;
#pragma unroll
      for (int t2 = 0; t2 < D / 32; ++t2)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[t2][r] *= alpha;
      l_run *= alpha;
      ls = expblock(s, pf);
    }
    l_run += ls;
  };
  auto whole = [&](int jr) __attribute__((always_inline)) {  // every row sees the whole block
    const int k0 = sp.kb(j0 + jr) * ATT_KEYS;
    return jr < n && k0 + ATT_KEYS - 1 <= sp.pa && k0 + ATT_KEYS <= sp.hi && (k0 > sp.pb - a.window || k0 + ATT_KEYS <= a.sinks) && !missing;
  };

  f32x16 sA, sB;
  B8 pA[2][NP], pB[2][NP];
#pragma unroll
  for (int j = 0; j < 2; ++j)
#pragma unroll
    for (int e = 0; e < 8; ++e) put_weight<NP>(pB[j], e, 0.f);
  // the end of an iteration: what was read is stored, the next is read
  auto move_on = [&](int jr) __attribute__((always_inline)) {
    store_k(jr + 2);
    store_v(jr);
    lds_barrier();
    load_k(jr + 3);
    load_v(jr + 1);
  };
  // Iteration jr, one body for all: the values of the block before (of zeros before
  // the first), the scores of the one behind (of zeros past the last), the softmax of
  // this one.  The last, jr = n, adds the last block's values.
  auto step = [&](int jr, f32x16 &cur, f32x16 &nxt, B8 (&prev)[2][NP], B8 (&now)[2][NP]) __attribute__((always_inline)) {
    if (!whole(jr)) mask(cur, jr);
    qk_pv(KR + ((jr + 1) & 1) * TB, nxt, VR + ((jr + 1) & 1) * TB, prev);
    const float ls = expblock(cur, now);
    raise(cur, now, ls);
    move_on(jr);
  };

  if (n > 0) {
    look_up(0);
    __syncthreads();
    load_k(0);
    load_v(-1);  // (zeros)
    store_k(0);
    store_v(1);
    load_k(1);
    store_k(1);
    load_k(2);
    load_v(0);
    lds_barrier();
    if (active) {
#pragma unroll
      for (int r = 0; r < 16; ++r) sA[r] = 0.f;
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) qk1(KR, sA, kk);
    }
    lds_barrier();  // (block 0 is read before its slot is refilled)
    auto ahead = [&](int jr) __attribute__((always_inline)) {
      if (jr % ATT8_AHEAD == 0) {
        const int32_t *f = lost + (jr / ATT8_AHEAD & 1) * 4;
        missing = __builtin_amdgcn_readfirstlane(f[0] | f[1] | f[2] | f[3]);
        // (the other half was last read an iteration, and a barrier, ago)
        if (jr + ATT8_AHEAD < n) look_up(jr / ATT8_AHEAD + 1);
      }
    };
    if (active) {
      for (int jr = 0;; jr += 2) {
        ahead(jr);
        step(jr, sA, sB, pB, pA);
        if (jr + 1 > n) break;
        step(jr + 1, sB, sA, pA, pB);
        if (jr + 2 > n) break;
      }
    } else {  // rows past the sequence's: the moves only
      for (int jr = 0; jr <= n; ++jr) {
        ahead(jr);
        move_on(jr);
      }
    }
  }

  const int row = row0 + l32, rld = min(row, rows - 1), qi = rld / rep, h = g * rep + rld % rep;
  const bool ok = klim >= 0;
  l_run += __shfl_xor(l_run, 32, 64);
  const int64_t nr = (int64_t)a.N * a.Hq;
  const int64_t orow = ((int64_t)(sq.lo + qi)) * a.Hq + h;
  float *wo = a.ws + (split * nr + orow) * D, *wm = a.ws + (int64_t)a.nsplit * nr * D + (split * nr + orow) * 2;
  uint16_t *o = (uint16_t *)a.o + orow * D;

  // whether this row, if it has no weight, sees any key of these blocks, pages aside
  bool sees = false;
  if (__any(ok && l_run == 0.f)) {
    auto part = [&](int a0, int a1) __attribute__((always_inline)) {  // (blocks that follow each other)
      const int lo = sp.kb(a0) * ATT_KEYS, hi = min(sp.kb(a1 - 1) * ATT_KEYS + ATT_KEYS - 1, klim);
      sees |= a0 < a1 && (max(lo, p - a.window + 1) <= hi || lo <= min(hi, a.sinks - 1));
    };
    part(j0, min(j1, sp.ns));
    part(max(j0, sp.ns), j1);
  }

  // rows that a NaN value may have spoiled, and those whose offset is too large to
  // cancel: s c - m is then off by half a step of m.  A row without weight still has
  // the offset it began with: where it sees keys their scores are below that, or -inf.
  float z = l_run * 0.f;
#pragma unroll
  for (int t2 = 0; t2 < D / 32; ++t2)
#pragma unroll
    for (int r = 0; r < 16; ++r) z = __builtin_fmaf(acc[t2][r], 0.f, z);
  uint64_t spoiled = __ballot(ok && (z != 0.f || (fabsf(m_run) >= 0x1p24f && (l_run != 0.f || sees))));
  spoiled = (spoiled | spoiled >> 32) & 0xffffffffull;
  const bool put = row < rows && !(spoiled >> l32 & 1);
  if (put && pieces == 1) {
    const float inv = ok && l_run != 0.f ? 1.0f / l_run : 0.f;
#pragma unroll
    for (int t2 = 0; t2 < D / 32; ++t2)
#pragma unroll
      for (int gq = 0; gq < 4; ++gq) {
        T y[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) Elt<T>::store(y, e, inv == 0.f ? 0.f : acc[t2][gq * 4 + e] * inv);
        uint2 u;
        __builtin_memcpy(&u, y, 8);
        *reinterpret_cast<uint2 *>(o + t2 * 32 + gq * 8 + lhi * 4) = u;
      }
  } else if (put) {
#pragma unroll
    for (int t2 = 0; t2 < D / 32; ++t2)
#pragma unroll
      for (int gq = 0; gq < 4; ++gq)
        *reinterpret_cast<float4 *>(wo + t2 * 32 + gq * 8 + lhi * 4) =
            ok ? make_float4(acc[t2][gq * 4], acc[t2][gq * 4 + 1], acc[t2][gq * 4 + 2], acc[t2][gq * 4 + 3]) : make_float4(0.f, 0.f, 0.f, 0.f);
    if (lhi == 0) wm[0] = m_run, wm[1] = ok ? l_run : 0.f;
  }
  // these again, reading only what they see
  while (spoiled) {
    const int src = __builtin_ctzll(spoiled);
    spoiled &= spoiled - 1;
    float m, l, x[D / 64];
    att8_row<T, D>(a, sq, sp, b, __shfl(qi, src, 64), __shfl(h, src, 64), j0, j1, m, l, x);
    const int64_t at = __shfl((int)orow, src, 64);  // (rows are below 2^31)
#pragma unroll
    for (int e = 0; e < D / 64; ++e) {
      if (pieces == 1) {
        Elt<T>::store((T *)a.o + at * D, lane + 64 * e, l == 0.f ? 0.f : x[e] / l);
      } else {
        a.ws[(split * nr + at) * D + lane + 64 * e] = x[e];
      }
    }
    if (pieces > 1 && lane == 0) {
      float *y = a.ws + (int64_t)a.nsplit * nr * D + (split * nr + at) * 2;
      y[0] = fmaxf(m * LOG2E, ATT8_LOWEST);
      y[1] = l;
    }
  }
}
#define NK_TILE8(T, name, D, OCC)                                                                          \
  extern "C" __global__ __launch_bounds__(256, OCC) void nk_attend8_tile_##name##_d##D(Attend8Args a) {    \
    attend8_tile_body<T, D>(a);                                                                            \
  }
NK_TILE8(bf16, bf16, 128, 2)
NK_TILE8(f16, f16, 128, 1)  // (under a bound of two, registers in memory)
NK_TILE8(bf16, bf16, 64, 2)
NK_TILE8(f16, f16, 64, 2)
