// The other steps of a serving loop: keys and values rotated into a paged
// cache, and the draw of the next token.

#include "common.h"

using namespace nk;

// ---------------------------------------------------------------------------
// Rotation and append.
//
//   y_i = x_i c_i - x_{i+r/2} s_i,  y_{i+r/2} = x_i s_i + x_{i+r/2} c_i,   i < r/2
//
// with row p of the tables for the token at position p, in fp32 and rounded
// once to the storage type; elements past r are copied.  k and v go to row
// p % page of page tables[b][p / page].  Bound by memory: every element is
// read and written once.  One workgroup per token: its sequence, position and
// page are found once and its heads share the tables' row.  A thread moves E
// elements of each half of a pair (16 bytes with E = 8).
// ---------------------------------------------------------------------------
struct AppendArgs {
  const void *q, *k, *v;
  void *oq, *ok, *ov;  // (N, Hq, D); the caches (pages, page, Hkv, D); null: that part is left out
  const float *cos, *sin;  // (P, half)
  const int32_t *tables, *lens, *starts;
  int64_t q_ss, q_sh, k_ss, k_sh, v_ss, v_sh;  // element strides of rows and heads
  int32_t B, N, Hq, Hkv, D, half, P;
  int32_t page, pages, width;
};

template <typename T, int E> struct Piece {  // E consecutive elements
  static NK_DEVICE void load(const T *p, float (&x)[E]) {
    if constexpr (E == 8) {
      Vec8<T>::load(p, x);
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e) x[e] = Elt<T>::load(p, e);
    }
  }
  static NK_DEVICE void store(T *p, const float (&x)[E]) {
    if constexpr (E == 8) {
      Vec8<T>::store(p, x);
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e) Elt<T>::store(p, e, x[e]);
    }
  }
};
// bits unchanged, signalling NaN included
template <typename T, int E>
NK_DEVICE void copy_piece(const T *x, T *y) {
  if constexpr (E == 8) {
    Raw8<T> r;
    r.template load<false>(x);
    r.template store<false>(y);
  } else {
#pragma unroll
    for (int e = 0; e < E; ++e) y[e] = x[e];
  }
}

template <typename T, int E>
__device__ __forceinline__ void rotary_append_body(const AppendArgs &a) {
  const int t = blockIdx.x, lane = threadIdx.x & 63;
  int b = t, lo = t, n = 1;
  if (a.starts) {
    // the last sequence that begins at or before this token
    int c = 0;
    for (int b0 = 0; b0 < a.B; b0 += 64) c += __popcll(__ballot(b0 + lane < a.B && a.starts[min(b0 + lane, a.B - 1)] <= t));
    b = c - 1;
    if (b >= 0) {
      lo = max(a.starts[b], 0);
      n = min(a.starts[b + 1], a.N) - lo;
    }
  }
  int p = -1;
  if (b >= 0 && t - lo < n) p = min(max(a.lens[b], 0), 1 << 30) - n + (t - lo);
  const bool in = p >= 0 && p < a.P;
  int64_t row = -1;  // the cache row
  if (in && a.tables && p / a.page < a.width) {
    const int pg = a.tables[(int64_t)b * a.width + p / a.page];
    if (pg >= 0 && pg < a.pages) row = (int64_t)pg * a.page + p % a.page;
  }
  const int turns = a.half / E, copies = (a.D - 2 * a.half) / E, per = turns + copies, vper = a.D / E;
  const int nq = a.oq ? a.Hq * per : 0, nk = row >= 0 && a.ok ? a.Hkv * per : 0, nv = row >= 0 && a.ov ? a.Hkv * vper : 0;
  const float *cr = a.cos + (int64_t)(in ? p : 0) * a.half, *sr = a.sin + (int64_t)(in ? p : 0) * a.half;
  for (int x = threadIdx.x; x < nq + nk + nv; x += 256) {
    if (x >= nq + nk) {
      const int h = (x - nq - nk) / vper, d = (x - nq - nk) % vper * E;
      copy_piece<T, E>((const T *)a.v + t * a.v_ss + h * a.v_sh + d, (T *)a.ov + (row * a.Hkv + h) * a.D + d);
      continue;
    }
    const bool isq = x < nq;
    const int y = isq ? x : x - nq, h = y / per, c = y % per;
    const T *src = isq ? (const T *)a.q + t * a.q_ss + h * a.q_sh : (const T *)a.k + t * a.k_ss + h * a.k_sh;
    T *dst = isq ? (T *)a.oq + ((int64_t)t * a.Hq + h) * a.D : (T *)a.ok + (row * a.Hkv + h) * a.D;
    if (c >= turns) {
      const int d = 2 * a.half + (c - turns) * E;
      if (in) {
        copy_piece<T, E>(src + d, dst + d);
      } else {
        const float z[E] = {};
        Piece<T, E>::store(dst + d, z);
      }
      continue;
    }
    float x0[E], x1[E], cc[E], ss[E];
    Piece<T, E>::load(src + c * E, x0);
    Piece<T, E>::load(src + a.half + c * E, x1);
    Piece<float, E>::load(cr + c * E, cc);
    Piece<float, E>::load(sr + c * E, ss);
    float y0[E], y1[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
      y0[e] = in ? x0[e] * cc[e] - x1[e] * ss[e] : 0.f;
      y1[e] = in ? x0[e] * ss[e] + x1[e] * cc[e] : 0.f;
    }
    Piece<T, E>::store(dst + c * E, y0);
    Piece<T, E>::store(dst + a.half + c * E, y1);
  }
}
#define NK_APPEND(T, name)                                                                    \
  extern "C" __global__ __launch_bounds__(256) void nk_rotary_append_##name(AppendArgs a) {   \
    rotary_append_body<T, 8>(a);                                                              \
  }                                                                                           \
  extern "C" __global__ __launch_bounds__(256) void nk_rotary_append1_##name(AppendArgs a) {  \
    rotary_append_body<T, 1>(a);                                                              \
  }
NK_APPEND(bf16, bf16)
NK_APPEND(f16, f16)
NK_APPEND(float, f32)

// ---------------------------------------------------------------------------
// The draw of a token.
//
// Weights w = 2^t, t = (x - max) log2(e) / T, are kept as whole numbers of
// 2^-40: sums of them are exact in 64 bits, so no order of additions or atomics
// changes a result, and what rounds to 0 (below 2^-41 of the largest, 4e-13)
// takes no part.  All three filters keep a beginning of the order (value
// descending, then index), so they come down to one border, the last (value,
// index) that stays, and the row is never sorted.
//
// Long rows take three launches, two of them over segments of the row, so that
// a few rows fill the chip:
//   top    each segment's largest value;
//   hist   each segment's counts and weights over BINS equal steps of t;
//   pick   one workgroup per row: the segments' histograms added, the bin in
//          which the count (top_k) or the weight (top_p) is reached, and the
//          values that matter listed in LDS: everything down to that bin, if
//          that is up to LIST values, and the border and the draw are searched
//          there; else that bin alone for the border, then the segment that holds
//          uniform x the kept weight, by the segments' sums.
// Rows of up to LIST tokens are one launch: the list is the row.
//
// A search (smp_select) finds where the running count or weight of a list in
// descending order of a key reaches a goal: histograms of 1024 steps of what is
// left of the keys' range, until a step is one key.  The key is the value for a
// border, the index for ties and for the draw.  A bin of more than LIST values
// (ties, a narrow spread) is searched in the row itself.
//
// Bound by one read of the logits and, in hist, by about 30 instructions per
// logit; with few rows by the latency of its launches.
// ---------------------------------------------------------------------------
struct SampleArgs {
  const void *x;
  const float *u;
  int32_t *out;
  const float *temp;     // per row; null: c_temp (likewise below)
  const int32_t *topk;
  const float *topp, *minp;
  uint64_t *tops;        // (rows, nseg): largest key and the complement of its index
  uint64_t *sums;        // (rows, nseg, BINS + 1): weights per bin, then their sum
  uint32_t *cnts;        // (rows, nseg, BINS)
  int64_t ld;            // elements from row to row
  int32_t rows, vocab, seg, nseg;  // seg: tokens of a segment
  float c_temp;
  int32_t c_topk;        // below 1: all
  float c_topp, c_minp;  // 1, 0: all
};

#define SMP_BLOCK 1024
#define SMP_SEG_BLOCK 256
#define SMP_BINS 512
#define SMP_LIST 8192
#define SMP_STEPS 1024
typedef unsigned long long u64;

// order of the values as whole numbers; -0 and 0 tie
NK_DEVICE uint32_t smp_key(float x) {
  const uint32_t u = __float_as_uint(x + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
NK_DEVICE float smp_value(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }

struct SmpRow {
  float best, c;  // largest logit, log2(e) / T
  NK_DEVICE void set(float b, float temp) {
    best = b;
    c = fminf(1.44269504088896340736f / temp, 3.4e38f);
  }
  // log2 of the weight; the largest logit has 0 also where it is infinite
  NK_DEVICE float depth(float x) const { return x == best ? 0.f : (x - best) * c; }
};
// weight in steps of 2^-40; 0 for NaN.  The hardware's 2^t is within an ulp, 1e-7
// of the weight.
NK_DEVICE u64 smp_weight(float t) {
  if (!(t > -42.f)) return 0;
  const float w = __builtin_amdgcn_exp2f(t) * 0x1p40f;
  const uint32_t hi = (uint32_t)(w * 0x1p-16f);
  const float rest = __builtin_fmaf((float)hi, -0x1p16f, w);  // exact: below 2^16
  return ((u64)hi << 16) + (u64)(uint32_t)__builtin_rintf(rest);
}
// (a weight above 0 has t >= -41: bin 492 at most)
NK_DEVICE int smp_bin(float t) { return min(SMP_BINS - 1, (int)(t * -12.f)); }

// Logits lo .. hi-1 of a row in pieces of 16 aligned bytes: f(index, value) by
// THREADS threads.  The pieces at the ends are read element by element.
template <typename T, int THREADS, typename F>
NK_DEVICE void smp_each(const T *x, int lo, int hi, F f) {
  constexpr int E = 16 / sizeof(T);
  const int off = (int)(((uintptr_t)(x + lo) & 15) / sizeof(T));  // elements of the first piece before lo
  for (int i = lo - off + threadIdx.x * E; i < hi; i += THREADS * E) {
    if (i >= lo && i + E <= hi) {
      const uint4 u = *reinterpret_cast<const uint4 *>(x + i);
      T v[E];
      __builtin_memcpy(v, &u, 16);
#pragma unroll
      for (int e = 0; e < E; ++e) f(i + e, Elt<T>::load(v, e));
    } else {
#pragma unroll 1
      for (int e = max(0, lo - i); e < min(E, hi - i); ++e) f(i + e, Elt<T>::load(x, i + e));
    }
  }
}

template <int WAVES>
NK_DEVICE u64 smp_max(u64 v, u64 *red) {
#pragma unroll
  for (int o = 32; o; o >>= 1) v = max(v, (u64)__shfl_xor(v, o, 64));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < WAVES; ++i) v = max(v, red[i]);
  return v;
}
template <int WAVES>
NK_DEVICE u64 smp_sum(u64 v, u64 *red) {
#pragma unroll
  for (int o = 32; o; o >>= 1) v += (u64)__shfl_xor(v, o, 64);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  v = 0;
#pragma unroll
  for (int i = 0; i < WAVES; ++i) v += red[i];
  return v;
}
// largest value of a stretch and its lowest index, as one number; 0 where all
// are NaN or -inf
template <typename T, int THREADS>
NK_DEVICE u64 smp_top(const T *x, int lo, int hi, u64 *red) {
  u64 top = 0;
  smp_each<T, THREADS>(x, lo, hi, [&](int i, float v) {
    if (v > -INFINITY) top = max(top, (u64)smp_key(v) << 32 | (uint32_t)~i);
  });
  return smp_max<THREADS / 64>(top, red);
}

template <typename T>
__device__ __forceinline__ void sample_top_body(const SampleArgs &a) {
  __shared__ u64 red[SMP_SEG_BLOCK / 64];
  const int r = blockIdx.x / a.nseg, s = blockIdx.x % a.nseg;
  const u64 top = smp_top<T, SMP_SEG_BLOCK>((const T *)a.x + r * a.ld, s * a.seg, min(a.vocab, (s + 1) * a.seg), red);
  if (threadIdx.x == 0) a.tops[blockIdx.x] = top;
}
template <int THREADS>
NK_DEVICE u64 smp_row_top(const SampleArgs &a, int r, u64 *red) {
  u64 top = 0;
  for (int i = threadIdx.x; i < a.nseg; i += THREADS) top = max(top, (u64)a.tops[(int64_t)r * a.nseg + i]);
  return smp_max<THREADS / 64>(top, red);
}
// its settings; false where there is nothing to weigh: no logit to draw, or no
// temperature
NK_DEVICE bool smp_settings(const SampleArgs &a, int r, u64 top, SmpRow &row) {
  const float temp = a.temp ? a.temp[r] : a.c_temp;
  row.set(smp_value((uint32_t)(top >> 32)), temp);
  return top && temp > 0.f;
}

template <typename T>
__device__ __forceinline__ void sample_hist_body(const SampleArgs &a) {
  __shared__ u64 sum[SMP_BINS];
  __shared__ uint32_t cnt[SMP_BINS];
  __shared__ u64 red[SMP_SEG_BLOCK / 64];
  const int r = blockIdx.x / a.nseg, s = blockIdx.x % a.nseg, tid = threadIdx.x;
  for (int i = tid; i < SMP_BINS; i += SMP_SEG_BLOCK) sum[i] = 0, cnt[i] = 0;
  SmpRow row;
  if (!smp_settings(a, r, smp_row_top<SMP_SEG_BLOCK>(a, r, red), row)) return;
  u64 all = 0;
  const bool bins = a.topk || a.topp || a.minp || a.c_topk > 0 || a.c_topp < 1.f || a.c_minp > 0.f;
  smp_each<T, SMP_SEG_BLOCK>((const T *)a.x + r * a.ld, s * a.seg, min(a.vocab, (s + 1) * a.seg), [&](int, float v) {
    const float t = row.depth(v);
    const u64 w = smp_weight(t);
    all += w;
    if (bins && w) {
      const int b = smp_bin(t);
      atomicAdd(&cnt[b], 1u);
      atomicAdd(&sum[b], w);
    }
  });
  all = smp_sum<SMP_SEG_BLOCK / 64>(all, red);  // (and the histogram is whole)
  uint64_t *so = a.sums + (int64_t)blockIdx.x * (SMP_BINS + 1);
  uint32_t *co = a.cnts + (int64_t)blockIdx.x * SMP_BINS;
  if (bins)
    for (int i = tid; i < SMP_BINS; i += SMP_SEG_BLOCK) so[i] = sum[i], co[i] = cnt[i];
  if (tid == 0) so[SMP_BINS] = all;
}

struct SmpShared {
  u64 hsum[SMP_BINS];      // the row's histogram
  u64 sum[SMP_STEPS];      // a search's
  uint32_t hcnt[SMP_BINS];
  uint32_t cnt[SMP_STEPS];
  uint32_t key[SMP_LIST], idx[SMP_LIST];
  u64 red[SMP_BLOCK / 64], sw[SMP_BLOCK / 64];
  uint32_t sc[SMP_BLOCK / 64];
  uint32_t n, kmin, kmax;
  // where a running sum reached its goal: step, and count and weight before and with it
  uint32_t bin, cb, ca;
  u64 wb, wa;
};

// Running sums of one count and weight per thread, on top of cb and wb: the
// first to reach `need` (COUNT) or `goal`.
template <bool COUNT>
NK_DEVICE void smp_search(SmpShared &s, uint32_t c, u64 w, uint32_t cb, u64 wb, uint32_t need, u64 goal) {
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
  uint32_t ci = c;
  u64 wi = w;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const uint32_t cu = __shfl_up(ci, o, 64);
    const u64 wu = __shfl_up(wi, o, 64);
    if (lane >= o) ci += cu, wi += wu;
  }
  __syncthreads();
  if (lane == 63) s.sc[wid] = ci, s.sw[wid] = wi;
  __syncthreads();
  ci += cb, wi += wb;
#pragma unroll
  for (int i = 0; i < SMP_BLOCK / 64; ++i)
    if (i < wid) ci += s.sc[i], wi += s.sw[i];
  if (COUNT ? ci - c < need && ci >= need : wi - w < goal && wi >= goal)
    s.bin = threadIdx.x, s.cb = ci - c, s.ca = ci, s.wb = wi - w, s.wa = wi;
  __syncthreads();
}

// where a search ended: the key, how many of its elements are in, and the weight
// up to and with them
struct SmpBorder {
  uint32_t key, ties;
  u64 upto;
};
// Of elements 0 .. n-1, f(i, key, weight) says which take part.  Those of one
// key weigh the same.
template <bool COUNT, typename F>
NK_DEVICE SmpBorder smp_select(SmpShared &s, int n, F f, uint32_t cb, u64 wb, uint32_t need, u64 goal) {
  const int tid = threadIdx.x;
  __syncthreads();
  if (tid == 0) s.kmin = 0xffffffffu, s.kmax = 0;
  __syncthreads();
  uint32_t mn = 0xffffffffu, mx = 0, k;
  u64 w;
  for (int i = tid; i < n; i += SMP_BLOCK)
    if (f(i, k, w)) mn = min(mn, k), mx = max(mx, k);
#pragma unroll
  for (int o = 32; o; o >>= 1) mn = min(mn, (uint32_t)__shfl_xor(mn, o, 64)), mx = max(mx, (uint32_t)__shfl_xor(mx, o, 64));
  if ((tid & 63) == 0) atomicMin(&s.kmin, mn), atomicMax(&s.kmax, mx);
  __syncthreads();
  uint32_t klo = s.kmin, khi = s.kmax;
  SmpBorder b;
  while (true) {
    const uint32_t range = max(khi, klo) - klo;
    const int shift = range < SMP_STEPS ? 0 : 22 - __builtin_clz(range);
    s.cnt[tid] = 0, s.sum[tid] = 0;
    __syncthreads();
    for (int i = tid; i < n; i += SMP_BLOCK)
      if (f(i, k, w) && k >= klo && k <= khi) {
        atomicAdd(&s.cnt[(khi - k) >> shift], 1u);
        atomicAdd(&s.sum[(khi - k) >> shift], w);
      }
    __syncthreads();
    smp_search<COUNT>(s, s.cnt[tid], s.sum[tid], cb, wb, need, goal);
    const uint32_t at = s.bin;
    cb = s.cb, wb = s.wb;
    if (shift == 0) {
      const u64 each = (s.wa - wb) / max(s.ca - cb, 1u);
      b.key = khi - at;
      b.ties = COUNT ? need - cb : (uint32_t)((goal - wb + each - 1) / max(each, (u64)1));
      b.upto = wb + b.ties * each;
      return b;
    }
    const uint32_t top = khi - (at << shift);
    klo = top - klo < (1u << shift) ? klo : top - (1u << shift) + 1;
    khi = top;
  }
}

// the elements of a stretch for which f holds, into the list
template <typename T, typename F>
NK_DEVICE int smp_gather(SmpShared &s, const T *x, int lo, int hi, F f) {
  __syncthreads();
  if (threadIdx.x == 0) s.n = 0;
  __syncthreads();
  smp_each<T, SMP_BLOCK>(x, lo, hi, [&](int i, float v) {
    if (f(i, v)) {
      const uint32_t at = atomicAdd(&s.n, 1u);
      if (at < SMP_LIST) s.key[at] = smp_key(v), s.idx[at] = i;
    }
  });
  __syncthreads();
  return s.n;
}

template <bool B> struct SmpFlag {
  static constexpr bool value = B;
};
// SMALL: the row is one segment of up to LIST tokens, and this its only launch
template <typename T, bool SMALL>
__device__ __forceinline__ void sample_pick_body(const SampleArgs &a) {
  __shared__ SmpShared s;
  const int tid = threadIdx.x, r = blockIdx.x;
  const T *x = (const T *)a.x + r * a.ld;
  const u64 top = SMALL ? smp_top<T, SMP_BLOCK>(x, 0, a.vocab, s.red) : smp_row_top<SMP_BLOCK>(a, r, s.red);
  SmpRow row;
  if (!smp_settings(a, r, top, row)) {
    if (tid == 0) a.out[r] = top ? (int32_t)~(uint32_t)top : -1;
    return;
  }
  const int topk = a.topk ? a.topk[r] : a.c_topk;
  const float topp = a.topp ? a.topp[r] : a.c_topp, minp = a.minp ? a.minp[r] : a.c_minp;
  const bool by_k = topk > 0 && topk < a.vocab, by_p = topp < 1.f, by_m = minp > 0.f;
  const float tmin = by_m ? log2f(fminf(minp, 1.f)) : -INFINITY;  // the least depth that min_p keeps

  // a listed or stored element's weight
  auto listed = [&](int i, uint32_t &k, u64 &w) {
    k = s.key[i];
    w = smp_weight(row.depth(smp_value(k)));
    return true;
  };
  auto stored = [&](int i, uint32_t &k, u64 &w) {
    const float v = Elt<T>::load(x, i);
    k = smp_key(v);
    w = smp_weight(row.depth(v));
    return w != 0;
  };
  const uint64_t *sums = a.sums + (int64_t)r * a.nseg * (SMP_BINS + 1);
  const uint32_t *cnts = a.cnts + (int64_t)r * a.nseg * SMP_BINS;
  bool whole = SMALL;      // the list holds all that is kept
  u64 total = 0;           // weight of the row
  int n = 0;
  uint32_t cbin = 0;       // the border's bin, count and weight before it (not whole)
  int last = SMP_BINS - 1; // bins up to here can be kept
  if (SMALL) {
    n = smp_gather(s, x, 0, a.vocab, [&](int, float v) { return smp_weight(row.depth(v)) != 0; });
    if (by_p && !(by_k && n >= topk)) {
      for (int i = tid; i < n; i += SMP_BLOCK) {
        uint32_t k;
        u64 w;
        listed(i, k, w);
        total += w;
      }
      total = smp_sum<SMP_BLOCK / 64>(total, s.red);
    }
  } else if (by_k || by_p || by_m) {
    uint32_t c = 0;
    u64 w = 0;
    const int bin = tid % SMP_BINS;
    for (int i = tid / SMP_BINS; i < a.nseg; i += SMP_BLOCK / SMP_BINS) {
      c += cnts[(int64_t)i * SMP_BINS + bin];
      w += sums[(int64_t)i * (SMP_BINS + 1) + bin];
    }
    if (tid < SMP_BINS) s.hcnt[bin] = c, s.hsum[bin] = w;
    __syncthreads();
    if (tid >= SMP_BINS) s.hcnt[bin] += c, s.hsum[bin] += w;
    total = smp_sum<SMP_BLOCK / 64>(w, s.red);  // (and the histogram is whole)
  }
  auto bin_of_row = [&](bool count, uint32_t need, u64 goal) {
    const uint32_t c = tid < SMP_BINS ? s.hcnt[tid] : 0;
    const u64 w = tid < SMP_BINS ? s.hsum[tid] : 0;
    __syncthreads();
    if (tid == 0) s.bin = SMP_BINS, s.cb = 0, s.ca = 0, s.wb = 0, s.wa = 0;
    if (count) smp_search<true>(s, c, w, 0, 0, need, goal);
    else smp_search<false>(s, c, w, 0, 0, need, goal);
  };
  auto share = [&](u64 of) {  // whole steps: at least topp of it, at least one
    return min(max((u64)ceil((double)fmaxf(topp, 0.f) * (double)of), (u64)1), of);
  };
  bool k_cuts = by_k, p_cuts = by_p;
  if (SMALL) {
    k_cuts = by_k && n >= topk;
  } else if (by_k || by_p || by_m) {
    // the bin that holds the first border; a top_k past the row's weights cuts nothing
    if (by_k) {
      bin_of_row(true, topk, 0);
      k_cuts = s.bin < SMP_BINS;
    }
    if (!k_cuts && by_p) bin_of_row(false, 0, share(total));
    if (k_cuts || by_p) last = s.bin;
    if (by_m && !(k_cuts && by_p) && smp_bin(tmin) < last) {
      last = smp_bin(tmin);  // min_p ends before either: their border is of no use
      k_cuts = p_cuts = false;
    }
    // everything down to there, where the list can hold it
    const uint32_t upto = (uint32_t)smp_sum<SMP_BLOCK / 64>(tid <= last ? s.hcnt[tid] : 0, s.red);
    if (upto <= SMP_LIST) {
      const float least = -((float)last + 1.01f) / 12.f;
      n = smp_gather(s, x, 0, a.vocab, [&](int, float v) {
        const float t = row.depth(v);
        return t > least && smp_bin(t) <= last && smp_weight(t) != 0;
      });
      whole = true;
    }
  }

  // the border: the last (value, index) kept
  uint32_t bkey = 0, bidx = 0xffffffffu;
  auto tie_break = [&](const SmpBorder &b, int len, auto each, auto index) {
    bkey = b.key;
    // the highest index of its ties that stays: by count, lowest first
    bidx = ~smp_select<true>(s, len, [&](int i, uint32_t &k, u64 &w) {
      const bool in = each(i, k, w) && k == b.key;
      k = ~index(i);
      return in;
    }, 0, 0, b.ties, 0).key;
  };
  int held = -1;  // the bin that the list holds
  auto in_list = [&](int i) { return s.idx[i]; };
  auto in_row = [&](int i) { return (uint32_t)i; };
  if (whole) {
    if (k_cuts || p_cuts) {
      SmpBorder b;
      if (k_cuts) b = smp_select<true>(s, n, listed, 0, 0, topk, 0);
      if (p_cuts) b = smp_select<false>(s, n, listed, 0, 0, 0, share(k_cuts ? b.upto : total));
      tie_break(b, n, listed, in_list);
    }
  } else if (k_cuts || p_cuts) {
    SmpBorder b;
    // the values of one bin, from the list or, too many, from the row
    bool fits = false;
    auto find = [&](auto count, uint32_t need, u64 goal) {
      const int bin = s.bin;
      const uint32_t cb = s.cb;
      const u64 wb = s.wb;
      cbin = bin;
      auto of_bin = [&](int i, uint32_t &k, u64 &w) { return stored(i, k, w) && smp_bin(row.depth(smp_value(k))) == bin; };
      if (bin != held) {
        fits = s.ca - cb <= SMP_LIST;
        if (fits) n = smp_gather(s, x, 0, a.vocab, [&](int, float v) {
          const float t = row.depth(v);
          return smp_bin(t) == bin && smp_weight(t) != 0;
        });
        held = fits ? bin : -1;
      }
      constexpr bool COUNT = decltype(count)::value;
      b = fits ? smp_select<COUNT>(s, n, listed, cb, wb, need, goal) : smp_select<COUNT>(s, a.vocab, of_bin, cb, wb, need, goal);
    };
    if (k_cuts) find(SmpFlag<true>{}, topk, 0);
    if (p_cuts) {
      const u64 goal = share(k_cuts ? b.upto : total);
      bin_of_row(false, 0, goal);
      find(SmpFlag<false>{}, 0, goal);
    }
    if (fits) tie_break(b, n, listed, in_list);
    else tie_break(b, a.vocab, stored, in_row);
  }
  auto kept = [&](uint32_t k, uint32_t i, float t) { return (k > bkey || (k == bkey && i <= bidx)) && t >= tmin; };

  // the draw: the first kept index up to and with which the weights exceed
  // uniform x their sum, that is, reach the whole number behind it
  const float uni = a.u[r];
  auto goal_of = [&](u64 all) {
    const u64 g = uni > 0.f ? (u64)(fmin((double)uni, 1.) * (double)all) : 0;
    return !(uni < 1.f) || g >= all ? all : g + 1;  // (NaN too: the last kept)
  };
  auto draw = [&](u64 goal, u64 before) {
    const uint32_t at = ~smp_select<false>(s, n, [&](int i, uint32_t &k, u64 &w) {
      listed(i, k, w);
      const bool in = kept(k, s.idx[i], row.depth(smp_value(k)));
      k = ~s.idx[i];
      return in;
    }, 0, before, 0, goal).key;
    if (tid == 0) a.out[r] = at;
  };
  if (whole) {
    u64 all = 0;
    for (int i = tid; i < n; i += SMP_BLOCK) {
      uint32_t k;
      u64 w;
      listed(i, k, w);
      if (kept(k, s.idx[i], row.depth(smp_value(k)))) all += w;
    }
    draw(goal_of(smp_sum<SMP_BLOCK / 64>(all, s.red)), 0);
    return;
  }
  // by segments: bins before the border's are kept whole; of the one it is in,
  // what is kept is added value by value
  const int edge = min(k_cuts || p_cuts ? (int)cbin : SMP_BINS, by_m ? smp_bin(tmin) : SMP_BINS);
  u64 *seg = s.sum;  // (up to STEPS segments)
  __syncthreads();
  seg[tid] = 0;
  __syncthreads();
  if (edge == SMP_BINS) {
    for (int i = tid; i < a.nseg; i += SMP_BLOCK) seg[i] = sums[(int64_t)i * (SMP_BINS + 1) + SMP_BINS];
  } else {
    for (int i = tid >> 6; i < a.nseg; i += SMP_BLOCK / 64) {  // a wave for each
      u64 w = 0;
      for (int b = tid & 63; b < edge; b += 64) w += sums[(int64_t)i * (SMP_BINS + 1) + b];
#pragma unroll
      for (int o = 32; o; o >>= 1) w += (u64)__shfl_xor(w, o, 64);
      if ((tid & 63) == 0) atomicAdd(&seg[i], w);
    }
    if (held == edge) {
      for (int i = tid; i < n; i += SMP_BLOCK) {
        const float t = row.depth(smp_value(s.key[i]));
        if (kept(s.key[i], s.idx[i], t)) atomicAdd(&seg[s.idx[i] / a.seg], smp_weight(t));
      }
    } else {
      smp_each<T, SMP_BLOCK>(x, 0, a.vocab, [&](int i, float v) {
        const float t = row.depth(v);
        if (!(t > -42.f) || smp_bin(t) != edge) return;
        const u64 w = smp_weight(t);
        if (w && kept(smp_key(v), i, t)) atomicAdd(&seg[i / a.seg], w);
      });
    }
  }
  __syncthreads();
  const u64 mine = tid < a.nseg ? seg[tid] : 0;
  const u64 goal = goal_of(smp_sum<SMP_BLOCK / 64>(mine, s.red));
  smp_search<false>(s, 0, mine, 0, 0, 0, goal);
  const int at = s.bin;
  const u64 before = s.wb;
  n = smp_gather(s, x, at * a.seg, min(a.vocab, (at + 1) * a.seg), [&](int i, float v) {
    const float t = row.depth(v);
    return smp_weight(t) != 0 && kept(smp_key(v), i, t);
  });
  draw(goal, before);
}
#define NK_SAMPLE(T, name)                                                                          \
  extern "C" __global__ __launch_bounds__(SMP_SEG_BLOCK) void nk_sample_top_##name(SampleArgs a) {  \
    sample_top_body<T>(a);                                                                          \
  }                                                                                                 \
  extern "C" __global__ __launch_bounds__(SMP_SEG_BLOCK) void nk_sample_hist_##name(SampleArgs a) { \
    sample_hist_body<T>(a);                                                                         \
  }                                                                                                 \
  extern "C" __global__ __launch_bounds__(SMP_BLOCK) void nk_sample_pick_##name(SampleArgs a) {     \
    sample_pick_body<T, false>(a);                                                                  \
  }                                                                                                 \
  extern "C" __global__ __launch_bounds__(SMP_BLOCK) void nk_sample_row_##name(SampleArgs a) {      \
    sample_pick_body<T, true>(a);                                                                   \
  }
NK_SAMPLE(bf16, bf16)
NK_SAMPLE(f16, f16)
NK_SAMPLE(float, f32)
