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
// Weights w = exp((x - max) / T) are kept as whole numbers of 2^-40: sums of
// them are exact in 64 bits, so no order of additions or atomics changes a
// result, and what rounds to 0 (below 2^-41 of the largest, 4e-13) takes no
// part.  All three filters keep a beginning of the order (value, then index),
// so they come down to one border: a value, and how many of its ties stay,
// lowest index first.  The border is found without sorting the row:
//   1. the largest logit;
//   2. a histogram of counts and weights over BINS equal steps of (x - max) / T;
//   3. the bin in which the count (top_k) or the weight (top_p) is reached;
//   4. that bin's few values ranked against each other in LDS; a bin of more
//      than LIST values (many ties, a narrow spread) is first cut down by
//      further histograms over its range of values.
// Then the kept weights are summed over tiles of the row in index order, the
// tile holding uniform x total is found, and the token in it.
// ---------------------------------------------------------------------------
struct SampleArgs {
  const void *x;
  const float *u;
  int32_t *out;
  const float *temp;     // per row; null: c_temp (likewise below)
  const int32_t *topk;
  const float *topp, *minp;
  int64_t ld;            // elements from row to row
  int32_t rows, vocab;
  float c_temp;
  int32_t c_topk;        // below 1: all
  float c_topp, c_minp;  // 1, 0: all
};

#define SMP_BLOCK 1024
#define SMP_BINS 2048
#define SMP_LIST 2048
#define SMP_TILES 1024  // tiles of a row, at most
typedef unsigned long long u64;

// order of the values as whole numbers; -0 and 0 tie
NK_DEVICE uint32_t smp_key(float x) {
  const uint32_t u = __float_as_uint(x + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
struct SmpRow {
  float best, temp;
  // (x - best) / temp; the largest is 0 also where it is infinite
  NK_DEVICE float depth(float x) const { return x == best ? 0.f : (x - best) / temp; }
};
// weight in steps of 2^-40; 0 for NaN
NK_DEVICE u64 smp_weight(float d) {
  if (!(d > -29.f)) return 0;
  const float w = exp_acc(d) * 0x1p40f;  // at most 2^40 and a few ulp
  const uint32_t hi = (uint32_t)(w * 0x1p-16f);
  const float rest = w - (float)hi * 0x1p16f;  // exact: below 2^16
  return ((u64)hi << 16) + (u64)(uint32_t)__builtin_rintf(rest);
}
// the deepest weight above 0 is at 28.42: bin 2046
NK_DEVICE int smp_bin(float d) { return min(SMP_BINS - 1, (int)(d * -72.f)); }

template <typename V>
NK_DEVICE V smp_shfl_up(V v, int n) {
  return __shfl_up(v, n, 64);
}
// exclusive sums of c and w over the workgroup's threads, and the totals
NK_DEVICE void smp_scan(uint32_t c, u64 w, uint32_t &ce, u64 &we, uint32_t &ct, u64 &wt, uint32_t *sc, u64 *sw) {
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
  if (lane == 63) sc[wid] = ci, sw[wid] = wi;
  __syncthreads();
  ct = 0, wt = 0;
  uint32_t cb = 0;
  u64 wb = 0;
#pragma unroll
  for (int i = 0; i < SMP_BLOCK / 64; ++i) {
    if (i < wid) cb += sc[i], wb += sw[i];
    ct += sc[i], wt += sw[i];
  }
  ce = cb + ci - c;
  we = wb + wi - w;
}

struct SmpShared {
  uint32_t cnt[2][SMP_BINS];
  u64 sum[2][SMP_BINS];
  uint32_t key[SMP_LIST], idx[SMP_LIST];
  u64 w[SMP_LIST];
  uint32_t skey[SMP_LIST];
  uint32_t sc[SMP_BLOCK / 64];
  u64 sw[SMP_BLOCK / 64];
  u64 red[SMP_BLOCK / 64];
  uint32_t n, kmin, kmax;
  // what a search found
  uint32_t bin, cb, key_at, ties;
  u64 wb, upto;
};

// Where the running count reaches `need` (COUNT) or the running weight `goal`,
// over the SMP_BINS entries of a histogram or the SMP_LIST of a ranked list
// (two per thread); false where neither does.
template <bool COUNT>
NK_DEVICE bool smp_search(SmpShared &s, const uint32_t *cnt, const u64 *sum, uint32_t cb, u64 wb, uint32_t need, u64 goal) {
  const int i = 2 * threadIdx.x;
  const uint32_t c0 = cnt ? cnt[i] : 1, c1 = cnt ? cnt[i + 1] : 1;
  const u64 w0 = sum[i], w1 = sum[i + 1];
  uint32_t ce, ct;
  u64 we, wt;
  smp_scan(c0 + c1, w0 + w1, ce, we, ct, wt, s.sc, s.sw);
  ce += cb, we += wb;
  const bool before0 = COUNT ? ce < need : we < goal;
  const bool in0 = COUNT ? ce + c0 >= need : we + w0 >= goal;
  const bool in1 = COUNT ? ce + c0 + c1 >= need : we + w0 + w1 >= goal;
  if (before0 && in1) {
    s.bin = in0 ? i : i + 1;
    s.cb = in0 ? ce : ce + c0;
    s.wb = in0 ? we : we + w0;
    s.upto = in0 ? we + w0 : we + w0 + w1;
  }
  __syncthreads();
  return COUNT ? cb + ct >= need : wb + wt >= goal;
}

// The border in bin `s.bin` of the first histogram: the key of the last value
// kept, how many of its ties are (s.key_at, s.ties), and the weight up to and
// with it (s.upto).
template <typename T, bool COUNT>
NK_DEVICE void smp_border(SmpShared &s, const T *x, int vocab, const SmpRow &r, uint32_t need, u64 goal) {
  const int tid = threadIdx.x;
  const int bin = s.bin;
  uint32_t cb = s.cb;
  u64 wb = s.wb;
  uint32_t klo = 0, khi = 0xffffffffu;  // the keys left
  bool by_bin = true;
  while (true) {
    __syncthreads();
    if (tid == 0) s.n = 0, s.kmin = 0xffffffffu, s.kmax = 0;
    __syncthreads();
    uint32_t mn = 0xffffffffu, mx = 0;
    for (int i = tid; i < vocab; i += SMP_BLOCK) {
      const float v = Elt<T>::load(x, i);
      const float d = r.depth(v);
      const uint32_t k = smp_key(v);
      if (!(d > -29.f) || (by_bin ? smp_bin(d) != bin : k < klo || k > khi)) continue;
      const u64 w = smp_weight(d);
      if (!w) continue;
      mn = min(mn, k), mx = max(mx, k);
      const uint32_t at = atomicAdd(&s.n, 1u);
      if (at < SMP_LIST) s.key[at] = k, s.idx[at] = i, s.w[at] = w;
    }
    atomicMin(&s.kmin, mn);
    atomicMax(&s.kmax, mx);
    __syncthreads();
    const uint32_t n = s.n;
    klo = s.kmin, khi = s.kmax;
    if (n <= SMP_LIST) break;
    // too many: a histogram of their range of keys, one key a bin once it is
    // narrow enough
    by_bin = false;
    int shift = 0;
    while (((khi - klo) >> shift) >= SMP_BINS) ++shift;
    for (int i = tid; i < SMP_BINS; i += SMP_BLOCK) s.cnt[1][i] = 0, s.sum[1][i] = 0;
    __syncthreads();
    for (int i = tid; i < vocab; i += SMP_BLOCK) {
      const float v = Elt<T>::load(x, i);
      const float d = r.depth(v);
      const uint32_t k = smp_key(v);
      if (!(d > -29.f) || k < klo || k > khi) continue;
      const u64 w = smp_weight(d);
      if (!w) continue;
      atomicAdd(&s.cnt[1][(khi - k) >> shift], 1u);
      atomicAdd(&s.sum[1][(khi - k) >> shift], w);
    }
    __syncthreads();
    smp_search<COUNT>(s, s.cnt[1], s.sum[1], cb, wb, need, goal);
    const uint32_t sub = s.bin;
    cb = s.cb, wb = s.wb;
    if (shift == 0) {  // one key: its ties share a weight
      if (tid == 0) {
        const u64 w = s.sum[1][sub] / s.cnt[1][sub];
        s.key_at = khi - sub;
        s.ties = COUNT ? need - cb : (uint32_t)((goal - wb + w - 1) / w);
        s.upto = wb + s.ties * w;
      }
      __syncthreads();
      return;
    }
    const uint32_t top = khi - (sub << shift), low = top - ((1u << shift) - 1);
    klo = low > top ? klo : max(klo, low);
    khi = top;
  }
  // rank the list: larger keys first, then lower indices
  const uint32_t n = s.n;
  uint32_t myk[SMP_LIST / SMP_BLOCK], rank[SMP_LIST / SMP_BLOCK];
  u64 myw[SMP_LIST / SMP_BLOCK];
#pragma unroll
  for (int e = 0; e < SMP_LIST / SMP_BLOCK; ++e) {
    const uint32_t i = tid + e * SMP_BLOCK;
    rank[e] = i;
    myk[e] = 0, myw[e] = 0;
    if (i < n) {
      const uint32_t k = s.key[i], ix = s.idx[i];
      uint32_t c = 0;
      for (uint32_t j = 0; j < n; ++j) c += s.key[j] > k || (s.key[j] == k && s.idx[j] < ix);
      rank[e] = c;
      myk[e] = k, myw[e] = s.w[i];
    }
  }
  __syncthreads();
#pragma unroll
  for (int e = 0; e < SMP_LIST / SMP_BLOCK; ++e) s.skey[rank[e]] = myk[e], s.w[rank[e]] = myw[e];
  __syncthreads();
  smp_search<COUNT>(s, nullptr, s.w, cb, wb, need, goal);
  if (tid == 0) {
    const uint32_t at = min(s.bin, n - 1), k = s.skey[at];
    uint32_t ties = 1;
    while (ties <= at && s.skey[at - ties] == k) ++ties;
    s.key_at = k;
    s.ties = ties;
  }
  __syncthreads();
}

template <typename T>
__device__ __forceinline__ void sample_body(const SampleArgs &a) {
  __shared__ SmpShared s;
  const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6, r = blockIdx.x;
  const T *x = (const T *)a.x + (int64_t)r * a.ld;
  SmpRow row;
  row.temp = a.temp ? a.temp[r] : a.c_temp;
  // 1. the largest logit and its lowest index
  u64 top = 0;
  for (int i = tid; i < a.vocab; i += SMP_BLOCK) {
    const float v = Elt<T>::load(x, i);
    if (v > -INFINITY) top = max(top, (u64)smp_key(v) << 32 | (uint32_t)~i);
  }
#pragma unroll
  for (int o = 32; o; o >>= 1) top = max(top, (u64)__shfl_xor(top, o, 64));
  if (lane == 0) s.red[wid] = top;
  __syncthreads();
  for (int i = 0; i < SMP_BLOCK / 64; ++i) top = max(top, s.red[i]);
  const int32_t first = top ? (int32_t)~(uint32_t)top : -1;
  if (first < 0 || !(row.temp > 0.f)) {
    if (tid == 0) a.out[r] = first;
    return;
  }
  row.best = Elt<T>::load(x, first);
  const int topk = a.topk ? a.topk[r] : a.c_topk;
  const float topp = a.topp ? a.topp[r] : a.c_topp, minp = a.minp ? a.minp[r] : a.c_minp;
  const bool by_k = topk > 0 && topk < a.vocab, by_p = topp < 1.f;
  uint32_t border = 0, ties = 0xffffffffu;
  if (by_k || by_p) {
    // 2. the histogram
    for (int i = tid; i < SMP_BINS; i += SMP_BLOCK) s.cnt[0][i] = 0, s.sum[0][i] = 0;
    __syncthreads();
    u64 all = 0;
    for (int i = tid; i < a.vocab; i += SMP_BLOCK) {
      const float d = row.depth(Elt<T>::load(x, i));
      const u64 w = smp_weight(d);
      if (!w) continue;
      const int b = smp_bin(d);
      all += w;
      atomicAdd(&s.cnt[0][b], 1u);
      atomicAdd(&s.sum[0][b], w);
    }
    // 3. and 4., first by the count, then by the weight of what it left
    uint32_t ce, ct;
    u64 we, total;
    smp_scan(0, all, ce, we, ct, total, s.sc, s.sw);
    if (by_k && smp_search<true>(s, s.cnt[0], s.sum[0], 0, 0, topk, 0)) {
      smp_border<T, true>(s, x, a.vocab, row, topk, 0);
      border = s.key_at, ties = s.ties, total = s.upto;
    }
    if (by_p) {
      // whole steps: at least topp of the total, at least one
      const double g = ceil((double)fmaxf(topp, 0.f) * (double)total);
      const u64 goal = min(max((u64)g, (u64)1), total);
      __syncthreads();
      smp_search<false>(s, s.cnt[0], s.sum[0], 0, 0, 0, goal);
      smp_border<T, false>(s, x, a.vocab, row, 0, goal);
      border = s.key_at, ties = s.ties;
    }
  }
  // the kept weights of each tile, in index order; ties of the border apart,
  // as how many of them stay depends on the tiles before
  const int tile = max(256, (a.vocab + SMP_TILES * 256 - 1) / (SMP_TILES * 256) * 256);
  const int tiles = (a.vocab + tile - 1) / tile;
  const float floor_w = fminf(minp, 1.f);
  u64 *tw = s.sum[1];
  uint32_t *tt = s.cnt[1];
  auto weigh = [&](int i, uint32_t &tie) -> u64 {
    const float v = Elt<T>::load(x, i);
    const float d = row.depth(v);
    const u64 w = smp_weight(d);
    const uint32_t k = smp_key(v);
    tie = 0;
    if (!w || k < border || (floor_w > 0.f && !(exp_acc(d) >= floor_w))) return 0;
    if (k == border) {
      tie = 1;
      return 0;
    }
    return w;
  };
  // (a border of 0, the whole row, is no value's key)
  const float best_border = border ? __uint_as_float(border & 0x80000000u ? border & 0x7fffffffu : ~border) : 0.f;
  u64 tie_w = border ? smp_weight(row.depth(best_border)) : 0;
  __syncthreads();
  for (int t = wid; t < tiles; t += SMP_BLOCK / 64) {
    u64 w = 0;
    uint32_t c = 0;
    for (int i = t * tile + lane; i < min(a.vocab, (t + 1) * tile); i += 64) {
      uint32_t tie;
      w += weigh(i, tie);
      c += tie;
    }
#pragma unroll
    for (int o = 32; o; o >>= 1) w += (u64)__shfl_xor(w, o, 64), c += __shfl_xor(c, o, 64);
    if (lane == 0) tw[t] = w, tt[t] = c;
  }
  __syncthreads();
  uint32_t c = tid < tiles ? tt[tid] : 0, ce, ct;
  u64 w = tid < tiles ? tw[tid] : 0, we, wt;
  smp_scan(c, w, ce, we, ct, wt, s.sc, s.sw);
  // weights with the ties that stay
  we += min(ce, ties) * tie_w;
  w += (min(ce + c, ties) - min(ce, ties)) * tie_w;
  wt += min(ct, ties) * tie_w;
  const float uni = a.u[r];
  u64 goal = uni > 0.f ? (u64)(fmin((double)uni, 1.) * (double)wt) : 0;
  if (!(uni < 1.f) || goal >= wt) goal = wt - 1;  // (NaN too: the last kept)
  if (we <= goal && goal < we + w) s.bin = tid, s.cb = ce, s.wb = we;
  __syncthreads();
  if (wid) return;
  const int t0 = s.bin * tile, t1 = min(a.vocab, t0 + tile);
  uint32_t cb = s.cb;
  u64 wb = s.wb;
  for (int i0 = t0; i0 < t1; i0 += 64) {
    uint32_t tie = 0;
    u64 mine = i0 + lane < t1 ? weigh(i0 + lane, tie) : 0;
    const u64 tied = __ballot(tie);
    const uint32_t before = cb + __popcll(tied & ((1ull << lane) - 1));
    if (tie && before < ties) mine = tie_w;
    u64 run = mine;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const u64 up = __shfl_up(run, o, 64);
      if (lane >= o) run += up;
    }
    const u64 hit = __ballot(wb + run > goal);
    if (hit) {
      if (lane == 0) a.out[r] = i0 + __builtin_ctzll(hit);
      return;
    }
    cb += __popcll(tied);
    wb += (u64)__shfl(run, 63, 64);
  }
}
extern "C" __global__ __launch_bounds__(SMP_BLOCK) void nk_sample_bf16(SampleArgs a) { sample_body<bf16>(a); }
extern "C" __global__ __launch_bounds__(SMP_BLOCK) void nk_sample_f16(SampleArgs a) { sample_body<f16>(a); }
extern "C" __global__ __launch_bounds__(SMP_BLOCK) void nk_sample_f32(SampleArgs a) { sample_body<float>(a); }
