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
// elements of each half of a pair (16 bytes with E = 8).  8000 tokens of 32 / 8
// heads of 128, bf16: 40 us, 5.0 TB/s, over inputs that change from call to call; 31
// over the same ones, which the last-level cache then holds in part.  In single
// elements (20 of 128 rotated) 120.
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
// 2^-36: sums of them are exact in 64 bits, so no order of additions or atomics
// changes a result, and what rounds to 0 (below 2^-37 of the largest, 7e-12)
// takes no part.  All three filters keep a beginning of the order (value
// descending, then index), so they come down to one border, the last (value,
// index) that stays, and the row is never sorted.
//
// Long rows take three launches, two of them over segments of the row, so that
// eight rows and more fill the chip (fewer stay on as many XCDs, one each: smp_place):
//   top    each segment's largest value, and those of its parts, some lanes' each;
//   hist   each segment's counts and weights over BINS equal steps of t, a bin's
//          both in one word (14 bits count up to 8192 tokens, 50 the weight), so
//          that a logit costs one LDS atomic, whose answer is its place among
//          the tokens in the order of their bins, which are written too.  A row
//          with top_k takes no histogram: the k-th of its parts' largest values
//          is not above the k-th value, and the segments list what is not below;
//   pick   one workgroup per row: the segments' histograms added, the bin in
//          which the count (top_k) or the weight (top_p) is reached, and the
//          values that matter listed in LDS: everything down to that bin, if
//          that is up to LIST values, and the border and the draw are searched
//          there; else that bin alone for the border, then the segment that holds
//          uniform x the kept weight, by the segments' sums.
// Rows of up to LIST tokens are one launch, read once: the list is the row, cut
// down to the bins that may be kept where those hold few (15 rows of 4546 with
// top_k and top_p 13 us, 29 with searches of the whole row).
//
// A list of up to FEW is ranked value against value.  Else a search (smp_select)
// finds where the running count or weight, in descending order of a key, reaches
// a goal: histograms of 1024 steps of what is left of the keys' range, until a
// step has up to a wave's elements, which it ranks, or is one key.  The key is
// the value for a border, the index for ties and for the draw.  A bin of more
// than LIST values (ties, a narrow spread) is searched in the row itself, and a
// top_k row whose lists overflow is read again by pick.
//
// Bound by the latency of one CU's steps in pick, by about 30 instructions per
// logit in hist, and by one read of the logits (top, hist, pick in us): 64 rows of
// 151936 bf16 with every filter 6, 11, 16, by nucleus alone 7, 20, 40; 17 rows of
// 128257 fp32 by nucleus 5, 12, 34; one row of 32000 with top_k 3, 8, 9.
// ---------------------------------------------------------------------------
struct SampleArgs {
  const void *x;
  const float *u;
  int32_t *out;
  const float *temp;     // per row; null: c_temp (likewise below)
  const int32_t *topk;
  const float *topp, *minp;
  uint64_t *tops;        // (rows, nseg): largest key and the complement of its index
  uint64_t *hist;        // (rows, nseg, BINS + 1): weight and count per bin, then the weight in all
  uint16_t *order;       // (rows, nseg, seg): a segment's tokens by bin, or a few of the largest
  uint16_t *places;      // (rows, nseg, BINS + 2): where each bin's begin, and the last one's end; or how many
  uint16_t *subs;        // (rows, nseg, sub): high halves of the keys of parts' largest values
  int64_t ld;            // elements from row to row
  double c_topp;         // 1: all (64 bits: the share that was given, where ties hold it exactly)
  int32_t rows, vocab, seg, nseg, sub;  // seg: tokens of a segment; sub: parts of one, at most 64
  float c_temp;
  int32_t c_topk;        // below 1: all
  float c_minp;          // 0: all
};

#define SMP_BLOCK 1024
#define SMP_SEG_BLOCK 256
#define SMP_BINS 512
#define SMP_LIST 8192
#define SMP_STEPS 1024
#define SMP_FEW 512
#define SMP_SEG_LIST 512
// copies of a bin, so that lanes of one wave meet less often; with four, 33 KB of
// LDS, one workgroup less fits a CU (64 rows of 151936: 27 us, 21 with two)
#define SMP_COPIES 2
#define SMP_SUBS 1024  // parts of a row at most
typedef unsigned long long u64;

// order of the values as whole numbers, of 16 bits for the 16-bit types; -0 and
// 0 tie
template <typename T> struct SmpKey {
  static NK_DEVICE uint32_t of(float x) {
    uint16_t h;
    T v;
    Elt<T>::store(&v, 0, x + 0.f);  // (exact: x is such a value)
    __builtin_memcpy(&h, &v, 2);
    return h & 0x8000u ? (uint16_t)~h : h | 0x8000u;
  }
  static NK_DEVICE float value(uint32_t k) {
    const uint16_t h = k & 0x8000u ? k & 0x7fffu : (uint16_t)~k;
    T v;
    __builtin_memcpy(&v, &h, 2);
    return Elt<T>::load(&v, 0);
  }
  static NK_DEVICE uint32_t high(uint32_t k) { return k; }
  static NK_DEVICE uint32_t from_high(uint32_t k) { return k; }
};
template <> struct SmpKey<float> {
  static NK_DEVICE uint32_t of(float x) {
    const uint32_t u = __float_as_uint(x + 0.f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
  }
  static NK_DEVICE float value(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }
  static NK_DEVICE uint32_t high(uint32_t k) { return k >> 16; }
  static NK_DEVICE uint32_t from_high(uint32_t k) { return k << 16; }
};

struct SmpRow {
  float best, c;  // largest logit, log2(e) / T
  NK_DEVICE void set(float b, float temp) {
    best = b;
    c = fminf(1.44269504088896340736f / temp, 3.4e38f);
  }
  // what is below this weighs nothing
  NK_DEVICE float floor() const { return fmaxf(best - 38.5f / c, -3.40282347e38f); }
  // log2 of the weight; the largest logit has 0 also where it is infinite
  NK_DEVICE float depth(float x) const { return x == best ? 0.f : (x - best) * c; }
};
// Weight in steps of 2^-36, as hi 2^18 + lo; 0 for NaN.  The hardware's 2^t is
// within an ulp, 1e-7 of the weight.
struct SmpWeight {
  uint32_t hi, lo;
  NK_DEVICE SmpWeight(float t) {
    const float p = t > -38.f ? __builtin_amdgcn_exp2f(t) * 0x1p18f : 0.f;
    hi = (uint32_t)p;
    lo = min((uint32_t)__builtin_fmaf(p - (float)hi, 0x1p18f, 0.5f), 0x3ffffu);  // (the difference is exact)
  }
  NK_DEVICE u64 sum() const { return ((u64)hi << 18) + lo; }
  NK_DEVICE u64 counted() const { return (u64)hi << 32 | lo << 14 | 1; }  // sum() 2^14 + 1
};
NK_DEVICE u64 smp_weight(float t) { return SmpWeight(t).sum(); }
// (a weight above 0 has t >= -37: bin 481 at most)
#define SMP_RATE 13.f  // bins per unit of t
NK_DEVICE int smp_bin(float t) { return min(SMP_BINS - 1, (int)(t * -SMP_RATE)); }

// Logits lo .. hi-1 of a row in pieces of 16 aligned bytes, U of a thread in
// flight at once: f(index, value) by THREADS threads.  The pieces at the ends
// are read element by element.
template <typename T, int THREADS, int U, typename F>
NK_DEVICE void smp_each(const T *x, int lo, int hi, F f) {
  constexpr int E = 16 / sizeof(T);
  const int off = (int)(((uintptr_t)(x + lo) & 15) / sizeof(T));  // elements of the first piece before lo
  for (int i0 = lo - off + threadIdx.x * E; i0 < hi; i0 += U * THREADS * E) {
    uint4 w[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u * THREADS * E;
      if (i >= lo && i + E <= hi) w[u] = *reinterpret_cast<const uint4 *>(x + i);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u * THREADS * E;
      if (i >= lo && i + E <= hi) {
        T v[E];
        __builtin_memcpy(v, &w[u], 16);
#pragma unroll
        for (int e = 0; e < E; ++e) f(i + e, Elt<T>::load(v, e));
      } else {
#pragma unroll 1
        for (int e = max(0, lo - i); e < min(E, hi - i); ++e) f(i + e, Elt<T>::load(x, i + e));
      }
    }
  }
}

// running sum over the lanes of a wave, this one's included: row shifts of 1, 2,
// 4, 8 lanes, then the rows' ends broadcast
template <int CTRL, int ROWS>
NK_DEVICE u64 smp_dpp(u64 v) {
  const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)v, CTRL, ROWS, 0xF, false);
  const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(v >> 32), CTRL, ROWS, 0xF, false);
  return (u64)hi << 32 | lo;
}
NK_DEVICE u64 smp_running(u64 v) {
  v += smp_dpp<0x111, 0xF>(v);
  v += smp_dpp<0x112, 0xF>(v);
  v += smp_dpp<0x114, 0xF>(v);
  v += smp_dpp<0x118, 0xF>(v);
  v += smp_dpp<0x142, 0xA>(v);
  v += smp_dpp<0x143, 0xC>(v);
  return v;
}
NK_DEVICE uint32_t smp_running(uint32_t v) {
  v += __builtin_amdgcn_update_dpp(0, (int)v, 0x111, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, (int)v, 0x112, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, (int)v, 0x114, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, (int)v, 0x118, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, (int)v, 0x142, 0xA, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, (int)v, 0x143, 0xC, 0xF, false);
  return v;
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
  v = smp_running(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 63) red[threadIdx.x >> 6] = v;
  __syncthreads();
  v = 0;
#pragma unroll
  for (int i = 0; i < WAVES; ++i) v += red[i];
  return v;
}
// largest value of a stretch and its lowest index, as one number; 0 where all
// are NaN or -inf; own(a thread's largest key)
template <typename T, int THREADS, typename F>
NK_DEVICE u64 smp_top(const T *x, int lo, int hi, u64 *red, F own) {
  float best = -INFINITY;
  int at = -1;
  smp_each<T, THREADS, 4>(x, lo, hi, [&](int i, float v) {  // (a thread's indices rise)
    if (v > best) best = v, at = i;
  });
  const u64 top = at < 0 ? 0 : (u64)SmpKey<T>::of(best) << 32 | (uint32_t)~at;
  own((uint32_t)(top >> 32));
  return smp_max<THREADS / 64>(top, red);
}

// The elements low <= v <= top of a stretch: their indices, those past LIMIT left
// out, and how many they are.  The two comparisons are all that an element costs.  A
// wave takes places for a few pieces of all its threads at once, with all reads in
// flight.
template <typename T, int THREADS, int LIMIT>
NK_DEVICE int smp_list(uint32_t *count, uint32_t *idx, const T *x, int lo, int hi, float low, float top) {
  constexpr int E = 16 / sizeof(T), U = 4;
  const int lane = threadIdx.x & 63;
  const int off = (int)(((uintptr_t)(x + lo) & 15) / sizeof(T));
  __syncthreads();
  if (threadIdx.x == 0) *count = 0;
  __syncthreads();
  auto fetch = [&](uint4 (&w)[U], int i0) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u * THREADS * E;
      if (i >= lo && i + E <= hi) w[u] = *reinterpret_cast<const uint4 *>(x + i);
    }
  };
  const int first = lo - off + (threadIdx.x - lane) * E;
  uint4 next[U];
  fetch(next, first + lane * E);
  // (every lane of a wave takes part in every round)
  for (int w0 = first; w0 < hi; w0 += U * THREADS * E) {
    const int i0 = w0 + lane * E;
    uint4 w[U];
    uint32_t in = 0;  // a bit for each of U E elements, the first the highest
#pragma unroll
    for (int u = 0; u < U; ++u) w[u] = next[u];
    fetch(next, i0 + U * THREADS * E);
    // (the middle of the three is y itself within the bounds, and not for NaN)
    auto inside = [&](float y) { return __builtin_amdgcn_fmed3f(y, low, top) == y; };
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u * THREADS * E;
      if (i >= lo && i + E <= hi) {
        T v[E];
        __builtin_memcpy(v, &w[u], 16);
#pragma unroll
        for (int e = 0; e < E; ++e) in += in + (inside(Elt<T>::load(v, e)) ? 1 : 0);
      } else {  // the ends, element by element
#pragma unroll 1
        for (int e = 0; e < E; ++e)
          in += in + (i + e >= lo && i + e < hi && inside(Elt<T>::load(x, max(lo, min(i + e, hi - 1)))) ? 1 : 0);
      }
    }
    if (!__any(in != 0)) continue;
    const uint32_t c = __popc(in), run = smp_running(c);
    uint32_t at = 0;
    if (lane == 63) at = atomicAdd(count, run);
    at = __builtin_amdgcn_readlane(at, 63) + run - c;
    for (; in; in &= in - 1, ++at) {
      const int bit = U * E - 1 - __builtin_ctz(in);
      if (at < LIMIT) idx[at] = i0 + bit / E * THREADS * E + bit % E;
    }
  }
  __syncthreads();
  return *count;
}

// Workgroup i runs on XCD i % 8: a row's segments go where the workgroup of its
// last launch reads the row again, so that it finds it in that XCD's cache.
// Grid: 8 nseg ceil(rows / 8).
NK_DEVICE void smp_place(const SampleArgs &a, int &r, int &s) {
  const int i = blockIdx.x >> 3;
  r = (i / a.nseg << 3) + (blockIdx.x & 7);
  s = i % a.nseg;
}
template <typename T>
__device__ __forceinline__ void sample_top_body(const SampleArgs &a) {
  __shared__ u64 red[SMP_SEG_BLOCK / 64];
  int r, s;
  smp_place(a, r, s);
  if (r >= a.rows) return;
  const u64 top = smp_top<T, SMP_SEG_BLOCK>((const T *)a.x + r * a.ld, s * a.seg, min(a.vocab, (s + 1) * a.seg), red,
                                            [&](uint32_t k) {
    k = SmpKey<T>::high(k);
    const int lanes = SMP_SEG_BLOCK / max(a.sub, SMP_SEG_BLOCK / 64);  // of a part
    for (int o = 1; o < lanes; o <<= 1) k = max(k, (uint32_t)__shfl_xor(k, o, 64));
    if (a.sub && threadIdx.x % lanes == 0) a.subs[((int64_t)r * a.nseg + s) * a.sub + threadIdx.x / lanes] = k;
  });
  if (threadIdx.x == 0) a.tops[(int64_t)r * a.nseg + s] = top;
}
template <int THREADS>
NK_DEVICE u64 smp_row_top(const SampleArgs &a, int r, u64 *red) {
  u64 top = 0;
  for (int i = threadIdx.x; i < a.nseg; i += THREADS) top = max(top, (u64)a.tops[(int64_t)r * a.nseg + i]);
  return smp_max<THREADS / 64>(top, red);
}
// its settings; false where there is nothing to weigh: no logit to draw, or no
// temperature
template <typename T>
NK_DEVICE bool smp_settings(const SampleArgs &a, int r, u64 top, SmpRow &row) {
  const float temp = a.temp ? a.temp[r] : a.c_temp;
  row.set(SmpKey<T>::value((uint32_t)(top >> 32)), temp);
  return top && temp > 0.f;
}

// The least key's high half that `need` parts of a row reach: as many values are
// not below it.  A wave's work; the keys in its lanes' registers.
NK_DEVICE uint32_t smp_reached(const SampleArgs &a, int r, int need) {
  const int lane = threadIdx.x & 63, n = a.nseg * a.sub;
  const uint16_t *p = a.subs + (int64_t)r * n;
  uint32_t k[SMP_SUBS / 64];
#pragma unroll
  for (int j = 0; j < SMP_SUBS / 64; ++j) k[j] = j * 64 + lane < n ? p[j * 64 + lane] : 0;
  uint32_t at = 0;
#pragma unroll 1
  for (uint32_t bit = 0x8000; bit; bit >>= 1) {
    int c = 0;
#pragma unroll
    for (int j = 0; j < SMP_SUBS / 64; ++j) c += __popcll(__ballot(k[j] >= (at | bit)));
    if (c >= need) at |= bit;
  }
  return at;
}
// Whether a row's top_k values are listed without a histogram: the parts' largest
// values bound them from below, closely while k is not near the parts' number.
NK_DEVICE bool smp_by_parts(const SampleArgs &a, int topk) {
  return topk > 0 && topk < a.vocab && topk <= a.nseg * a.sub * 3 / 4;
}
NK_DEVICE int smp_topk(const SampleArgs &a, int r) { return a.topk ? a.topk[r] : a.c_topk; }

// A segment's weights by bin (its histogram) to ho, its tokens in the order of
// their bins to `order`, where each bin begins to `places`.  The histogram's
// atomics return a token's place within its bin.
template <typename T>
NK_DEVICE void smp_segment(u64 (*bins)[SMP_COPIES], uint16_t *ord, u64 *red, const T *x, int n, const SmpRow &row, uint64_t *ho,
                           uint16_t *order, uint16_t *places) {
  constexpr int THREADS = SMP_SEG_BLOCK;
  static_assert(SMP_BINS == 2 * THREADS, "two bins of a thread");
  constexpr int E = 16 / sizeof(T), U = (SMP_LIST + E + THREADS * E - 1) / (THREADS * E);
  const int tid = threadIdx.x;
  __syncthreads();
  for (int i = tid; i < SMP_BINS * SMP_COPIES; i += THREADS) (&bins[0][0])[i] = 0;
  __syncthreads();
  const int off = (int)(((uintptr_t)x & 15) / sizeof(T)), i0 = tid * E - off;  // (as in smp_each)
  uint4 w[U];
  uint32_t at[U * E];  // bin and place
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int i = i0 + u * THREADS * E;
    if (i >= 0 && i + E <= n) {
      w[u] = *reinterpret_cast<const uint4 *>(x + i);
    } else if (i < n) {  // an end: element by element, -inf beyond
      u64 p[2] = {0, 0};
#pragma unroll 1
      for (int e = 0; e < E; ++e) {
        T v;
        Elt<T>::store(&v, 0, -INFINITY);
        if (i + e >= 0 && i + e < n) v = x[i + e];
        u64 bits = 0;
        __builtin_memcpy(&bits, &v, sizeof(T));
        p[0] = p[0] >> (8 * sizeof(T)) | p[1] << (64 - 8 * sizeof(T));
        p[1] = p[1] >> (8 * sizeof(T)) | bits << (64 - 8 * sizeof(T));
      }
      w[u] = make_uint4((uint32_t)p[0], (uint32_t)(p[0] >> 32), (uint32_t)p[1], (uint32_t)(p[1] >> 32));
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    T v[E];
    __builtin_memcpy(v, &w[u], 16);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const float t = row.depth(Elt<T>::load(v, e));
      const SmpWeight y(t);
      at[u * E + e] = ~0u;
      if ((y.hi | y.lo) && i0 + u * THREADS * E < n) {
        const int bin = smp_bin(t);
        at[u * E + e] = bin << 16 | ((uint32_t)atomicAdd(&bins[bin][tid % SMP_COPIES], y.counted()) & 0x3fff);
      }
    }
  }
  __syncthreads();
  // two bins of a thread: added up, then replaced by where their parts begin
  u64 all = 0;
  uint32_t c[2 * SMP_COPIES], mine = 0;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    u64 h = 0;
#pragma unroll
    for (int q = 0; q < SMP_COPIES; ++q) {
      const u64 y = bins[2 * tid + j][q];
      h += y;
      c[SMP_COPIES * j + q] = mine;
      mine += (uint32_t)y & 0x3fff;
    }
    all += h >> 14;
    ho[2 * tid + j] = h;
  }
  uint32_t run = smp_running(mine);
  all = smp_sum<THREADS / 64>(all, red);
  __syncthreads();
  if ((tid & 63) == 63) red[tid >> 6] = run;
  __syncthreads();
  run -= mine;
  uint32_t total = 0;
#pragma unroll
  for (int i = 0; i < THREADS / 64; ++i) {
    if (i < tid >> 6) run += (uint32_t)red[i];
    total += (uint32_t)red[i];
  }
#pragma unroll
  for (int q = 0; q < 2 * SMP_COPIES; ++q) bins[2 * tid + q / SMP_COPIES][q % SMP_COPIES] = run + c[q];
  places[2 * tid] = run, places[2 * tid + 1] = run + c[SMP_COPIES];
  if (tid == 0) ho[SMP_BINS] = all, places[SMP_BINS] = total;
  __syncthreads();
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const uint32_t k = at[u * E + e];
      if (k != ~0u) ord[(uint32_t)bins[k >> 16][tid % SMP_COPIES] + (k & 0xffff)] = i0 + u * THREADS * E + e;
    }
  __syncthreads();
  for (int i = tid; i < (int)total; i += THREADS) order[i] = ord[i];
}

template <typename T>
__device__ __forceinline__ void sample_hist_body(const SampleArgs &a) {
  __shared__ u64 bins[SMP_BINS][SMP_COPIES];
  __shared__ u64 red[SMP_SEG_BLOCK / 64];
  __shared__ uint16_t ord[SMP_LIST];
  __shared__ uint32_t count, reach;
  const int tid = threadIdx.x;
  int r, s;
  smp_place(a, r, s);
  if (r >= a.rows) return;
  SmpRow row;
  if (!smp_settings<T>(a, r, smp_row_top<SMP_SEG_BLOCK>(a, r, red), row)) return;
  const int lo = s * a.seg, n = min(a.vocab - lo, a.seg), topk = smp_topk(a, r);
  const T *x = (const T *)a.x + r * a.ld + lo;
  const int64_t at = (int64_t)r * a.nseg + s;
  uint64_t *ho = a.hist + at * (SMP_BINS + 1);
  uint16_t *order = a.order + at * a.seg, *places = a.places + at * (SMP_BINS + 2);
  if (smp_by_parts(a, topk)) {
    if (tid < 64) {
      const uint32_t k = smp_reached(a, r, topk);
      if (tid == 0) reach = k;
    }
    __syncthreads();
    // (a key past -inf's is a NaN, which fmaxf drops)
    const float low = fmaxf(row.floor(), SmpKey<T>::value(SmpKey<T>::from_high(reach)));
    const int c = smp_list<T, SMP_SEG_BLOCK, SMP_SEG_LIST>(&count, (uint32_t *)bins, x, 0, n, low, row.best);
    for (int i = tid; i < min(c, SMP_SEG_LIST); i += SMP_SEG_BLOCK) order[i] = ((uint32_t *)bins)[i];
    if (tid == 0) places[0] = c;
  } else if (a.topk || a.topp || a.minp || a.c_topk > 0 || a.c_topp < 1.0 || a.c_minp > 0.f) {
    smp_segment<T>(bins, ord, red, x, n, row, ho, order, places);
  } else {
    u64 all = 0;
    smp_each<T, SMP_SEG_BLOCK, 4>(x, 0, n, [&](int, float v) { all += smp_weight(row.depth(v)); });
    all = smp_sum<SMP_SEG_BLOCK / 64>(all, red);
    if (tid == 0) ho[SMP_BINS] = all;
  }
}

struct SmpShared {
  u64 hsum[SMP_BINS];      // the row's histogram
  u64 sum[SMP_STEPS];      // a search's
  uint32_t hcnt[SMP_BINS];
  uint32_t cnt[SMP_STEPS];
  uint32_t place[SMP_STEPS];
  u64 w[SMP_LIST];         // the list: weights, keys, indices
  uint32_t key[SMP_LIST], idx[SMP_LIST];
  u64 red[SMP_BLOCK / 64], sw[SMP_BLOCK / 64];
  uint32_t sc[SMP_BLOCK / 64];
  u64 cw[64];              // a search's last elements
  uint32_t ck[64];
  uint32_t n, few;
  uint32_t rkey, rties, rof;
  u64 rupto;
  // where a running sum reached its goal: step, and count and weight before and with it
  uint32_t bin, cb, ca;
  u64 wb, wa;
};

// Running sums of one count and weight per thread, on top of cb and wb: the
// first to reach `need` (COUNT) or `goal`.
template <bool COUNT>
NK_DEVICE void smp_search(SmpShared &s, uint32_t c, u64 w, uint32_t cb, u64 wb, uint32_t need, u64 goal) {
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
  uint32_t ci = smp_running(c);
  u64 wi = smp_running(w);
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

// where a search ended: the key, how many of its elements are in, how many there
// are, and the weight up to and with those in
struct SmpBorder {
  uint32_t key, ties, of;
  u64 upto;
};
// Of elements 0 .. n-1, key(i, k) says which take part, if weight(i) is not 0;
// their keys are in klo .. khi.  Those of one key weigh the same.
template <bool COUNT, typename K, typename W>
NK_DEVICE SmpBorder smp_select(SmpShared &s, int n, K key, W weight, uint32_t klo, uint32_t khi, uint32_t cb, u64 wb,
                               uint32_t need, u64 goal) {
  const int tid = threadIdx.x, lane = tid & 63;
  // a list stands nearly in the order of indices: neighbouring lanes take
  // elements apart, or they would meet in one step
  const int per = n <= SMP_LIST ? (n + SMP_BLOCK - 1) / SMP_BLOCK | 1 : 1, begin = tid * per;  // (odd: the lanes' banks)
  const int step = n <= SMP_LIST ? 1 : SMP_BLOCK, end = n <= SMP_LIST ? min(n, begin + per) : n;
  uint32_t k;
  SmpBorder b;
  while (true) {
    const uint32_t range = khi - klo;
    const int shift = range < SMP_STEPS ? 0 : 22 - __builtin_clz(range);
    __syncthreads();
    s.cnt[tid] = 0, s.sum[tid] = 0;
    if (tid == 0) s.few = 0;
    __syncthreads();
    for (int i = begin; i < end; i += step)
      if (key(i, k) && k >= klo && k <= khi) {
        const u64 w = weight(i);
        if (w) {
          atomicAdd(&s.cnt[(khi - k) >> shift], 1u);
          atomicAdd(&s.sum[(khi - k) >> shift], w);
        }
      }
    __syncthreads();
    smp_search<COUNT>(s, s.cnt[tid], s.sum[tid], cb, wb, need, goal);
    const uint32_t at = s.bin, left = s.ca - s.cb;
    cb = s.cb, wb = s.wb;
    if (shift == 0) {
      b.of = max(left, 1u);
      const u64 each = (s.wa - wb) / b.of;
      b.key = khi - at;
      b.ties = COUNT ? need - cb : (uint32_t)((goal - wb + each - 1) / max(each, (u64)1));
      b.upto = wb + b.ties * each;
      return b;
    }
    const uint32_t top = khi - (at << shift);
    klo = top - klo < (1u << shift) ? klo : top - (1u << shift) + 1;
    khi = top;
    if (left > 64) continue;
    // the rest by one wave
    for (int i = begin; i < end; i += step)
      if (key(i, k) && k >= klo && k <= khi) {
        const u64 w = weight(i);
        if (w) {
          const uint32_t to = atomicAdd(&s.few, 1u);
          if (to < 64) s.ck[to] = k, s.cw[to] = w;
        }
      }
    __syncthreads();
    if (tid < 64) {
      const bool in = lane < left;
      const uint32_t mk = in ? s.ck[lane] : 0;
      const u64 mw = in ? s.cw[lane] : 0;
      uint32_t c = cb, of = 0;
      u64 w = wb;
      for (int j = 0; j < left; ++j) {
        const uint32_t kj = __builtin_amdgcn_readlane(mk, j);
        if (kj > mk) ++c, w += s.cw[j];
        of += kj == mk;
      }
      if (in && (COUNT ? c < need && c + of >= need : w < goal && w + of * mw >= goal)) {  // (its ties agree)
        s.rkey = mk, s.rof = of;
        s.rties = COUNT ? need - c : (uint32_t)((goal - w + mw - 1) / mw);
        s.rupto = w + s.rties * mw;
      }
    }
    __syncthreads();
    b.key = s.rkey, b.ties = s.rties, b.of = s.rof, b.upto = s.rupto;
    return b;
  }
}

// The least key of a float for which f holds, if it holds for `top` and for every
// key above one it holds for; it should be above `out` and not above `in`.  Each
// lane of a wave tries a key of its own.
template <typename F>
NK_DEVICE uint32_t smp_least(uint32_t out, uint32_t in, uint32_t top, F f) {
  const int lane = threadIdx.x & 63;
  const u64 guess = __ballot(f(lane ? in : out));
  if (guess & 1 || out >= in) out = 0;
  if (!(guess & 2) || in > top) in = top;
  while (in - out > 1) {
    const uint32_t step = max((in - out) / 64, 1u), k = out + (lane + 1) * step;
    const u64 hit = __ballot(k < in && f(k));
    const uint32_t at = hit ? __builtin_ctzll(hit) : min(64u, (in - out - 1) / step);  // (lanes below `in`)
    if (hit) in = out + (at + 1) * step;
    out += at * step;
  }
  return in;
}
// the largest float below that of a key
NK_DEVICE float smp_below(uint32_t k) { return SmpKey<float>::value(k == 0x80000000u ? 0x7ffffffeu : k - 1); }
// those of a stretch with low <= v <= top, with keys and weights
template <typename T>
NK_DEVICE int smp_gather(SmpShared &s, const T *x, int lo, int hi, float low, float top, const SmpRow &row) {
  const int n = smp_list<T, SMP_BLOCK, SMP_LIST>(&s.n, s.idx, x, lo, hi, low, top);
#pragma unroll
  for (int j = 0; j < SMP_LIST / SMP_BLOCK; ++j) {
    const int i = j * SMP_BLOCK + threadIdx.x;
    if (i < n) {
      const float v = Elt<T>::load(x, s.idx[i]);
      s.key[i] = SmpKey<T>::of(v);
      s.w[i] = smp_weight(row.depth(v));
    }
  }
  __syncthreads();
  return n;
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
  constexpr int U = SMP_LIST / SMP_BLOCK;  // elements of a thread, all reads in flight
  T held_row[U];                           // (SMALL: the row)
  u64 top = 0;
  if (SMALL) {
#pragma unroll
    for (int j = 0; j < U; ++j) {
      const int i = j * SMP_BLOCK + tid;
      Elt<T>::store(&held_row[j], 0, -INFINITY);
      if (i < a.vocab) held_row[j] = x[i];
    }
#pragma unroll
    for (int j = 0; j < U; ++j) {
      const float f = Elt<T>::load(&held_row[j], 0);
      if (f > -INFINITY) top = max(top, (u64)SmpKey<T>::of(f) << 32 | (uint32_t)~(j * SMP_BLOCK + tid));
    }
    top = smp_max<SMP_BLOCK / 64>(top, s.red);
  } else {
    top = smp_row_top<SMP_BLOCK>(a, r, s.red);
  }
  SmpRow row;
  if (!smp_settings<T>(a, r, top, row)) {
    if (tid == 0) a.out[r] = top ? (int32_t)~(uint32_t)top : -1;
    return;
  }
  const int topk = smp_topk(a, r);
  const double topp = a.topp ? (double)a.topp[r] : a.c_topp;
  const float minp = a.minp ? a.minp[r] : a.c_minp;
  const bool by_k = topk > 0 && topk < a.vocab, by_p = topp < 1.0, by_m = minp > 0.f;
  const float tmin = by_m ? log2f(fminf(minp, 1.f)) : -INFINITY;  // the least depth that min_p keeps

  const uint64_t *hist = a.hist + (int64_t)r * a.nseg * (SMP_BINS + 1);
  // a value `at` bins below the largest, as a key: near there, and past every
  // value of a bin with a fiftieth of a bin to spare and a key on either side
  auto near = [&](float at) -> uint32_t {
    const float v = row.best - at / (SMP_RATE * row.c);
    return v > -3e38f ? SmpKey<float>::of(fminf(v, row.best)) : 0;
  };
  // the least float of bins up to `bin` that weighs anything, as its key: as the
  // arithmetic of the bins has it
  auto least = [&](int bin) -> uint32_t {
    return smp_least(near(bin + 1.02f), near(bin + 0.98f), SmpKey<float>::of(row.best), [&](uint32_t k) {
      const float t = row.depth(SmpKey<float>::value(k));
      const SmpWeight w(t);
      return (w.hi | w.lo) && smp_bin(t) <= bin;
    });
  };
  const bool cuts = by_k || by_p || by_m;
  bool whole = SMALL;  // the list holds all that may be kept
  u64 total = 0;       // weight of the row
  int n = 0;
  // Into the list: c tokens of segment `tid`, those from place `from` of its order on.
  auto pull = [&](uint32_t from, uint32_t c) __attribute__((always_inline)) {
    uint32_t run = smp_running(c);
    __syncthreads();
    if ((tid & 63) == 63) s.sc[tid >> 6] = run;
    __syncthreads();
    uint32_t all = 0;
#pragma unroll
    for (int i = 0; i < SMP_BLOCK / 64; ++i) {
      if (i < tid >> 6) run += s.sc[i];
      all += s.sc[i];
    }
    s.cnt[tid] = run - c;                      // its first place in the list
    s.place[tid] = from;                       // and that in its order
    __syncthreads();
    n = min((int)all, SMP_LIST);
    uint32_t at[U];  // a segment, the last that begins by this place; then the token
    T v[U];
#pragma unroll
    for (int j = 0; j < U; ++j) at[j] = 0;
#pragma unroll 1
    for (int step = SMP_STEPS / 2; step; step >>= 1) {
      if (step >= a.nseg) continue;
#pragma unroll
      for (int j = 0; j < U; ++j) {
        if (j * SMP_BLOCK >= n) continue;
        const int to = min((int)at[j] + step, a.nseg - 1);  // (past the last segment: the last)
        if (s.cnt[to] <= (uint32_t)(j * SMP_BLOCK + tid)) at[j] = to;
      }
    }
#pragma unroll
    for (int j = 0; j < U; ++j) {
      const int i = j * SMP_BLOCK + tid;
      if (i < n) {
        const uint32_t place = s.place[at[j]] + (i - s.cnt[at[j]]);
        at[j] = at[j] * a.seg + a.order[((int64_t)r * a.nseg + at[j]) * a.seg + place];
      }
    }
#pragma unroll
    for (int j = 0; j < U; ++j)
      if (j * SMP_BLOCK + tid < n) v[j] = x[at[j]];
#pragma unroll
    for (int j = 0; j < U; ++j) {
      const int i = j * SMP_BLOCK + tid;
      if (i < n) {
        const float f = Elt<T>::load(&v[j], 0);
        s.key[i] = SmpKey<T>::of(f), s.idx[i] = at[j], s.w[i] = smp_weight(row.depth(f));
      }
    }
    __syncthreads();
  };
  const uint16_t *places = a.places + ((int64_t)r * a.nseg + tid) * (SMP_BINS + 2);  // (where tid < nseg)
  const bool parts = !SMALL && smp_by_parts(a, topk);
  // the tokens of bins b0 .. b1; from the row where its segments have no order
  auto pull_bins = [&](int b0, int b1) __attribute__((always_inline)) {
    if (parts) {
      n = smp_gather(s, x, 0, a.vocab, SmpKey<float>::value(least(b1)), b0 ? smp_below(least(b0 - 1)) : row.best, row);
    } else {
      const uint32_t from = tid < a.nseg ? places[b0] : 0;
      pull(from, tid < a.nseg ? places[b1 + 1] - from : 0);
    }
  };
  auto clear_bins = [&]() {
    if (tid < SMP_BINS) s.hcnt[tid] = 0, s.hsum[tid] = 0;
    __syncthreads();
  };
  auto add_bin = [&](float t, u64 w) {
    const int bin = smp_bin(t);
    total += w;
    atomicAdd(&s.hcnt[bin], 1u);
    atomicAdd(&s.hsum[bin], w);
  };
  if (parts) {
    const uint32_t c = tid < a.nseg ? places[0] : 0;
    const u64 all = smp_sum<SMP_BLOCK / 64>((u64)(c > SMP_SEG_LIST) << 32 | c, s.red);
    whole = all <= SMP_LIST;
    if (whole) {
      pull(0, c);
    } else {  // many alike, or one segment has most: the row's histogram after all
      clear_bins();
      smp_each<T, SMP_BLOCK, 1>(x, 0, a.vocab, [&](int, float v) {
        const float t = row.depth(v);
        const u64 w = smp_weight(t);
        if (w) add_bin(t, w);
      });
      total = smp_sum<SMP_BLOCK / 64>(total, s.red);
    }
  }
  if (SMALL) {
    n = a.vocab;
#pragma unroll
    for (int j = 0; j < U; ++j) {
      const int i = j * SMP_BLOCK + tid;
      if (i < n) {
        const float f = Elt<T>::load(&held_row[j], 0);
        const u64 w = smp_weight(row.depth(f));
        s.key[i] = w ? SmpKey<T>::of(f) : 0, s.idx[i] = i, s.w[i] = w;  // (what weighs nothing, NaN too, comes last)
      }
    }
    __syncthreads();
  }
  // (a few listed values are ranked below, and need no bins)
  const bool ranked = (SMALL || parts) && whole && n <= SMP_FEW;
  if (whole && !ranked) {
    if (cuts) {
      clear_bins();
      for (int i = tid; i < n; i += SMP_BLOCK)
        if (s.w[i]) add_bin(row.depth(SmpKey<T>::value(s.key[i])), s.w[i]);
      total = smp_sum<SMP_BLOCK / 64>(total, s.red);  // (and the histogram is whole)
    }
  } else if (cuts && !whole && !parts) {
    uint32_t c = 0;
    u64 w = 0;
    const int bin = tid % SMP_BINS;
    for (int i0 = tid / SMP_BINS; i0 < a.nseg; i0 += 16) {  // (eight segments' loads at once)
      u64 h[8];
#pragma unroll
      for (int j = 0; j < 8; ++j)
        h[j] = hist[(int64_t)min(i0 + j * (SMP_BLOCK / SMP_BINS), a.nseg - 1) * (SMP_BINS + 1) + bin];
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (i0 + j * (SMP_BLOCK / SMP_BINS) < a.nseg) c += (uint32_t)h[j] & 0x3fff, w += h[j] >> 14;
    }
    if (tid < SMP_BINS) s.hcnt[bin] = c, s.hsum[bin] = w;
    __syncthreads();
    if (tid >= SMP_BINS) s.hcnt[bin] += c, s.hsum[bin] += w;
    total = smp_sum<SMP_BLOCK / 64>(w, s.red);  // (and the histogram is whole)
  }
  // the bin where the row's running count or weight gets there (s.bin; BINS: in none)
  auto bin_of_row = [&](bool count, uint32_t need, u64 goal) {
    const uint32_t c = tid < SMP_BINS ? s.hcnt[tid] : 0;
    const u64 w = tid < SMP_BINS ? s.hsum[tid] : 0;
    __syncthreads();
    if (tid == 0) s.bin = SMP_BINS;
    if (count) smp_search<true>(s, c, w, 0, 0, need, goal);
    else smp_search<false>(s, c, w, 0, 0, need, goal);
  };
  auto share = [&](u64 of) {  // whole steps: at least topp of it, at least one
    return min(max((u64)ceil(fmax(topp, 0.0) * (double)of), (u64)1), of);
  };
  bool k_cuts = by_k, p_cuts = by_p;
  if (cuts && !ranked) {
    int last = SMP_BINS - 1;  // bins up to here may be kept
    // the first border's bin; a top_k past the row's weights cuts nothing
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
    if (!whole && smp_sum<SMP_BLOCK / 64>(tid <= last ? s.hcnt[tid % SMP_BINS] : 0, s.red) <= SMP_LIST) {
      pull_bins(0, last);
      whole = true;
    }
    // a long list of which a few may be kept: those alone
    if (whole && n > SMP_FEW && smp_sum<SMP_BLOCK / 64>(tid <= last ? s.hcnt[tid % SMP_BINS] : 0, s.red) <= SMP_FEW) {
      if (tid == 0) s.n = 0;
      __syncthreads();
      for (int i = tid; i < n; i += SMP_BLOCK)
        if (s.w[i] && smp_bin(row.depth(SmpKey<T>::value(s.key[i]))) <= last) {
          const uint32_t at = atomicAdd(&s.n, 1u);
          s.cnt[at] = s.key[i], s.place[at] = s.idx[i];
        }
      __syncthreads();
      n = s.n;
      if (tid < n) s.key[tid] = s.cnt[tid], s.idx[tid] = s.place[tid];
      __syncthreads();
    }
  }
  // the draw: the first kept index up to and with which the weights exceed
  // uniform x their sum, that is, reach the whole number behind it
  const float uni = a.u[r];
  auto goal_of = [&](u64 all) {
    const u64 g = uni > 0.f ? (u64)(fmin((double)uni, 1.) * (double)all) : 0;
    return !(uni < 1.f) || g >= all ? all : g + 1;  // (NaN too: the last kept)
  };

  // A few values: ranked against each other, everything else is in their order.
  if (whole && n <= SMP_FEW) {
    static_assert(SMP_BLOCK == 2 * SMP_FEW, "two threads a value");
    const int e = tid >> 1, half = tid & 1;  // each half of the others
    const u64 mine = e < n ? (u64)s.key[e] << 32 | (uint32_t)~s.idx[e] : 0;
    if (e < n) s.sum[e] = mine;
    __syncthreads();
    uint32_t rank = 0;
    if (e < n) {
#pragma unroll 8
      for (int j = half; j < n; j += 2) rank += s.sum[j] > mine;
    }
    rank += __shfl_xor(rank, 1, 64);
    __syncthreads();
    if (e < n && !half) s.sum[rank] = mine;
    __syncthreads();
    const bool in = tid < n;
    const u64 it = in ? s.sum[tid] : 0;
    const float t = in ? row.depth(SmpKey<T>::value((uint32_t)(it >> 32))) : 0.f;
    const u64 w = in ? smp_weight(t) : 0;
    u64 run = smp_running(w);
    if ((tid & 63) == 63) s.sw[tid >> 6] = run;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < SMP_FEW / 64; ++i)
      if (i < tid >> 6) run += s.sw[i];
    uint32_t keep = k_cuts ? min(topk, n) : n;
    if (in) s.hsum[tid] = run;
    __syncthreads();
    if (p_cuts) {
      const u64 goal = share(k_cuts || ranked ? s.hsum[keep - 1] : total);
      keep = min(keep, 1 + (uint32_t)smp_sum<SMP_BLOCK / 64>(in && run < goal, s.red));
    }
    if (by_m) keep = min(keep, (uint32_t)smp_sum<SMP_BLOCK / 64>(in && t >= tmin, s.red));
    const u64 goal = goal_of(s.hsum[keep - 1]);
    __syncthreads();
    if (in) s.hsum[tid] = w;
    __syncthreads();
    if (e < keep) {
      const uint32_t at = (uint32_t)s.sum[e];
      u64 upto = 0;  // the weight of indices up to this one's (complements order them backwards)
#pragma unroll 8
      for (int j = half; j < keep; j += 2) upto += (uint32_t)s.sum[j] >= at ? s.hsum[j] : 0;
      upto += (u64)__shfl_xor(upto, 1, 64);
      if (!half && upto >= goal && upto - s.hsum[e] < goal) a.out[r] = ~at;
    }
    return;
  }

  // the border: the last (value, index) kept
  uint32_t bkey = 0, bidx = 0xffffffffu;
  int edge = SMP_BINS;  // its bin
  int held = -1;        // the bin whose values the list holds
  if (k_cuts || p_cuts) {
    SmpBorder b;
    // the values of the bin found last: from the list, or too many for it, from the row
    bool listing = whole;
    auto find = [&](auto count, uint32_t need, u64 goal) {
      constexpr bool COUNT = decltype(count)::value;
      const uint32_t cb = s.cb, many = s.ca - s.cb;
      const u64 wb = s.wb;
      edge = s.bin;
      if (!whole && edge != held) {
        listing = many <= SMP_LIST;
        held = listing ? edge : -1;
        if (listing) pull_bins(edge, edge);
      }
      const uint32_t low = near(edge + 1.02f), top = near(edge - 0.02f);
      const uint32_t klo = low ? max(SmpKey<T>::of(SmpKey<float>::value(low)), 1u) - 1 : 0;
      const uint32_t khi = SmpKey<T>::of(top ? SmpKey<float>::value(top) : row.best) + 1;
      if (listing) {
        b = smp_select<COUNT>(s, n, [&](int i, uint32_t &k) {
          k = s.key[i];
          return smp_bin(row.depth(SmpKey<T>::value(k))) == edge;
        }, [&](int i) { return s.w[i]; }, klo, khi, cb, wb, need, goal);
      } else {
        b = smp_select<COUNT>(s, a.vocab, [&](int i, uint32_t &k) {
          const float v = Elt<T>::load(x, i);
          k = SmpKey<T>::of(v);
          return smp_bin(row.depth(v)) == edge;
        }, [&](int i) { return smp_weight(row.depth(Elt<T>::load(x, i))); }, klo, khi, cb, wb, need, goal);
      }
    };
    if (k_cuts) find(SmpFlag<true>{}, topk, 0);
    if (p_cuts) {
      const u64 goal = share(k_cuts ? b.upto : total);
      bin_of_row(false, 0, goal);
      find(SmpFlag<false>{}, 0, goal);
    }
    bkey = b.key;
    // the highest index of its ties that stays: by count, lowest first
    if (b.ties < b.of) {
      const uint32_t klo = ~(uint32_t)(a.vocab - 1);
      auto one = [](int) -> u64 { return 1; };
      if (listing) {
        bidx = ~smp_select<true>(s, n, [&](int i, uint32_t &k) {
          k = ~s.idx[i];
          return s.key[i] == bkey;
        }, one, klo, ~0u, 0, 0, b.ties, 0).key;
      } else {
        bidx = ~smp_select<true>(s, a.vocab, [&](int i, uint32_t &k) {
          k = ~i;
          const float v = Elt<T>::load(x, i);
          return v == v && SmpKey<T>::of(v) == bkey;
        }, one, klo, ~0u, 0, 0, b.ties, 0).key;
      }
    }
  }
  auto kept = [&](uint32_t k, uint32_t i, float t) { return (k > bkey || (k == bkey && i <= bidx)) && t >= tmin; };

  // a listed element's weight, 0 where it is not kept
  auto weigh = [&](int i) -> u64 {
    return kept(s.key[i], s.idx[i], row.depth(SmpKey<T>::value(s.key[i]))) ? s.w[i] : 0;
  };
  auto draw = [&](u64 goal, u64 before, int lo, int hi) {
    const uint32_t at = ~smp_select<false>(s, n, [&](int i, uint32_t &k) {
      k = ~s.idx[i];
      return true;
    }, weigh, ~(uint32_t)(hi - 1), ~(uint32_t)lo, 0, before, 0, goal).key;
    if (tid == 0) a.out[r] = at;
  };
  if (whole) {
    u64 all = 0;
    for (int i = tid; i < n; i += SMP_BLOCK) all += weigh(i);
    draw(goal_of(smp_sum<SMP_BLOCK / 64>(all, s.red)), 0, 0, a.vocab);
    return;
  }
  // by segments: bins before the border's are kept whole; of the one it is in,
  // what is kept is added value by value
  if (by_m) edge = min(edge, smp_bin(tmin));
  u64 *seg = s.sum;  // (up to STEPS segments)
  __syncthreads();
  seg[tid] = 0;
  __syncthreads();
  if (edge == SMP_BINS && !parts) {
    for (int i = tid; i < a.nseg; i += SMP_BLOCK) seg[i] = hist[(int64_t)i * (SMP_BINS + 1) + SMP_BINS];
  } else {
    for (int i = tid >> 6; !parts && i < a.nseg; i += SMP_BLOCK / 64) {  // a wave for each
      u64 w = 0;
      for (int b = tid & 63; b < edge; b += 64) w += hist[(int64_t)i * (SMP_BINS + 1) + b] >> 14;
#pragma unroll
      for (int o = 32; o; o >>= 1) w += (u64)__shfl_xor(w, o, 64);
      if ((tid & 63) == 0) atomicAdd(&seg[i], w);
    }
    if (held == edge && !parts) {
      for (int i = tid; i < n; i += SMP_BLOCK) atomicAdd(&seg[s.idx[i] / a.seg], weigh(i));
    } else {
      smp_each<T, SMP_BLOCK, 4>(x, 0, a.vocab, [&](int i, float v) {
        const float t = row.depth(v);
        if (!(t > -38.f) || (!parts && smp_bin(t) != edge)) return;
        const u64 w = smp_weight(t);
        if (w && kept(SmpKey<T>::of(v), i, t)) atomicAdd(&seg[i / a.seg], w);
      });
    }
  }
  __syncthreads();
  const u64 mine = tid < a.nseg ? seg[tid] : 0;
  const u64 goal = goal_of(smp_sum<SMP_BLOCK / 64>(mine, s.red));
  smp_search<false>(s, 0, mine, 0, 0, 0, goal);
  const int at = s.bin;
  const u64 before = s.wb;
  n = min(a.vocab - at * a.seg, a.seg);  // the segment
  for (int i = tid; i < n; i += SMP_BLOCK) {
    const float f = Elt<T>::load(x, at * a.seg + i);
    s.key[i] = SmpKey<T>::of(f), s.idx[i] = at * a.seg + i, s.w[i] = smp_weight(row.depth(f));
  }
  __syncthreads();
  draw(goal, before, at * a.seg, min(a.vocab, (at + 1) * a.seg));
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
