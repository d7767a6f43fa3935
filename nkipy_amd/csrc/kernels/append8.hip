// Keys and values rotated and quantised into a paged cache of e4m3 codes.

#include "cache8.h"

using namespace nk;

// ---------------------------------------------------------------------------
// With row p of the tables for the token at position p, and one exponent e for
// the rows of a page and head:
//
//   y_i = x_i c_i - x_{i+r/2} s_i,  y_{i+r/2} = x_i s_i + x_{i+r/2} c_i,   i < r/2
//   code = e4m3(y 2^-e),  e the least with max |y| <= 448 2^e (and none below the
//   page's where rows written earlier stay)
//
// in fp32, every product and sum rounded by itself, so that the largest magnitude,
// and with it e, is what the same steps give anywhere.  Workgroups: one for the queries
// of a token or of four; one for each (page that a sequence writes, keys or values, some
// heads), as many as its threads can keep between the largest magnitude and the codes
// (large pages, odd sizes and heads rotated in part: read again, mostly from cache).
// Maxima are of whole numbers (bits), so no order changes them.  Bound by memory (8000
// tokens of 32 / 8 heads of 128, 184 MB: 40 us, 4.6 TB/s; the queries alone take 27, keys
// and values 16; in fp32, 344 MB, 70; with 64 of the 128 elements rotated, keys read
// twice, 63), single tokens by latency (8 of them: 4.5 us).
// ---------------------------------------------------------------------------
struct Append8Args {
  const void *q, *k, *v;
  void *oq;                // (N, Hq, D); null: left out
  uint8_t *kc, *vc;        // (pages, page, Hkv, D)
  int32_t *ke, *ve;        // (pages, Hkv)
  const float *cos, *sin;  // (P, half)
  const int32_t *tables, *lens, *starts;
  int64_t q_ss, q_sh, k_ss, k_sh, v_ss, v_sh;  // element strides of rows and heads
  int32_t B, N, Hq, Hkv, D, half, P;
  int32_t page, pages, width;
  int32_t heads;  // of a workgroup, up to A8_HEADS
  int32_t blocks;  // workgroups of keys and values
  int32_t qwaves;  // waves of a token's queries: 1 or 4
};
#define A8_HEADS 64
#define A8_ITEMS 4  // pairs of pieces that a thread keeps

// the sequence of token or tile t, by its first one: the last that begins at or before
template <typename F>
NK_DEVICE int a8_find(int n, int t, F f) {
  const int lane = threadIdx.x & 63;
  int c = 0;
  for (int b0 = 0; b0 < n; b0 += 64) c += __popcll(__ballot(b0 + lane < n && f(min(b0 + lane, n - 1)) <= t));
  return c - 1;
}
struct A8Seq {
  int lo, n, len;
};
NK_DEVICE A8Seq a8_seq(const Append8Args &a, int b) {
  A8Seq s;
  s.lo = b, s.n = 1;
  if (a.starts) {
    s.lo = min(max(a.starts[b], 0), a.N);
    s.n = min(max(a.starts[b + 1], s.lo), a.N) - s.lo;
  }
  s.len = min(max(a.lens[b], 0), 1 << 30);
  return s;
}
// Pages that a sequence writes are tiles floor(start / page) + 2 b ...: room for
// the n / page + 2 that n tokens may touch.
NK_DEVICE int a8_tile0(const Append8Args &a, int b) { return min(max(a.starts[b], 0), a.N) / a.page + 2 * b; }

// E elements of both halves of a piece, rotated
template <int E>
NK_DEVICE void a8_turn(const float (&x0)[E], const float (&x1)[E], const float (&c)[E], const float (&s)[E], float (&y0)[E],
                       float (&y1)[E]) {
#pragma clang fp contract(off)
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const float p0 = x0[e] * c[e], p1 = x1[e] * s[e], p2 = x0[e] * s[e], p3 = x1[e] * c[e];
    y0[e] = p0 - p1;
    y1[e] = p2 + p3;
  }
}
template <typename T, int E>
NK_DEVICE void a8_turn(const T *x, const float *cr, const float *sr, int half, float (&y0)[E], float (&y1)[E]) {
  float x0[E], x1[E], c[E], s[E];
  Piece<T, E>::load(x, x0);
  Piece<T, E>::load(x + half, x1);
  Piece<float, E>::load(cr, c);
  Piece<float, E>::load(sr, s);
  a8_turn<E>(x0, x1, c, s, y0, y1);
}

// The queries of a token, by `qwaves` waves; 4 / qwaves tokens to a workgroup.  Heads
// rotated as a whole, of a power of two of pieces: a lane keeps its place in the head
// and its angles, with A8_ITEMS heads on their way at once (8000 tokens of 32 / 8 heads
// of 128, keys and values with them: 42 us with a head at a time, 40 so).
template <typename T, int E>
__device__ __forceinline__ void append8_queries(const Append8Args &a, int blk) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int t = blk * (4 / a.qwaves) + wave / a.qwaves, place = wave % a.qwaves * 64 + lane, step = 64 * a.qwaves;
  if (t >= a.N) return;
  int b = t;
  if (a.starts) b = a8_find(a.B, t, [&](int x) { return a.starts[x]; });
  int p = -1;
  if (b >= 0) {
    const A8Seq s = a8_seq(a, b);
    if (t - s.lo < s.n) p = s.len - s.n + (t - s.lo);
  }
  const bool in = p >= 0 && p < a.P;
  const int turns = a.half / E, per = turns + (a.D - 2 * a.half) / E;
  const float *cr = a.cos + (int64_t)(in ? p : 0) * a.half, *sr = a.sin + (int64_t)(in ? p : 0) * a.half;
  const T *const q = (const T *)a.q + t * a.q_ss;
  T *const o = (T *)a.oq + (int64_t)t * a.Hq * a.D;
  if (E == 8 && in && per == turns && (turns & (turns - 1)) == 0 && turns <= 64) {
    const int d = place % turns * E, hs = step / turns;
    float c[E], s[E];
    Piece<float, E>::load(cr + d, c);
    Piece<float, E>::load(sr + d, s);
    for (int h0 = place / turns; h0 < a.Hq; h0 += A8_ITEMS * hs) {
      float x[A8_ITEMS][2][E];
#pragma unroll
      for (int i = 0; i < A8_ITEMS; ++i) {
        const T *src = q + min(h0 + i * hs, a.Hq - 1) * a.q_sh + d;
        Piece<T, E>::load(src, x[i][0]);
        Piece<T, E>::load(src + a.half, x[i][1]);
      }
#pragma unroll
      for (int i = 0; i < A8_ITEMS; ++i) {
        float y0[E], y1[E];
        if (h0 + i * hs >= a.Hq) break;
        a8_turn<E>(x[i][0], x[i][1], c, s, y0, y1);
        T *dst = o + (int64_t)(h0 + i * hs) * a.D + d;
        Piece<T, E>::store(dst, y0);
        Piece<T, E>::store(dst + a.half, y1);
      }
    }
    return;
  }
  for (int x = place; x < a.Hq * per; x += step) {
    const int h = x / per, c = x % per;
    const T *src = q + h * a.q_sh;
    T *dst = o + (int64_t)h * a.D;
    if (!in) {
      const float z[E] = {};
      const int d = c < turns ? c * E : 2 * a.half + (c - turns) * E;
      Piece<T, E>::store(dst + d, z);
      if (c < turns) Piece<T, E>::store(dst + a.half + d, z);
    } else if (c >= turns) {
      copy_piece<T, E>(src + 2 * a.half + (c - turns) * E, dst + 2 * a.half + (c - turns) * E);
    } else {
      float y0[E], y1[E];
      a8_turn<T, E>(src + c * E, cr + c * E, sr + c * E, a.half, y0, y1);
      Piece<T, E>::store(dst + c * E, y0);
      Piece<T, E>::store(dst + a.half + c * E, y1);
    }
  }
}

template <typename T, int E>
__device__ __forceinline__ void append8_body(const Append8Args &a) {
  __shared__ uint32_t top[A8_HEADS];
  __shared__ int32_t now[A8_HEADS], old[A8_HEADS];
  const int tid = threadIdx.x;
  // (keys and values first: they take longer)
  if ((int)blockIdx.x >= a.blocks) {
    append8_queries<T, E>(a, blockIdx.x - a.blocks);
    return;
  }
  const int parts = (a.Hkv + a.heads - 1) / a.heads;
  int w = blockIdx.x;
  const int h0 = w % parts * a.heads, hn = min(a.heads, a.Hkv - h0);
  w /= parts;
  const bool values = w & 1;
  const int t = w >> 1;
  int b = t, i = 0;
  if (a.starts) {
    b = a8_find(a.B, t, [&](int x) { return a8_tile0(a, x); });
    if (b < 0) return;
    i = t - a8_tile0(a, b);
  }
  const A8Seq s = a8_seq(a, b);
  const int p0 = s.len - s.n;              // of the first new token
  const int g = max(p0, 0) / a.page + i;   // page of the sequence
  if (i < 0 || g >= a.width) return;
  const int lo = max(g * a.page, max(p0, 0)), hi = min(min(g * a.page + a.page, s.len), a.P);  // positions written
  if (lo >= hi) return;
  const int pg = a.tables[(int64_t)b * a.width + g];
  if (pg < 0 || pg >= a.pages) return;
  const int first = lo - g * a.page, n = hi - lo;
  int32_t *const exps = (values ? a.ve : a.ke) + (int64_t)pg * a.Hkv + h0;
  uint8_t *const codes = (values ? a.vc : a.kc) + ((int64_t)pg * a.page * a.Hkv + h0) * a.D;
  const T *const src = values ? (const T *)a.v + (int64_t)(s.lo + lo - p0) * a.v_ss + h0 * a.v_sh
                              : (const T *)a.k + (int64_t)(s.lo + lo - p0) * a.k_ss + h0 * a.k_sh;
  const int64_t ss = values ? a.v_ss : a.k_ss, sh = values ? a.v_sh : a.k_sh;
  const int half = values ? 0 : a.half;
  const int turns = half / E, per = turns + (a.D - 2 * half) / E;

  if (tid < hn) top[tid] = 0, old[tid] = first ? c8_clip(exps[tid]) : C8_MIN;
  __syncthreads();
  auto larger = [&](uint32_t most, const float (&y)[E]) __attribute__((always_inline)) {
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const uint32_t u = __float_as_uint(y[e]) & 0x7fffffffu;
      most = u < 0x7f800000u ? max(most, u) : most;
    }
    return most;
  };
  auto settle = [&]() __attribute__((always_inline)) {  // the heads' exponents
    __syncthreads();
    if (tid < hn) {
      const int e = max(c8_exponent(__uint_as_float(top[tid])), old[tid]);
      now[tid] = e;
      exps[tid] = e;
    }
    __syncthreads();
  };
  if (E == 8 && n * hn * a.D <= 1024 * A8_ITEMS * 4 && a.D % 16 == 0 && (values || 2 * half == a.D)) {
    // read once: a thread's pairs of pieces, the same place of both halves of a head
    const int pc = a.D / 16, total = n * hn * pc;
    const bool side = (pc & (pc - 1)) == 0 && pc <= 64;  // a head's pieces lie with neighbouring lanes
    auto once = [&](auto count) __attribute__((always_inline)) {
      constexpr int I = decltype(count)::value;
      float y[I][2][E];
      int64_t at[I];
      int head[I];
#pragma unroll
      for (int i = 0; i < I; ++i) {
        const int x = min(tid + 256 * i, total - 1), r = x / (hn * pc), z = x % (hn * pc), h = z / pc, c = z % pc;
        const T *from = src + r * ss + h * sh + c * E;
        head[i] = h, at[i] = ((int64_t)(first + r) * a.Hkv + h) * a.D + c * E;
        if (values) {
          Piece<T, E>::load(from, y[i][0]);
          Piece<T, E>::load(from + a.D / 2, y[i][1]);
        } else {
          const int64_t turn = (int64_t)(lo + r) * half + c * E;
          a8_turn<T, E>(from, a.cos + turn, a.sin + turn, half, y[i][0], y[i][1]);
        }
      }
#pragma unroll
      for (int i = 0; i < I; ++i) {
        const bool is = tid + 256 * i < total;
        uint32_t most = is ? larger(larger(0, y[i][0]), y[i][1]) : 0;
        if (side) {
          for (int o = 1; o < pc; o <<= 1) most = max(most, (uint32_t)__shfl_xor(most, o, 64));
          if (tid % pc == 0 && most) atomicMax(&top[head[i]], most);
        } else if (most) {
          atomicMax(&top[head[i]], most);
        }
      }
      settle();
#pragma unroll
      for (int i = 0; i < I; ++i) {
        if (tid + 256 * i >= total) break;
        const float scale = c8_power(-now[head[i]]);
        c8_store<E>(codes + at[i], y[i][0], scale);
        c8_store<E>(codes + at[i] + a.D / 2, y[i][1], scale);
      }
    };
    if (total <= 256) {
      once(Count<1>{});
    } else {
      once(Count<A8_ITEMS>{});
    }
  } else {
    // every piece of these rows: f(row, head, first element, whether it is a pair, its values)
    auto each = [&](auto f) __attribute__((always_inline)) {
      for (int x = tid; x < n * hn * per; x += 256) {
        const int r = x / (hn * per), y = x % (hn * per), h = y / per, c = y % per;
        const T *from = src + r * ss + h * sh;
        float y0[E], y1[E];
        if (c < turns) {
          const int64_t at = (int64_t)(lo + r) * half + c * E;
          a8_turn<T, E>(from + c * E, a.cos + at, a.sin + at, half, y0, y1);
          f(r, h, c * E, true, y0, y1);
        } else {
          const int d = 2 * half + (c - turns) * E;
          Piece<T, E>::load(from + d, y0);
          f(r, h, d, false, y0, y0);
        }
      }
    };
    each([&](int, int h, int, bool, const float (&y0)[E], const float (&y1)[E]) __attribute__((always_inline)) {
      const uint32_t most = larger(larger(0, y0), y1);
      if (most) atomicMax(&top[h], most);
    });
    settle();
    each([&](int r, int h, int d, bool pair, const float (&y0)[E], const float (&y1)[E]) __attribute__((always_inline)) {
      const float scale = c8_power(-now[h]);
      uint8_t *to = codes + ((int64_t)(first + r) * a.Hkv + h) * a.D + d;
      c8_store<E>(to, y0, scale);
      if (pair) c8_store<E>(to + half, y1, scale);
    });
  }
  // the rows before, where the scale grew
  for (int h = 0; h < hn && first; ++h) {
    const int by = old[h] - now[h];
    if (by == 0) continue;
    const float scale = c8_power(max(by, -126));
    for (int x = tid; x < first * (a.D / E); x += 256) {
      uint8_t *at = codes + ((int64_t)(x / (a.D / E)) * a.Hkv + h) * a.D + x % (a.D / E) * E;
      float y[E];
      c8_load<E>(at, y);
      c8_store<E>(at, y, scale);
    }
  }
}
#define NK_APPEND8(T, name)                                                                                       \
  extern "C" __global__ __launch_bounds__(256) void nk_append8_##name(Append8Args a) { append8_body<T, 8>(a); }   \
  extern "C" __global__ __launch_bounds__(256) void nk_append81_##name(Append8Args a) { append8_body<T, 1>(a); }
NK_APPEND8(bf16, bf16)
NK_APPEND8(f16, f16)
NK_APPEND8(float, f32)
