// Attention of queries at known positions to keys in a paged cache or in
// plain tensors, with a sliding window and visible first tokens: arguments,
// the sequences of a packed batch and the keys that a tile of queries sees.
//
//   o = sum_j p_j v_j / sum_j p_j,   p_j = exp(scale q . k_j - m),
//   over the keys j <= p with p - j < window or j < sinks, j below the
//   sequence's length and (paged) on a page of the cache.
//
// Rows: the queries of one sequence and KV head, heads fastest:
// row = token * rep + head within the group.  A tile is ATT_ROWS rows: its
// queries share the keys, so one pass over them serves the whole group, and
// few tokens span few positions, which keeps the masked blocks few.
#pragma once

#include "common.h"

#define ATT_ROWS 128  // rows per tile
#define ATT_KEYS 32   // keys per block

struct AttendArgs {
  const void *q, *k, *v;
  void *o;                 // (N, Hq, D), contiguous
  const int32_t *tables;   // (B, width) page numbers; null: plain tensors
  const int32_t *lens;     // (B,) tokens (plain: keys) of a sequence; null: T
  const int32_t *starts;   // (B + 1,) first row of each sequence; null: S rows each
  const int32_t *first;    // (B,) position of a sequence's first query (plain); null: T - S
  float *ws;               // splits: (nsplit, N, Hq, D) sums, then (nsplit, N, Hq, 2) offset and weight
  const void *zeros;       // one row of zeros
  int64_t q_sb, q_ss, q_sh;  // element strides: sequence (plain), row, head
  int64_t k_sb, k_ss, k_sh;
  int64_t v_sb, v_ss, v_sh;
  int32_t B, S, N, T;        // sequences, rows per sequence (no starts), rows in all, keys (plain)
  int32_t Hq, Hkv, D;
  int32_t page, pages, width, pitch;  // pitch: rows from one page to the next
  int32_t window, sinks;     // window 2^30: none
  int32_t nsplit, min_blocks, tiles;  // tiles per KV head
  float scale;
};

namespace nk {

struct AttSeq {
  int lo, n;   // first row in the batch, rows
  int p0;      // position of row lo
  int len;     // tokens: queries at or past it see nothing
  int cap;     // keys that have a place
};

// (a start or length out of its range counts as the nearest end: every access
// stays inside the tensors whatever the arrays hold)
NK_DEVICE AttSeq att_seq(const AttendArgs &a, int b) {
  AttSeq s;
  if (a.tables) {
    s.lo = b, s.n = 1;
    if (a.starts) {
      s.lo = min(max(a.starts[b], 0), a.N);
      s.n = min(max(a.starts[b + 1], s.lo), a.N) - s.lo;
    }
    s.len = min(max(a.lens[b], 0), 1 << 30);
    s.p0 = s.len - s.n;
    s.cap = min(s.len, a.width * a.page);
  } else {
    s.lo = b * a.S, s.n = a.S;
    s.len = a.lens ? min(max(a.lens[b], 0), a.T) : a.T;
    s.p0 = a.first ? min(max(a.first[b], -(1 << 30)), 1 << 30) : a.T - a.S;
    s.cap = s.len;
  }
  return s;
}

// Tiles of a packed batch: sequence b's begin at floor(starts[b] rep / ROWS) + b,
// which leaves room for ceil(n rep / ROWS) of them and needs no sum over the
// sequences before it.
NK_DEVICE int att_tile0(const AttendArgs &a, int b) {
  const int rep = a.Hq / a.Hkv;
  return (int)((int64_t)min(max(a.starts[b], 0), a.N) * rep / ATT_ROWS) + b;
}

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

// Blocks of ATT_KEYS keys that the rows of one tile see: block j is keys
// 32 kb(j) ...: the sinks' blocks first, then those of the window.
struct AttSpan {
  int pa, pb;      // positions of the first and last query that sees anything
  int lo, hi;      // keys lo .. hi-1 (and the sinks) are seen by some query
  int ns, shift;   // block j < ns is block j of the sequence, else j + shift
  int nb;          // blocks
  NK_DEVICE int kb(int j) const { return j < ns ? j : j + shift; }
};

NK_DEVICE AttSpan att_span(const AttendArgs &a, const AttSeq &s, int tile) {
  const int rep = a.Hq / a.Hkv;
  AttSpan t;
  const int i0 = tile * ATT_ROWS / rep, i1 = min(s.n - 1, (tile * ATT_ROWS + ATT_ROWS - 1) / rep);
  t.pa = max(s.p0 + i0, 0);
  t.pb = min(s.p0 + i1, s.len - 1);
  t.lo = t.hi = t.ns = t.shift = t.nb = 0;
  if (i0 >= s.n || t.pb < t.pa) return t;
  t.hi = min(t.pb + 1, s.cap);
  t.lo = max(0, t.pa - a.window + 1);
  const int ns = (min(min(a.sinks, t.lo), t.hi) + ATT_KEYS - 1) / ATT_KEYS;
  const int b0 = t.lo / ATT_KEYS, b1 = (t.hi + ATT_KEYS - 1) / ATT_KEYS;
  t.ns = min(ns, b0);
  t.shift = b0 - t.ns;
  t.nb = t.ns + max(0, b1 - b0);
  return t;
}

// the part of a tile's blocks that split s takes: a multiple of min_blocks, so few
// splits of a short sequence have any; returns their number
NK_DEVICE int att_split(const AttendArgs &a, int nb, int s, int &j0, int &j1) {
  const int per = max((nb + a.nsplit * a.min_blocks - 1) / (a.nsplit * a.min_blocks), 1) * a.min_blocks;
  j0 = min(s * per, nb);
  j1 = min(j0 + per, nb);
  return max(1, (nb + per - 1) / per);
}

NK_DEVICE bool att_sees(const AttendArgs &a, const AttSeq &s, int p, int key) {
  return key <= p && p < s.len && key < s.cap && (p - key < a.window || key < a.sinks);
}

// row of the cache (or tensor) that holds a key of sequence b; -1: none
NK_DEVICE int att_place(const AttendArgs &a, int b, int key) {
  if (!a.tables) return key;
  const int pg = a.tables[(int64_t)b * a.width + key / a.page];
  return pg >= 0 && pg < a.pages ? pg * a.pitch + key % a.page : -1;
}

// One query row by one wave, over blocks j0 .. j1-1 of its tile's span: eight
// lanes share a key's product, 64 keys a step; then the lanes share the head's
// elements, d = lane + 64 e.  Only the keys that the row sees are read.
template <typename T>
NK_DEVICE void att_row(const AttendArgs &a, const AttSeq &sq, const AttSpan &sp, int b, int i, int h, int j0, int j1,
                       float &m, float &l, float (&acc)[4]) {
  const int lane = threadIdx.x & 63, c = lane & 7;
  const int g = h / (a.Hq / a.Hkv), p = sq.p0 + i, per = (a.D + 7) / 8;
  const int64_t qrow = a.tables ? (int64_t)(sq.lo + i) * a.q_ss : (int64_t)b * a.q_sb + (int64_t)i * a.q_ss;
  const T *q = (const T *)a.q + qrow + (int64_t)h * a.q_sh;
  const T *k = (const T *)a.k + (a.tables ? 0 : (int64_t)b * a.k_sb) + (int64_t)g * a.k_sh;
  const T *v = (const T *)a.v + (a.tables ? 0 : (int64_t)b * a.v_sb) + (int64_t)g * a.v_sh;
  float qc[32];
#pragma unroll
  for (int e = 0; e < 32; ++e) {
    const int d = c * per + e;
    qc[e] = e < per && d < a.D ? Elt<T>::load(q, d) * a.scale : 0.f;
  }
  m = -INFINITY, l = 0.f;
#pragma unroll
  for (int e = 0; e < 4; ++e) acc[e] = 0.f;
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
        for (int e = 0; e < 32; ++e)
          if (e < per && c * per + e < a.D) d = fmaf(qc[e], Elt<T>::load(kr, c * per + e), d);
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
    for (int e = 0; e < 4; ++e) acc[e] *= alpha;
    while (todo) {
      const int n = __builtin_ctzll(todo);
      todo &= todo - 1;
      const float wn = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(w), n));
      const T *vr = v + (int64_t)__builtin_amdgcn_readlane(row, n) * a.v_ss;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (lane + 64 * e < a.D) acc[e] = fmaf(wn, Elt<T>::load(vr, lane + 64 * e), acc[e]);
    }
  }
}

}  // namespace nk
