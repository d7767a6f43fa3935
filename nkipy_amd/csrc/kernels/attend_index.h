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
//
// This file is integer arithmetic alone: it compiles for the host as well, where
// NK_DEVICE, min, max and att_find are given.
#pragma once

#include <stdint.h>

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

// the sequence of row t of the batch and the row's place i in it; false for none
NK_DEVICE bool att_query(const AttendArgs &a, int t, int &b, AttSeq &s, int &i) {
  b = a.starts ? att_find(a.B, t, [&](int x) { return a.starts[x]; }) : t / a.S;
  if (b < 0) return false;
  s = att_seq(a, b);
  i = t - s.lo;
  return i >= 0 && i < s.n;  // (below 0: starts that decrease)
}

// Tiles of a packed batch: sequence b's begin at floor(starts[b] rep / ROWS) + b,
// which leaves room for ceil(n rep / ROWS) of them and needs no sum over the
// sequences before it.
NK_DEVICE int att_tile0(const AttendArgs &a, int b) {
  const int rep = a.Hq / a.Hkv;
  return (int)((int64_t)min(max(a.starts[b], 0), a.N) * rep / ATT_ROWS) + b;
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

// Workgroups run round-robin over the eight XCDs: with the KV head fastest, the
// tiles of one head (eight heads, or a multiple) share an XCD's cache.  The last
// tiles of a sequence, the longest without a window, go first; splits that only
// the longest sequences have come last, and so leave no CU with two workgroups
// while others have none (256 tokens behind 4000: 70 us with the splits of a tile
// side by side, 48 so).
struct AttWork {
  int g, split, b, tile;
};
template <bool PAGED>
NK_DEVICE AttWork att_work(const AttendArgs &a, int w) {
  AttWork k;
  const int rep = a.Hq / a.Hkv;
  k.g = w % a.Hkv;
  w /= a.Hkv;
  const int t = a.tiles - 1 - w % a.tiles;
  k.split = w / a.tiles;
  if (PAGED && a.starts) {
    k.b = att_find(a.B, t, [&](int x) { return att_tile0(a, x); });
    k.tile = k.b < 0 ? 0 : t - att_tile0(a, k.b);
  } else {
    const int per = (a.S * rep + ATT_ROWS - 1) / ATT_ROWS;
    k.b = t / per, k.tile = t % per;
  }
  return k;
}
// Workgroup w's work and its sequence; false where it has no rows.  (Starts that
// decrease find sequences whose first tile lies behind this one: none of theirs.)
template <bool PAGED>
NK_DEVICE bool att_tile(const AttendArgs &a, int w, AttWork &k, AttSeq &s) {
  k = att_work<PAGED>(a, w);
  if (k.b < 0 || k.tile < 0) return false;
  s = att_seq(a, k.b);
  return (int64_t)k.tile * ATT_ROWS < (int64_t)s.n * (a.Hq / a.Hkv);
}

}  // namespace nk
