// Attention of packed queries over a paged cache of e4m3 codes: tiles on matrix
// instructions (attend_index.h holds what a query sees and the layout of the work).

#include "attend8.h"

using namespace nk;

// ---------------------------------------------------------------------------
// 16-bit queries, head dim 64 or 128.  One workgroup of four waves per (tile of 128
// rows, KV head, split); a wave owns 32 rows.  S^T = K Q^T and O^T = V^T P^T by
// 32x32x16 products, so that a lane owns one row and the weights leave the first
// product in the order the second one takes them.
//
// The codes of a block of 32 keys go through registers, where a thread converts what
// it read into bf16 values once for all four waves, into two LDS slots each for K and
// V: iteration j has the scores of block j + 1, the values of block j - 1 and the
// softmax of block j, and stores K of block j + 2 and V of block j, with one barrier;
// what it stores was read in the iteration before.  The rows and scales of 16 blocks are
// looked up while the 16 before are worked on, in three steps four iterations apart,
// so that no read of them is waited for (each block's by one wave as it came: 326 us
// for 2100 tokens of 24 sequences of up to 6000, 263 so).  A key that is not seen by
// any row, or has no page, is read as some row: its scores are masked, and its scale
// of 2^-127 leaves nothing of its values (but for NaN codes: see below).
//
// Softmax: p = 2^(s c - m), c = scale log2(e), with an offset m per row that starts
// below any ordinary score and is raised (sums rescaled, block recomputed) when a
// lane's 16 weights of a block exceed LIMIT: the common block takes no maximum.  m
// divides out.  Under bf16 queries a weight is one bf16 number in the values and 32 bits
// in the sum that divides them.  Two numbers a weight, as single tokens have them, leave
// results off by their own rounding, 1.66e-3 of their norm, where one leaves 2.33e-3; but
// they cost a product of the values and the instructions of a second rounding more: 219
// us for 176 (2100 tokens of 24 sequences), 112 for 100 (2048 of 8, heads of 64).  The sum
// of the rounded weights below would cost 2 us and give 2.28e-3, but a result is then off
// by up to 2^-8 sum w |v - o|, up to twice the 2^-8 sum w |v| that it is off by so.
// Masks are applied only to blocks that some row does not see whole.
// Rows whose sums are not finite (a NaN value that other rows of the tile see), or
// whose offset is too large to cancel, are computed again at the end, a wave each.
// ---------------------------------------------------------------------------
#define ATT8_AHEAD 16  // blocks whose rows are looked up at once
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

// Workgroup w's work and its sequence; false where it has no rows.  The KV head
// fastest, as in att_work; the sequences of most keys first (up to 256 of them: a
// thread ranks each against all), a sequence's last tiles first, the second splits
// behind all first ones, so that the longest work begins first (2100 tokens of 24
// sequences of up to 6000: 324 us so, 382 in the order of the batch, both with the
// look-up of a wave).
NK_DEVICE bool att8_tile(const Attend8Args &a, int w, int32_t *lds, AttWork &k, AttSeq &s) {
  if (a.B > 256) return att_tile<true>(a, w, k, s);
  const int tid = threadIdx.x, lane = tid & 63, rep = a.Hq / a.Hkv;
  int32_t *const len = lds, *const count = lds + 256, *const which = lds + 512;
  int tiles = 0, mine = -1;
  if (tid < a.B) {
    s = att_seq(a, tid);
    tiles = (int)(((int64_t)s.n * rep + ATT_ROWS - 1) / ATT_ROWS);
    mine = s.len;
  }
  len[tid] = mine, count[tid] = 0;
  __syncthreads();
  int rank = 0;
  for (int x = 0; x < a.B; ++x) rank += len[x] > mine || (len[x] == mine && x < tid) ? 1 : 0;
  if (tid < a.B) count[rank] = tiles, which[rank] = tid;
  __syncthreads();
  k.g = w % a.Hkv;
  w /= a.Hkv;
  const int t = w % a.tiles;
  k.split = w / a.tiles;
  int before = 0;
  k.b = -1;
  for (int x = 0; x < a.B; x += 64) {
    const int c = count[x + lane];
    int upto = c;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int y = __shfl_up(upto, o, 64);
      upto += lane >= o ? y : 0;
    }
    const uint64_t past = __ballot(before + upto > t);
    if (past) {
      const int f = __builtin_ctzll(past);
      k.b = __builtin_amdgcn_readfirstlane(which[x + f]);
      k.tile = before + __builtin_amdgcn_readlane(upto, f) - 1 - t;
      break;
    }
    before += __builtin_amdgcn_readlane(upto, 63);
  }
  __syncthreads();  // (the memory has another use now)
  if (k.b < 0) return false;
  s = att_seq(a, k.b);
  return true;
}

template <typename T, int D>
__device__ __forceinline__ void attend8_tile_body(const Attend8Args &a) {
  constexpr int NP = Parts<T>::N;
  constexpr int RB = D * 2, TB = ATT_KEYS * RB;  // bytes of a row, of a block, as bf16
  constexpr int LPR = D / 16;                    // threads that read a key's codes
  constexpr bool BOTH = ATT_KEYS * LPR == 256;   // every thread reads keys and values (else half of them each)
  __shared__ __attribute__((aligned(1024))) uint8_t KR[2 * TB];
  __shared__ __attribute__((aligned(1024))) uint8_t VR[2 * TB];
  __shared__ __attribute__((aligned(16))) int32_t ent[2 * ATT8_AHEAD * ATT_KEYS];  // rows, below 0: none
  __shared__ uint16_t exps[2 * ATT8_AHEAD * ATT_KEYS];                            // exponents + 127, a key's below its value's
  __shared__ int32_t lost[2 * ATT8_AHEAD];                                        // some key of the block has no page

  static_assert(ATT8_AHEAD * ATT_KEYS == 512, "two keys of a thread");

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l32 = lane & 31, lhi = lane >> 5;
  const int rep = a.Hq / a.Hkv;

  att8_zero_rest<T>(a, blockIdx.x, a.tiles * a.Hkv * a.nsplit);
  AttWork wk;
  AttSeq sq;
  if (!att8_tile(a, blockIdx.x, reinterpret_cast<int32_t *>(KR), wk, sq)) return;
  // (one for the workgroup, in scalar registers: read behind stores, they came to vector ones)
  auto uniform = [](int x) __attribute__((always_inline)) { return __builtin_amdgcn_readfirstlane(x); };
  sq.lo = uniform(sq.lo), sq.n = uniform(sq.n), sq.len = uniform(sq.len), sq.p0 = uniform(sq.p0), sq.cap = uniform(sq.cap);
  const int g = wk.g, split = wk.split, b = uniform(wk.b), tile = uniform(wk.tile);
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

  // Looking up the rows of blocks 16 c ... in three steps: two keys' pages of a thread,
  // their exponents, and both to LDS.  (A row of -1: not seen, -2: no page.)
  // (Reads without a branch around them: in one, they would be waited for at its end.)
  int page_now[2], in_now[2], kexp_now[2], vexp_now[2];
  auto find_pages = [&](int c) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int x = tid + 256 * i, j = j0 + c * ATT8_AHEAD + x / ATT_KEYS, key = sp.kb(j) * ATT_KEYS + x % ATT_KEYS;
      const int y = (int)((uint32_t)key / (uint32_t)a.page);
      page_now[i] = a.tables[(int64_t)b * a.width + min(y, a.width - 1)];
      in_now[i] = j < j1 && key < sp.hi && (key >= sp.lo || key < a.sinks) ? key - y * a.page : -1;
    }
  };
  auto find_exps = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const bool is = page_now[i] >= 0 && page_now[i] < a.pages;
      const int64_t at = (int64_t)(is ? page_now[i] : 0) * a.Hkv + g;
      kexp_now[i] = a.ke[at];
      vexp_now[i] = a.ve[at];
      in_now[i] = in_now[i] < 0 ? -1 : is ? page_now[i] * a.pitch + in_now[i] : -2;
    }
  };
  auto put_rows = [&](int c) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int x = (c & 1) * ATT8_AHEAD * ATT_KEYS + tid + 256 * i;
      ent[x] = in_now[i];
      exps[x] = (uint16_t)(in_now[i] >= 0 ? (c8_clip(kexp_now[i]) + 127) | (c8_clip(vexp_now[i]) + 127) << 8 : 0);
      // (half a wave has a block's keys)
      const uint64_t gone = __ballot(in_now[i] == -2);
      if (l32 == 0) lost[x / ATT_KEYS] = (uint32_t)(gone >> (lane & 32)) != 0;
    }
  };

  // a thread's codes of a block: row rr, elements 16 cc ..., of K and V or of one of them
  const int rr = (BOTH ? tid : tid & 127) / LPR, cc = tid % LPR;
  const bool keys = BOTH || wave < 2;
  const uint8_t *const kp = (keys ? (const uint8_t *)a.k + (int64_t)g * a.k_sh : (const uint8_t *)a.v + (int64_t)g * a.v_sh);
  const uint8_t *const vp = (const uint8_t *)a.v + (int64_t)g * a.v_sh;
  const int64_t kss = keys ? a.k_ss : a.v_ss;
  struct Codes {
    uint4 w;
    float scale;
  };
  Codes ck, cv;
  // K of block jr + 2 and V of block jr: where they lie, then their codes
  int kat, vat;
  uint32_t kex, vex;
  int gone;  // whether some key of block jr has no page
  auto look = [&](int jr) __attribute__((always_inline)) {
    const int e = ((keys ? jr + 2 : jr) & (2 * ATT8_AHEAD - 1)) * ATT_KEYS + rr;
    kat = ent[e], kex = exps[e];
    if constexpr (BOTH) {
      const int f = (jr & (2 * ATT8_AHEAD - 1)) * ATT_KEYS + rr;
      vat = ent[f], vex = exps[f];
    }
    gone = lost[jr & (2 * ATT8_AHEAD - 1)];
  };
  auto fetch = [&]() __attribute__((always_inline)) {
    ck.scale = __uint_as_float((keys ? kex & 0xff : kex >> 8) << 23);
    ck.w = *reinterpret_cast<const uint4 *>(kp + (max(kat, 0) * kss + cc * 16));
    if constexpr (BOTH) {
      cv.scale = __uint_as_float((vex >> 8) << 23);
      cv.w = *reinterpret_cast<const uint4 *>(vp + (max(vat, 0) * a.v_ss + cc * 16));
    }
  };
  auto put = [&](const Codes &x, uint8_t *to, int swz) __attribute__((always_inline)) {
    *reinterpret_cast<B8 *>(to + rr * RB + (((2 * cc) ^ swz) << 4)) = codes8(x.w.x, x.w.y, x.scale);
    *reinterpret_cast<B8 *>(to + rr * RB + (((2 * cc + 1) ^ swz) << 4)) = codes8(x.w.z, x.w.w, x.scale);
  };
  // both go to slot jr & 1
  auto store_k = [&](int slot) __attribute__((always_inline)) { put(ck, (keys ? KR : VR) + slot * TB, keys ? kswz(rr) : vswz(rr)); };
  auto store_v = [&](int slot) __attribute__((always_inline)) {
    if constexpr (BOTH) put(cv, VR + slot * TB, vswz(rr));
  };

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
  auto read_k = [&](const uint8_t *K, int kk) __attribute__((always_inline)) {
    return *reinterpret_cast<const B8 *>(K + kbase + ((kk << 5) ^ kx));
  };
  auto read_v = [&](const uint8_t *Vt, int j, int dt) __attribute__((always_inline)) {
    s16x4 v[2];
#pragma unroll
    for (int si = 0; si < 2; ++si)
      v[si] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          (lds_s16x4 *)(Vt + (16 * j + 8 * si) * RB + vbase + ((dt << 6) ^ vx)));
    return __builtin_bit_cast(B8, __builtin_shufflevector(v[0], v[1], 0, 1, 2, 3, 4, 5, 6, 7));
  };
  // The scores of one block, the values of another and the weights of a third, in turns
  // (each product of the scores waits for the one before it; the weights, and what
  // `between` does, go on beside the products), with what a step reads on its way two
  // steps before.  Returns the sum of the weights 2^(s c - m).  2100 tokens of 24
  // sequences, us as traced: 265 with the weights behind all products and the codes
  // stored behind those, 240 with the weights in turns, 227 with the sequence's numbers
  // in scalar registers.  The codes' stores and reads in turns as well, at a raised
  // priority (of two workgroups' waves one is at its products then), took queued calls
  // from 198 to 173 .. 181; traced, launches of 199 to 228 (median 221).
  auto work = [&](const uint8_t *K, B8 k0, f32x16 &nxt, const uint8_t *Vt, B8 v0, const B8 (&prev)[2][NP],
                  const f32x16 &cur, B8 (&now)[2][NP], auto between) __attribute__((always_inline)) {
    constexpr int STEPS = D / 16, W = 16 / STEPS;
    float s0 = 0.f, s1 = 0.f;
    constexpr int DI = 2;
    B8 kf[DI + 1], vf[DI + 1];
    kf[0] = k0, vf[0] = v0, kf[1] = read_k(K, 1), vf[1] = read_v(Vt, 1 / (D / 32), 1 % (D / 32));
#pragma unroll
    for (int r = 0; r < 16; ++r) nxt[r] = 0.f;
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
      if (i + DI < STEPS) kf[(i + DI) % (DI + 1)] = read_k(K, i + DI), vf[(i + DI) % (DI + 1)] = read_v(Vt, (i + DI) / (D / 32), (i + DI) % (D / 32));
#pragma unroll
      for (int u = 0; u < NP; ++u) nxt = mul32(kf[i % (DI + 1)], qf[i][u], nxt);
#pragma unroll
      for (int u = 0; u < NP; ++u) acc[i % (D / 32)] = mul32(vf[i % (DI + 1)], prev[i / (D / 32)][u], acc[i % (D / 32)]);
#pragma unroll
      for (int e = i * W; e < i * W + W; ++e) {
        const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(cur[e], sl2, -m_run));
        if (e & 1) s1 += x; else s0 += x;
        put_weight<NP>(now[e / 8], e % 8, x);
      }
      between(i);
      __builtin_amdgcn_sched_barrier(0);
    }
    return s0 + s1;
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
  // What no row sees of block jr out of its scores; past the last block, all of it.
  // Element r of a lane is key 32 kb + 8 (r / 4) + 4 lhi + r % 4.
  auto mask = [&](f32x16 &s, int jr, bool missing) __attribute__((always_inline)) {
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

  f32x16 sA, sB;
  B8 pA[2][NP], pB[2][NP];
#pragma unroll
  for (int j = 0; j < 2; ++j)
#pragma unroll
    for (int e = 0; e < 8; ++e) put_weight<NP>(pB[j], e, 0.f);
  // Iteration jr, in slot i = jr & 1, one body for all: the values of the block before
  // (of zeros before the first), the scores of the one behind (of zeros past the last),
  // the softmax of this one.  The last, jr = n, adds the last block's values.
  // (waves without rows have a loop of their own, with the same barriers: one body would
  // branch around the products, and what is read in a branch is waited for at its end)
  auto step = [&](auto act, auto slot, int jr, f32x16 &cur, f32x16 &nxt, B8 (&prev)[2][NP],
                  B8 (&now)[2][NP]) __attribute__((always_inline)) {
    constexpr int I = decltype(slot)::value;
    if constexpr (decltype(act)::value) {
      // (the first products' factors before all else: what they wait for)
      const uint8_t *const K = KR + (I ^ 1) * TB, *const Vt = VR + (I ^ 1) * TB;
      const B8 k0 = read_k(K, 0), v0 = read_v(Vt, 0, 0);
      const bool missing = __builtin_amdgcn_readfirstlane(gone) != 0;
      look(jr + 1);
      const int key = sp.kb(j0 + jr) * ATT_KEYS;
      if (!(jr < n && key + ATT_KEYS - 1 <= sp.pa && key + ATT_KEYS <= sp.hi && (key > sp.pb - a.window || key + ATT_KEYS <= a.sinks) && !missing))
        mask(cur, jr, missing);  // (else every row sees the whole block)
      __builtin_amdgcn_s_setprio(1);
      const float ls = work(K, k0, nxt, Vt, v0, prev, cur, now, [&](int i) __attribute__((always_inline)) {
        constexpr int AT = D / 16 / 4;
        if (i == AT) store_k(I);
        if (i == AT + 1) store_v(I);
        if (i == AT + 1 + (D == 128)) fetch();
      });
      __builtin_amdgcn_s_setprio(0);
      raise(cur, now, ls);
    } else {
      look(jr + 1);
      store_k(I);
      store_v(I);
      fetch();
    }
    lds_barrier();
  };

  if (n > 0) {
    find_pages(0);
    find_exps();
    put_rows(0);
    in_now[0] = in_now[1] = -1;  // (what stands for the blocks before the first)
    put_rows(1);
    lds_barrier();
    // K of blocks 0 and 1; V of block -1 is zeros
    look(-2);
    fetch();
    if (keys) put(ck, KR, kswz(rr));
    look(-1);
    fetch();
    if (keys) put(ck, KR + TB, kswz(rr));
    if (BOTH || !keys) {
      const Codes none = {make_uint4(0, 0, 0, 0), 0.f};
      put(none, VR + TB, vswz(rr));
    }
    look(0);
    fetch();
    lds_barrier();
    if (active) {
#pragma unroll
      for (int r = 0; r < 16; ++r) sA[r] = 0.f;
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) qk1(KR, sA, kk);
    }
    lds_barrier();  // (block 0 is read before its slot is refilled)
    auto run = [&](auto act) __attribute__((always_inline)) {
      for (int jr = 0;; jr += 2) {
        // (the other half was last read an iteration, and a barrier, ago)
        if (jr % ATT8_AHEAD == 0) {
          find_pages(jr / ATT8_AHEAD + 1);
        } else if (jr % ATT8_AHEAD == 4) {
          find_exps();
        } else if (jr % ATT8_AHEAD == 8) {
          put_rows(jr / ATT8_AHEAD + 1);
        }
        step(act, Count<0>{}, jr, sA, sB, pB, pA);
        if (jr + 1 > n) break;
        step(act, Count<1>{}, jr + 1, sB, sA, pA, pB);
        if (jr + 2 > n) break;
      }
    };
    if (active) run(Count<1>{});
    else run(Count<0>{});
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
  const bool fine = row < rows && !(spoiled >> l32 & 1);
  if (fine && pieces == 1) {
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
  } else if (fine) {
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
NK_TILE8(f16, f16, 128, 1)
NK_TILE8(bf16, bf16, 64, 2)
NK_TILE8(f16, f16, 64, 2)
