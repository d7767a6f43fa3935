// Attention over a paged cache or plain tensors with a window and sinks
// (attend_index.h holds the definition and the layout of the work).

#include "attend.h"

using namespace nk;

// ---------------------------------------------------------------------------
// Any head dim to 256, any strides and addresses, fp32 operands: one wave per
// query row.  It reads each key for each query head apart and uses no matrix
// instructions; the 16-bit types of head dims 64 and 128 have the tiled form.  64
// sequences of up to 8192 tokens, 32 / 8 heads: 8.1 ms with 80 bf16, 11.1 with 128
// fp32, 21.2 with 256 bf16; one prompt of 1000: 2.24 ms with 80 bf16, 4.2 with 128 fp32.
// ---------------------------------------------------------------------------
template <typename T>
__device__ __forceinline__ void attend_rows_body(const AttendArgs &a) {
  const int lane = threadIdx.x & 63;
  const int64_t r = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (r >= (int64_t)a.N * a.Hq) return;
  const int t = (int)(r / a.Hq), h = (int)(r % a.Hq);
  int b, i;
  AttSeq sq;
  float m, l = 0.f, acc[4];
  if (att_query(a, t, b, sq, i)) {
    const AttSpan sp = att_span(a, sq, (i * (a.Hq / a.Hkv) + h % (a.Hq / a.Hkv)) / ATT_ROWS);
    att_row<T, false>(a, sq, sp, b, i, h, 0, sp.nb, m, l, acc);
    float z = 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) z = fmaf(acc[e], 0.f, z);
    if (__any(z != 0.f)) att_row<T, true>(a, sq, sp, b, i, h, 0, sp.nb, m, l, acc);
  }
  T *o = (T *)a.o + r * a.D;
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (lane + 64 * e < a.D) Elt<T>::store(o, lane + 64 * e, l == 0.f ? 0.f : acc[e] / l);
}
extern "C" __global__ __launch_bounds__(256) void nk_attend_rows_bf16(AttendArgs a) { attend_rows_body<bf16>(a); }
extern "C" __global__ __launch_bounds__(256) void nk_attend_rows_f16(AttendArgs a) { attend_rows_body<f16>(a); }
extern "C" __global__ __launch_bounds__(256) void nk_attend_rows_f32(AttendArgs a) { attend_rows_body<float>(a); }

// ---------------------------------------------------------------------------
// The tiled form: 16-bit operands, head dim 64 or 128, 16-byte aligned rows.
//
// One workgroup of four waves per (tile of 128 rows, KV head, split); a wave
// owns 32 rows.  S^T = K Q^T and O^T = V^T P^T by 32x32x16 matrix
// instructions, so that a lane owns one row: its softmax offset and sum stay
// in its own registers (the two lanes that hold a row meet at the end), and the
// weights leave the first product in the order the second one takes them.
//
// Keys move in blocks of 32 through rings of four LDS slots each for K and V,
// by loads straight into LDS; iteration j has the scores of block j + 1, the
// values of block j - 1 and the softmax of block j in one basic block, and
// moves K of block j + 4 and V of block j + 2 into the slots freed before it: one
// barrier per block, three iterations for a move to land.  A key's row is
// looked up once per workgroup: the rows of 32 blocks ahead stand in LDS, -1
// where no query of the tile sees the key or it has no page.  Those rows are
// zeros in LDS, so nothing of them enters a product; a value that is
// not finite and seen by some rows of a tile only would still meet the others'
// weights of 0, and the rows it spoils are computed again one by one.
//
// Scores of blocks that some row does not see in full (the diagonal, the window's
// end, the sinks' last block, missing pages) are masked ahead of that body, which
// is one for all blocks.
//
// Softmax: p = 2^(s c - m), c = scale log2(e), with an offset m per row that
// starts TOP below the first block's largest score and is raised (sums
// rescaled, block recomputed) when a lane's 16 weights of a block exceed LIMIT:
// the common block takes no maximum.  m divides out.  Sums are fp32; weights
// enter the second product rounded to the operands' type, the one rounding
// beside the result's own.  f16 weights start at 2^10 and stay below 2^14,
// which leaves 2^34 between the largest and the least one that is kept.
// ---------------------------------------------------------------------------
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

template <typename T> struct Mat;
template <> struct Mat<bf16> {
  typedef __bf16 E;
  typedef __bf16 V __attribute__((ext_vector_type(8)));
  static constexpr float LIMIT = 65536.f, TOP = 0.f;
  static NK_DEVICE f32x16 mul(V a, V b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
};
template <> struct Mat<f16> {
  typedef _Float16 E;
  typedef _Float16 V __attribute__((ext_vector_type(8)));
  static constexpr float LIMIT = 16384.f, TOP = 10.f;
  static NK_DEVICE f32x16 mul(V a, V b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
};
#define ATT_LOWEST -3.40282347e38f  // the least finite offset
template <int N> struct Slot {
  static constexpr int value = N;
};

// lane l of the wave fills LDS bytes lds + 16 l (lds uniform) from p; waits
// for these moves are explicit
NK_DEVICE void move16(const void *p, uint32_t lds) {
  const uint32_t m = __builtin_amdgcn_readfirstlane(lds);
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off"
               :: "v"((uint64_t)p), "s"(m) : "memory", "m0");
}

#define ATT_AHEAD 32  // blocks whose rows are looked up at once
// offset of a row that is not there: past the end of any buffer resource, also
// with a place in a row added
#define ATT_NOWHERE 0xfffff000u

// rows outside every sequence: zeros, shared out over the grid
template <typename T>
NK_DEVICE void att_zero_rest(const AttendArgs &a, int wg, int nwg) {
  const int s0 = min(max(a.starts[0], 0), a.N), s1 = min(max(a.starts[a.B], s0), a.N);
  const int n = a.Hq * a.D;
  for (int x = wg; x < s0 + a.N - s1; x += nwg) {
    T *o = (T *)a.o + (int64_t)(x < s0 ? x : x - s0 + s1) * n;
    for (int e = threadIdx.x; e < n; e += 256) o[e] = T{};
  }
}

// FAR: keys or values over 4 GiB, or keys and values of different row strides in
// one cache: 64-bit addresses, and a row of zeros for what has no use.  Else offsets
// into a buffer resource, past whose end a move writes zeros.
template <typename T, int D, bool PAGED, bool FAR>
__device__ __forceinline__ void attend_tile_body(const AttendArgs &a) {
  typedef typename Mat<T>::V V8;
  constexpr int RB = D * 2, TB = ATT_KEYS * RB;  // bytes of a row, of a block
  constexpr int LPR = RB / 16, RPM = 64 / LPR;   // lanes per row, rows per move
  constexpr int NM = ATT_KEYS / RPM / 4;         // moves per wave and block
  __shared__ __attribute__((aligned(1024))) uint8_t KR[4 * TB];
  __shared__ __attribute__((aligned(1024))) uint8_t VR[4 * TB];
  __shared__ __attribute__((aligned(16))) int32_t ent[PAGED ? 2 * ATT_AHEAD * ATT_KEYS : 4];
  __shared__ int32_t lost[8];  // per half of ent and wave: some key has no page

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l32 = lane & 31, lhi = lane >> 5;
  const int rep = a.Hq / a.Hkv;

  if (PAGED && a.starts) att_zero_rest<T>(a, blockIdx.x, a.tiles * a.Hkv * a.nsplit);
  AttWork wk;
  AttSeq sq;
  if (!att_tile<PAGED>(a, blockIdx.x, wk, sq)) return;
  const int g = wk.g, split = wk.split, b = wk.b, tile = wk.tile;
  const AttSpan sp = att_span(a, sq, tile);
  int j0, j1;
  const int pieces = att_split(a, sp.nb, split, j0, j1);
  if (split >= pieces) return;
  const int n = j1 - j0;  // blocks of this workgroup

  // this lane's row
  const int row0 = tile * ATT_ROWS + wave * 32, rows = sq.n * rep;
  const bool active = row0 < rows;
  V8 qf[D / 16];
  int p, klim;  // its position and last key
  {
    const int rld = min(row0 + l32, rows - 1), qi = rld / rep, h = g * rep + rld % rep;
    p = sq.p0 + qi;
    klim = row0 + l32 < rows && p >= 0 && p < sq.len ? min(p, sq.cap - 1) : -1;
    const uint16_t *q = (const uint16_t *)a.q + (PAGED ? (int64_t)(sq.lo + qi) * a.q_ss : (int64_t)b * a.q_sb + (int64_t)qi * a.q_ss)
                        + (int64_t)h * a.q_sh;
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk) qf[kk] = *reinterpret_cast<const V8 *>(q + kk * 16 + lhi * 8);
  }
  const uint16_t *kp = (const uint16_t *)a.k + (PAGED ? 0 : (int64_t)b * a.k_sb) + (int64_t)g * a.k_sh;
  const uint16_t *vp = (const uint16_t *)a.v + (PAGED ? 0 : (int64_t)b * a.v_sb) + (int64_t)g * a.v_sh;

  f32x16 acc[D / 32];
#pragma unroll
  for (int t2 = 0; t2 < D / 32; ++t2)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[t2][r] = 0.f;
  float m_run = -1e30f, l_run = 0.f;  // (finite: a masked score gives p = 0; scores below it: see `sees`)
  const float sl2 = a.scale * 1.44269504088896340736f;

  // swizzles: 16-byte chunk c of row r stands at chunk c ^ kswz / vswz, so that
  // 16 rows of a K fragment, and the four rows of a transposing V read, cover
  // all banks
  auto kswz = [](int r) __attribute__((always_inline)) { return D == 128 ? r & 15 : (r >> 1) & 7; };
  auto vswz = [](int r) __attribute__((always_inline)) { return D == 128 ? (r & 3) << 2 : ((r >> 1) & 1) << 2; };

  // look up the rows of blocks 32 c .. 32 c + 31 of this workgroup
  auto look_up = [&](int c) __attribute__((always_inline)) {
    if constexpr (PAGED) {
      bool miss = false;
#pragma unroll 1
      for (int x = tid; x < ATT_AHEAD * ATT_KEYS; x += 256) {
        const int j = j0 + c * ATT_AHEAD + x / ATT_KEYS;
        const int key = sp.kb(j) * ATT_KEYS + x % ATT_KEYS;
        int at = -1;
        if (j < j1 && key < sp.hi && (key >= sp.lo || key < a.sinks)) {
          at = att_place(a, b, key);
          miss |= at < 0;
        }
        if constexpr (!FAR) at = at < 0 ? (int)ATT_NOWHERE : (int)((uint32_t)at * (uint32_t)a.k_ss * 2);
        ent[(c & 1) * ATT_AHEAD * ATT_KEYS + x] = at;
      }
      const bool any = __ballot(miss) != 0;
      if (lane == 0) lost[(c & 1) * 4 + wave] = any;
      __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
    }
  };
  const uint32_t k_lds = lds_addr(KR) + wave * 1024, v_lds = lds_addr(VR) + wave * 1024;
  const int64_t rows_there = PAGED ? (int64_t)a.pages * a.pitch : sp.hi;
  const i32x4_t rk = rsrc_words(kp, (rows_there - 1) * a.k_ss * 2 + RB), rv = rsrc_words(vp, (rows_there - 1) * a.v_ss * 2 + RB);
  const int r0 = wave * RPM + lane / LPR;
  const uint32_t kown = r0 * (uint32_t)a.k_ss * 2 + (((lane % LPR) ^ kswz(r0)) << 4);
  const uint32_t vown = r0 * (uint32_t)a.v_ss * 2 + (((lane % LPR) ^ vswz(r0)) << 4);
  // move i of block j0 + jr: row r, 16-byte chunk c of this lane, which are `own`
  // bytes into the block for i = 0
  auto move = [&](const uint16_t *base, i32x4_t rsrc, int64_t ss, int jr, int i, int r, int c, uint32_t own, uint32_t lds)
      __attribute__((always_inline)) {
    const int k0 = sp.kb(j0 + jr) * ATT_KEYS;
    if constexpr (!FAR) {
      uint32_t off;
      if constexpr (PAGED) {
        off = jr < n ? (uint32_t)ent[(jr & (2 * ATT_AHEAD - 1)) * ATT_KEYS + r] : ATT_NOWHERE;
      } else {
        // (the block's part is uniform; past the last key the resource ends)
        off = own + (uint32_t)(k0 + i * 4 * RPM) * (uint32_t)ss * 2;
        rsrc[2] = jr < n ? rsrc[2] : 0;
        if (k0 < sp.lo && k0 + ATT_KEYS > a.sinks) off = k0 + r < sp.lo && k0 + r >= a.sinks ? ATT_NOWHERE : off;
      }
      dma16_asm(rsrc, lds, PAGED ? off + c * 16 : off);
    } else {
      int at = -1;
      if constexpr (PAGED) {
        if (jr < n) at = ent[(jr & (2 * ATT_AHEAD - 1)) * ATT_KEYS + r];
      } else {
        if (jr < n && k0 + r < sp.hi && (k0 + r >= sp.lo || k0 + r < a.sinks)) at = k0 + r;
      }
      move16((at < 0 ? (const uint8_t *)a.zeros : (const uint8_t *)(base + (int64_t)at * ss)) + c * 16, lds);
    }
  };
  auto load_k = [&](auto sl, int jr) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < NM; ++i) {
      int l = lane;
      if constexpr (PAGED && FAR) asm volatile("" : "+v"(l));  // (registers: found again every time)
      const int r = (i * 4 + wave) * RPM + l / LPR;
      move(kp, rk, a.k_ss, jr, i, r, (l % LPR) ^ kswz(r), kown, k_lds + (decltype(sl)::value & 3) * TB + i * 4096);
    }
  };
  auto load_v = [&](auto sl, int jr) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < NM; ++i) {
      int l = lane;
      if constexpr (PAGED && FAR) asm volatile("" : "+v"(l));  // (registers: found again every time)
      const int r = (i * 4 + wave) * RPM + l / LPR;
      move(vp, rv, a.v_ss, jr, i, r, (l % LPR) ^ vswz(r), vown, v_lds + (decltype(sl)::value & 3) * TB + i * 4096);
    }
  };
  // an iteration leaves the moves of the last two outstanding
  auto wait_moves = [&](auto count) __attribute__((always_inline)) {
    static_assert(decltype(count)::value < 16, "vmcnt field");
    __builtin_amdgcn_s_waitcnt(0x0F70 | decltype(count)::value);
  };

  // K fragment kk: row l32, chunk 2 kk + lhi
  const int kbase = l32 * RB + ((lhi ^ (kswz(l32) & 1)) << 4), kx = (kswz(l32) & ~1) << 4;
  auto qk = [&](const uint8_t *K, f32x16 &s) __attribute__((always_inline)) {
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = 0.f;
    int x = kx;
    asm volatile("" : "+v"(x));  // (eight sums kept through the loop would cost as many registers)
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk)
      s = Mat<T>::mul(*reinterpret_cast<const V8 *>(K + kbase + ((kk << 5) ^ x)), qf[kk], s);
  };
  // transposing V read (group lane / 16, i = lane % 16): row 16 j + 8 si + 4 (group / 2) + i / 4,
  // columns 32 dt + 16 (group % 2) + 4 (i % 4)
  int vbase, vx;
  {
    const int grp = lane >> 4, gi = lane & 15, r = 4 * (grp >> 1) + (gi >> 2);
    vbase = r * RB + (((grp & 1) * 2 + ((gi & 3) >> 1)) << 4) + (gi & 1) * 8;
    vx = vswz(r) << 4;
  }
  auto pv1 = [&](const uint8_t *Vt, const V8 (&pf)[2], int j, int dt) __attribute__((always_inline)) {
    s16x4 v[2];
#pragma unroll
    for (int si = 0; si < 2; ++si)
      v[si] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          (lds_s16x4 *)(Vt + (16 * j + 8 * si) * RB + vbase + ((dt << 6) ^ vx)));
    const s16x8 vf = __builtin_shufflevector(v[0], v[1], 0, 1, 2, 3, 4, 5, 6, 7);
    acc[dt] = Mat<T>::mul(__builtin_bit_cast(V8, vf), pf[j], acc[dt]);
  };
  // The scores of one block and the values of another, in turns: each product of
  // the scores waits for the one before it, the values' are apart.
  auto qk_pv = [&](const uint8_t *K, f32x16 &s, const uint8_t *Vt, const V8 (&pf)[2]) __attribute__((always_inline)) {
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = 0.f;
#pragma unroll
    for (int i = 0; i < D / 16; ++i) {
      s = Mat<T>::mul(*reinterpret_cast<const V8 *>(K + kbase + ((i << 5) ^ kx)), qf[i], s);
      pv1(Vt, pf, i / (D / 32), i % (D / 32));
    }
  };
  auto expblock = [&](const f32x16 &s, V8 (&pf)[2]) __attribute__((always_inline)) {
    float s0 = 0.f, s1 = 0.f;
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(s[8 * j + e], sl2, -m_run));
        if (e & 1) s1 += x; else s0 += x;
        pf[j][e] = (typename Mat<T>::E)x;
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
    if (PAGED && missing) {
      const int32_t *en = ent + (jr & (2 * ATT_AHEAD - 1)) * ATT_KEYS + lhi * 4;
#pragma unroll
      for (int r = 0; r < 16; r += 4) {
        const int4 e = *reinterpret_cast<const int4 *>(en + r * 2);
        asm volatile("" ::: "memory");  // (one at a time: registers)
        auto gone = [](int x) { return FAR ? x < 0 : (uint32_t)x >= ATT_NOWHERE; };
        s[r] = gone(e.x) ? -INFINITY : s[r];
        s[r + 1] = gone(e.y) ? -INFINITY : s[r + 1];
        s[r + 2] = gone(e.z) ? -INFINITY : s[r + 2];
        s[r + 3] = gone(e.w) ? -INFINITY : s[r + 3];
      }
    }
  };
  auto raise = [&](f32x16 &s, V8 (&pf)[2], float ls) __attribute__((always_inline)) {
    if (__builtin_expect(__builtin_amdgcn_ballot_w64(!(ls <= Mat<T>::LIMIT)) != 0, 0)) {
      float bm = s[0];
#pragma unroll
      for (int r = 1; r < 16; ++r) bm = fmaxf(bm, s[r]);
      bm = fmaxf(bm, __shfl_xor(bm, 32, 64));
      const float m_new = fmaxf(m_run, bm * sl2 - Mat<T>::TOP);
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
  V8 pA[2], pB[2];
#pragma unroll
  for (int j = 0; j < 2; ++j)
#pragma unroll
    for (int e = 0; e < 8; ++e) pB[j][e] = (typename Mat<T>::E)0.f;
  // the end of an iteration: the next moves, behind its matrix instructions
  auto move_on = [&](auto sl, int jr) __attribute__((always_inline)) {
    load_k(sl, jr + 4);
    load_v(Slot<decltype(sl)::value + 2>{}, jr + 2);
    wait_moves(Slot<4 * NM>{});
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
  // Iteration jr, one body for all: the values of the block before (of zeros
  // before the first), the scores of the one behind (of zeros past the last), the
  // softmax of this one.  The last, jr = n, adds the last block's values.
  auto step = [&](auto sl, int jr, f32x16 &cur, f32x16 &nxt, V8 (&prev)[2], V8 (&now)[2]) __attribute__((always_inline)) {
    constexpr int SL = decltype(sl)::value;
    if (!whole(jr)) mask(cur, jr);
    qk_pv(KR + ((SL + 1) & 3) * TB, nxt, VR + ((SL + 3) & 3) * TB, prev);
    const float ls = expblock(cur, now);
    // Six LDS reads ahead, then in turns a matrix instruction, the reads of a later
    // one and a share of the softmax.  One 16384-token prompt in a 4096 window:
    // 892 us; in source order 897, every read first 926, the scores' products in
    // two sums 927, all scores before all values 921 to 980 (all on one card; others
    // take 914 and 927 for the first).
    __builtin_amdgcn_sched_group_barrier(0x100, 6, 0);
    __builtin_amdgcn_sched_group_barrier(0x002, 6, 0);
#pragma unroll
    for (int i = 0; i < D / 8; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
      __builtin_amdgcn_sched_group_barrier(0x002, 3 * 128 / D, 0);
    }
    raise(cur, now, ls);
    move_on(sl, jr);
  };

  if (n > 0) {
    look_up(0);
    __syncthreads();
    load_v(Slot<3>{}, n);  // (zeros)
    load_k(Slot<0>{}, 0);
    load_k(Slot<1>{}, 1);
    load_k(Slot<2>{}, 2);
    load_v(Slot<0>{}, 0);
    load_k(Slot<3>{}, 3);
    load_v(Slot<1>{}, 1);
    wait_moves(Slot<4 * NM>{});
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    if (active) qk(KR, sA);
    __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0): block 0 is read before its slot is refilled
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    auto ahead = [&](int jr) __attribute__((always_inline)) {
      if (PAGED && jr % ATT_AHEAD == 0) {
        const int32_t *f = lost + (jr / ATT_AHEAD & 1) * 4;
        missing = __builtin_amdgcn_readfirstlane(f[0] | f[1] | f[2] | f[3]);
        // (the other half was last read an iteration, and a barrier, ago)
        if (jr + ATT_AHEAD < n) look_up(jr / ATT_AHEAD + 1);
      }
    };
    if (active) {
      for (int jr = 0;; jr += 4) {
        ahead(jr);
        step(Slot<0>{}, jr, sA, sB, pB, pA);
        if (jr + 1 > n) break;
        step(Slot<1>{}, jr + 1, sB, sA, pA, pB);
        if (jr + 2 > n) break;
        step(Slot<2>{}, jr + 2, sA, sB, pB, pA);
        if (jr + 3 > n) break;
        step(Slot<3>{}, jr + 3, sB, sA, pA, pB);
        if (jr + 4 > n) break;
      }
    } else {  // rows past the sequence's: the moves only
      for (int jr = 0; jr <= n; jr += 4) {
        ahead(jr);
        move_on(Slot<0>{}, jr);
        if (jr + 1 <= n) move_on(Slot<1>{}, jr + 1);
        if (jr + 2 <= n) move_on(Slot<2>{}, jr + 2);
        if (jr + 3 <= n) move_on(Slot<3>{}, jr + 3);
      }
    }
    wait_moves(Slot<0>{});  // no move outlives the workgroup
  }

  // (the row's place is found again: kept through the loop it costs registers)
  int again = l32;
  asm volatile("" : "+v"(again));
  const int row = row0 + again, rld = min(row, rows - 1), qi = rld / rep, h = g * rep + rld % rep;
  const bool ok = klim >= 0;
  l_run += __shfl_xor(l_run, 32, 64);
  const int64_t nr = (int64_t)a.N * a.Hq;
  const int64_t orow = ((int64_t)(PAGED ? sq.lo + qi : b * a.S + qi)) * a.Hq + h;
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

  // rows that a value which is not finite may have spoiled
  float z = l_run * 0.f;
#pragma unroll
  for (int t2 = 0; t2 < D / 32; ++t2)
#pragma unroll
    for (int r = 0; r < 16; ++r) z = __builtin_fmaf(acc[t2][r], 0.f, z);
  // and those whose offset is too large to cancel: s c - m is then off by half a
  // step of m.  A row without weight still has the offset it began with: where it
  // sees keys their scores are below that, or -inf.
  uint64_t spoiled = __ballot(ok && (z != 0.f || (fabsf(m_run) >= 0x1p24f && (l_run != 0.f || sees))));
  spoiled = (spoiled | spoiled >> 32) & 0xffffffffull;
  const bool mine = spoiled >> l32 & 1;
  const bool put = row < rows && !mine;
  if (put && pieces == 1) {
    const float inv = ok && l_run != 0.f ? 1.0f / l_run : 0.f;
#pragma unroll
    for (int t2 = 0; t2 < D / 32; ++t2)
#pragma unroll
      for (int gq = 0; gq < 4; ++gq) {
        float x[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = inv == 0.f ? 0.f : acc[t2][gq * 4 + e] * inv;
        T y[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) Elt<T>::store(y, e, x[e]);
        uint2 u;
        __builtin_memcpy(&u, y, 8);
        *reinterpret_cast<uint2 *>(o + t2 * 32 + gq * 8 + lhi * 4) = u;
      }
  } else if (put) {
#pragma unroll
    for (int t2 = 0; t2 < D / 32; ++t2)
#pragma unroll
      for (int gq = 0; gq < 4; ++gq) {
        float4 x;
        x.x = ok ? acc[t2][gq * 4] : 0.f;
        x.y = ok ? acc[t2][gq * 4 + 1] : 0.f;
        x.z = ok ? acc[t2][gq * 4 + 2] : 0.f;
        x.w = ok ? acc[t2][gq * 4 + 3] : 0.f;
        *reinterpret_cast<float4 *>(wo + t2 * 32 + gq * 8 + lhi * 4) = x;
      }
    if (lhi == 0) wm[0] = m_run, wm[1] = ok ? l_run : 0.f;
  }
  // These again, reading only what they see.  (The arguments are read anew, so
  // that none of them takes a register through the loop above for this.)
  while (spoiled) {
    typedef const __attribute__((address_space(4))) AttendArgs *Kernarg;
    Kernarg args = (Kernarg)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(args));
    const AttendArgs &a2 = *(const AttendArgs *)args;
    const AttWork wk2 = att_work<PAGED>(a2, blockIdx.x);
    const AttSeq sq2 = att_seq(a2, wk2.b);
    const AttSpan sp2 = att_span(a2, sq2, wk2.tile);
    const int64_t nr2 = (int64_t)a2.N * a2.Hq;
    int k0, k1;
    const int pieces2 = att_split(a2, sp2.nb, wk2.split, k0, k1);
    const int src = __builtin_ctzll(spoiled);
    spoiled &= spoiled - 1;
    float m, l, x[D / 64];
    att_row<T, true, D>(a2, sq2, sp2, wk2.b, __shfl(qi, src, 64), __shfl(h, src, 64), k0, k1, m, l, x);
    const int64_t at = __shfl((int)orow, src, 64);  // (rows are below 2^31)
#pragma unroll
    for (int e = 0; e < D / 64; ++e) {
      if (pieces2 == 1) {
        Elt<T>::store((T *)a2.o + at * D, lane + 64 * e, l == 0.f ? 0.f : x[e] / l);
      } else {
        a2.ws[(wk2.split * nr2 + at) * D + lane + 64 * e] = x[e];
      }
    }
    if (pieces2 > 1 && lane == 0) {
      float *q = a2.ws + (int64_t)a2.nsplit * nr2 * D + (wk2.split * nr2 + at) * 2;
      q[0] = fmaxf(m * 1.44269504088896340736f, ATT_LOWEST);
      q[1] = l;
    }
  }
}

#define NK_TILE(T, name, D, OCC, MORE)                                                                             \
  extern "C" __global__ __launch_bounds__(256, OCC) void nk_attend_tile_paged_##name##_d##D(AttendArgs a) {        \
    attend_tile_body<T, D, true, false>(a);                                                                      \
  }                                                                                                              \
  extern "C" __global__ __launch_bounds__(256, MORE) void nk_attend_tile_plain_##name##_d##D(AttendArgs a) {        \
    attend_tile_body<T, D, false, false>(a);                                                                     \
  }                                                                                                              \
  extern "C" __global__ __launch_bounds__(256, OCC) void nk_attend_tile_paged_far_##name##_d##D(AttendArgs a) {    \
    attend_tile_body<T, D, true, true>(a);                                                                       \
  }                                                                                                              \
  extern "C" __global__ __launch_bounds__(256, MORE) void nk_attend_tile_plain_far_##name##_d##D(AttendArgs a) {    \
    attend_tile_body<T, D, false, true>(a);                                                                      \
  }
// (workgroups per CU, paged and plain: what LDS and registers hold; 4 sequences of
// 2000 with 16 heads of 64 in a window of 512: 40 us; the body takes 122 registers
// under a bound of three as well)
NK_TILE(bf16, bf16, 128, 2, 2)
NK_TILE(f16, f16, 128, 2, 2)
NK_TILE(bf16, bf16, 64, 3, 4)
NK_TILE(f16, f16, 64, 3, 4)

// ---------------------------------------------------------------------------
// One new token per sequence (16-bit operands, head dim 64 or 128): bound by the
// read of the keys and values, so the waves of a workgroup take blocks of 32 keys
// of their own, no barrier between them, and meet at the end.
//
// A wave has up to 16 heads of the group as the columns of 16x16x32 products,
// S^T = K Q^T and O^T = V^T P^T.  K fragments come straight from memory (16 bytes
// of a row per lane); V goes to an LDS slot of the wave's own, from which
// transposing reads take four keys of a column.  Every head sees the same keys.
// 64 sequences of up to 8192 tokens, 32 / 8 heads of 128: 240 us, 4.6 TB/s.
// ---------------------------------------------------------------------------
typedef float f32x4 __attribute__((ext_vector_type(4)));
NK_DEVICE f32x4 mul16(Mat<bf16>::V a, Mat<bf16>::V b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
NK_DEVICE f32x4 mul16(Mat<f16>::V a, Mat<f16>::V b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }

template <typename T, int D, bool PAGED>
__device__ __forceinline__ void attend_step_body(const AttendArgs &a) {
  typedef typename Mat<T>::V V8;
  constexpr int RB = D * 2, TB = ATT_KEYS * RB, LPR = RB / 16, RPM = 64 / LPR, NM = ATT_KEYS / RPM;
  constexpr int NW = 4;
  constexpr int SUM = NW * 16 * (D + 2) * 4;  // the waves' sums
  __shared__ __attribute__((aligned(1024))) uint8_t lds[NW * TB > SUM ? NW * TB : SUM];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l16 = lane & 15, grp = lane >> 4;
  const int rep = a.Hq / a.Hkv, per = (rep + 15) / 16;
  int w = blockIdx.x;
  const int g = w % a.Hkv;
  w /= a.Hkv;
  const int split = w / a.tiles, h0 = w % a.tiles % per * 16, b = w % a.tiles / per;  // (h0: first head of the group's)
  const AttSeq sq = att_seq(a, b);
  const AttSpan sp = att_span(a, sq, 0);
  int j0, j1;
  const int pieces = att_split(a, sp.nb, split, j0, j1);
  if (split >= pieces) return;
  const int p = sq.p0, klim = min(p, sq.cap - 1);

  V8 qf[D / 32];
  {
    const uint16_t *q = (const uint16_t *)a.q + (PAGED ? (int64_t)b * a.q_ss : (int64_t)b * a.q_sb) +
                        (int64_t)(g * rep + min(h0 + l16, rep - 1)) * a.q_sh;
#pragma unroll
    for (int kk = 0; kk < D / 32; ++kk) qf[kk] = *reinterpret_cast<const V8 *>(q + kk * 32 + grp * 8);
  }
  const uint16_t *kp = (const uint16_t *)a.k + (PAGED ? 0 : (int64_t)b * a.k_sb) + (int64_t)g * a.k_sh;
  const uint16_t *vp = (const uint16_t *)a.v + (PAGED ? 0 : (int64_t)b * a.v_sb) + (int64_t)g * a.v_sh;
  const uint8_t *zeros = (const uint8_t *)a.zeros;

  f32x4 acc[D / 16];
#pragma unroll
  for (int t = 0; t < D / 16; ++t) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m_run = ATT_LOWEST, l_run = 0.f;  // (the offset of the scores themselves: large ones cancel exactly)
  const float sl2 = a.scale * 1.44269504088896340736f;

  // 16 rows of a transposing read, two chunks each, cover all banks
  auto swz = [](int r) __attribute__((always_inline)) { return D == 128 ? (r & 7) << 1 : ((r >> 1) & 3) << 1; };
  uint8_t *const slot = lds + wave * TB;
  const uint32_t slot_lds = lds_addr(lds) + wave * TB;
  // lane l looks up key l % 32 of a block: its row, -1 where it is not seen
  auto place = [&](int j) __attribute__((always_inline)) {
    const int key = sp.kb(j) * ATT_KEYS + (lane & 31);
    return j < j1 && key <= klim && (key > p - a.window || key < a.sinks) ? att_place(a, b, key) : -1;
  };

  int ent = place(j0 + wave);
  for (int j = j0 + wave; j < j1; j += NW) {
#pragma unroll
    for (int i = 0; i < NM; ++i) {
      const int r = i * RPM + lane / LPR, c = ((lane % LPR) ^ swz(r)) * 16;
      const int at = __shfl(ent, r, 64);
      move16((at < 0 ? zeros : (const uint8_t *)(vp + (int64_t)at * a.v_ss)) + c, slot_lds + i * 1024);
    }
    V8 kf[2][D / 32];
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) {
      const int at = __shfl(ent, kt * 16 + l16, 64);
      const uint16_t *k = at < 0 ? (const uint16_t *)zeros : kp + (int64_t)at * a.k_ss;
#pragma unroll
      for (int kk = 0; kk < D / 32; ++kk) kf[kt][kk] = *reinterpret_cast<const V8 *>(k + kk * 32 + grp * 8);
    }
    const uint32_t seen = (uint32_t)__ballot(ent >= 0);
    ent = place(j + NW);  // (on its way while this block is worked on)
    f32x4 s[2];
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) {
      s[kt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int kk = 0; kk < D / 32; ++kk) s[kt] = mul16(kf[kt][kk], qf[kk], s[kt]);
    }
    // element r of tile kt is key 16 kt + 4 grp + r
    const uint32_t mine = seen >> (grp * 4);
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
      for (int r = 0; r < 4; ++r) s[kt][r] = mine >> (kt * 16 + r) & 1 ? s[kt][r] : -INFINITY;
    V8 pf;
    auto weigh = [&]() __attribute__((always_inline)) {
      float sum = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(s[e >> 2][e & 3] - m_run, sl2, Mat<T>::TOP));
        sum += x;
        pf[e] = (typename Mat<T>::E)x;
      }
      return sum;
    };
    float ls = weigh();
    if (__builtin_amdgcn_ballot_w64(!(ls <= Mat<T>::LIMIT)) != 0) {
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
    __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): V is there
    asm volatile("" ::: "memory");
#pragma unroll
    for (int t = 0; t < D / 16; ++t) {
      s16x4 v[2];
#pragma unroll
      for (int si = 0; si < 2; ++si) {
        const int r = 16 * si + 4 * grp + (l16 >> 2);
        const int c = (t * 2 + ((l16 & 3) >> 1)) ^ swz(r);
        v[si] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(slot + r * RB + c * 16 + (l16 & 1) * 8));
      }
      const s16x8 vf = __builtin_shufflevector(v[0], v[1], 0, 1, 2, 3, 4, 5, 6, 7);
      acc[t] = mul16(__builtin_bit_cast(V8, vf), pf, acc[t]);
    }
    __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0): the slot is read before it is refilled
    asm volatile("" ::: "memory");
  }

  // The waves' sums: their offsets meet, then each row's sums are added in the
  // waves' order.
  l_run += __shfl_xor(l_run, 16, 64);
  l_run += __shfl_xor(l_run, 32, 64);
  float *so = reinterpret_cast<float *>(lds), *sm = so + NW * 16 * D;  // (NW, 16, D) sums; (NW, 16) weights, (16) in all
  // a bit for each row with a sum that is not finite under weights that are (those of
  // a NaN score are NaN, and so is all of the row)
  __shared__ uint32_t spoiled[NW];
  float z = 0.f;
#pragma unroll
  for (int t = 0; t < D / 16; ++t)
#pragma unroll
    for (int r = 0; r < 4; ++r) z = __builtin_fmaf(acc[t][r], 0.f, z);
  uint64_t bits = __ballot(z != 0.f && l_run == l_run);
  bits |= bits >> 32;
  if (lane == 0) spoiled[wave] = (uint32_t)(bits | bits >> 16) & 0xffffu;
  __syncthreads();
  if (grp == 0) so[wave * 16 + l16] = m_run;
  __syncthreads();
  const float m = fmaxf(fmaxf(so[l16], so[16 + l16]), fmaxf(so[32 + l16], so[48 + l16]));
  __syncthreads();
  // (an infinite score's offset is infinite: its sums are NaN already)
  const float f = m_run == m ? 1.f : __builtin_amdgcn_exp2f((m_run - m) * sl2);
#pragma unroll
  for (int t = 0; t < D / 16; ++t)
    *reinterpret_cast<float4 *>(so + (wave * 16 + l16) * D + t * 16 + grp * 4) =
        make_float4(acc[t][0] * f, acc[t][1] * f, acc[t][2] * f, acc[t][3] * f);
  if (grp == 0) sm[wave * 16 + l16] = l_run * f;
  __syncthreads();
  const int64_t nr = (int64_t)a.N * a.Hq, r0 = (int64_t)b * a.Hq + g * rep + h0;
  auto weight = [&](int r) __attribute__((always_inline)) { return (sm[r] + sm[16 + r]) + (sm[32 + r] + sm[48 + r]); };
  const uint32_t again = __builtin_amdgcn_readfirstlane(spoiled[0] | spoiled[1] | spoiled[2] | spoiled[3]);
#pragma unroll
  for (int x = 0; x < 16 * D / 256; ++x) {
    const int e = x * 256 + tid, r = e / D;
    if (h0 + r >= rep) break;  // (rows rise)
    if (again >> r & 1) continue;
    const float o = (so[e] + so[16 * D + e]) + (so[2 * 16 * D + e] + so[3 * 16 * D + e]), l = weight(r);
    if (pieces == 1) {
      Elt<T>::store((T *)a.o + r0 * D, e, l == 0.f ? 0.f : o / l);
    } else {
      a.ws[(split * nr + r0) * D + e] = o;
    }
  }
  float *wm = a.ws + (int64_t)a.nsplit * nr * D + (split * nr + r0) * 2;
  if (pieces > 1 && wave == 0 && grp == 0 && h0 + l16 < rep && !(again >> l16 & 1))
    wm[2 * l16] = fmaxf(m * sl2, ATT_LOWEST), wm[2 * l16 + 1] = weight(l16);
  // Values that are not finite under weights that rounded to 0: those rows again, a
  // wave for each.
  for (uint32_t left = again; left; left &= left - 1) {
    const int r = __builtin_ctz(left);
    if (h0 + r >= rep) break;
    if (r % NW != wave) continue;
    float mr, lr, x[D / 64];
    att_row<T, true, D>(a, sq, sp, b, 0, g * rep + h0 + r, j0, j1, mr, lr, x);
#pragma unroll
    for (int e = 0; e < D / 64; ++e) {
      if (pieces == 1) {
        Elt<T>::store((T *)a.o + (r0 + r) * D, lane + 64 * e, lr == 0.f ? 0.f : x[e] / lr);
      } else {
        a.ws[(split * nr + r0 + r) * D + lane + 64 * e] = x[e];
      }
    }
    // (the step's weights are 2^TOP of these)
    if (pieces > 1 && lane == 0) wm[2 * r] = fmaxf(mr * 1.44269504088896340736f, ATT_LOWEST) + Mat<T>::TOP, wm[2 * r + 1] = lr;
  }
}
#define NK_STEP(T, name, D)                                                                                 \
  extern "C" __global__ __launch_bounds__(256, 2) void nk_attend_step_paged_##name##_d##D(AttendArgs a) {   \
    attend_step_body<T, D, true>(a);                                                                        \
  }                                                                                                         \
  extern "C" __global__ __launch_bounds__(256, 2) void nk_attend_step_plain_##name##_d##D(AttendArgs a) {   \
    attend_step_body<T, D, false>(a);                                                                       \
  }
NK_STEP(bf16, bf16, 128)
NK_STEP(f16, f16, 128)
NK_STEP(bf16, bf16, 64)
NK_STEP(f16, f16, 64)

// ---------------------------------------------------------------------------
// The splits of a row joined, in their order: o = sum 2^(m_s - M) o_s / sum
// 2^(m_s - M) l_s, over the splits with any weight.  Up to 64 splits, a lane each for
// their offsets; bound by the latency of its reads.  One wave per row, or (W = 4) a workgroup, each wave a
// quarter of the splits, all of its reads in flight at once.  Rows that one split
// had are written already.
// ---------------------------------------------------------------------------
template <typename T, int D, int W>
__device__ __forceinline__ void attend_join_body(const AttendArgs &a) {
  __shared__ float part[W == 1 ? 1 : W][D];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t r = W == 1 ? (int64_t)blockIdx.x * 4 + wave : blockIdx.x, nr = (int64_t)a.N * a.Hq;
  if (r >= nr) return;
  const int t = (int)(r / a.Hq), h = (int)(r % a.Hq), rep = a.Hq / a.Hkv;
  int b, i;
  AttSeq sq;
  if (!att_query(a, t, b, sq, i)) return;
  int j0, j1;
  const int pieces = att_split(a, att_span(a, sq, (i * rep + h % rep) / ATT_ROWS).nb, 0, j0, j1);
  if (pieces == 1) return;
  const float *wm = a.ws + (int64_t)a.nsplit * nr * D;
  const int w0 = W == 1 ? 0 : wave;  // this wave's splits: w0, w0 + W, ...
  constexpr int U = W == 1 ? 4 : 16;
  float acc[D / 64], x[U][D / 64];
  auto fetch = [&](int s0) __attribute__((always_inline)) {
#pragma unroll
    for (int s = 0; s < U; ++s)  // (past the last piece: the last again, unused)
#pragma unroll
      for (int e = 0; e < D / 64; ++e)
        x[s][e] = a.ws[((int64_t)min(s0 + s * W, pieces - 1) * nr + r) * D + lane + 64 * e];
  };
  fetch(w0);
  float m = -INFINITY, l = 0.f;
  if (lane < pieces) {
    const float2 v = *reinterpret_cast<const float2 *>(wm + (lane * nr + r) * 2);
    l = v.y;
    if (l != 0.f) m = v.x;
  }
  const float top = wave_max(m), w = l != 0.f ? __builtin_amdgcn_exp2f(m - top) : 0.f;
  const float total = wave_sum(w * l);
  const float inv = total == 0.f ? 0.f : 1.f / total;
  auto add = [&](auto f) __attribute__((always_inline)) {
#pragma unroll
    for (int e = 0; e < D / 64; ++e) acc[e] = 0.f;
    for (int s0 = w0; s0 < pieces; s0 += U * W) {
      if (s0 != w0) fetch(s0);
#pragma unroll
      for (int s = 0; s < U; ++s) {
        if (s0 + s * W >= pieces) break;
        const float ws = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(w), s0 + s * W));
#pragma unroll
        for (int e = 0; e < D / 64; ++e) acc[e] = f(ws, x[s][e], acc[e]);
      }
    }
  };
  add([](float ws, float y, float c) { return fmaf(ws, y, c); });
  bool whole = true;
#pragma unroll
  for (int e = 0; e < D / 64; ++e) whole &= __builtin_isfinite(acc[e]);
  if (__builtin_expect(__any(!whole), 0)) {  // (0 x inf: a split's sum is not finite, and its weight is nothing beside the others')
    fetch(w0);
    add(att_add);
  }
  if constexpr (W > 1) {
#pragma unroll
    for (int e = 0; e < D / 64; ++e) part[wave][lane + 64 * e] = acc[e];
    __syncthreads();
    if (wave) return;
#pragma unroll
    for (int e = 0; e < D / 64; ++e) {
      const int d = lane + 64 * e;
      acc[e] = (part[0][d] + part[1][d]) + (part[2][d] + part[3][d]);
    }
  }
#pragma unroll
  for (int e = 0; e < D / 64; ++e) Elt<T>::store((T *)a.o + r * D, lane + 64 * e, total == 0.f ? 0.f : acc[e] * inv);
}
#define NK_JOIN(T, name, D)                                                                          \
  extern "C" __global__ __launch_bounds__(256) void nk_attend_join_##name##_d##D(AttendArgs a) {     \
    attend_join_body<T, D, 1>(a);                                                                    \
  }                                                                                                  \
  extern "C" __global__ __launch_bounds__(256) void nk_attend_join4_##name##_d##D(AttendArgs a) {    \
    attend_join_body<T, D, 4>(a);                                                                    \
  }
NK_JOIN(bf16, bf16, 128)
NK_JOIN(f16, f16, 128)
NK_JOIN(bf16, bf16, 64)
NK_JOIN(f16, f16, 64)
