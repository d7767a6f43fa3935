// A generation loop around its kernels: block tables and slots from lengths, the
// choice of a beam search's beams, and the paged caches that follow them.

#include "common.h"

using namespace nk;

typedef unsigned long long u64;

// running sums over the lanes of a wave, this one's included: within rows of 16 lanes,
// then from the rows before
template <int CTRL, int ROWS>
NK_DEVICE int64_t lanes_before(int64_t v) {
  const int lo = __builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xf, false);
  const int hi = __builtin_amdgcn_update_dpp(0, (int)(v >> 32), CTRL, ROWS, 0xf, false);
  return (int64_t)((u64)(uint32_t)hi << 32 | (uint32_t)lo);
}
NK_DEVICE int64_t running(int64_t v) {
  v += lanes_before<0x111, 0xf>(v);  // row_shr 1, 2, 4, 8
  v += lanes_before<0x112, 0xf>(v);
  v += lanes_before<0x114, 0xf>(v);
  v += lanes_before<0x118, 0xf>(v);
  v += lanes_before<0x142, 0xa>(v);  // row_bcast 15: lane 15 of rows 0 and 2
  v += lanes_before<0x143, 0xc>(v);  // row_bcast 31: lane 31
  return v;
}
NK_DEVICE int64_t lane_of(int64_t v, int lane) {
  return (int64_t)((u64)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), lane) << 32
                   | (uint32_t)__builtin_amdgcn_readlane((int)v, lane));
}
// and of two numbers over a workgroup of W waves; `all`: the whole sums
template <int W>
NK_DEVICE void running_block(int64_t (&v)[2], int64_t (*red)[W], int64_t (&all)[2]) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  v[0] = running(v[0]), v[1] = running(v[1]);
  __syncthreads();
  if (lane == 63) red[0][wave] = v[0], red[1][wave] = v[1];
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    // (the waves' sums again by a running sum: W registers less)
    const int64_t w = running(lane < W ? red[k][lane] : 0);
    all[k] = lane_of(w, W - 1);
    if (wave) v[k] += lane_of(w, wave - 1);
  }
}

// ---------------------------------------------------------------------------
// Block tables.
//
// Row b holds ceil((len - new) / page) pages; those of all rows are marked in a
// bitmap in LDS.  What is not marked is free, and the r-th free page goes to the
// r-th entry that wants one: r by running sums over the rows, the page by running
// counts over the bitmap.  Marks are ORs and sums are whole numbers, so no order
// changes a result.
//
// Bound by latency.  Small batches are one launch of one workgroup; larger ones
// three: workgroups that mark some rows each, into bitmaps of their own; one that
// joins the bitmaps, sums up and lists the free pages that are wanted; and as many as
// there are rows and tokens for the entries and slots (500 rows of up to 375 pages,
// 20000 tokens: 83 us by the one workgroup, 19 so; 64 rows of up to 250 by the one: 9.4).
// ---------------------------------------------------------------------------
struct AssignArgs {
  int32_t *tables;  // (rows, width)
  const int32_t *lens, *news;
  int32_t *starts, *slots, *free;
  int32_t *wants;   // (rows) pages wanted by the rows before
  int32_t *list;    // the free pages that are wanted, in order; -1 behind the last
  uint32_t *marks;  // (parts, words in fours) bitmaps of some rows each
  int32_t rows, width, page, pages, tokens, parts;
};
#define ASG_BLOCK 1024
#define ASG_WORDS 32768  // of 32 pages

struct AsgRow {
  int len, fresh, held, need;
};
NK_DEVICE AsgRow asg_row(const AssignArgs &a, int len, int fresh) {
  AsgRow r;
  r.len = min(max(len, 0), 1 << 30);
  r.fresh = min(max(fresh, 0), 1 << 30);
  // (sums below 2^31: page is at most 2^30)
  r.held = min((int)(((uint32_t)max(r.len - r.fresh, 0) + (uint32_t)a.page - 1) / (uint32_t)a.page), a.width);
  r.need = min((int)(((uint32_t)r.len + (uint32_t)a.page - 1) / (uint32_t)a.page), a.width);
  return r;
}
NK_DEVICE AsgRow asg_row(const AssignArgs &a, int b) { return asg_row(a, a.lens[b], a.news[b]); }

// The pages that rows b0, b0 + step, ... hold, marked by a wave: four rows' entries
// on their way at once.
NK_DEVICE void asg_mark(const AssignArgs &a, uint32_t *used, int b0, int step) {
  const int lane = threadIdx.x & 63;
  auto mark = [&](int pg) __attribute__((always_inline)) {
    if (pg >= 0 && pg < a.pages) atomicOr(&used[pg >> 5], 1u << (pg & 31));
  };
  for (int c0 = b0; c0 < a.rows; c0 += 64 * step) {
    const int64_t b = c0 + (int64_t)lane * step;  // (a lane's row of the next 64)
    const int held = b < a.rows ? asg_row(a, (int)b).held : 0;
    for (int r = 0; r < 64 && c0 + (int64_t)r * step < a.rows; r += 4) {
      int pg[4][4], n[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        n[u] = __builtin_amdgcn_readlane(held, r + u);
        const int32_t *t = a.tables + min(c0 + (int64_t)(r + u) * step, (int64_t)a.rows - 1) * a.width;
#pragma unroll
        for (int k = 0; k < 4; ++k) pg[u][k] = k * 64 + lane < n[u] ? t[k * 64 + lane] : -1;
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
#pragma unroll
        for (int k = 0; k < 4; ++k) mark(pg[u][k]);
        const int32_t *t = a.tables + min(c0 + (int64_t)(r + u) * step, (int64_t)a.rows - 1) * a.width;
        for (int i = 256 + lane; i < n[u]; i += 64) mark(t[i]);
      }
    }
  }
}

// Starts and wanted pages of the rows, and from the bitmap the free pages before each
// thread's words; returns (pages wanted, pages free).
NK_DEVICE void asg_sums(const AssignArgs &a, const uint32_t *used, int32_t *before, int64_t (*red)[ASG_BLOCK / 64],
                        int64_t &wanted, int64_t &free) {
  const int tid = threadIdx.x;
  const int words = (a.pages + 31) / 32;
  const int per = (words + ASG_BLOCK - 1) / ASG_BLOCK, w0 = min(tid * per, words), w1 = min(w0 + per, words);
  int count = 0;
  for (int i = w0; i < w1; ++i) count += __popc(~used[i]);
  int64_t starts = 0, wants = 0, v[2], all[2];
  for (int b0 = 0; b0 < a.rows; b0 += ASG_BLOCK) {
    const int b = b0 + tid;
    int n = 0, w = 0;
    if (b < a.rows) {
      const AsgRow r = asg_row(a, b);
      n = r.fresh, w = max(r.need - r.held, 0);
    }
    // (what is wanted in the upper bits: below 2^40 in all; free pages: up to 2^20)
    v[0] = n, v[1] = (int64_t)w << 21 | (b0 ? 0 : count);
    running_block(v, red, all);
    if (b0 == 0) before[tid] = (int)(v[1] & 0x1fffff) - count, free = all[1] & 0x1fffff;
    if (b < a.rows) {
      a.starts[b] = (int32_t)min(starts + v[0] - n, (int64_t)0x7fffffff);
      a.wants[b] = (int32_t)min(wants + (v[1] >> 21) - w, (int64_t)a.pages);
    }
    starts += all[0], wants += all[1] >> 21;
  }
  if (tid == 0) {
    a.starts[a.rows] = (int32_t)min(starts, (int64_t)0x7fffffff);
    a.free[0] = (int32_t)max(free - wants, (int64_t)-0x7fffffff);
  }
  wanted = wants;
}
// the wanted free pages of a thread's words
NK_DEVICE void asg_list(const AssignArgs &a, const uint32_t *used, int before, int64_t wanted, int64_t free) {
  const int words = (a.pages + 31) / 32;
  const int per = (words + ASG_BLOCK - 1) / ASG_BLOCK, w0 = min((int)threadIdx.x * per, words), w1 = min(w0 + per, words);
  const int most = (int)min(wanted, (int64_t)a.pages);
  for (int i = w0, k = before; i < w1 && k < most; ++i)
    for (uint32_t bits = ~used[i]; bits && k < most; bits &= bits - 1, ++k) a.list[k] = i * 32 + __builtin_ctz(bits);
  for (int k = (int)free + threadIdx.x; k < most; k += ASG_BLOCK) a.list[k] = -1;
}
// the page of entry i of a row
NK_DEVICE int asg_entry(const AssignArgs &a, int64_t b, const AsgRow &r, int first, int i) {
  if (i < r.held) return a.tables[b * a.width + i];
  const int k = first + (i - r.held);
  return i < r.need && k < a.pages ? a.list[k] : -1;
}
// the entries of row b that it does not hold, by `threads` from t on
NK_DEVICE void asg_fill(const AssignArgs &a, int b, int t, int threads) {
  const AsgRow r = asg_row(a, b);
  const int first = a.wants[b];
  for (int i = r.held + t; i < a.width; i += threads) a.tables[(int64_t)b * a.width + i] = asg_entry(a, b, r, first, i);
}

// Slots of 64 tokens t0 ..: the rows that begin among them are read side by side.
NK_DEVICE void asg_slots(const AssignArgs &a, int t0) {
  const int lane = threadIdx.x & 63, t = t0 + lane;
  int b0 = 0;  // rows that begin at or before t0
#pragma unroll 4
  for (int b = 0; b < a.rows; b += 64) b0 += __popcll(__ballot(b + lane < a.rows && a.starts[min(b + lane, a.rows - 1)] <= t0));
  int b = b0 - 1;
  for (int x = b0;; x += 64) {
    const int s = x + lane < a.rows ? a.starts[x + lane] : 0x7fffffff;
    int more = 0;
#pragma unroll 8
    for (int k = 0; k < 64; ++k) more += __builtin_amdgcn_readlane(s, k) <= t ? 1 : 0;
    b += more;
    if (!__any(more == 64)) break;
  }
  if (t >= a.tokens) return;
  int slot = -1;
  if (b >= 0 && t < a.starts[b + 1]) {
    const AsgRow r = asg_row(a, b);
    const int p = r.len - r.fresh + (t - a.starts[b]);
    if (p >= 0 && p / a.page < a.width) {
      const int pg = asg_entry(a, b, r, a.wants[b], p / a.page);
      if (pg >= 0 && pg < a.pages) slot = pg * a.page + p % a.page;
    }
  }
  a.slots[t] = slot;
}

extern "C" __global__ __launch_bounds__(ASG_BLOCK) void nk_assign_pages(AssignArgs a) {
  __shared__ uint32_t used[ASG_WORDS];
  __shared__ int32_t before[ASG_BLOCK];
  __shared__ int64_t red[2][ASG_BLOCK / 64];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, words = (a.pages + 31) / 32;
  for (int i = tid; i < words; i += ASG_BLOCK) used[i] = i == words - 1 && (a.pages & 31) ? ~0u << (a.pages & 31) : 0;  // (no pages)
  __syncthreads();
  asg_mark(a, used, wave, ASG_BLOCK / 64);
  __syncthreads();
  int64_t wanted, free;
  asg_sums(a, used, before, red, wanted, free);
  asg_list(a, used, before[tid], wanted, free);
  __threadfence_block();
  __syncthreads();
  for (int t = wave * 64; t < a.tokens; t += ASG_BLOCK) asg_slots(a, t);
  for (int b = wave; b < a.rows; b += ASG_BLOCK / 64) asg_fill(a, b, lane, 64);
}
// the bitmap of a share of the rows
extern "C" __global__ __launch_bounds__(ASG_BLOCK) void nk_assign_mark(AssignArgs a) {
  __shared__ uint32_t used[ASG_WORDS];
  const int tid = threadIdx.x, wave = tid >> 6, words = (a.pages + 31) / 32;
  for (int i = tid; i < words; i += ASG_BLOCK) used[i] = i == words - 1 && (a.pages & 31) ? ~0u << (a.pages & 31) : 0;
  __syncthreads();
  asg_mark(a, used, blockIdx.x * (ASG_BLOCK / 64) + wave, a.parts * (ASG_BLOCK / 64));
  __syncthreads();
  for (int i = tid; i < words; i += ASG_BLOCK) a.marks[(int64_t)blockIdx.x * ((words + 3) & ~3) + i] = used[i];
}
extern "C" __global__ __launch_bounds__(ASG_BLOCK) void nk_assign_plan(AssignArgs a) {
  __shared__ __attribute__((aligned(16))) uint32_t used[ASG_WORDS];
  __shared__ int32_t before[ASG_BLOCK];
  __shared__ int64_t red[2][ASG_BLOCK / 64];
  const int tid = threadIdx.x, words = (a.pages + 31) / 32, pitch = (words + 3) & ~3;
  for (int i = tid * 4; i < words; i += ASG_BLOCK * 4) {
    u32x4 u = {0, 0, 0, 0};
#pragma unroll 8
    for (int p = 0; p < a.parts; ++p) u |= *reinterpret_cast<const u32x4 *>(a.marks + (int64_t)p * pitch + i);
    *reinterpret_cast<u32x4 *>(used + i) = u;
  }
  __syncthreads();
  int64_t wanted, free;
  asg_sums(a, used, before, red, wanted, free);
  asg_list(a, used, before[tid], wanted, free);
}
// a workgroup for each row's entries, then for 256 tokens each
extern "C" __global__ __launch_bounds__(256) void nk_assign_fill(AssignArgs a) {
  if ((int)blockIdx.x < a.rows) {
    asg_fill(a, blockIdx.x, threadIdx.x, 256);
  } else {
    const int t = ((blockIdx.x - a.rows) * 4 + (threadIdx.x >> 6)) * 64;
    if (t < a.tokens) asg_slots(a, t);
  }
}

// ---------------------------------------------------------------------------
// The choice of beams.
//
// Two launches.  The first reads the logits once: a wave has 2048 of a row in
// registers, their largest value m, sum of 2^((x - m) log2 e) and the K best (K:
// beams); a workgroup joins its waves' lists.  The K best of a wave: the K-th largest
// of its lanes' largest values bounds them from below; what is not below it (a few more
// than K) is listed in LDS and ranked one against the other; more than LIST of them
// (ties) are taken in K rounds.
//
// The second, a workgroup per group, ranks the segments' best by score, value and
// place; an entry with j before it in a list whose best has rank r has r + j
// better ones, so K (K + 1) / 2 entries are left to rank.
//
// 16 groups of 8 beams of 151936 logits (bf16): 16 and 7.6 us; one of 4 of 32000 (fp32): 6
// and 4.6.  The first is bound by the instructions of a wave's 2048 logits (a quarter of
// those beams have ended and are not read: 29 MB, 1.8 TB/s; 64 groups of 32 of 30000 in
// fp32, none ended, 4.3), the second by its chain: two reads, two rankings.
// ---------------------------------------------------------------------------
struct SelectArgs {
  const void *x;
  const float *scores;
  const int32_t *ended;
  int32_t *tokens, *parents;
  float *out;
  int32_t *ends;
  float2 *sums;   // (rows, nseg): largest value, sum
  float2 *best;   // (rows, nseg, K): value, token (as bits); tokens of -1: no more
  int64_t ld;
  int32_t groups, beams, vocab, nseg, end;
};
#define SEL_WAVE 2048
#define SEL_LIST 256
#define SEL_BEAMS 32

// A value and its place as one number: the larger value first, then the lower place.
// (No number, and infinitely little, are below SEL_LEAST.)
#define SEL_LEAST ((u64)0x00800000u << 32)
NK_DEVICE uint32_t sel_order(float v) {
  const uint32_t u = __float_as_uint(v + 0.f);  // (one zero)
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
NK_DEVICE u64 sel_key(float v, int i) { return (u64)sel_order(v) << 32 | (uint32_t)~i; }

template <typename T>
__device__ __forceinline__ void select_top_body(const SelectArgs &a) {
  constexpr int E = 16 / sizeof(T), U = 32 / E;  // elements of a piece, pieces of a lane
  __shared__ u64 list[4][SEL_LIST];
  __shared__ u64 best[4][SEL_BEAMS];
  __shared__ float2 ms[4];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = blockIdx.x / a.nseg, seg = blockIdx.x % a.nseg, K = a.beams;
  if (a.ended[r] != 0) return;  // (not read)
  const T *x = (const T *)a.x + r * a.ld;
  const int off = (int)(((uintptr_t)x & 15) / sizeof(T));  // elements of the first piece before the row
  const int i0 = (seg * 4 + wave) * SEL_WAVE - off + lane * E;
  float v[32];
  float top = -INFINITY;
  {
    uint4 w[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u * 64 * E;
      if (i >= 0 && i + E <= a.vocab) w[u] = *reinterpret_cast<const uint4 *>(x + i);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u * 64 * E;
      if (i >= 0 && i + E <= a.vocab) {
        T y[E];
        __builtin_memcpy(y, &w[u], 16);
#pragma unroll
        for (int e = 0; e < E; ++e) v[u * E + e] = Elt<T>::load(y, e);
      } else {  // an end
#pragma unroll
        for (int e = 0; e < E; ++e) v[u * E + e] = i + e >= 0 && i + e < a.vocab ? Elt<T>::load(x, i + e) : -INFINITY;
      }
    }
  }
#pragma unroll
  for (int e = 0; e < 32; ++e) top = fmaxf(top, v[e]);  // (fmaxf drops NaN)
  const float m = wave_max(top);
  float sum = 0.f;
  if (fabsf(m) < INFINITY) {
    // 2^(x L - c), with c = RN(m L): what c is off by, d = m L - c, is a factor 2^-d of all.
    // From |c| = 2^24 on d may be 1 and more, and later so large that the terms overflow
    // or vanish: the differences there, as with NaN logits and ones past fp32's range times L.
    const float L = 1.44269504088896340736f, c = m * L, d = __builtin_fmaf(m, L, -c);
#pragma unroll
    for (int e = 0; e < 32; ++e) sum += __builtin_amdgcn_exp2f(__builtin_fmaf(v[e], L, -c));
    sum *= __builtin_amdgcn_exp2f(-d);
    if (__any(sum != sum) || !(fabsf(d) < 1.f)) {
      sum = 0.f;
#pragma unroll
      for (int e = 0; e < 32; ++e) sum += v[e] == v[e] ? __builtin_amdgcn_exp2f((v[e] - m) * L) : 0.f;
    }
  } else if (m > 0.f) {  // infinite logits share the weight
#pragma unroll
    for (int e = 0; e < 32; ++e) sum += v[e] == m ? 1.f : 0.f;
  }
  sum = wave_sum(sum);
  // the K-th largest of the lanes' largest values, its key's high half: as many values
  // are not below it
  const uint32_t key = sel_order(top) >> 16;
  uint32_t kth = 0;
#pragma unroll
  for (uint32_t bit = 0x8000; bit; bit >>= 1) kth |= __popcll(__ballot(key >= (kth | bit))) >= K ? bit : 0;
  kth <<= 16;
  float low = __uint_as_float(kth & 0x80000000u ? kth & 0x7fffffffu : ~kth);
  low = low > -3.40282347e38f ? low : -3.40282347e38f;  // (-inf, or what is no number, is listed nowhere)
  int total = 0;
#pragma unroll
  for (int e = 0; e < 32; ++e) {
    const bool in = v[e] >= low;
    const u64 those = __ballot(in);
    if (those == 0) continue;
    const int at = total + __builtin_amdgcn_mbcnt_hi((uint32_t)(those >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)those, 0));
    if (in && at < SEL_LIST) list[wave][at] = sel_key(v[e], i0 + e / E * 64 * E + e % E);
    total += __popcll(those);
  }
  const int count = min(total, K);
  if (total <= SEL_LIST) {
    __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0): the wave's own list
    asm volatile("" ::: "memory");
    for (int k = lane; k < total; k += 64) {
      const u64 y = list[wave][k];
      int before = 0;
#pragma unroll 8
      for (int q = 0; q < total; ++q) before += list[wave][q] > y ? 1 : 0;
      if (before < K) best[wave][before] = y;
    }
  } else {
    u64 last = ~0ull;  // taken
    for (int k = 0; k < count; ++k) {
      u64 y = 0;
#pragma unroll
      for (int e = 0; e < 32; ++e) {
        const u64 z = v[e] >= low ? sel_key(v[e], i0 + e / E * 64 * E + e % E) : 0;
        y = z < last && z > y ? z : y;
      }
#pragma unroll
      for (int o = 32; o; o >>= 1) y = max(y, (u64)__shfl_xor(y, o, 64));
      if (lane == 0) best[wave][k] = y;
      last = y;
    }
  }
  if (lane >= count && lane < K) best[wave][lane] = (u64)(4 * SEL_BEAMS - wave * SEL_BEAMS - lane);  // (nothing, in order)
  if (lane == 0) ms[wave] = make_float2(m, sum);
  __syncthreads();
  const int64_t at = (int64_t)r * a.nseg + seg;
  if (threadIdx.x < 4 * K) {
    const int w = threadIdx.x / K, k = threadIdx.x % K;
    const u64 y = best[w][k];
    int before = k;
    // (of another list as many as are before this one)
#pragma unroll
    for (int o = 1; o < 4; ++o) {
      const int u = (w + o) & 3;
      int lo = 0, hi = K;
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (best[u][mid] > y) lo = mid + 1; else hi = mid;
      }
      before += lo;
    }
    if (before < K) {
      const uint32_t u = (uint32_t)(y >> 32);
      const bool is = y >= SEL_LEAST;
      a.best[at * K + before] = make_float2(is ? __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u) : -INFINITY,
                                            __int_as_float(is ? (int)~(uint32_t)y : -1));
    }
  }
  if (threadIdx.x == 0) {
    const float t = fmaxf(fmaxf(ms[0].x, ms[1].x), fmaxf(ms[2].x, ms[3].x));
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) s += ms[w].x == t ? ms[w].y : ms[w].x == -INFINITY ? 0.f : ms[w].y * exp_acc(ms[w].x - t);
    a.sums[at] = make_float2(t, s);
  }
}
extern "C" __global__ __launch_bounds__(256) void nk_select_top_bf16(SelectArgs a) { select_top_body<bf16>(a); }
extern "C" __global__ __launch_bounds__(256) void nk_select_top_f16(SelectArgs a) { select_top_body<f16>(a); }
extern "C" __global__ __launch_bounds__(256) void nk_select_top_f32(SelectArgs a) { select_top_body<float>(a); }

#define SEL_BLOCK 1024
#define SEL_HEADS 2048  // beams x segments at most
#define SEL_LEFT (SEL_BEAMS * (SEL_BEAMS + 1) / 2)
#define SEL_NONE 0xffffffffu

// a score in its order among all, places packed as beam * 2^22 + token
NK_DEVICE bool sel_better(double s, uint32_t p, double t, uint32_t q) { return (s > t) | ((s == t) & (p < q)); }

// sums over 2, 4, 8 and 16 neighbouring lanes by lane moves, one after the other: with the
// neighbour, the other pair, and mirrored in halves of a row and in a row
template <int CTRL>
NK_DEVICE int lanes_swapped(int v) { return __builtin_amdgcn_update_dpp(0, v, CTRL, 0xf, 0xf, false); }
template <int CTRL>
NK_DEVICE double lanes_swapped(double v) {
  const u64 u = __double_as_longlong(v);
  const uint32_t lo = lanes_swapped<CTRL>((int)(uint32_t)u), hi = lanes_swapped<CTRL>((int)(uint32_t)(u >> 32));
  return __longlong_as_double((u64)hi << 32 | lo);
}
NK_DEVICE double sel_wave_sum(double v) {
  v += lanes_swapped<0xB1>(v);   // quad_perm 1 0 3 2
  v += lanes_swapped<0x4E>(v);   // quad_perm 2 3 0 1
  v += lanes_swapped<0x141>(v);  // row_half_mirror
  v += lanes_swapped<0x140>(v);  // row_mirror
  const int64_t u = __double_as_longlong(v);
  return (__longlong_as_double(lane_of(u, 0)) + __longlong_as_double(lane_of(u, 16))) +
         (__longlong_as_double(lane_of(u, 32)) + __longlong_as_double(lane_of(u, 48)));
}

// order[r]: the entry of rank r < K of n (those with a place), by a workgroup.  Up to
// DIRECT are ranked each against all, some threads side by side.  Of more, the first
// wave lists those that can count, as above: what is not below the K-th largest of its
// lanes' largest, by the upper halves (152 lists of 8 beams: 13 us for the launch with
// each against all, 8.7 so, of 36 entries or 64 lists no less; 992 lists of 32 beams: 153
// and 16).  S threads rank an entry; 16 at most, as their sums are a chain (4 beams: 6.3 us
// with 64, 4.6 so).
#define SEL_DIRECT 64
struct SelFew {
  uint16_t list[SEL_HEADS];
  uint32_t n;
};
NK_DEVICE void sel_rank(const double *s, const uint32_t *p, int n, int K, int32_t *order, SelFew &few) {
  const int tid = threadIdx.x, lane = tid & 63;
  const bool all = n <= SEL_DIRECT;
  int c = n;
  if (!all) {
    if (tid < 64) {
      auto key = [&](int i) __attribute__((always_inline)) {
        const uint32_t u = (uint32_t)__double2hiint(s[i] + 0.0);
        return p[i] != SEL_NONE ? max(u & 0x80000000u ? ~u : u | 0x80000000u, 1u) : 0u;
      };
      uint32_t top = 0, low = 0;
#pragma unroll 4
      for (int i = lane; i < n; i += 64) top = max(top, key(i));
#pragma unroll
      for (uint32_t bit = 0x80000000u; bit; bit >>= 1) low |= __popcll(__ballot(top >= (low | bit))) >= K ? bit : 0;
      low = max(low, 1u);
      uint32_t at = 0;
#pragma unroll 4
      for (int i0 = 0; i0 < n; i0 += 64) {
        const bool in = i0 + lane < n && key(min(i0 + lane, n - 1)) >= low;
        const u64 those = __ballot(in);
        if (in) few.list[at + __popcll(those & ((1ull << lane) - 1))] = (uint16_t)(i0 + lane);
        at += __popcll(those);
      }
      if (lane == 0) few.n = at;
    }
    __syncthreads();
    c = few.n;
  }
  auto id = [&](int x) { return all ? x : (int)few.list[x]; };
  int S = 1;
  while (S < 16 && c * S * 2 <= SEL_BLOCK) S *= 2;
  for (int x = tid; x < (c * S + 63) / 64 * 64; x += SEL_BLOCK) {
    const int i = id(min(x / S, c - 1));
    const double y = s[i];
    const uint32_t z = p[i];
    int rank = 0;
#pragma unroll 4
    for (int q = x % S; q < c; q += S) rank += (p[id(q)] != SEL_NONE) & sel_better(s[id(q)], p[id(q)], y, z) ? 1 : 0;
    if (S > 1) rank += lanes_swapped<0xB1>(rank);
    if (S > 2) rank += lanes_swapped<0x4E>(rank);
    if (S > 4) rank += lanes_swapped<0x141>(rank);
    if (S > 8) rank += lanes_swapped<0x140>(rank);
    if (x % S == 0 && x / S < c && z != SEL_NONE && rank < K) order[rank] = i;
  }
  __syncthreads();
}

extern "C" __global__ __launch_bounds__(SEL_BLOCK) void nk_select_pick(SelectArgs a) {
  __shared__ SelFew few;
  __shared__ double hs[SEL_HEADS];
  __shared__ uint32_t hp[SEL_HEADS];
  __shared__ double cs[SEL_LEFT];
  __shared__ uint32_t cp[SEL_LEFT];
  __shared__ double base[SEL_BEAMS];
  __shared__ float largest[SEL_BEAMS];
  __shared__ int32_t order[SEL_BEAMS];  // the lists of the K best heads; -1: none
  __shared__ int32_t kind[SEL_BEAMS];  // 0: nothing, 1: its logits, 2: ended
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = blockIdx.x, K = a.beams, heads = K * a.nseg;
  // the lists' best are on their way meanwhile
  float2 mine[SEL_HEADS / SEL_BLOCK];
#pragma unroll
  for (int i = 0; i < SEL_HEADS / SEL_BLOCK; ++i)
    mine[i] = a.best[((int64_t)g * heads + min(tid + i * SEL_BLOCK, heads - 1)) * K];
  for (int b = wave; b < K; b += SEL_BLOCK / 64) {
    const int r = g * K + b;
    const float s = a.scores[r];
    const bool over = a.ended[r] != 0;
    int what = s == s && s > -INFINITY ? (over ? 2 : 1) : 0;
    double z = (double)s;
    float m = -INFINITY;
    if (what == 1) {
      for (int i = lane; i < a.nseg; i += 64) m = fmaxf(m, a.sums[(int64_t)r * a.nseg + i].x);
      m = wave_max(m);
      if (m == -INFINITY) what = 0;
      double sum = 0.0;
      for (int i = lane; i < a.nseg; i += 64) {
        const float2 y = a.sums[(int64_t)r * a.nseg + i];
        sum += y.x == m ? (double)y.y : y.x == -INFINITY ? 0.0 : (double)y.y * exp_acc(y.x - m);
      }
      z -= log(sel_wave_sum(sum));
    }
    if (lane == 0) base[b] = z, largest[b] = m, kind[b] = what;
  }
  for (int i = tid; i < K * (K + 1) / 2; i += SEL_BLOCK) cp[i] = SEL_NONE;
  if (tid < K) order[tid] = -1;
  __syncthreads();
  // entry y, j-th of list h: false where there is none
  auto entry = [&](int h, int j, float2 y, double &s, uint32_t &p) {
    const int b = h / a.nseg, i = h % a.nseg;
    if (kind[b] == 0 || (kind[b] == 2 && (i || j))) return false;
    if (kind[b] == 2) {
      s = base[b], p = (uint32_t)b << 22 | (uint32_t)max(a.end, 0);
      return true;
    }
    const int t = __float_as_int(y.y);
    if (t < 0 || (y.x != largest[b] && largest[b] == INFINITY)) return false;
    s = base[b] + (y.x == largest[b] ? 0.0 : (double)y.x - (double)largest[b]), p = (uint32_t)b << 22 | (uint32_t)t;
    return true;
  };
#pragma unroll
  for (int i = 0; i < SEL_HEADS / SEL_BLOCK; ++i) {
    const int h = tid + i * SEL_BLOCK;
    double s;
    uint32_t p;
    if (h >= heads) break;
    const bool is = entry(h, 0, mine[i], s, p);
    hs[h] = is ? s : 0.0;
    hp[h] = is ? p : SEL_NONE;
  }
  __syncthreads();
  sel_rank(hs, hp, heads, K, order, few);
  // entry j of the list whose best has rank r: a thread for each r + j < K
  for (int c = tid; c < K * K; c += SEL_BLOCK) {
    const int r = c / K, j = c % K;
    if (r + j >= K || order[r] < 0) continue;
    double t;
    uint32_t q;
    if (!entry(order[r], j, a.best[((int64_t)g * heads + order[r]) * K + j], t, q)) continue;
    const int to = r * K - r * (r - 1) / 2 + j;
    cs[to] = t, cp[to] = q;
  }
  __syncthreads();
  const int n = K * (K + 1) / 2;
  if (tid < K) order[tid] = -1;
  __syncthreads();
  sel_rank(cs, cp, n, K, order, few);
  if (tid < K && order[tid] >= 0) {
    const double s = cs[order[tid]];
    const uint32_t p = cp[order[tid]];
    const int b = p >> 22, t = kind[b] == 2 ? a.end : (int)(p & 0x3fffff), to = g * K + tid;
    a.tokens[to] = t;
    a.parents[to] = b;
    a.out[to] = (float)s;
    a.ends[to] = kind[b] == 2 || t == a.end ? 1 : 0;
  } else if (tid < K) {  // too few continuations
    a.tokens[g * K + tid] = -1;
    a.parents[g * K + tid] = tid;
    a.out[g * K + tid] = -INFINITY;
    a.ends[g * K + tid] = a.ended[g * K + tid] != 0;
  }
}

// ---------------------------------------------------------------------------
// Caches behind their parents.
//
// A thread has one place (an entry of the tables, 16 bytes of a page) of every
// beam of a group: it reads what all of them come from, then writes, so no
// thread reads what another has written.  Beams that are their own parents move
// nothing.  Bound by memory (32 groups of 8 beams with parents at random, pages of 128
// rows of 1024 codes: each parent read once and each beam with another parent written,
// 56 MB in 12 us, 4.7 TB/s), small ones by two dependent reads (4 beams: 3.6 us).
// ---------------------------------------------------------------------------
struct ReorderArgs {
  const int32_t *parents, *lens;
  int32_t *tables;
  void *k, *v;
  int32_t *ke, *ve;   // null: none
  int64_t row;        // bytes of a cache row
  int32_t groups, beams, width, page, pages, hkv;
  int32_t tblocks, kblocks;  // workgroups of a group for the tables and for each cache
};

template <int K, typename U>
__device__ __forceinline__ void reorder_body(const ReorderArgs &a) {
  __shared__ int32_t up[K], from[K], to[K];  // a beam's parent; pages, -1 where nothing moves
  const int per = a.tblocks + 2 * a.kblocks + (a.ke ? 1 : 0), tid = threadIdx.x;
  const int g = blockIdx.x / per, part = blockIdx.x % per;
  const int len = (int)min((int64_t)max(a.lens[(int64_t)g * a.beams], 0), (int64_t)a.width * a.page);
  const int full = len / a.page, tail = len % a.page;
  int32_t *table = a.tables + (int64_t)g * a.beams * a.width;
  if (part < a.tblocks ? part * 256 >= full : tail == 0) return;
  if (tid < K) {
    const int b = min(tid, a.beams - 1), p = a.parents[(int64_t)g * a.beams + b];
    const bool moves = tid < a.beams && p >= 0 && p < a.beams && p != b;
    up[tid] = moves ? p : tid;
    int x = -1, y = -1;
    if (moves && part >= a.tblocks) {  // (full is below width: the length leaves a page in part filled)
      x = table[(int64_t)p * a.width + full], y = table[(int64_t)b * a.width + full];
      if (x < 0 || x >= a.pages || y < 0 || y >= a.pages) x = y = -1;  // (no page, on either side)
    }
    from[tid] = x, to[tid] = y;
  }
  __syncthreads();
  if (part < a.tblocks) {
    const int j = part * 256 + tid;
    if (j >= full) return;
    int32_t x[K];
#pragma unroll
    for (int b = 0; b < K; ++b) {
      x[b] = table[(int64_t)min(__builtin_amdgcn_readfirstlane(up[b]), a.beams - 1) * a.width + j];
    }
#pragma unroll
    for (int b = 0; b < K; ++b)
      if (__builtin_amdgcn_readfirstlane(up[b]) != b) table[(int64_t)b * a.width + j] = x[b];
    return;
  }
  const int which = (part - a.tblocks) / a.kblocks;  // 0: keys, 1: values, 2: exponents
  // (a page's address is uniform, the place in it 32 bits of a lane; what moves
  // nothing reads page 0, since a read in a branch would be waited for at its end)
  auto move = [&](auto *x, int64_t pitch, uint32_t at) __attribute__((always_inline)) {
    typename std::remove_reference<decltype(*x)>::type y[K];
#pragma unroll
    for (int b = 0; b < K; ++b) {
      const auto *src = x + __builtin_amdgcn_readfirstlane(max(from[b], 0)) * pitch;
      y[b] = src[at];
    }
#pragma unroll
    for (int b = 0; b < K; ++b) {
      const int p = __builtin_amdgcn_readfirstlane(to[b]);
      auto *dst = x + p * pitch;
      if (p >= 0) dst[at] = y[b];
    }
  };
  if (which < 2) {
    const int64_t at = (int64_t)((part - a.tblocks) % a.kblocks) * 256 + tid, units = a.row / (int64_t)sizeof(U);  // (of a row)
    if (at < tail * units) move((U *)(which ? a.v : a.k), a.page * units, (uint32_t)at);
  } else {
    for (int h = tid; h < 2 * a.hkv; h += 256) move(h < a.hkv ? a.ke : a.ve, a.hkv, h < a.hkv ? h : h - a.hkv);
  }
}
#define NK_REORDER(K)                                                                                                    \
  extern "C" __global__ __launch_bounds__(256) void nk_beam_reorder16_k##K(ReorderArgs a) { reorder_body<K, u32x4>(a); }  \
  extern "C" __global__ __launch_bounds__(256) void nk_beam_reorder1_k##K(ReorderArgs a) { reorder_body<K, uint8_t>(a); }
NK_REORDER(4)
NK_REORDER(8)
NK_REORDER(32)
