// Attention over a paged cache or plain tensors with a window and sinks
// (attend.h holds the definition and the layout of the work).

#include "attend.h"

using namespace nk;

// ---------------------------------------------------------------------------
// Any head dim to 256, any strides and addresses, fp32 operands: one wave per
// query row.  It reads each key for each query head apart and uses no matrix
// instructions; the 16-bit types of head dims 64 and 128 have the tiled form.
// ---------------------------------------------------------------------------
template <typename T>
__device__ __forceinline__ void attend_rows_body(const AttendArgs &a) {
  const int lane = threadIdx.x & 63;
  const int64_t r = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (r >= (int64_t)a.N * a.Hq) return;
  const int t = (int)(r / a.Hq), h = (int)(r % a.Hq);
  const int b = a.starts ? att_find(a.B, t, [&](int x) { return a.starts[x]; }) : t / a.S;
  float m, l = 0.f, acc[4];
  if (b >= 0) {
    const AttSeq sq = att_seq(a, b);
    const int i = t - sq.lo;
    if (i < sq.n) {
      const AttSpan sp = att_span(a, sq, (i * (a.Hq / a.Hkv) + h % (a.Hq / a.Hkv)) / ATT_ROWS);
      att_row<T>(a, sq, sp, b, i, h, 0, sp.nb, m, l, acc);
    }
  }
  T *o = (T *)a.o + r * a.D;
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (lane + 64 * e < a.D) Elt<T>::store(o, lane + 64 * e, l == 0.f ? 0.f : acc[e] / l);
}
extern "C" __global__ __launch_bounds__(256) void nk_attend_rows_bf16(AttendArgs a) { attend_rows_body<bf16>(a); }
extern "C" __global__ __launch_bounds__(256) void nk_attend_rows_f16(AttendArgs a) { attend_rows_body<f16>(a); }
extern "C" __global__ __launch_bounds__(256) void nk_attend_rows_f32(AttendArgs a) { attend_rows_body<float>(a); }
