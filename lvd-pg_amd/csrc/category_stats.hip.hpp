// What the forward kernels on rows of scores share: sums of exponentials above a moving maximum, and results of a row.
//
// A row's sums are held relative to the running maximum m, in base 2: with c = m log2 e,
//   s = sum 2^(x log2 e - c),   t = sum 2^(d) d, d = x log2 e - c,
// so that an entry costs one fused multiply-add, one exponential and two or three additions.  c is rounded, but it is the same
// c in every term, and r = c - m log2 e is found exactly by one fused multiply-add at the end:
//   log Z = m + r ln 2 + log s,   log p[g] = (x[g] log2 e - c) ln 2 - log s,   H = log s - t ln 2 / s.
// Entries that count as masks never move m off its start, masked_from<T>(), where c = 0 and their terms underflow to 0.
#pragma once

#include "category_rows.hpp"

namespace pcm {

struct ScoreOut {
  float *logp, *log_sum, *entropy, *top_logp;
  int32_t* top;
};

// Short rows and rows that lie side by side; false: not rows of that kind, nothing done.  `ckpt` only with stride_cat == 1.
template <typename T>
bool category_scores_short(const RowsRef& x, const RowsShape& shape, const GivenRef& given, int top, const ScoreOut& out, const CkptRef& ckpt,
                           hipStream_t stream);

#ifdef __HIPCC__
template <typename T>
struct RowSums {
  float m = masked_from<T>(), c = 0.f, s = 0.f, t = 0.f;
  __device__ __forceinline__ void raise(float to) {   // m and c to a larger maximum, the sums with them
    const float c1 = to * kLog2e, dc = m > masked_from<T>() ? fmaxf(c - c1, -200.f) : -200.f, al = __builtin_amdgcn_exp2f(dc);
    t = al * (t + s * dc);
    s *= al;
    m = to;
    c = c1;
  }
  template <bool kEnt>
  __device__ __forceinline__ void add(float x, float& gs, float& gt) const {   // to a group's own sums
    const float d = fmaf(x, kLog2e, -c), e = __builtin_amdgcn_exp2f(d);
    gs += e;
    if (kEnt) gt = fmaf(e, fmaxf(d, -200.f), gt);   // (0 where e is: d may be -inf)
  }
  // the sums of a row from those that every lane of the wave holds (m, s, t) of other entries
  __device__ __forceinline__ void join_lanes(float4 o) {
    m = over_lanes<64>(o.x, Larger());
    c = m > masked_from<T>() ? m * kLog2e : 0.f;
    const float d = o.x > masked_from<T>() ? fmaxf(o.x * kLog2e - c, -200.f) : -200.f, al = __builtin_amdgcn_exp2f(d);
    t = over_lanes<64>(al * (o.z + o.y * d), Sum());
    s = over_lanes<64>(o.y * al, Sum());
  }
};

template <typename T>
struct RowResult {
  bool nan, none;
  float c, ls, z;
  __device__ __forceinline__ explicit RowResult(const RowSums<T>& q) {
    // (beyond 2^127 c would pass the range of float)
    nan = !(q.s < INFINITY) || q.m > 1.7014118e38f;
    none = !nan && !(q.m > masked_from<T>());
    c = q.c;
    ls = logf(q.s);
    z = q.m + fmaf(fmaf(-q.m, kLog2e, q.c), kLn2, ls);
  }
  __device__ __forceinline__ float log_sum() const { return nan ? NAN : none ? -INFINITY : z; }
  __device__ __forceinline__ float entropy(const RowSums<T>& q) const { return nan || none ? NAN : fmaf(-q.t / q.s, kLn2, ls); }
  __device__ __forceinline__ float logp(float x) const {   // of an entry of the row that is seen as x
    return nan ? NAN : none || x <= masked_from<T>() ? -INFINITY : fmaf(fmaf(x, kLog2e, -c), kLn2, -ls);
  }
  template <typename Load>
  __device__ __forceinline__ float given(int64_t g, int32_t cats, Load&& load) const {
    return g < 0 ? 0.f : g >= cats || nan ? NAN : logp(load(g));
  }
};
#endif

}  // namespace pcm
