// What the forward kernels on rows of scores share: sums of exponentials above a moving maximum, and results of a row.
//
// A row's sums are held relative to the running maximum m, in base 2: with k = log2 e and c = m k,
//   s = sum 2^(x k - c),   t = sum 2^(d) d, d = x k - c,
// so that an entry costs one fused multiply-add, one exponential and two or three additions.  c is rounded, but it is the same
// c in every term.  In the end all is taken relative to m itself, by the term of m (u = ln 2):
//   dm = m k - c,   q = log(s / 2^dm),   log Z = m + q,   log p[g] = (x[g] k - c - dm) u - q,   H = q - u (t - s dm) / s,
// where a row of one category comes out as 0, 0 exactly.
// From |m| = 2^30 on dm could pass the range of the exponential.  There entries that are not m lie 64 or more below it and
// count for nothing; k = u = 1 takes the differences exactly, and s becomes the number of entries that are m.
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
// (in every step below c is the product as rounded, never fused into what it is subtracted from)
template <typename T>
struct RowSums {
  float m = masked_from<T>(), c = 0.f, k = kLog2e, s = 0.f, t = 0.f;
  static __device__ __forceinline__ bool far(float m) { return masked_from<T>() < -1e30f && fabsf(m) >= 1073741824.f; }
  __device__ __forceinline__ void set(float to) {     // m, where nothing is summed yet
#pragma clang fp contract(off)
    m = to;
    k = far(to) ? 1.f : kLog2e;
    c = to * k;
  }
  __device__ __forceinline__ void raise(float to) {   // m and c to a larger maximum, the sums with them
#pragma clang fp contract(off)
    const bool near = m > masked_from<T>() && !far(m) && !far(to);
    const float c0 = c;
    set(to);
    const float dc = near ? fmaxf(c0 - c, -200.f) : -200.f, al = __builtin_amdgcn_exp2f(dc);
    t = al * (t + s * dc);
    s *= al;
  }
  template <bool kEnt>
  __device__ __forceinline__ void add(float x, float& gs, float& gt) const {   // to a group's own sums
    const float d = fmaf(x, k, -c), e = __builtin_amdgcn_exp2f(d);
    gs += e;
    if (kEnt) gt = fmaf(e, fmaxf(d, -200.f), gt);   // (0 where e is: d may be -inf)
  }
  // the sums of a row from those that every lane of the wave holds (m, s, t) of other entries
  __device__ __forceinline__ void join_lanes(float4 o) {
#pragma clang fp contract(off)
    m = over_lanes<64>(o.x, Larger());
    if (m > masked_from<T>()) set(m);
    const float d0 = o.x * kLog2e - c;
    const float d = o.x == m ? 0.f : o.x > masked_from<T>() && !far(o.x) && !far(m) ? fmaxf(d0, -200.f) : -200.f, al = __builtin_amdgcn_exp2f(d);
    t = over_lanes<64>(al * (o.z + o.y * d), Sum());
    s = over_lanes<64>(o.y * al, Sum());
  }
};

template <typename T>
struct RowResult {
  bool nan, none;
  float c, k, u, dm, q, z;
  __device__ __forceinline__ explicit RowResult(const RowSums<T>& sum) {
    nan = !(sum.s < INFINITY);
    none = !nan && !(sum.m > masked_from<T>());
    c = sum.c;
    k = sum.k;
    u = RowSums<T>::far(sum.m) ? 1.f : kLn2;
    dm = fmaf(sum.m, k, -c);
    q = logf(sum.s / __builtin_amdgcn_exp2f(dm));
    z = sum.m + q;
  }
  __device__ __forceinline__ float log_sum() const { return nan ? NAN : none ? -INFINITY : z; }
  __device__ __forceinline__ float entropy(const RowSums<T>& sum) const {
    const float one = __builtin_amdgcn_exp2f(dm);   // (of one category alone: its term, in both sums)
    const float t = sum.s == one && sum.t == one * dm ? 0.f : fmaf(-sum.s, dm, sum.t);
    return nan || none ? NAN : fmaf(-t / sum.s, u, q);
  }
  __device__ __forceinline__ float logp(float x) const {   // of an entry of the row that is seen as x
    return nan ? NAN : none || x <= masked_from<T>() ? -INFINITY : fmaf(fmaf(x, k, -c) - dm, u, -q);
  }
  template <typename Load>
  __device__ __forceinline__ float given(int64_t g, int32_t cats, Load&& load) const {
    return g < 0 ? 0.f : g >= cats || nan ? NAN : logp(load(g));
  }
};
#endif

}  // namespace pcm
