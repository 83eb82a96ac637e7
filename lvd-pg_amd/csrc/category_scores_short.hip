// Short rows of scores, and rows that lie side by side (stride 1 from row to row, as a forest's forward pass leaves them).
#include "category_stats.hip.hpp"

namespace pcm {

namespace {
// Rows of up to 256 neighbouring categories: 16 lanes a row, all of it in registers, four rows a wave.  A lane holds kGroups
// times 16 bytes; the sums need no running maximum.  The likeliest are found one after the other: the largest entry of 16 lanes
// (four steps), the lowest index that has it (four), and out it goes.
template <typename T, int kGroups, bool kTop, bool kCkpt>
__global__ __launch_bounds__(256) void score_short_kernel(RowsRef x, RowsShape shape, GivenRef given, int top, ScoreOut out, CkptRef ckpt) {
  constexpr int kVec = 16 / (int)sizeof(T), kEntries = kGroups * kVec;
  const int lane = threadIdx.x & 15;
  const int64_t rows = shape.rows(), step = (int64_t)gridDim.x * 16;
  const int64_t pitch = (shape.cats + 15) / 16 * 16, blocks = (shape.cats + kCkptBlock - 1) / kCkptBlock;
  for (int64_t r0 = (int64_t)blockIdx.x * 16; r0 < rows; r0 += step) {   // (the same number of turns for all lanes of the workgroup)
    const int64_t own = r0 + (threadIdx.x >> 4);
    const bool mine = own < rows;
    const uint32_t r = (uint32_t)(mine ? own : rows - 1);
    const int64_t e = shape.vars == 1 ? r : r / (uint32_t)shape.vars, v = shape.vars == 1 ? 0 : r % (uint32_t)shape.vars;
    const T* const row = static_cast<const T*>(x.p) + e * x.stride_ex + v * x.stride_var;
    float y[kGroups][kVec];
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
      const int c = (g * 16 + lane) * kVec;
      raw4 raw;
      if (c + kVec <= shape.cats) raw = load16(row + c);
      else {
        T w[kVec];
#pragma unroll
        for (int i = 0; i < kVec; ++i) w[i] = c + i < shape.cats ? row[c + i] : (T)-INFINITY;
        raw = __builtin_bit_cast(raw4, w);
      }
      unpack(raw, y[g], T());
    }
    RowSums<T> sum;
    float largest = -INFINITY;
#pragma unroll
    for (int g = 0; g < kGroups; ++g)
#pragma unroll
      for (int i = 0; i < kVec; ++i) largest = fmaxf(largest, y[g][i]);
    largest = over_lanes<16>(largest, Larger());
    if (largest > masked_from<T>()) {
      sum.m = largest;
      sum.c = largest * kLog2e;
    }
    float s = 0.f, t = 0.f;
#pragma unroll
    for (int g = 0; g < kGroups; ++g)
#pragma unroll
      for (int i = 0; i < kVec; ++i) sum.template add<true>(y[g][i], s, t);
    sum.s = over_lanes<16>(s, Sum());
    sum.t = over_lanes<16>(t, Sum());
    const RowResult<T> res(sum);
    if (mine) {
      for (int j = lane; j < given.slots; j += 16)
        out.logp[(int64_t)r * given.slots + j] = res.given(given_at(given, e, v, j), shape.cats, [&](int64_t g) { return seen(row[g]); });
      if (lane == 0) {
        if (out.log_sum) out.log_sum[r] = res.log_sum();
        if (out.entropy) out.entropy[r] = res.entropy(sum);
      }
    }
    if constexpr (kCkpt) {
#pragma unroll
      for (int g = 0; g < kGroups; ++g) {
        const int c = (g * 16 + lane) * kVec;
        const BlockCodes<kVec> k = encode_block<T>(y[g]);
        if (mine) store_codes(ckpt, k, r, c, shape.cats, pitch, blocks);
      }
    }
    if constexpr (kTop) {
      int32_t index = -1;
      float value = -INFINITY;
      for (int j = 0; j < top; ++j) {
        float best = -INFINITY;
        int at = 0x7fffffff;
#pragma unroll
        for (int g = 0; g < kGroups; ++g)
#pragma unroll
          for (int i = 0; i < kVec; ++i)
            if (y[g][i] > best) {
              best = y[g][i];
              at = (g * 16 + lane) * kVec + i;
            }
        const float w = over_lanes<16>(best, Larger());
        uint32_t low = best == w ? (uint32_t)at : 0x7fffffffu;
        low = min(low, (uint32_t)__builtin_amdgcn_mov_dpp(low, 0xB1, 0xf, 0xf, false));
        low = min(low, (uint32_t)__builtin_amdgcn_mov_dpp(low, 0x4E, 0xf, 0xf, false));
        low = min(low, (uint32_t)__builtin_amdgcn_mov_dpp(low, 0x141, 0xf, 0xf, false));
        low = min(low, (uint32_t)__builtin_amdgcn_mov_dpp(low, 0x140, 0xf, 0xf, false));
        const bool some = w > masked_from<T>();
        if (lane == j) {
          index = some ? (int32_t)low : -1;
          value = some ? w : -INFINITY;
        }
#pragma unroll
        for (int g = 0; g < kGroups; ++g)
#pragma unroll
          for (int i = 0; i < kVec; ++i)
            if (low == (uint32_t)((g * 16 + lane) * kVec + i)) y[g][i] = -INFINITY;
      }
      if (mine && lane < top) {
        out.top[(int64_t)r * top + lane] = res.nan ? -1 : index;
        out.top_logp[(int64_t)r * top + lane] = index < 0 && !res.nan ? -INFINITY : res.logp(value);
      }
    }
  }
}

// A lane per row: rows that lie side by side, and rows of a few categories.  `parts` waves share the categories of 64 rows and
// meet in LDS; each lane keeps its sums and, sorted in, its kList likeliest.
template <typename T, int kList>
__global__ __launch_bounds__(1024) void score_column_kernel(RowsRef x, RowsShape shape, GivenRef given, int top, ScoreOut out, int parts,
                                                            bool examples_first) {
  constexpr int kStep = 8, kWords = 3 + 2 * kList;
  extern __shared__ float column_lds[];   // [waves][kWords][64]
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int sets = (blockDim.x >> 6) / parts, set = wave / parts, q = wave % parts;
  const int64_t rows = shape.rows();
  const int len = ((shape.cats + parts - 1) / parts + kStep - 1) / kStep * kStep;
  const int first = min(q * len, shape.cats), end = min(first + len, shape.cats);
  for (int64_t n0 = (int64_t)blockIdx.x * sets * 64; n0 < rows; n0 += (int64_t)gridDim.x * sets * 64) {
    const int64_t at = n0 + set * 64 + lane;
    const bool mine = at < rows;
    const uint32_t n = (uint32_t)(mine ? at : rows - 1);
    uint32_t e, v;
    if (examples_first) {
      v = n / (uint32_t)shape.examples;
      e = n - v * (uint32_t)shape.examples;
    } else {
      e = shape.vars == 1 ? n : n / (uint32_t)shape.vars;
      v = n - e * (uint32_t)shape.vars;
    }
    const T* const row = static_cast<const T*>(x.p) + e * x.stride_ex + v * x.stride_var;
    RowSums<T> sum;
    float value[kList ? kList : 1];
    int32_t index[kList ? kList : 1];
#pragma unroll
    for (int j = 0; j < kList; ++j) {
      value[j] = masked_from<T>();
      index[j] = -1;
    }
    // behind those that are as large: they have lower indices
    auto sort_in = [&](float w, int32_t i) {
#pragma unroll
      for (int j = kList - 1; j >= 0; --j) {
        const bool here = w > value[j], above = j > 0 && w > value[j ? j - 1 : 0];
        value[j] = above ? value[j ? j - 1 : 0] : here ? w : value[j];
        index[j] = above ? index[j ? j - 1 : 0] : here ? i : index[j];
      }
    };
    for (int c0 = first; c0 < end; c0 += kStep) {
      float y[kStep], largest = -INFINITY, s = 0.f, t = 0.f;
#pragma unroll
      for (int i = 0; i < kStep; ++i) y[i] = c0 + i < end ? seen(row[(int64_t)(c0 + i) * x.stride_cat]) : -INFINITY;
#pragma unroll
      for (int i = 0; i < kStep; ++i) largest = fmaxf(largest, y[i]);
      if (largest > sum.m) sum.raise(largest);
#pragma unroll
      for (int i = 0; i < kStep; ++i) sum.template add<true>(y[i], s, t);
      sum.s += s;
      sum.t += t;
      if constexpr (kList > 0)
        if (largest > value[kList - 1])
#pragma unroll
          for (int i = 0; i < kStep; ++i)
            if (y[i] > value[kList - 1]) sort_in(y[i], c0 + i);
    }
    if (parts > 1) {
      float* const own = column_lds + (size_t)wave * kWords * 64 + lane;
      if (q > 0) {
        own[0] = sum.m;
        own[64] = sum.s;
        own[128] = sum.t;
#pragma unroll
        for (int j = 0; j < kList; ++j) {
          own[(3 + j) * 64] = value[j];
          own[(3 + kList + j) * 64] = __builtin_bit_cast(float, index[j]);
        }
      }
      __syncthreads();
      if (q == 0) {
        float m = sum.m;
        for (int p = 1; p < parts; ++p) m = fmaxf(m, own[(size_t)p * kWords * 64]);
        if (m > sum.m) sum.raise(m);
        for (int p = 1; p < parts; ++p) {
          const float* const o = own + (size_t)p * kWords * 64;
          RowSums<T> other;
          other.m = o[0];
          other.c = o[0] > masked_from<T>() ? o[0] * kLog2e : 0.f;
          other.s = o[64];
          other.t = o[128];
          if (m > other.m) other.raise(m);
          sum.s += other.s;
          sum.t += other.t;
#pragma unroll 1
          for (int j = 0; j < kList; ++j) {
            const float w = o[(3 + j) * 64];
            if (w > value[kList ? kList - 1 : 0]) sort_in(w, __builtin_bit_cast(int32_t, o[(3 + kList + j) * 64]));
          }
        }
      }
      __syncthreads();   // (the next rows' sums go where these were read)
    }
    if (q == 0 && mine) {
      const RowResult<T> res(sum);
      const int64_t r = (int64_t)e * shape.vars + v;
      for (int j = 0; j < given.slots; ++j)
        out.logp[r * given.slots + j] =
            res.given(given_at(given, e, v, j), shape.cats, [&](int64_t g) { return seen(row[g * x.stride_cat]); });
      if (out.log_sum) out.log_sum[r] = res.log_sum();
      if (out.entropy) out.entropy[r] = res.entropy(sum);
#pragma unroll
      for (int j = 0; j < kList; ++j)
        if (j < top) {
          out.top[r * top + j] = res.nan ? -1 : index[j];
          out.top_logp[r * top + j] = index[j] < 0 && !res.nan ? -INFINITY : res.logp(value[j]);
        }
    }
  }
}

template <typename T, int kGroups>
void launch_short(const RowsRef& x, const RowsShape& shape, const GivenRef& given, int top, const ScoreOut& out, const CkptRef& ckpt,
                  hipStream_t stream) {
  const dim3 grid((unsigned)std::min<int64_t>((shape.rows() + 15) / 16, 1 << 20));
  auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(256), 0, stream, x, shape, given, top, out, ckpt); };
  if (ckpt.codes) top ? launch(score_short_kernel<T, kGroups, true, true>) : launch(score_short_kernel<T, kGroups, false, true>);
  else top ? launch(score_short_kernel<T, kGroups, true, false>) : launch(score_short_kernel<T, kGroups, false, false>);
}

template <typename T, int kList>
void launch_column(const RowsRef& x, const RowsShape& shape, const GivenRef& given, int top, const ScoreOut& out, hipStream_t stream) {
  const int64_t sets = (shape.rows() + 63) / 64;
  const int most = kList > 8 ? 4 : kList > 4 ? 8 : 16;   // (LDS)
  int parts = 1;
  while (parts < most && sets * parts < 4096 && shape.cats / parts >= 32) parts *= 2;
  const int waves = std::max(4, parts), per = waves / parts;
  const int lds = parts > 1 ? waves * (3 + 2 * kList) * 64 * 4 : 0;
  const bool examples_first = shape.vars > 1 && (x.stride_ex == 1 || x.stride_ex == -1);
  hipLaunchKernelGGL((score_column_kernel<T, kList>), dim3((unsigned)std::min<int64_t>((sets + per - 1) / per, 1 << 20)), dim3(64 * waves), lds,
                     stream, x, shape, given, top, out, parts, examples_first);
}
}  // namespace

template <typename T>
bool category_scores_short(const RowsRef& x, const RowsShape& shape, const GivenRef& given, int top, const ScoreOut& out, const CkptRef& ckpt,
                           hipStream_t stream) {
  const bool neighbours = x.stride_cat == 1;
  const bool side_by_side = !neighbours && ((shape.examples > 1 && std::abs(x.stride_ex) == 1) || (shape.vars > 1 && std::abs(x.stride_var) == 1));
  if (top > 16) return false;
  if (side_by_side || (shape.cats <= 16 && !ckpt.codes)) {
    if (top == 0) launch_column<T, 0>(x, shape, given, top, out, stream);
    else if (top <= 4) launch_column<T, 4>(x, shape, given, top, out, stream);
    else if (top <= 8) launch_column<T, 8>(x, shape, given, top, out, stream);
    else launch_column<T, 16>(x, shape, given, top, out, stream);
    return true;
  }
  if (!neighbours || shape.cats > 256) return false;
  constexpr int kGroup = 256 / (int)sizeof(T);   // categories of 16 lanes times 16 bytes
  if (shape.cats <= kGroup) launch_short<T, 1>(x, shape, given, top, out, ckpt, stream);
  else if (shape.cats <= 2 * kGroup) launch_short<T, 2>(x, shape, given, top, out, ckpt, stream);
  else if constexpr (sizeof(T) == 4) launch_short<T, 4>(x, shape, given, top, out, ckpt, stream);
  return true;
}

template bool category_scores_short<float>(const RowsRef&, const RowsShape&, const GivenRef&, int, const ScoreOut&, const CkptRef&, hipStream_t);
template bool category_scores_short<bf16>(const RowsRef&, const RowsShape&, const GivenRef&, int, const ScoreOut&, const CkptRef&, hipStream_t);
template bool category_scores_short<f16>(const RowsRef&, const RowsShape&, const GivenRef&, int, const ScoreOut&, const CkptRef&, hipStream_t);

}  // namespace pcm
