// Short rows of scores, many rows, and rows that lie side by side (stride 1 from row to row, as a forest's forward pass leaves them).
#include "category_stats.hip.hpp"

namespace pcm {

namespace {
// Rows of neighbouring categories that go a lane each: as many as fill the device with 64 a wave.  Times in us, a lane a row / 16 lanes a
// row (up to 256 categories) or a wave a row: 65536 rows of 128 (f32, 4 likeliest) 17 / 17, 262144 37 / 59, 524288 66 / 113; 32768 rows of
// 512 24 / 56, 65536 of 1000 68 / 118, 65536 of 2000 (bf16) 85 / 144, 8192 of 2000 43 / 24.
constexpr int kShortCats = 256;
constexpr int64_t kLaneRowsShort = 65536, kLaneRows = 32768;   // fewest rows, up to and beyond kShortCats categories
constexpr int kLaneCats = 2048;                                // most categories
// Rows that lie side by side: as many as fill the device with 64 a wave, too; fewer go a wave or more each, which read the same lines at
// the same time.  A lane a row / waves a row, us, f32, entropy, no list: 1024 rows of 128 6.2 / 4.3, 4096 6.4 / 5.8; 1024 of 1000 14 / 8,
// 4096 14 / 30; 1024 of 5000 38 / 34, 4096 40 / 172; 64 of 50000 295 / 25, 1024 298 / 283.  The lines are drawn for rows without a list: with
// 8 likeliest some 4096 rows of 300 take 21 / 16, of 1000 33 / 33, of 5000 92 / 151, of 50000 645 / 2144.
constexpr int64_t kSideRowsShort = 6144, kSideRows = 2048;

// Rows of up to 256 neighbouring categories: 16 lanes a row, all of it in registers, four rows a wave.  A lane holds kGroups
// times 16 bytes; the sums need no running maximum.  The likeliest are found one after the other: the largest entry of 16 lanes
// (four steps), the lowest index that has it (four), and out it goes.  50176 rows of 256 f32 with entropy and checkpoint: 19 us, 3.4 TB/s, one
// round of workgroups.
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
    if (largest > masked_from<T>()) sum.set(largest);
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

// A lane per row: no step across lanes, and what a row costs once is shared by 64.  Rows that lie side by side are read as they are;
// rows of neighbouring categories go through LDS, 128 bytes of each of the wave's 64 rows at a time (kStaged).  A lane takes kStep
// entries: their maximum, their sums, and which of them lie above the last of its kList likeliest, kept sorted.  Those, a few once the
// list has filled, are sorted in one of every lane at a time, a median and a comparison per place.  `parts` waves share the categories
// of 64 rows and meet in LDS.  524288 rows of 128 f32 (kStaged), 4 likeliest, entropy: 65 us, 4.1 TB/s, half of it vector instructions; 32768
// of them side by side: 13 us.
template <typename T, int kList, bool kStaged>
__global__ __launch_bounds__(kStaged ? 256 : 1024, kStaged ? kList > 4 ? 3 : 4 : 1) void score_lane_kernel(RowsRef x, RowsShape shape, GivenRef given, int top, ScoreOut out, int parts,
                                                                         bool examples_first) {
  constexpr int kStep = 16, kWords = 3 + 2 * kList, kVec = 16 / (int)sizeof(T), kTile = 8 * kVec, kPitch = 36;   // (words of a row in LDS)
  extern __shared__ float lane_lds[];   // per wave a tile [64][kPitch] (kStaged); then, of several parts, [waves][kWords][64]
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int sets = (blockDim.x >> 6) / parts, set = wave / parts, q = wave % parts;
  const int64_t rows = shape.rows();
  const int len = ((shape.cats + parts - 1) / parts + kTile - 1) / kTile * kTile;
  const int first = min(q * len, shape.cats), end = min(first + len, shape.cats);
  float* const tile = lane_lds + (size_t)wave * 64 * kPitch;
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
    // behind those that are as large: they have lower indices (w lies above the last)
    auto sort_in = [&](float w, int32_t i) {
#pragma unroll
      for (int j = kList - 1; j > 0; --j) {
        index[j] = w > value[j - 1] ? index[j - 1] : w > value[j] ? i : index[j];
        value[j] = __builtin_amdgcn_fmed3f(w, value[j - 1], value[j]);
      }
      index[0] = w > value[0] ? i : index[0];
      value[0] = fmaxf(w, value[0]);
    };
    // the entries of a step, and one of them by its place
    auto work = [&](const float (&y)[kStep], int c0, auto&& entry) {
      float largest = y[0], s = 0.f, t = 0.f;
#pragma unroll
      for (int i = 1; i < kStep; ++i) largest = __builtin_elementwise_maximum(largest, y[i]);
      if (largest > sum.m) sum.raise(largest);
      if constexpr (kList > 0) {
        uint32_t hit = 0;
#pragma unroll
        for (int i = 0; i < kStep; ++i) hit |= y[i] > value[kList - 1] ? 1u << i : 0u;
        if (__any(__popc(hit) > kStep / 2)) {        // (a list that fills, entries that rise)
#pragma unroll
          for (int i = 0; i < kStep; ++i)
            if (y[i] > value[kList - 1]) sort_in(y[i], c0 + i);
          hit = 0;
        }
        while (hit) {
          const int i = __builtin_ctz(hit);
          hit &= hit - 1;
          const float w = entry(i);
          if (w > value[kList - 1]) sort_in(w, c0 + i);
        }
      }
#pragma unroll
      for (int i = 0; i < kStep; ++i) sum.template add<true>(y[i], s, t);
      sum.s += s;
      sum.t += t;
    };
    if constexpr (kStaged) {
      // rows lie stride_ex apart (one variable); eight lanes hold 128 bytes of a row, a request eight rows
      const int64_t r0 = n0 + set * 64;
      const int in = (lane & 7) * kVec;
      raw4 raw[8];
      auto request = [&](int c0) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int64_t r = min(r0 + i * 8 + (lane >> 3), rows - 1);
          const T* const from = static_cast<const T*>(x.p) + r * x.stride_ex;
          if (c0 + in + kVec <= end) raw[i] = load16(from + c0 + in);
          else {
            T w[kVec];
#pragma unroll
            for (int k = 0; k < kVec; ++k) w[k] = c0 + in + k < end ? from[c0 + in + k] : (T)-INFINITY;
            raw[i] = __builtin_bit_cast(raw4, w);
          }
        }
      };
      if (first < end) request(first);
      for (int c0 = first; c0 < end; c0 += kTile) {
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int i = 0; i < 8; ++i) *reinterpret_cast<raw4*>(tile + (i * 8 + (lane >> 3)) * kPitch + (lane & 7) * 4) = raw[i];
        __builtin_amdgcn_wave_barrier();
        if (c0 + kTile < end) request(c0 + kTile);
        const float* const own = tile + lane * kPitch;
#pragma unroll 1
        for (int h = 0; h < kTile && c0 + h < end; h += kStep) {
          const float* const half = own + h * (int)sizeof(T) / 4;
          float y[kStep];
#pragma unroll
          for (int i = 0; i < kStep / kVec; ++i) {
            float z[kVec];
            unpack(*reinterpret_cast<const raw4*>(half + 4 * i), z, T());
#pragma unroll
            for (int k = 0; k < kVec; ++k) y[i * kVec + k] = z[k];
          }
          work(y, c0 + h, [&](int i) { return seen(reinterpret_cast<const T*>(half)[i]); });
        }
      }
    } else {
      float y[kStep];
      T next[kStep];
      auto request = [&](int c0) {
        const T* const from = row + (int64_t)c0 * x.stride_cat;
#pragma unroll
        for (int i = 0; i < kStep; ++i) next[i] = c0 + i < end ? from[(int64_t)i * x.stride_cat] : (T)-INFINITY;
      };
      request(first);
      for (int c0 = first; c0 < end; c0 += kStep) {
#pragma unroll
        for (int i = 0; i < kStep; ++i) y[i] = seen(next[i]);
        request(c0 + kStep);
        work(y, c0, [&](int i) {
          float a[kStep];
#pragma unroll
          for (int k = 0; k < kStep; ++k) a[k] = y[k];
#pragma unroll
          for (int w = kStep / 2; w > 0; w /= 2)
#pragma unroll
            for (int k = 0; k < w; ++k) a[k] = i & w ? a[k + w] : a[k];
          return a[0];
        });
      }
    }
    if (parts > 1) {
      __syncthreads();                      // (tiles are done with)
      float* const own = lane_lds + (size_t)wave * kWords * 64 + lane;
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
          if (o[0] > masked_from<T>()) other.set(o[0]);
          other.s = o[64];
          other.t = o[128];
          if (m > other.m) other.raise(m);
          sum.s += other.s;
          sum.t += other.t;
          if constexpr (kList > 0)
#pragma unroll 1
            for (int j = 0; j < kList; ++j) {
              const float w = o[(3 + j) * 64];
              if (w > value[kList - 1]) sort_in(w, __builtin_bit_cast(int32_t, o[(3 + kList + j) * 64]));
            }
        }
      }
      __syncthreads();   // (the next rows' tiles and sums go where these were read)
    }
    if (q == 0 && mine) {
      const RowResult<T> res(sum);
      const int64_t r = (int64_t)e * shape.vars + v;
      const int64_t ge = kStaged && given.vars > 1 ? r / given.vars : e, gv = kStaged && given.vars > 1 ? r - ge * given.vars : v;
      for (int j = 0; j < given.slots; ++j)
        out.logp[r * given.slots + j] =
            res.given(given_at(given, ge, gv, j), shape.cats, [&](int64_t g) { return seen(row[g * x.stride_cat]); });
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
void launch_lane(const RowsRef& x, const RowsShape& shape, const GivenRef& given, int top, const ScoreOut& out, bool staged, hipStream_t stream) {
  const int64_t sets = (shape.rows() + 63) / 64;
  const int most = staged || kList > 8 ? 4 : kList > 4 ? 8 : 16;   // (LDS)
  int parts = 1;
  while (parts < most && sets * parts < 4096 && shape.cats / parts >= 64) parts *= 2;
  const int waves = std::max(4, parts), per = waves / parts;
  const int lds = std::max(staged ? waves * 64 * 36 * 4 : 0, parts > 1 ? waves * (3 + 2 * kList) * 64 * 4 : 0);
  const bool examples_first = examples_side_by_side(x, shape);
  const dim3 grid((unsigned)std::min<int64_t>((sets + per - 1) / per, 1 << 20)), block(64 * waves);
  auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, block, lds, stream, x, shape, given, top, out, parts, examples_first); };
  staged ? launch(score_lane_kernel<T, kList, true>) : launch(score_lane_kernel<T, kList, false>);
}
}  // namespace

template <typename T>
bool category_scores_short(const RowsRef& x, const RowsShape& shape, const GivenRef& given, int top, const ScoreOut& out, const CkptRef& ckpt,
                           hipStream_t stream) {
  if (top > 16) return false;
  const bool neighbours = x.stride_cat == 1;
  const bool side = !neighbours && side_by_side(x, shape) && shape.rows() >= (shape.cats <= kShortCats ? kSideRowsShort : kSideRows);
  // rows of neighbouring categories one stride apart: their examples and variables are one axis
  const bool even = shape.vars == 1 || x.stride_ex == (int64_t)shape.vars * x.stride_var;
  const bool staged = neighbours && even && shape.cats > 16 && shape.cats <= kLaneCats &&
                      shape.rows() >= (shape.cats <= kShortCats ? kLaneRowsShort : kLaneRows) && !ckpt.codes;
  if (side || staged || (shape.cats <= 16 && !ckpt.codes)) {
    RowsRef y = x;
    RowsShape one = shape;
    GivenRef g = given;
    if (staged) {
      g.vars = shape.vars;
      y.stride_ex = shape.vars == 1 ? x.stride_ex : x.stride_var;
      one = {shape.rows(), 1, shape.cats};
    }
    if (top == 0) launch_lane<T, 0>(y, one, g, top, out, staged, stream);
    else if (top <= 4) launch_lane<T, 4>(y, one, g, top, out, staged, stream);
    else if (top <= 8) launch_lane<T, 8>(y, one, g, top, out, staged, stream);
    else launch_lane<T, 16>(y, one, g, top, out, staged, stream);
    return true;
  }
  if (!neighbours || shape.cats > kShortCats) return false;
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
