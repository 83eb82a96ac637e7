// How the kernels that turn rows into rows, entry by entry, deal them out: G lanes a row (a power of two, up to the workgroup's 256),
// each with up to kTileGroups groups of 16 bytes at a time; a workgroup holds 256 / G short rows, or one of the `segments` of a long
// one, in `turns`.
#pragma once

#include "category_rows.hpp"

namespace pcm {

constexpr int kTileThreads = 256, kTileGroups = 4;

struct Tiles {
  int lanes_log2;      // log2 G
  int segments;        // of a row
  int turns;           // of a segment
  int64_t jobs;        // workgroups' worth of work
};
// `vec` entries a group, at least `least` lanes a row; a segment takes several turns where there are more than `wanted_jobs` jobs without
inline Tiles tiles_of(const RowsShape& shape, int vec, int least, int64_t wanted_jobs = INT64_MAX) {
  const int64_t groups = ((int64_t)shape.cats + vec - 1) / vec, wanted = (groups + kTileGroups - 1) / kTileGroups;
  Tiles t{0, 1, 1, 0};
  while ((1 << t.lanes_log2) < kTileThreads && (1 << t.lanes_log2) < std::max<int64_t>(wanted, least)) ++t.lanes_log2;
  const int64_t held = (int64_t)kTileGroups << t.lanes_log2;
  const int64_t all = (groups + held - 1) / held, rows = std::max<int64_t>(shape.rows(), 1);
  t.turns = (int)std::max<int64_t>(1, all / std::max<int64_t>(1, (std::min(wanted_jobs, rows * all) + rows - 1) / rows));
  t.segments = (int)((all + t.turns - 1) / t.turns);
  const int64_t per = kTileThreads >> t.lanes_log2;
  t.jobs = (shape.rows() + per - 1) / per * t.segments;
  return t;
}
inline dim3 tile_grid(const Tiles& t) { return dim3((unsigned)std::min<int64_t>(t.jobs, 1 << 22)); }

#ifdef __HIPCC__
// The n-th row, counted examples first or variables first
struct RowAt {
  int64_t e, v, r;
};
__device__ __forceinline__ RowAt row_at(const RowsShape& shape, uint32_t n, bool examples_first) {
  const uint32_t by = examples_first ? (uint32_t)shape.examples : (uint32_t)shape.vars, hi = n / by, lo = n - hi * by;
  const int64_t e = examples_first ? lo : hi, v = examples_first ? hi : lo;
  return {e, v, e * shape.vars + v};
}

struct TileAt {        // of a lane in a job
  int64_t row;         // may lie behind the last one
  int first, step;     // group u holds the categories from (first + u * step) * vec
};
__device__ __forceinline__ TileAt tile_at(const Tiles& t, int64_t job) {
  const int lanes = 1 << t.lanes_log2, in = threadIdx.x & (lanes - 1), of = threadIdx.x >> t.lanes_log2;
  if (t.segments == 1) return {(job << (8 - t.lanes_log2)) + of, in, lanes};
  const int64_t row = job / t.segments;   // (one row a workgroup)
  return {row, (int)(job - row * t.segments) * t.turns * kTileGroups * lanes + in, lanes};
}

// A group of 16 bytes from categories c.. of a row of `cats`; -inf behind its end
template <typename T>
__device__ __forceinline__ raw4 load_group(const T* row, int64_t c, int cats) {
  constexpr int kVec = 16 / (int)sizeof(T);
  if (c + kVec <= cats) return load16(row + c);
  T w[kVec];
#pragma unroll
  for (int i = 0; i < kVec; ++i) w[i] = c + i < cats ? row[c + i] : (T)-INFINITY;
  return __builtin_bit_cast(raw4, w);
}
// ... of a row whose categories are not neighbours
template <typename T>
__device__ __forceinline__ raw4 gather_group(const T* row, int64_t c, int cats, int64_t stride) {
  constexpr int kVec = 16 / (int)sizeof(T);
  T w[kVec];
#pragma unroll
  for (int i = 0; i < kVec; ++i) w[i] = c + i < cats ? row[(c + i) * stride] : (T)-INFINITY;
  return __builtin_bit_cast(raw4, w);
}
template <typename T>
__device__ __forceinline__ void scatter_group(T* row, int64_t c, int cats, int64_t stride, const T (&w)[16 / (int)sizeof(T)]) {
#pragma unroll
  for (int i = 0; i < 16 / (int)sizeof(T); ++i)
    if (c + i < cats) row[(c + i) * stride] = w[i];
}
template <typename T>
__device__ __forceinline__ void store_group(T* row, int64_t c, int cats, const T (&w)[16 / (int)sizeof(T)]) {
  constexpr int kVec = 16 / (int)sizeof(T);
  if (c + kVec <= cats) {
    store16(row + c, __builtin_bit_cast(raw4, w));
    return;
  }
#pragma unroll
  for (int i = 0; i < kVec; ++i)
    if (c + i < cats) row[c + i] = w[i];
}
// The codes of a group (c is a multiple of its size, the codes' pitch of 16)
template <int kVec>
struct Codes {
  uint32_t w[kVec / 4];
  __device__ __forceinline__ float operator[](int i) const { return (float)(w[i / 4] >> (8 * (i % 4)) & 0xffu); }
};
template <int kVec>
__device__ __forceinline__ Codes<kVec> load_codes(const uint8_t* at) {
  Codes<kVec> k;
  if constexpr (kVec == 4) k.w[0] = *reinterpret_cast<const uint32_t*>(at);
  else {
    const uint2 v = *reinterpret_cast<const uint2*>(at);
    k.w[0] = v.x;
    k.w[1] = v.y;
  }
  return k;
}
// the entries that they stand for
template <int kVec>
__device__ __forceinline__ void decode(const Codes<kVec>& k, const BlockUnit& u, float (&y)[kVec]) {
  if (__any(u.masks)) {
#pragma unroll
    for (int i = 0; i < kVec; ++i) y[i] = block_entry_or_mask(u, k[i]);
  } else {
#pragma unroll
    for (int i = 0; i < kVec; ++i) y[i] = block_entry(u, k[i]);
  }
}
#endif

}  // namespace pcm
