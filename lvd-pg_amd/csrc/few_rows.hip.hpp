// Products of a long matrix (weights: categories or channels) with a few rows: bound by reading the long one once.
//
// A workgroup takes 32 rows of the long matrix, its eight waves every eighth piece of 128 bytes of them each, straight from memory into the
// cores' operands: whatever the rows' length and alignment, nothing is laid out.  The waves' sums meet in LDS.
#pragma once

#include "float_tiles.hip.hpp"

namespace pcm {

constexpr int kFewRowsMost = 64;             // rows that are few
constexpr int kFewTile = 32;                 // rows of the long matrix of a workgroup
struct FewOperand {                          // rows of neighbouring entries
  const void* p;
  int64_t stride_ex, stride_var;             // in entries
  int32_t vars;
};

#ifdef __HIPCC__
typedef float v4sums __attribute__((ext_vector_type(4)));
// 16 x 16 sums over 64 bytes of both operands' rows: lane l gives 16 bytes of row l % 16, of its quarter; of the sums it gets, as entry
// i, row 4 (l / 16) + i of a and row l % 16 of b
template <typename T>
struct FewCores;
template <>
struct FewCores<bf16> {
  typedef v4sums Sums;
  static __device__ __forceinline__ v4sums mma(v4i a, v4i b, v4sums c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), c, 0, 0, 0);
  }
};
template <>
struct FewCores<f16> {
  typedef v4sums Sums;
  static __device__ __forceinline__ v4sums mma(v4i a, v4i b, v4sums c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
  }
};
template <>
struct FewCores<int8_t> {
  typedef v4i Sums;
  static __device__ __forceinline__ v4i mma(v4i a, v4i b, v4i c) { return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0); }
};

// A lane's 32 bytes of a row's piece, 64 apart: of 16-bit and 8-bit types a step's operand each, of float one step's
template <typename T>
struct FewPiece {
  static constexpr int entries = 128 / sizeof(T);
  raw4 v[2];
  __device__ __forceinline__ void load(const T* row) {
    const int quarter = (threadIdx.x & 63) / 16;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if constexpr (sizeof(T) == 1) v[i] = *reinterpret_cast<const raw4*>(row + i * 64 + quarter * 16);
      else v[i] = load16(row + (i * 64 + quarter * 16) / sizeof(T));
    }
  }
  // with `left` entries left in the row
  __device__ __forceinline__ void load_end(const T* row, int left) {
    const int quarter = (threadIdx.x & 63) / 16;
    constexpr int each = 16 / sizeof(T);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      T e[each];
#pragma unroll
      for (int k = 0; k < each; ++k) {
        const int at = (i * 64 + quarter * 16) / (int)sizeof(T) + k;
        e[k] = at < left ? row[at] : (T)0;
      }
      v[i] = __builtin_bit_cast(raw4, e);
    }
  }
};
template <typename T>
struct FewParts {                            // ... as operands of the cores
  v4i p[sizeof(T) == 4 ? 3 : 2];
  __device__ __forceinline__ explicit FewParts(const FewPiece<T>& x) {
    if constexpr (sizeof(T) == 4) {          // three parts of eight floats
      float w[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) w[k] = as_float(x.v[k / 4][k % 4]);
#pragma unroll
      for (int q = 0; q < 3; ++q)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t two = pair_of<bf16>(w[2 * k], w[2 * k + 1]);
          p[q][k] = (int)two;
          if (q < 2) {
            w[2 * k] -= as_float(two << 16);
            w[2 * k + 1] -= as_float(two & 0xffff0000u);
          }
        }
    } else {
      p[0] = __builtin_bit_cast(v4i, x.v[0]);
      p[1] = __builtin_bit_cast(v4i, x.v[1]);
    }
  }
};

// Sums of rows [32 blockIdx.x, + 32) of a with all (16 kGroups at most) rows of b over `length` entries: sum of rows m and n of the tile at
// lds[m][n], 32 bits (whole numbers: their bits), after a barrier.  Parts of the pieces by blockIdx.y.
template <int kGroups>
constexpr int kFewPitch = 16 * kGroups + 1;
template <typename T, int kGroups>
__device__ __forceinline__ void few_sums(const FewOperand& a, const FewOperand& b, int64_t m, int64_t n, int length, int parts,
                                         float (&lds)[8][kFewTile][kFewPitch<kGroups>]) {
  typedef typename std::conditional<sizeof(T) == 4, bf16, T>::type Core;
  constexpr int kPiece = FewPiece<T>::entries;
  const int lane = threadIdx.x & 63, wave = threadIdx.x / 64;
  const T *at_a[2], *at_b[kGroups];
#pragma unroll
  for (int g = 0; g < 2; ++g) at_a[g] = static_cast<const T*>(a.p) + min((int64_t)blockIdx.x * kFewTile + 16 * g + (lane & 15), m - 1) * a.stride_ex;
#pragma unroll
  for (int g = 0; g < kGroups; ++g) {
    const int64_t r = min((int64_t)(16 * g + (lane & 15)), n - 1);
    at_b[g] = static_cast<const T*>(b.p) + r / b.vars * b.stride_ex + r % b.vars * b.stride_var;
  }
  typename FewCores<Core>::Sums sums[2][kGroups] = {};
  auto multiply = [&](const FewPiece<T> (&pa)[2], const FewPiece<T> (&pb)[kGroups]) {
    const FewParts<T> fa[2] = {FewParts<T>(pa[0]), FewParts<T>(pa[1])};
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
      const FewParts<T> fb(pb[g]);
      if constexpr (sizeof(T) == 4) {
        constexpr int of_a[6] = {0, 2, 1, 0, 1, 0}, of_b[6] = {2, 0, 1, 1, 0, 0};   // hl lh mm hm mh hh
#pragma unroll
        for (int q = 0; q < 6; ++q)
#pragma unroll
          for (int i = 0; i < 2; ++i) sums[i][g] = FewCores<Core>::mma(fa[i].p[of_a[q]], fb.p[of_b[q]], sums[i][g]);
      } else {
#pragma unroll
        for (int q = 0; q < 2; ++q)
#pragma unroll
          for (int i = 0; i < 2; ++i) sums[i][g] = FewCores<Core>::mma(fa[i].p[q], fb.p[q], sums[i][g]);
      }
    }
  };
  // whole pieces first, the wave's next one on its way while one is multiplied; then what is left
  const int whole = length / kPiece, pieces = (length + kPiece - 1) / kPiece;
  const int first = (int)((int64_t)pieces * blockIdx.y / parts), last = (int)((int64_t)pieces * (blockIdx.y + 1) / parts);
  const int end = min(last, whole);
  FewPiece<T> pa[2][2], pb[2][kGroups];
  auto load = [&](int set, int piece) {
#pragma unroll
    for (int g = 0; g < 2; ++g) pa[set][g].load(at_a[g] + (int64_t)piece * kPiece);
#pragma unroll
    for (int g = 0; g < kGroups; ++g) pb[set][g].load(at_b[g] + (int64_t)piece * kPiece);
  };
  int piece = first + wave;
  if (piece < end) {
    load(0, piece);
    for (; piece < end; piece += 16) {
      load(1, min(piece + 8, end - 1));      // (past the end the last one once more, not used)
      multiply(pa[0], pb[0]);
      if (piece + 8 >= end) break;
      load(0, min(piece + 16, end - 1));
      multiply(pa[1], pb[1]);
    }
  }
  if (last > end && wave == 7) {
    const int left = length - whole * kPiece;
#pragma unroll
    for (int g = 0; g < 2; ++g) pa[0][g].load_end(at_a[g] + (int64_t)whole * kPiece, left);
#pragma unroll
    for (int g = 0; g < kGroups; ++g) pb[0][g].load_end(at_b[g] + (int64_t)whole * kPiece, left);
    multiply(pa[0], pb[0]);
  }
#pragma unroll
  for (int g = 0; g < kGroups; ++g)
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const auto sum = sums[i][g][r];        // (a bit cast of a vector's element takes the vector's first one)
        lds[wave][16 * i + 4 * (lane / 16) + r][16 * g + (lane & 15)] = __builtin_bit_cast(float, sum);
      }
  __syncthreads();
  for (int i = threadIdx.x; i < kFewTile * 16 * kGroups; i += 512) {
    const int r = i / (16 * kGroups), c = i % (16 * kGroups);
    if constexpr (sizeof(T) == 1) {
      int s = 0;
#pragma unroll
      for (int w = 0; w < 8; ++w) s += __builtin_bit_cast(int, lds[w][r][c]);
      lds[0][r][c] = __builtin_bit_cast(float, s);
    } else {
      float s = 0.f;
#pragma unroll
      for (int w = 0; w < 8; ++w) s += lds[w][r][c];
      lds[0][r][c] = s;
    }
  }
  __syncthreads();
}
#endif

}  // namespace pcm
