// Products of a long matrix (weights: categories or channels) with a few rows: bound by reading the long one once, and, with more than 16 rows, by
// each workgroup's reading the others from the caches: 50021 x 1001 f16 with 16 rows 34 us (3 TB/s), with 48 50 us.
//
// A workgroup takes 32 rows of the long matrix, its waves (eight, or four with more than 32 others) a piece of 128 bytes of them each in turns, whatever
// the rows' length and alignment: nothing is laid out.  The waves' sums meet in LDS.
#pragma once

#include "float_tiles.hip.hpp"

namespace pcm {

constexpr int kFewRowsMost = 64;             // rows that are few: those of a workgroup
constexpr int kFewTile = 32;                 // rows of the long matrix of a workgroup
struct FewOperand {                          // rows of neighbouring entries
  const void* p;
  int64_t stride_ex, stride_var;             // in entries
  int32_t vars;
};

// Whether a product of scores goes this way: few rows, or so few tiles of 128 x 128 that long sums are best cut among the waves of a workgroup (100 x
// 3000 x 500 f32: 111 us by tiles, 43 here).  Where rows can be read where they are, tiles of 128 categories stream faster once there
// are enough of them for the compute units, fewer the shorter the rows and the more of them there are, since a workgroup here takes its time to
// join sums (f16, tiles and here: 16 x 4096 x 15000 57 us, 38; 8 x 4096 x 50000 80, 124; 16 x 256 x 20000 11.4, 15.4; 64 x 1024 x 30000 26,
// 38; 64 x 4096 x 10000 56, 49; either way within some percent near the rule).
inline int64_t many_cats(int64_t rows, int64_t row_bytes) {
  return rows <= 32 ? 36000 * row_bytes / (row_bytes + 1200) : 24000 * row_bytes / (row_bytes + 2200);
}
bool takes_few(const Matrix2& f, const Matrix2& w);
bool takes_few8(int64_t rows, int64_t cats, int64_t length);
FewOperand few_operand(const Matrix2& x);

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

// A lane's 16 bytes of a piece of 128 bytes of a row, of which eight neighbouring lanes take one each
template <typename T>
struct FewChunk {
  raw4 v;
  uint32_t next;                             // 16-bit types: the word behind
  __device__ __forceinline__ void load(const T* at) {
    if constexpr (sizeof(T) == 1) {
      v = *reinterpret_cast<const raw4*>(at);
    } else if constexpr (sizeof(T) == 4) {
      v = load16(at);
    } else {                                 // whole words, of which the first and the last may hold a neighbour's entry
      const uint32_t* const p = reinterpret_cast<const uint32_t*>((uintptr_t)at & ~(uintptr_t)3);
      v = *reinterpret_cast<const raw4_by4*>(p);
      next = p[(uintptr_t)at & 2 ? 4 : 3];
    }
  }
  // of the `left` entries that are left there
  __device__ __forceinline__ void load_end(const T* at, int left) {
    constexpr int each = 16 / sizeof(T);
    T e[each];
#pragma unroll
    for (int k = 0; k < each; ++k) e[k] = k < left ? at[k] : (T)0;
    v = __builtin_bit_cast(raw4, e);
  }
  __device__ __forceinline__ raw4 get(const T* at) const {
    if constexpr (sizeof(T) != 2) return v;
    const uint32_t shift = ((uint32_t)(uintptr_t)at & 2) * 8;
    raw4 w;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint32_t hi = k < 3 ? v[k < 3 ? k + 1 : 3] : next, lo = v[k];
      w[k] = __builtin_amdgcn_alignbit(hi, lo, shift);
    }
    return w;
  }
};
template <typename T>
struct FewParts {                            // two chunks of a row, 64 bytes apart, as operands of the cores
  v4i p[sizeof(T) == 4 ? 3 : 2];
  __device__ __forceinline__ FewParts(raw4 x, raw4 y) {
    if constexpr (sizeof(T) == 4) {          // three parts of eight floats
      float w[8];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        w[k] = as_float(x[k]);
        w[4 + k] = as_float(y[k]);
      }
#pragma unroll
      for (int q = 0; q < 3; ++q)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t two = q ? pair_of<bf16>(w[2 * k], w[2 * k + 1]) : pair_of<bf16>(first_part(w[2 * k]), first_part(w[2 * k + 1]));
          p[q][k] = (int)two;
          if (q < 2) {
            w[2 * k] -= as_float(two << 16);
            w[2 * k + 1] -= as_float(two & 0xffff0000u);
          }
        }
    } else {
      p[0] = __builtin_bit_cast(v4i, x);
      p[1] = __builtin_bit_cast(v4i, y);
    }
  }
};

// Between a wave's writes to LDS and its other lanes' reads of them, and the other way round.  LDS takes a wave's requests in order, so the compiler's
// order is all that has to be held, and that of LDS alone.  (Before a turn's writes, not behind the products of the turn before: there registers
// spill, and 48 x 1001 x 50021 f16 takes 80 us instead of 65.)
__device__ __forceinline__ void lanes_share() { __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local"); }

template <int kGroups>
struct FewTile {                             // kGroups: of 16 rows of b
  static constexpr int rows = 16 * kGroups;
  static constexpr int longs = kFewTile;                      // rows of a
  static constexpr int waves = kGroups == 4 ? 4 : 8, threads = 64 * waves;   // (three workgroups fit a compute unit's LDS, with 17 to 32 rows two)
  static constexpr int wave_bytes = (longs + rows) * 128;     // a piece of each
  static constexpr int pitch = rows + 1;                      // of the sums
  static constexpr int sums_bytes = waves * longs * pitch * 4;
  static constexpr int lds = sums_bytes > waves * wave_bytes ? sums_bytes : waves * wave_bytes;
};
// Sums of rows [longs blockIdx.x, + longs) of a with rows [rows blockIdx.z, + rows) of b over `length` entries: sum of rows m and n of the tile
// at m * pitch + n of what is returned (LDS), 32 bits (whole numbers: their bits), after a barrier.  Parts of the pieces by blockIdx.y.
//
// A wave's piece goes through its own share of LDS: requested by eight lanes a row, read back as the cores' operands.  No barrier until the
// waves' sums meet; the next piece is requested before one is multiplied.
template <typename T, int kGroups>
__device__ __forceinline__ const float* few_sums(const FewOperand& a, const FewOperand& b, int64_t m, int64_t n, int length, int parts, char* lds) {
  typedef typename std::conditional<sizeof(T) == 4, bf16, T>::type Core;
  typedef FewTile<kGroups> S;
  constexpr int kPiece = 128 / sizeof(T), kEach = 16 / sizeof(T), kLongs = S::longs / 8, kRows = S::rows / 8, kCats = S::longs / 16;
  const int lane = threadIdx.x & 63, wave = threadIdx.x / 64;
  char* const mine = lds + wave * S::wave_bytes;
  const T *at_a[kLongs], *at_b[kRows];
#pragma unroll
  for (int g = 0; g < kLongs; ++g)
    at_a[g] = static_cast<const T*>(a.p) + min((int64_t)blockIdx.x * S::longs + 8 * g + lane / 8, m - 1) * a.stride_ex + lane % 8 * kEach;
#pragma unroll
  for (int g = 0; g < kRows; ++g) {
    const int64_t r = min((int64_t)blockIdx.z * S::rows + 8 * g + lane / 8, n - 1);
    at_b[g] = static_cast<const T*>(b.p) + r / b.vars * b.stride_ex + r % b.vars * b.stride_var + lane % 8 * kEach;
  }
  typename FewCores<Core>::Sums sums[kCats][kGroups] = {};
  FewChunk<T> ca[kLongs], cb[kRows];
  auto load = [&](int piece) {
#pragma unroll
    for (int g = 0; g < kLongs; ++g) ca[g].load(at_a[g] + (int64_t)piece * kPiece);
#pragma unroll
    for (int g = 0; g < kRows; ++g) cb[g].load(at_b[g] + (int64_t)piece * kPiece);
  };
  // chunk c of row r lies at c ^ (r / 2) % 8 of the row
  const int to = lane / 8 * 128 + ((lane & 7) ^ (lane >> 4 & 3)) * 16;     // (row r + 8 g: bits of g join below)
  auto put = [&](int g, raw4 v) { *reinterpret_cast<raw4*>(mine + g * 1024 + (to ^ (g & 1) * 64)) = v; };
  auto operand = [&](int group) {
    const int r = lane & 15, swap = r >> 1 & 7, quarter = lane / 16;
    const char* const row = mine + (16 * group + r) * 128;
    return FewParts<T>(*reinterpret_cast<const raw4*>(row + (quarter ^ swap) * 16), *reinterpret_cast<const raw4*>(row + ((quarter + 4) ^ swap) * 16));
  };
  auto multiply = [&] {
    constexpr int kParts = sizeof(T) == 4 ? 3 : 2;
    v4i fa[kCats][kParts];
#pragma unroll
    for (int i = 0; i < kCats; ++i) {
      const FewParts<T> x = operand(i);
#pragma unroll
      for (int q = 0; q < kParts; ++q) fa[i][q] = x.p[q];
    }
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
      const FewParts<T> fb = operand(kCats + g);
      if constexpr (sizeof(T) == 4) {
        constexpr int of_a[6] = {0, 2, 1, 0, 1, 0}, of_b[6] = {2, 0, 1, 1, 0, 0};   // hl lh mm hm mh hh
#pragma unroll
        for (int q = 0; q < 6; ++q)
#pragma unroll
          for (int i = 0; i < kCats; ++i) sums[i][g] = FewCores<Core>::mma(fa[i][of_a[q]], fb.p[of_b[q]], sums[i][g]);
      } else {
#pragma unroll
        for (int q = 0; q < 2; ++q)
#pragma unroll
          for (int i = 0; i < kCats; ++i) sums[i][g] = FewCores<Core>::mma(fa[i][q], fb.p[q], sums[i][g]);
      }
    }
  };
  // whole pieces first, then what is left
  const int whole = length / kPiece, pieces = (length + kPiece - 1) / kPiece;
  const int first = (int)((int64_t)pieces * blockIdx.y / parts), last = (int)((int64_t)pieces * (blockIdx.y + 1) / parts);
  const int end = min(last, whole);
  if (first + wave < end) {
    load(first + wave);
    for (int piece = first + wave; piece < end; piece += S::waves) {
      lanes_share();
#pragma unroll
      for (int g = 0; g < kLongs; ++g) put(g, ca[g].get(at_a[g]));
#pragma unroll
      for (int g = 0; g < kRows; ++g) put(kLongs + g, cb[g].get(at_b[g]));
      lanes_share();
      load(min(piece + S::waves, end - 1));         // (past the end the last one once more, not used)
      multiply();
    }
  }
  if constexpr (sizeof(T) > 1) {             // (8-bit rows are whole pieces)
    if (last > end && wave == S::waves - 1) {
      const int left = length - whole * kPiece - lane % 8 * kEach;
      lanes_share();
#pragma unroll
      for (int g = 0; g < kLongs + kRows; ++g) {
        __builtin_amdgcn_sched_barrier(0);   // one at a time: registers
        ca[0].load_end((g < kLongs ? at_a[g < kLongs ? g : 0] : at_b[g < kLongs ? 0 : g - kLongs]) + (int64_t)whole * kPiece, left);
        put(g, ca[0].v);
      }
      lanes_share();
      multiply();
    }
  }
  float* const out = reinterpret_cast<float*>(lds);
  __syncthreads();
#pragma unroll
  for (int g = 0; g < kGroups; ++g)
#pragma unroll
    for (int i = 0; i < kCats; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const auto sum = sums[i][g][r];        // (a bit cast of a vector's element takes the vector's first one)
        out[(wave * S::longs + 16 * i + 4 * (lane / 16) + r) * S::pitch + 16 * g + (lane & 15)] = __builtin_bit_cast(float, sum);
      }
  __syncthreads();
  for (int i = threadIdx.x; i < S::longs * S::rows; i += S::threads) {
    const int at = i / S::rows * S::pitch + i % S::rows;
    if constexpr (sizeof(T) == 1) {
      int s = 0;
#pragma unroll
      for (int w = 0; w < S::waves; ++w) {
        const float x = out[w * S::longs * S::pitch + at];
        s += __builtin_bit_cast(int, x);
      }
      out[at] = __builtin_bit_cast(float, s);
    } else {
      float s = 0.f;
#pragma unroll
      for (int w = 0; w < S::waves; ++w) s += out[w * S::longs * S::pitch + at];
      out[at] = s;
    }
  }
  __syncthreads();
  return out;
}
#endif

}  // namespace pcm
