// Products of two matrices whose rows are both neighbours along the summed axis, sum_k a[m][k] b[n][k], on the matrix cores: the tile
// loop that the kernels of linear_scores.hip, linear_gradient.hip and product8.hip share, each with what it does with the sums.
#pragma once

#include "linear_plan.hpp"
#include "linear_scores.hpp"

namespace pcm {

// Which planes of b are multiplied with a, one after the other: two bits each, the first product lowest
struct PlanePairs {
  int count;
  uint32_t b;
};
constexpr PlanePairs kOnePlane{1, 0}, kTwoOfB{2, 0x1};   // b in two parts: the smaller one first
// What a product sums over: `count` steps of 128 bytes for each pair of planes.  With parts > 1 part blockIdx.y takes its share of the steps.
struct Steps {
  int count;
  PlanePairs pairs;
  int parts;
};

#ifdef __HIPCC__
// The first of a float's three parts is its nearest bfloat16, but no infinity for a finite one: the second part has the rest (NaN comes back in it too)
__device__ __forceinline__ float first_part(float x) {
  constexpr float most = 0x1.fep127f;        // bfloat16's largest
  return __builtin_amdgcn_fmed3f(x, -most, most);
}
typedef int v4i __attribute__((ext_vector_type(4)));
typedef int v16i __attribute__((ext_vector_type(16)));
typedef float v16f __attribute__((ext_vector_type(16)));
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));

// 32 x 32 sums over 32 bytes of both operands' rows: lane l gives 16 bytes of row l % 32, of its half; it gets of the sums, as entry i,
// row 8 (i / 4) + 4 (l / 32) + i % 4 of a and row l % 32 of b.
template <typename T>
struct Cores;
template <>
struct Cores<bf16> {
  typedef v16f Sums;
  static __device__ __forceinline__ v16f mma(v4i a, v4i b, v16f c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), c, 0, 0, 0);
  }
};
template <>
struct Cores<f16> {
  typedef v16f Sums;
  static __device__ __forceinline__ v16f mma(v4i a, v4i b, v16f c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
  }
};
template <>
struct Cores<int8_t> {
  typedef v16i Sums;
  static __device__ __forceinline__ v16i mma(v4i a, v4i b, v16i c) { return __builtin_amdgcn_mfma_i32_32x32x32_i8(a, b, c, 0, 0, 0); }
};

// Sixteen bytes a lane from memory straight into LDS: lane l's from `base` (the first 48 bits of the descriptor) + at + k to lds + 16 l.
// Written out so that the compiler does not wait for it at the next read of LDS, whichever stage that is of: stage_barrier says when what
// is there.  It has no register to return to, and its address is taken when it is issued.
__device__ __forceinline__ void request_into_lds(const char* lds, v4i base, uint32_t at, uint32_t k) {
  const uint32_t to = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)lds);   // (an address in LDS is the lower half of one in memory's space)
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" ::"s"(to), "v"(at), "s"(base), "s"(k) : "m0");
}
// the descriptor of memory from p on; p is the same in all lanes
__device__ __forceinline__ v4i memory_at(const char* p) {
  const uint64_t v = (uint64_t)p;
  return v4i{(int)__builtin_amdgcn_readfirstlane((uint32_t)v), (int)(__builtin_amdgcn_readfirstlane((uint32_t)(v >> 32)) & 0xffffu), -1, 0x00020000};
}
// A barrier after which what the workgroup's waves have requested into LDS is there, but for the last `kOpen` requests of each wave: a barrier
// by itself says nothing of requests on their way.
template <int kOpen>
__device__ __forceinline__ void stage_barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt((kOpen & 15) | kOpen >> 4 << 14 | 7 << 4);   // vmcnt(kOpen) lgkmcnt(0)
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

template <int kBM, int kBN, int kWM, int kWN>
struct TileSizes {
  static constexpr int BM = kBM, BN = kBN, WM = kWM, WN = kWN;   // rows of a and of b, of a workgroup and of a wave
  static constexpr int waves_m = kBM / kWM, waves = waves_m * (kBN / kWN), threads = 64 * waves;
  static constexpr int FM = kWM / 32, FN = kWN / 32;
  static constexpr int stage = (kBM + kBN) * kKBytes;            // bytes in LDS
};

// A wave's share of a stage: requests of 1 KB, eight rows of 128 bytes, straight into LDS.  There chunk c (16 bytes) of row r lies at
// c ^ (r / 2) % 8 of the row, so that sixteen lanes reading one chunk of neighbouring rows meet all banks once.  Rows past the
// end are read from the last row; what they give is not used.
template <typename S>
struct TileLoader {
  static constexpr int each = S::stage / 1024 / S::waves;
  static_assert(each * 1024 * S::waves == S::stage && S::BM % 8 == 0 && S::BN % 8 == 0);
  const char *a0, *b0;
  int64_t plane_b;
  v4i a, b;
  uint32_t at[each];
  uint32_t k, begin, end;      // the bytes of a row that come next, and between which
  PlanePairs pairs;
  int wave, product = 0;

  __device__ __forceinline__ void choose_plane() {
    const int64_t pb = pairs.b >> 2 * product & 3;
    b = memory_at(b0 + pb * plane_b);
  }
  __device__ __forceinline__ TileLoader(const Operand& oa, const Operand& ob, int64_t m0, int64_t n0, int64_t m, int64_t n, int first, int count,
                                        const PlanePairs& of) : pairs(of) {
    wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    a0 = static_cast<const char*>(oa.p) + m0 * oa.pitch;
    b0 = static_cast<const char*>(ob.p) + n0 * ob.pitch;
    plane_b = ob.plane;
    k = begin = __builtin_amdgcn_readfirstlane((uint32_t)first * kKBytes);
    end = begin + __builtin_amdgcn_readfirstlane((uint32_t)count * kKBytes);
    a = memory_at(a0);
    choose_plane();
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int i = 0; i < each; ++i) {
      const int q = i * S::waves + wave;
      const bool of_a = q < S::BM / 8;
      const int row = (of_a ? q : q - S::BM / 8) * 8 + lane / 8;
      const int64_t last = (of_a ? m - m0 : n - n0) - 1;
      at[i] = (uint32_t)((row < last ? row : last) * (of_a ? oa.pitch : ob.pitch)) + ((lane & 7) ^ (row >> 1 & 7)) * 16;
    }
  }
  __device__ __forceinline__ void load(const char* lds) {
#pragma unroll
    for (int i = 0; i < each; ++i) {
      const int q = i * S::waves + wave;
      request_into_lds(lds + q * 1024, q < S::BM / 8 ? a : b, at[i], k);
    }
    k += kKBytes;
    if (k == end && product + 1 < pairs.count) {
      k = begin;
      ++product;
      choose_plane();
    }
  }
};

// The tile of workgroup blockIdx.x, of a launch over whole rows of tiles from row `first` of b on: each of the eight dies takes a run of tiles,
// four rows of b's tiles at a time, so that what its workgroups read at one time meets in its cache
struct TileAt {
  int64_t m0, n0;
};
template <typename S>
__device__ __forceinline__ TileAt tile_at(int64_t m, int64_t first) {
  const int all = gridDim.x, die = blockIdx.x % 8;
  const int tiles_m = (int)((m + S::BM - 1) / S::BM), tiles_n = all / tiles_m;
  const int id = die * (all / 8) + min(die, all % 8) + blockIdx.x / 8;
  constexpr int kRows = 4;
  const int group = id / (kRows * tiles_m), in = id % (kRows * tiles_m);
  const int rows = min(kRows, tiles_n - group * kRows);
  return {(int64_t)(in / rows) * S::BM, first + (int64_t)(group * kRows + in % rows) * S::BN};
}

// Sums of the tile at (m0, n0), of a launch over rows of b from first_n on, handed to done(sums, m, n, lds): sums[i][j] of the wave's rows
// m + 32 i of a and n + 32 j of b, and the first stage's LDS for its own use (after a barrier).
//
// Two stages of 128 bytes in LDS.  Fragments are read from LDS one step of 32 bytes ahead of their products, and the barrier at a stage's
// end stands before its last products: they run while the next stage's first fragments are on their way.  A stage's memory
// requests go out as soon as that barrier has freed its LDS, one stage ahead of their use.
template <typename T, typename S, typename Done>
__device__ __forceinline__ void product_tile(const Operand& a, const Operand& b, int64_t m, int64_t n, int64_t first_n, const Steps& steps, Done done) {
  __shared__ __attribute__((aligned(1024))) char s0[S::stage];
  __shared__ __attribute__((aligned(1024))) char s1[S::stage];
  const TileAt tile = tile_at<S>(m, first_n);
  const int part = blockIdx.y, first = (int)((int64_t)steps.count * part / steps.parts);
  const int count = (int)((int64_t)steps.count * (part + 1) / steps.parts) - first;
  TileLoader<S> from(a, b, tile.m0, tile.n0, m, n, first, count, steps.pairs);
  const int stages = count * steps.pairs.count;
  const int lane = threadIdx.x & 63, row = lane & 31, half = lane >> 5, swap = row >> 1 & 7;
  const int wm = from.wave % S::waves_m * S::WM, wn = from.wave / S::waves_m * S::WN;
  const int at_a = (wm + row) * kKBytes, at_b = (S::BM + wn + row) * kKBytes;
  typename Cores<T>::Sums sums[S::FM][S::FN] = {};
  v4i fa[2][S::FM], fb[2][S::FN];
  auto read = [&](const char* s, int step, int w) {
    const int c = ((2 * step + half) ^ swap) * 16;
#pragma unroll
    for (int j = 0; j < S::FN; ++j) fb[w][j] = *reinterpret_cast<const v4i*>(s + at_b + j * 32 * kKBytes + c);
#pragma unroll
    for (int i = 0; i < S::FM; ++i) fa[w][i] = *reinterpret_cast<const v4i*>(s + at_a + i * 32 * kKBytes + c);
  };
  auto multiply = [&](int w) {
#pragma unroll
    for (int i = 0; i < S::FM; ++i)
#pragma unroll
      for (int j = 0; j < S::FN; ++j) sums[i][j] = Cores<T>::mma(fa[w][i], fb[w][j], sums[i][j]);
  };
  auto mix = [] {   // a fragment's read between two products
#pragma unroll
    for (int i = 0; i < S::FM * S::FN; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      if (i < S::FM + S::FN) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
    }
  };
  auto stage = [&](char* mine, const char* next, int t) {
#pragma unroll
    for (int step = 1; step < 4; ++step) {
      read(mine, step, step & 1);
      multiply(~step & 1);
      mix();
    }
    stage_barrier<0>();
    if (t + 1 < stages) read(next, 0, 0);
    if (t + 2 < stages) from.load(mine);
    multiply(1);
  };
  if (stages > 0) {
    from.load(s0);
    if (stages > 1) {
      from.load(s1);
      stage_barrier<TileLoader<S>::each>();
    } else {
      stage_barrier<0>();
    }
    read(s0, 0, 0);
    for (int t = 0; t < stages; t += 2) {
      stage(s0, s1, t);
      if (t + 1 < stages) stage(s1, s0, t + 1);
    }
  }
  done(sums, tile.m0 + wm, tile.n0 + wn, s0);
}
#endif

}  // namespace pcm
