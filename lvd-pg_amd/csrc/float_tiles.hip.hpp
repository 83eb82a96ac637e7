// Products of float matrices on the matrix cores: each float as three bfloat16 parts, h + m + l, which hold all of its 24 bits (from 2^-110 on;
// smaller ones to 2^-134), and the six largest of the nine products of parts; what is left out (m l, l m, l l) is less than 2^-24 of the
// product.  An infinity has no such parts: a product with one is NaN, as may be one that passes float's range.
//
// A tile's floats come through registers, are taken apart there (some six instructions an entry) and lie in LDS as three planes, from which all
// six products are read: 12 fragments for 24 products of 32 x 32, so LDS is no bound, and the floats are read once, whatever
// their strides and alignment.  Either operand may be turned: summed over its rows.  The six products take six times a bfloat16 product's
// time, 2.4 TFLOP/s a compute unit at most against 0.6 of the cores' own float products.  Scores of 2048 x 32003 over 1024: 757 us, 177
// TFLOP/s (both operands turned: 946 us, where stores to LDS are of words; whole rows of four there, from requests of two, took more).
#pragma once

#include <type_traits>

#include "product_tiles.hip.hpp"

namespace pcm {

struct FloatOperand {
  const float* p;
  int64_t stride_ex, stride_var, stride;     // rows (example, variable), entries
  int32_t vars;
  bool turned;                               // summed over rows (else over entries)
  const int* skip;                           // turned: rows with kDeadRow here count as zeros, whatever they hold; null: none
};
// the matrix as an operand that is summed over its entries, or over its rows
FloatOperand float_operand(const Matrix2& x, bool turned, const int* skip = nullptr);

#ifdef __HIPCC__
typedef float v4f __attribute__((ext_vector_type(4)));
typedef v4f v4f_by4 __attribute__((aligned(4)));
typedef TileSizes<128, 128, 64, 64> FloatTile;
constexpr int kFloatSteps = 16;              // entries of the summed axis in a stage
constexpr int kFloatPitch = 48;              // bytes of a row of a plane: 32 and a gap that spreads rows over the banks
constexpr int kFloatPlane = (FloatTile::BM + FloatTile::BN) * kFloatPitch;

// A thread's part of an operand's stage: eight floats.  Summed over entries: four neighbours of two rows 64 apart; over rows (kTurned): a
// block of two rows and four neighbours, turned on the way to LDS.
template <bool kTurned>
struct FloatLoader {
  FloatOperand x;
  const float* at[2];                        // summed over entries: the thread's rows; over rows: its entries of row 0, and of row 1
  int64_t first;                             // the tile's first row (or entry)
  int64_t count;                             // rows (or entries) of the operand
  int row, step;                             // thread's place in the tile
  v4f v[2][2];                               // two stages
  int mark[2][2];                            // turned: of the rows
  __device__ __forceinline__ const float* row_at(int64_t r) const {
    return x.p + (x.vars == 1 ? r * x.stride_ex : r / x.vars * x.stride_ex + r % x.vars * x.stride_var);
  }
  __device__ __forceinline__ FloatLoader(const FloatOperand& o, int64_t first_, int64_t count_) : x(o), first(first_), count(count_) {
    if constexpr (kTurned) {
      step = threadIdx.x % 8 * 2;
      row = threadIdx.x / 8 * 4;
      // (blocks past the end take the last four entries, to where those belong)
      if (plain()) row = (int)min((int64_t)row, count - 4 - first);
      at[0] = x.p + (first + row) * x.stride;
    } else {
      step = threadIdx.x % 4 * 4;
      row = threadIdx.x / 4;
#pragma unroll
      for (int i = 0; i < 2; ++i) at[i] = row_at(min(first + row + 64 * i, count - 1));
    }
  }
  // whether all of the tile's requests are of four neighbours
  __device__ __forceinline__ bool plain() const {
    return x.stride == 1 && (!kTurned || (x.vars == 1 && count - first >= 4));
  }
  // steps [k, k + 16), all of them there
  template <int kSet>
  __device__ __forceinline__ void load_plain(int64_t k) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if constexpr (kTurned) {
        const int64_t r = k + step + i;
        // (without marks any word of the row is read, and not looked at)
        mark[kSet][i] = *(x.skip ? x.skip + r : reinterpret_cast<const int*>(x.p + r * x.stride_ex));
        v[kSet][i] = *reinterpret_cast<const v4f_by4*>(at[0] + r * x.stride_ex);
      } else {
        v[kSet][i] = *reinterpret_cast<const v4f_by4*>(at[i] + k + step);
      }
    }
  }
  // steps [k, k + 16) of those below end, any strides; into the first set
  __device__ __forceinline__ void load_any(int64_t k, int64_t end) {
    const int64_t s = k + step;
    const bool fours = plain();
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if constexpr (kTurned) {
        const bool some = s + i < end && !(x.skip && x.skip[s + i] == kDeadRow);
        mark[0][i] = 0;
        v[0][i] = v4f{0.f, 0.f, 0.f, 0.f};
        if (!some) continue;
        if (fours) v[0][i] = *reinterpret_cast<const v4f_by4*>(at[0] + (s + i) * x.stride_ex);
        else
#pragma unroll
          for (int e = 0; e < 4; ++e) v[0][i][e] = first + row + e < count ? row_at(s + i)[(first + row + e) * x.stride] : 0.f;
      } else if (fours && s + 4 <= end) {
        v[0][i] = *reinterpret_cast<const v4f_by4*>(at[i] + s);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[0][i][e] = s + e < end ? at[i][(s + e) * x.stride] : 0.f;
      }
    }
  }
  // one half of a set's floats to LDS, in three parts each
  template <int kSet, int kHalf>
  __device__ __forceinline__ void store(char* planes_of) const {
    if constexpr (!kTurned) {
      v4f w = v[kSet][kHalf];
      char* const to = planes_of + (row + 64 * kHalf) * kFloatPitch + step * 2;
#pragma unroll
      for (int p = 0; p < 3; ++p) {
        const uint32_t a = p ? pair_of<bf16>(w[0], w[1]) : pair_of<bf16>(first_part(w[0]), first_part(w[1]));
        const uint32_t b = p ? pair_of<bf16>(w[2], w[3]) : pair_of<bf16>(first_part(w[2]), first_part(w[3]));
        *reinterpret_cast<uint2*>(to + p * kFloatPlane) = make_uint2(a, b);
        if (p < 2) w -= v4f{as_float(a << 16), as_float(a & 0xffff0000u), as_float(b << 16), as_float(b & 0xffff0000u)};
      }
    } else {
      const bool none[2] = {x.skip && mark[kSet][0] == kDeadRow, x.skip && mark[kSet][1] == kDeadRow};
#pragma unroll
      for (int e = 2 * kHalf; e < 2 * kHalf + 2; ++e) {
        float u = none[0] ? 0.f : v[kSet][0][e], w = none[1] ? 0.f : v[kSet][1][e];
        char* const to = planes_of + (row + e) * kFloatPitch + step * 2;
#pragma unroll
        for (int p = 0; p < 3; ++p) {
          const uint32_t a = p ? pair_of<bf16>(u, w) : pair_of<bf16>(first_part(u), first_part(w));
          *reinterpret_cast<uint32_t*>(to + p * kFloatPlane) = a;
          if (p < 2) {
            u -= as_float(a << 16);
            w -= as_float(a & 0xffff0000u);
          }
        }
      }
    }
  }
};

// The tile loop.  Two stages in LDS: while one is multiplied the next is taken apart, instruction by instruction between the products,
// and the one after it is on its way to registers; one barrier a stage.
template <bool kTurnedA, bool kTurnedB>
__device__ __forceinline__ void float_stages(const FloatOperand& a, const FloatOperand& b, const TileAt& tile, int64_t m, int64_t n, int64_t k, int64_t first,
                                             int64_t last, char* lds, v16f (&sums)[FloatTile::FM][FloatTile::FN]) {
  typedef FloatTile S;
  FloatLoader<kTurnedA> from_a(a, tile.m0, m);
  FloatLoader<kTurnedB> from_b(b, tile.n0, n);
  const int lane = threadIdx.x & 63, row = lane & 31, half = lane >> 5, wave = threadIdx.x / 64;
  const int wm = wave % S::waves_m * S::WM, wn = wave / S::waves_m * S::WN;
  const int at_a = (wm + row) * kFloatPitch + half * 16, at_b = (S::BM + wn + row) * kFloatPitch + half * 16;
  auto load_any = [&](int64_t s) {
    from_a.load_any(s * kFloatSteps, k);
    from_b.load_any(s * kFloatSteps, k);
  };
  auto store = [&](char* to) {
    from_a.template store<0, 0>(to);
    from_a.template store<0, 1>(to);
    from_b.template store<0, 0>(to + S::BM * kFloatPitch);
    from_b.template store<0, 1>(to + S::BM * kFloatPitch);
  };
  v4i fa[3][S::FM], fb[3][S::FN];
  auto read = [&](const char* from) {
#pragma unroll
    for (int p = 0; p < 3; ++p) {
#pragma unroll
      for (int i = 0; i < S::FM; ++i) fa[p][i] = *reinterpret_cast<const v4i*>(from + at_a + p * kFloatPlane + i * 32 * kFloatPitch);
#pragma unroll
      for (int j = 0; j < S::FN; ++j) fb[p][j] = *reinterpret_cast<const v4i*>(from + at_b + p * kFloatPlane + j * 32 * kFloatPitch);
    }
  };
  auto multiply = [&](int p) {               // hl lh mm hm mh hh
    constexpr int of_a[6] = {0, 2, 1, 0, 1, 0}, of_b[6] = {2, 0, 1, 1, 0, 0};
#pragma unroll
    for (int i = 0; i < S::FM; ++i)
#pragma unroll
      for (int j = 0; j < S::FN; ++j) sums[i][j] = Cores<bf16>::mma(fa[of_a[p]][i], fb[of_b[p]][j], sums[i][j]);
  };
  char *mine = lds, *next = lds + 3 * kFloatPlane;
  auto swap = [&] {
    char* const was = mine;
    mine = next;
    next = was;
  };
  // stages that are there in whole, in requests of four neighbours
  const int64_t whole = from_a.plain() && from_b.plain() ? min(last, k / kFloatSteps) : first;
  auto load_plain = [&](auto set, int64_t s) {   // (past the end the last one once more, not used)
    const int64_t at = min(s, whole - 1) * kFloatSteps;
    from_a.template load_plain<set.value>(at);
    from_b.template load_plain<set.value>(at);
  };
  // stage s is in LDS, s + 1 in the other set of registers; s + 2 goes into `set`
  auto stage = [&](auto set, int64_t s) {
    constexpr int kOther = 1 - set.value;
    char* const to_b = next + S::BM * kFloatPitch;
    load_plain(set, s + 2);
    read(mine);
    multiply(0);
    from_a.template store<kOther, 0>(next);
    __builtin_amdgcn_sched_barrier(0);
    multiply(1);
    from_a.template store<kOther, 1>(next);
    __builtin_amdgcn_sched_barrier(0);
    multiply(2);
    from_b.template store<kOther, 0>(to_b);
    __builtin_amdgcn_sched_barrier(0);
    multiply(3);
    from_b.template store<kOther, 1>(to_b);
    __builtin_amdgcn_sched_barrier(0);
    multiply(4);
    multiply(5);
    __syncthreads();
    swap();
  };
  constexpr std::integral_constant<int, 0> kSet0{};
  constexpr std::integral_constant<int, 1> kSet1{};
  int64_t s = first;
  if (first + 1 < whole) {
    load_plain(kSet0, first);
    load_plain(kSet1, first + 1);
    store(mine);
    __syncthreads();
    for (; s + 2 < whole; s += 2) {
      stage(kSet0, s);
      stage(kSet1, s + 1);
    }
    if (s + 1 < whole) {
      stage(kSet0, s);
      ++s;
    }
  } else if (first < last) {
    load_any(first);
    store(mine);
    __syncthreads();
  }
  for (; s < last; ++s) {                  // stage s is in LDS
    if (s + 1 < last) load_any(s + 1);
    read(mine);
    if (s + 1 < last) store(next);
#pragma unroll
    for (int p = 0; p < 6; ++p) multiply(p);
    __syncthreads();
    swap();
  }
}

// Sums over steps [0, k) of a's rows (m) and b's (n), as product_tile; parts of the steps by blockIdx.y
template <typename Done>
__device__ __forceinline__ void float_tile(const FloatOperand& a, const FloatOperand& b, int64_t m, int64_t n, int64_t first_n, int64_t k, int parts, Done done) {
  typedef FloatTile S;
  __shared__ __attribute__((aligned(16))) char lds[6 * kFloatPlane];
  const TileAt tile = tile_at<S>(m, first_n);
  const int64_t stages = (k + kFloatSteps - 1) / kFloatSteps;
  const int64_t first = stages * blockIdx.y / parts, last = stages * (blockIdx.y + 1) / parts;
  v16f sums[S::FM][S::FN] = {};
  if (a.turned) {
    if (b.turned) float_stages<true, true>(a, b, tile, m, n, k, first, last, lds, sums);
    else float_stages<true, false>(a, b, tile, m, n, k, first, last, lds, sums);
  } else {
    if (b.turned) float_stages<false, true>(a, b, tile, m, n, k, first, last, lds, sums);
    else float_stages<false, false>(a, b, tile, m, n, k, first, last, lds, sums);
  }
  const int wave = threadIdx.x / 64;
  done(sums, tile.m0 + wave % S::waves_m * S::WM, tile.n0 + wave / S::waves_m * S::WN, lds);
}

// ---- scores of categories (a) under rows of features (b) -------------------------------------------------------
struct ScoreInputs {
  Operand w, f;
  FloatOperand fw, ff;       // ... of float, of fk entries
  int64_t fk;
  int64_t cats, rows;
  int64_t first_cat;         // the category that is row 0 of w (category 0 of bias and scale)
  int64_t first_row;         // the launch's first row of features, by tiles
  Steps steps;
  BiasRef bias;
  ScaleRef scale;
  GivenRef given;
};
template <typename T, typename S, typename Done>
__device__ __forceinline__ void score_sums(const ScoreInputs& t, Done done) {
  if constexpr (__is_same(T, float)) float_tile(t.fw, t.ff, t.cats, t.rows, t.first_row, t.fk, 1, done);
  else product_tile<T, S>(t.w, t.f, t.cats, t.rows, t.first_row, t.steps, done);
}
// bias and scales of the tile's categories into LDS, while its sums are on their way; a barrier before they are read
template <typename S>
__device__ __forceinline__ void tile_constants(const ScoreInputs& t, float* bias, float* scale) {
  const int64_t m0 = tile_at<S>(t.cats, 0).m0;
  for (int i = threadIdx.x; i < S::BM; i += S::threads) {
    bias[i] = bias_at(t.bias, m0 + i, t.cats);
    scale[i] = t.scale.m && m0 + i < t.cats ? t.scale.m[m0 + i] : 1.f;
  }
}
// The scores of the wave's j-th rows of features
template <typename S, typename Sums>
__device__ __forceinline__ void scores_of(const Sums (&sums)[S::FM][S::FN], int j, float scale_n, const float* bias, const float* scale, int half,
                                          float (&x)[S::FM][16]) {
#pragma unroll
  for (int i = 0; i < S::FM; ++i)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int at = 32 * i + 8 * q + 4 * half;
      const float4 b = *reinterpret_cast<const float4*>(bias + at);
      if constexpr (__is_same(Sums, v16i)) {
        const float4 s = *reinterpret_cast<const float4*>(scale + at);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[i][4 * q + e] = score_of((float)sums[i][j][4 * q + e] * scale_n * (&s.x)[e], (&b.x)[e]);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) x[i][4 * q + e] = score_of(sums[i][j][4 * q + e], (&b.x)[e]);
      }
    }
}
#endif

}  // namespace pcm
