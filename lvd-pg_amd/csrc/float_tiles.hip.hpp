// Products of float matrices on the matrix cores: each float as three bfloat16 parts, h + m + l, and the six largest of the nine
// products of parts; what is left out lies 2^-26 below a product.
//
// A tile's floats come through registers, are taken apart there (some six instructions an entry) and lie in LDS as three planes, from which all
// six products are read: 12 fragments for 24 products of 32 x 32, so LDS is no bound, and the floats are read once, whatever
// their strides and alignment.  Either operand may be turned: summed over its rows.  The six products take six times a bfloat16 product's
// time, 2.4 TFLOP/s a compute unit at most against 0.6 of the cores' own float products.
#pragma once

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
constexpr int kFloatSteps = 32;              // entries of the summed axis in a stage
constexpr int kFloatPitch = 80;              // bytes of a row of a plane: 64 and a gap that spreads rows over the banks
constexpr int kFloatPlane = (FloatTile::BM + FloatTile::BN) * kFloatPitch;

// A thread's part of an operand's stage: 4 x 4 floats.  Summed over entries: four neighbours of four rows 32 apart; over rows: a block of
// four rows and four neighbours, turned on the way to LDS.
struct FloatLoader {
  FloatOperand x;
  const float* at[4];                        // summed over entries: the thread's rows
  int64_t first;                             // the tile's first row (or entry)
  int64_t count;                             // rows (or entries) of the operand
  int row, step;                             // thread's place in the tile
  __device__ __forceinline__ const float* row_at(int64_t r) const {
    return x.p + (x.vars == 1 ? r * x.stride_ex : r / x.vars * x.stride_ex + r % x.vars * x.stride_var);
  }
  __device__ __forceinline__ FloatLoader(const FloatOperand& o, int64_t first_, int64_t count_) : x(o), first(first_), count(count_) {
    step = threadIdx.x % 8 * 4;
    row = threadIdx.x / 8;
    if (x.turned) row *= 4;
    else
#pragma unroll
      for (int i = 0; i < 4; ++i) at[i] = row_at(min(first + row + 32 * i, count - 1));
  }
  // steps [k, k + 32) of those below end
  __device__ __forceinline__ void load(v4f (&v)[4], int64_t k, int64_t end) const {
    const int64_t s = k + step;
    if (!x.turned) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float* const p = at[i] + s * x.stride;
        if (x.stride == 1 && s + 4 <= end) v[i] = *reinterpret_cast<const v4f_by4*>(p);
        else
#pragma unroll
          for (int e = 0; e < 4; ++e) v[i][e] = s + e < end ? p[e * x.stride] : 0.f;
      }
    } else {
      const int64_t m = first + row;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const bool some = s + i < end && !(x.skip && x.skip[s + i] == kDeadRow);
        v[i] = v4f{0.f, 0.f, 0.f, 0.f};
        if (!some) continue;
        const float* const p = row_at(s + i) + m * x.stride;
        if (x.stride == 1 && m + 4 <= count) v[i] = *reinterpret_cast<const v4f_by4*>(p);
        else
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (m + e < count) v[i][e] = p[e * x.stride];
      }
    }
  }
  __device__ __forceinline__ void store(const v4f (&v)[4], char* planes_of) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v4f w;
      if (x.turned) w = v4f{v[0][i], v[1][i], v[2][i], v[3][i]};
      else w = v[i];
      char* const to = planes_of + (row + (x.turned ? i : 32 * i)) * kFloatPitch + step * 2;
#pragma unroll
      for (int p = 0; p < 3; ++p) {
        const uint32_t a = pair_of<bf16>(w[0], w[1]), b = pair_of<bf16>(w[2], w[3]);
        *reinterpret_cast<uint2*>(to + p * kFloatPlane) = make_uint2(a, b);
        w -= v4f{as_float(a << 16), as_float(a & 0xffff0000u), as_float(b << 16), as_float(b & 0xffff0000u)};
      }
    }
  }
};

// Sums over steps [0, k) of a's rows (m) and b's (n), as product_tile; parts of the steps by blockIdx.y
template <typename Done>
__device__ __forceinline__ void float_tile(const FloatOperand& a, const FloatOperand& b, int64_t m, int64_t n, int64_t k, int parts, Done done) {
  typedef FloatTile S;
  __shared__ __attribute__((aligned(16))) char lds[3 * kFloatPlane];
  const TileAt tile = tile_at<S>(m, n);
  const int64_t stages = (k + kFloatSteps - 1) / kFloatSteps;
  const int64_t first = stages * blockIdx.y / parts, last = stages * (blockIdx.y + 1) / parts;
  const FloatLoader from_a(a, tile.m0, m), from_b(b, tile.n0, n);
  const int lane = threadIdx.x & 63, row = lane & 31, half = lane >> 5, wave = threadIdx.x / 64;
  const int wm = wave % S::waves_m * S::WM, wn = wave / S::waves_m * S::WN;
  const char* const at_a = lds + (wm + row) * kFloatPitch + half * 16;
  const char* const at_b = lds + (S::BM + wn + row) * kFloatPitch + half * 16;
  v16f sums[S::FM][S::FN] = {};
  v4f va[4], vb[4];
  if (first < last) {
    from_a.load(va, first * kFloatSteps, k);
    from_b.load(vb, first * kFloatSteps, k);
  }
  for (int64_t s = first; s < last; ++s) {
    from_a.store(va, lds);
    from_b.store(vb, lds + S::BM * kFloatPitch);
    __syncthreads();
    if (s + 1 < last) {
      from_a.load(va, (s + 1) * kFloatSteps, k);
      from_b.load(vb, (s + 1) * kFloatSteps, k);
    }
#pragma unroll
    for (int step = 0; step < 2; ++step) {
      v4i fa[3][S::FM], fb[3][S::FN];
#pragma unroll
      for (int p = 0; p < 3; ++p) {
#pragma unroll
        for (int i = 0; i < S::FM; ++i) fa[p][i] = *reinterpret_cast<const v4i*>(at_a + p * kFloatPlane + i * 32 * kFloatPitch + step * 32);
#pragma unroll
        for (int j = 0; j < S::FN; ++j) fb[p][j] = *reinterpret_cast<const v4i*>(at_b + p * kFloatPlane + j * 32 * kFloatPitch + step * 32);
      }
      constexpr int of_a[6] = {0, 2, 1, 0, 1, 0}, of_b[6] = {2, 0, 1, 1, 0, 0};   // hl lh mm hm mh hh
#pragma unroll
      for (int p = 0; p < 6; ++p)
#pragma unroll
        for (int i = 0; i < S::FM; ++i)
#pragma unroll
          for (int j = 0; j < S::FN; ++j) sums[i][j] = Cores<bf16>::mma(fa[of_a[p]][i], fb[of_b[p]][j], sums[i][j]);
    }
    __syncthreads();
  }
  done(sums, tile.m0 + wm, tile.n0 + wn, lds);
}

// ---- scores of categories (a) under rows of features (b) -------------------------------------------------------
struct ScoreInputs {
  Operand w, f;
  FloatOperand fw, ff;       // ... of float, of fk entries
  int64_t fk;
  int64_t cats, rows;
  Steps steps;
  BiasRef bias;
  ScaleRef scale;
  GivenRef given;
};
template <typename T, typename S, typename Done>
__device__ __forceinline__ void score_sums(const ScoreInputs& t, Done done) {
  if constexpr (__is_same(T, float)) float_tile(t.fw, t.ff, t.cats, t.rows, t.fk, 1, done);
  else product_tile<T, S>(t.w, t.f, t.cats, t.rows, t.steps, done);
}
// bias and scales of a tile's categories into LDS; barriers before and after
template <typename S>
__device__ __forceinline__ void tile_constants(const ScoreInputs& t, int64_t m0, float* bias, float* scale) {
  __syncthreads();
  for (int i = threadIdx.x; i < S::BM; i += S::threads) {
    bias[i] = bias_at(t.bias, m0 + i, t.cats);
    scale[i] = t.scale.m && m0 + i < t.cats ? t.scale.m[m0 + i] : 1.f;
  }
  __syncthreads();
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
