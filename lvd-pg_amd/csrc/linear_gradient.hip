// Gradients of log-probabilities and log-sums of scores that are products of features and weights, without keeping the scores.
//
//   dx[n][c] = sum_j gl[n][j] [c = g_j] - (sum_j gl[n][j] - gz[n]) p[n][c],  p = exp(x - Z)
//   features: dx w, weights: dx^T f, bias: sum_n dx
// The categories are taken in pieces: the scores of a piece once more (gradient_kernel), whose dx goes into the workspace in both
// orders, rounded to the operands' 16 bits (fewer than 1024 rows: in two parts; float: as it is, in one order), then the piece's two products.
// Half's dx is held as dx 2^(15 - e[n]), 2^e[n] the next power of two above what |dx| of the row can be, so that its range holds it whatever the
// loss's scale; its features are turned with 2^(e[n] - largest e) for the sum over rows, which is exact down to the type's least normal
// number (what lies below 2^-14 after it is off by 2^-25 at most).
//
// Bound by the matrix cores where sums are long: 4096 rows of 4096 bf16, a piece of 16384 categories: the scores and dx 500 us (1.10
// PFLOP/s; the scores alone go at 1.23), either product 460 to 480.  Few rows are bound by reading the weights twice and writing their gradients.
#include "product_out.hip.hpp"

namespace pcm {

namespace {
constexpr int kMostBlocks = 256;     // candidates of the largest exponent
constexpr int kFewRows = 1024;       // fewer: dx in two parts (Plan)

// Per row: the weight of p, and the exponent
__global__ __launch_bounds__(256) void row_terms_kernel(GivenRef given, const float* grad_logp, const float* grad_log_sum, const float* log_sum,
                                                        int64_t rows, int64_t cats, float* of_p, int* expo, int* most) {
  __shared__ int sub[256];
  int best = kDeadRow;
  for (int64_t n = (int64_t)blockIdx.x * 256 + threadIdx.x; n < rows; n += kMostBlocks * 256) {
    float total = 0.f, size = 0.f;
    bool past = false;
    for (int s = 0; s < given.slots; ++s) {
      const int64_t g = given_at(given, n / given.vars, n % given.vars, s);
      if (g < 0) continue;
      past |= g >= cats;
      const float by = grad_logp[n * given.slots + s];
      total += by;
      size += fabsf(by);
    }
    if (grad_log_sum) total -= grad_log_sum[n];
    size += fabsf(total);
    int e = kDeadRow;
    if (past) total = size = __builtin_nanf("");
    if (log_sum[n] == -INFINITY) size = 0.f;                        // no category: no gradient
    if (size != 0.f) e = size < INFINITY ? min(max(ilogbf(size) + 1, -100), 127) : 0;   // (NaN, inf: as they are)
    of_p[n] = total;
    expo[n] = e;
    best = max(best, e);
  }
  sub[threadIdx.x] = best;
  __syncthreads();
  for (int s = 128; s; s /= 2) {
    if (threadIdx.x < s) sub[threadIdx.x] = max(sub[threadIdx.x], sub[threadIdx.x + s]);
    __syncthreads();
  }
  if (threadIdx.x == 0) most[blockIdx.x] = sub[0];
}

struct GradientTask : ScoreInputs {   // of a piece of the categories
  const float *grad_logp, *log_sum, *of_p;
  const int* expo;
  float* dx;                         // float: dx [row][pitch_row]
  uint16_t* by_row;                  // dx [plane][row][pitch_row]; null: not needed
  uint16_t* by_cat;                  // dx [plane][category of the piece][pitch_cat]
  int64_t pitch_row, pitch_cat, plane_row, plane_cat;
  float* bias_parts;                 // [tile of rows][category of the piece]; null: none
};

// What dx of a row with exponent e is multiplied by on its way to the operands, 0 for a row without a gradient: only half's range needs it (bfloat16 has
// float's, and sums of scaled ones would leave that where weights or features are large)
template <typename T>
__device__ __forceinline__ float scale_of(int e) { return e == kDeadRow ? 0.f : __is_same(T, f16) ? ldexpf(1.f, 15 - e) : 1.f; }

// Numbers as the operands hold them, two to a word: the nearest ones, and with kParts > 1 the nearest ones to what is left
template <typename T, int kParts>
struct Coded {
  uint32_t p[kParts];
  __device__ __forceinline__ Coded(float u, float v) {
#pragma unroll
    for (int i = 0; i < kParts; ++i) {
      p[i] = pair_of<T>(u, v);
      u -= (float)__builtin_bit_cast(T, (uint16_t)(p[i] & 0xffffu));
      v -= (float)__builtin_bit_cast(T, (uint16_t)(p[i] >> 16));
    }
  }
};
// 4 x 4 entries of two bytes turned among four neighbouring lanes: lane i has row i as (0 1) and (2 3) and gets column i
__device__ __forceinline__ void turn(uint32_t& a, uint32_t& b) {
  const int lane = threadIdx.x;
  // pairs of lanes two apart exchange halves: the lower two keep columns 0 1, the upper two get 2 3
  const uint32_t give = lane & 2 ? a : b, got = lane_xor<2>(give);
  uint32_t u = lane & 2 ? got : a, v = lane & 2 ? b : got;      // rows (0 2) or (1 3) of two columns
  // neighbours exchange columns: u is of row i & 1, v of row (i & 1) + 2
  const uint32_t gu = lane_xor<1>(u), gv = lane_xor<1>(v);
  const uint32_t order = lane & 1 ? 0x03020706u : 0x05040100u;   // bytes of (own, other): odd lanes take the high halves, even the low ones
  u = __builtin_amdgcn_perm(gu, u, order);
  v = __builtin_amdgcn_perm(gv, v, order);
  a = u;
  b = v;
}

template <typename T, typename S, int kParts>
__device__ __forceinline__ void gradient_tile(const GradientTask& t) {
  __shared__ __attribute__((aligned(16))) float bias[S::BM], scale[S::BM];
  tile_constants<S>(t, bias, scale);
  score_sums<T, S>(t, [&](auto& sums, int64_t m, int64_t n, char* lds) {
    const int lane = threadIdx.x & 63, half = lane >> 5, wave = threadIdx.x / 64, wm = wave % S::waves_m * S::WM;
    float* const of_bias = reinterpret_cast<float*>(lds);                   // [waves_n][BM]
    __syncthreads();
#pragma unroll
    for (int j = 0; j < S::FN; ++j) {
      __builtin_amdgcn_sched_barrier(0);
      const int64_t row = n + 32 * j + (lane & 31);
      const bool valid = row < t.rows;
      const int64_t at = valid ? row : t.rows - 1;
      float dx[S::FM][16];
      scores_of<S>(sums, j, 1.f, bias + wm, scale + wm, half, dx);
      const float z = t.log_sum[at], of_p = t.of_p[at];
      const float by = scale_of<T>(valid ? t.expo[at] : kDeadRow);
#pragma unroll
      for (int i = 0; i < S::FM; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const float p = __builtin_amdgcn_exp2f((dx[i][r] - z) * kLog2e);
          dx[i][r] = by == 0.f ? 0.f : -of_p * p;
        }
      if (t.given.slots && by != 0.f) {
        const int64_t ex = row / t.given.vars, v = row % t.given.vars;
        for (int s = 0; s < t.given.slots; ++s) {
          const int64_t g = given_at(t.given, ex, v, s) - t.first_cat - m;
          if (g < 0 || g >= S::WM || (g >> 2 & 1) != half) continue;
          const float add = t.grad_logp[row * t.given.slots + s];
#pragma unroll
          for (int i = 0; i < S::FM; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r) dx[i][r] += (int)g == 32 * i + 8 * (r / 4) + 4 * half + r % 4 ? add : 0.f;
        }
      }
      if (t.bias_parts) {   // over the 32 lanes of a half
#pragma unroll
        for (int i = 0; i < S::FM; ++i)
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            float s = over_lanes<16>(dx[i][r], Sum());
            s += __shfl_xor(s, 16);
            float& to = of_bias[wave / S::waves_m * S::BM + wm + 32 * i + 8 * (r / 4) + 4 * half + r % 4];
            if ((lane & 31) == 0) to = j ? to + s : s;
          }
      }
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (__is_same(T, float)) {
        if (t.dx && valid) {
          float* const to = t.dx + row * t.pitch_row + m + 4 * half;
#pragma unroll
          for (int i = 0; i < S::FM; ++i)
#pragma unroll
            for (int q = 0; q < 4; ++q)
              if (m + 32 * i + 8 * q + 4 * half < t.pitch_row)
                *reinterpret_cast<float4*>(to + 32 * i + 8 * q) = make_float4(dx[i][4 * q], dx[i][4 * q + 1], dx[i][4 * q + 2], dx[i][4 * q + 3]);
        }
      } else {
      // by row: eight neighbouring categories a lane, from both halves' four; by category: four neighbouring rows, of a quad of lanes
      uint16_t* by_row = t.by_row + row * t.pitch_row + m + 8 * half;
      const int64_t row4 = row - (lane & 3);
      uint16_t* by_cat = t.by_cat + (m + 4 * half + (lane & 3)) * t.pitch_cat + row4;
#pragma unroll
      for (int i = 0; i < S::FM; ++i)
#pragma unroll
        for (int q = 0; q < 4; q += 2) {
          uint32_t code[kParts][4];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const Coded<T, kParts> two(dx[i][4 * q + 2 * k] * by, dx[i][4 * q + 2 * k + 1] * by);
#pragma unroll
            for (int part = 0; part < kParts; ++part) code[part][k] = two.p[part];
          }
          if (t.by_cat) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const int64_t c = m + 32 * i + 8 * (q + h) + 4 * half + (lane & 3);
#pragma unroll
              for (int part = 0; part < kParts; ++part) {
                uint32_t a = code[part][2 * h], b = code[part][2 * h + 1];
                turn(a, b);
                if (c < t.cats && row4 < t.pitch_cat) {
                  uint16_t* const to = by_cat + part * t.plane_cat;
                  *reinterpret_cast<uint2*>(to) = make_uint2(a, b);
                  if (S::BN < kKBytes / 2 && row4 + S::BN < t.pitch_cat)   // (one tile of rows, shorter than a step)
                    *reinterpret_cast<uint2*>(to + S::BN) = make_uint2(0, 0);
                }
              }
              by_cat += 8 * t.pitch_cat;
            }
          }
          if (t.by_row) {
#pragma unroll
            for (int part = 0; part < kParts; ++part) {
              const auto lo = __builtin_amdgcn_permlane32_swap(code[part][0], code[part][2], false, false);
              const auto hi = __builtin_amdgcn_permlane32_swap(code[part][1], code[part][3], false, false);
              if (valid && m + 32 * i + 8 * q + 8 * half < t.pitch_row)
                *reinterpret_cast<uint4*>(by_row + part * t.plane_row + 32 * i + 8 * q) = make_uint4(lo[0], hi[0], lo[1], hi[1]);
            }
          }
        }
      }
    }
    if (t.bias_parts) {
      __syncthreads();
      for (int i = threadIdx.x; i < S::BM; i += S::threads) {
        float s = 0.f;
#pragma unroll
        for (int w = 0; w < S::waves / S::waves_m; ++w) s += of_bias[w * S::BM + i];
        if (m - wm + i < t.cats) t.bias_parts[n / S::BN * t.cats + m - wm + i] = s;
      }
    }
  });
}
template <typename T, typename S, int kParts>
__global__ __launch_bounds__(S::threads, 2) void gradient_kernel(GradientTask t) {
  gradient_tile<T, S, kParts>(t);
}

// Few rows: dx of a tile of categories in LDS, then out in whichever orders are needed
template <typename T, int kGroups>
__global__ __launch_bounds__(FewTile<kGroups>::threads) void gradient_few_kernel(GradientTask t, FewOperand w, FewOperand f, int length) {
  typedef FewTile<kGroups> S;
  __shared__ __attribute__((aligned(16))) char lds[S::lds];
  float* const dx = const_cast<float*>(few_sums<T, kGroups>(w, f, t.cats, t.rows, length, 1, lds));
  constexpr int kLanes = S::threads / S::rows, kOwn = S::longs / kLanes;   // lanes to a row, and categories of each
  const int in = threadIdx.x % S::rows, lane = threadIdx.x / S::rows;
  const int64_t c0 = (int64_t)blockIdx.x * S::longs, n0 = (int64_t)blockIdx.z * S::rows, n = n0 + in, at_n = min(n, t.rows - 1);
  const float z = t.log_sum[at_n], of_p = t.of_p[at_n];
  const int e = n < t.rows ? t.expo[at_n] : kDeadRow;
  float own[kOwn];
#pragma unroll
  for (int i = 0; i < kOwn; ++i) {
    const int at = lane + i * kLanes;
    const float x = score_of(dx[at * S::pitch + in], bias_at(t.bias, c0 + at, t.cats));
    own[i] = e == kDeadRow ? 0.f : -of_p * __builtin_amdgcn_exp2f((x - z) * kLog2e);
  }
  if (e != kDeadRow)
    for (int s = 0; s < t.given.slots; ++s) {
      const int64_t g = given_at(t.given, n / t.given.vars, n % t.given.vars, s) - t.first_cat - c0;
      const float add = t.grad_logp[n * t.given.slots + s];
#pragma unroll
      for (int i = 0; i < kOwn; ++i) own[i] += g == lane + i * kLanes ? add : 0.f;
    }
#pragma unroll
  for (int i = 0; i < kOwn; ++i) dx[(lane + i * kLanes) * S::pitch + in] = own[i];
  __syncthreads();
  if (t.bias_parts && threadIdx.x < S::longs && c0 + threadIdx.x < t.cats) {
    float s = 0.f;
    for (int r = 0; r < S::rows; ++r) s += dx[threadIdx.x * S::pitch + r];
    t.bias_parts[blockIdx.z * t.cats + c0 + threadIdx.x] = s;
  }
  if constexpr (sizeof(T) == 4) {
    if (!t.dx) return;
    for (int i = threadIdx.x; i < S::longs * S::rows; i += S::threads) {
      const int c = i % S::longs, r = i / S::longs;
      if (n0 + r < t.rows && c0 + c < t.pitch_row) t.dx[(n0 + r) * t.pitch_row + c0 + c] = dx[c * S::pitch + r];
    }
  } else {                             // two at a time, in two parts; the turned rows up to a whole step
    if (t.by_row)
      for (int i = threadIdx.x; i < S::longs / 2 * S::rows; i += S::threads) {
        const int c = i % (S::longs / 2) * 2, r = i / (S::longs / 2);
        if (n0 + r >= t.rows || c0 + c >= t.pitch_row) continue;
        const float by = scale_of<T>(t.expo[n0 + r]);
        const Coded<T, 2> two(dx[c * S::pitch + r] * by, dx[(c + 1) * S::pitch + r] * by);
#pragma unroll
        for (int part = 0; part < 2; ++part) *reinterpret_cast<uint32_t*>(t.by_row + part * t.plane_row + (n0 + r) * t.pitch_row + c0 + c) = two.p[part];
      }
    if (t.by_cat)
      for (int i = threadIdx.x; i < S::longs * 32; i += S::threads) {
        const int r = i % 32 * 2, c = i / 32;
        if (c0 + c >= t.cats || n0 + r >= t.pitch_cat) continue;
        float v[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const float by = scale_of<T>(n0 + r + k < t.rows ? t.expo[n0 + r + k] : kDeadRow);
          v[k] = by == 0.f ? 0.f : dx[c * S::pitch + (r + k < S::rows ? r + k : 0)] * by;
        }
        const Coded<T, 2> two(v[0], v[1]);
#pragma unroll
        for (int part = 0; part < 2; ++part) *reinterpret_cast<uint32_t*>(t.by_cat + part * t.plane_cat + (c0 + c) * t.pitch_cat + n0 + r) = two.p[part];
      }
  }
}

// float: categories that the bias masks, whose weights have no part in the features' gradients
__global__ __launch_bounds__(256) void masked_kernel(BiasRef bias, int64_t cats, int* skip) {
  const int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (c < cats) skip[c] = bias_at(bias, c, cats) == -INFINITY ? kDeadRow : 0;
}

// 32 categories a workgroup, eight lanes to each
__global__ __launch_bounds__(256) void join_bias_kernel(const float* parts, int64_t count, int64_t cats, void* out, int type, int64_t first) {
  __shared__ float sub[8][32];
  const int in = threadIdx.x % 32, lane = threadIdx.x / 32;
  const int64_t c = (int64_t)blockIdx.x * 32 + in;
  float s = 0.f;
  if (c < cats)
    for (int64_t i = lane; i < count; i += 8) s += parts[i * cats + c];
  sub[lane][in] = s;
  __syncthreads();
  if (lane || c >= cats) return;
  for (int i = 1; i < 8; ++i) s += sub[i][in];
  store_as(out, type, first + c, s);
}

typedef TileSizes<256, 256, 128, 64> Wide;
typedef TileSizes<128, 128, 64, 64> Middle;
typedef TileSizes<128, 64, 64, 32> Slim;
typedef TileSizes<128, 32, 32, 32> Narrow;
int tile_rows(int64_t cats, int64_t rows, int64_t steps, bool of_float) {
  return of_float ? 128 : rows <= 64 ? (rows <= 32 ? 32 : 64) : wide_tiles(cats, rows, steps) ? 256 : 128;
}

template <typename T, typename S, int kParts>
void launch(const GradientTask& t, hipStream_t stream) {
  const int64_t tiles = ((t.cats + S::BM - 1) / S::BM) * ((t.rows + S::BN - 1) / S::BN);
  hipLaunchKernelGGL((gradient_kernel<T, S, kParts>), dim3((unsigned)tiles), dim3(S::threads), 0, stream, t);
}
template <typename T, int kParts>
void launch(const GradientTask& t, hipStream_t stream) {
  const int size = tile_rows(t.cats, t.rows, t.steps.count, false);
  if (size == 256) launch<T, Wide, kParts>(t, stream);
  else if (size == 128) launch<T, Middle, kParts>(t, stream);
  else if (size == 64) launch<T, Slim, kParts>(t, stream);
  else launch<T, Narrow, kParts>(t, stream);
}

template <typename T>
void launch_few(const GradientTask& t, const FewOperand& w, const FewOperand& f, int length, hipStream_t stream) {
  const int64_t each = kFewTile, cols = sizeof(T) == 4 ? t.cats : laid_length(t.cats);   // (what is behind the last category is written too)
  const dim3 grid((unsigned)((cols + each - 1) / each), 1, (unsigned)((t.rows + kFewRowsMost - 1) / kFewRowsMost)), block(t.rows > 32 ? 256 : 512);
  if (t.rows <= 16) hipLaunchKernelGGL((gradient_few_kernel<T, 1>), grid, block, 0, stream, t, w, f, length);
  else if (t.rows <= 32) hipLaunchKernelGGL((gradient_few_kernel<T, 2>), grid, block, 0, stream, t, w, f, length);
  else hipLaunchKernelGGL((gradient_few_kernel<T, 4>), grid, block, 0, stream, t, w, f, length);
}

// What the workspace holds, and how the categories are cut into pieces
struct Plan {
  bool of_float, few, lay_f, lay_w;
  int dx_planes;
  PlanePairs dx_pairs;
  int64_t rows, cats, length, piece, pieces, part, parts;     // part: rows of one
  bool features_direct, weight_direct;                        // whether a product gives them as they are
  int features_parts, weight_parts;
  int64_t of_p, expo, most, skip, f, f_turned, w, w_turned, by_row, by_cat, features, weight, bias, bytes;   // offsets

  Plan(const Matrix2& fm, const Matrix2& wm, bool of_features, bool of_weight, bool of_bias) {
    of_float = fm.type == PCM_F32;
    rows = fm.rows();
    cats = wm.examples;
    length = fm.length;
    few = takes_few(fm, wm);
    lay_f = !few && !readable(fm);
    lay_w = !few && !readable(wm);
    // Rounded once, dx is off by as much as rounding the results is, however many terms a sum has: bf16 gradients by 2.2e-3 to 2.3e-3 of their norm, where
    // the results' own rounding is 1.66e-3, half's by 2.8e-4 and 2.1e-4.  A second part takes that away, for twice the steps of two of the
    // four products.  Rows x 4096 x 50304 bf16, one part and two: 16 rows 559 us, 636; 64 568, 653; 256 786, 1014; 1000 1668, 2506; 4096
    // 4834, 7686; 32768 x 768 x 128 f16 124, 142.  So fewer than 1024 rows, where it is less than a millisecond, take two.
    dx_planes = !of_float && rows < kFewRows ? 2 : 1;
    dx_pairs = dx_planes == 2 ? kTwoOfB : kOnePlane;
    // (float's weights are read where they are)
    const int64_t most_cats = most_piece(rows, length, !of_float);
    piece = cats <= most_cats ? cats : piece_for(most_cats);
    pieces = (cats + piece - 1) / piece;
    part = part_rows(rows, fm.vars, piece);
    parts = (rows + part - 1) / part;
    const int64_t cat_steps = steps_of(piece), row_steps = steps_of(part);
    features_parts = (int)std::min<int64_t>(parts_for(length, part, cat_steps * dx_pairs.count, of_float), cat_steps);
    weight_parts = (int)std::min<int64_t>(parts_for(length, piece, row_steps * dx_pairs.count, of_float), row_steps);
    features_direct = pieces == 1 && features_parts == 1;
    weight_direct = parts == 1 && weight_parts == 1;
    int64_t at = 0;
    auto take = [&](bool needed, int64_t n) {
      const int64_t here = at;
      if (needed) at += round_up(n, 256);
      return here;
    };
    of_p = take(true, rows * 4);
    expo = take(true, rows * 4);
    most = take(true, kMostBlocks * 4);
    skip = take(of_float && of_features, cats * 4);
    f = take(lay_f, laid_bytes(rows, length, 1));
    f_turned = take(of_weight && !of_float, laid_bytes(length, rows, 1));
    w = take(lay_w, laid_bytes(piece, length, 1));
    w_turned = take(of_features && !of_float, laid_bytes(length, piece, 1));
    by_row = take(of_float ? of_features || of_weight : of_features, of_float ? part * round_up(piece, 4) * 4 : laid_bytes(part, piece, dx_planes));
    by_cat = take(of_weight && !of_float, laid_bytes(piece, part, dx_planes));
    features = take(of_features && !features_direct, features_parts * rows * length * 4);
    weight = take(of_weight && !weight_direct, weight_parts * piece * length * 4);
    bias = take(of_bias, (rows + 63) / 64 * piece * 4);       // (tiles have 64 rows or more, if there are as many)
    bytes = at;
  }
  // The size of pieces, of at most `most` categories: the one whose tiles take the fewest turns of the compute units (256 tiles of 256 x 256, or 512 of
  // 128 x 128), a quarter of a turn more for each piece's launches.  4096 rows of 4096 bf16, 50304 categories: four like pieces take 15 turns,
  // three of 16384 and a short one 13 (6.5 ms the step, 6.2).
  int64_t piece_for(int64_t most) const {
    const int64_t each = of_float ? 128 : 256, turn = of_float ? 512 : 256, row_tiles = (rows + each - 1) / each;
    auto turns = [&](int64_t n) { return n ? 4 * (((n + each - 1) / each * row_tiles + turn - 1) / turn) + 1 : 0; };
    int64_t best = most, least = -1;
    for (int64_t n = most; n > most / 2 && n > most - 64 * 256; n -= 256) {
      const int64_t all = cats / n * turns(n) + turns(cats % n);
      if (least < 0 || all < least) {
        least = all;
        best = n;
      }
    }
    return best;
  }
  // steps of a sum over n entries
  int64_t steps_of(int64_t n) const { return of_float ? (n + kFloatSteps - 1) / kFloatSteps : laid_length(n) * 2 / kKBytes; }
};
}  // namespace

int64_t linear_scores_backward_workspace(const Matrix2& f, const Matrix2& w, bool of_features, bool of_weight, bool of_bias) {
  return Plan(f, w, of_features, of_weight, of_bias).bytes;
}

void linear_scores_backward(const Matrix2& f, const Matrix2& w, const BiasRef& bias, const GivenRef& given_in, const float* d_grad_logp,
                            const float* d_grad_log_sum, const float* d_log_sum, const LinearGradients& out, void* d_work, int64_t work_bytes,
                            hipStream_t stream) {
  check_linear(f, w, bias, given_in, "gradient of linear scores");
  const int64_t rows = f.rows(), cats = w.examples;
  if (!rows) {   // sums of nothing, which need no workspace
    if (out.weight) join_parts(nullptr, 0, false, f.length, cats, Finish(), out.weight, f.type, f.length, stream);
    if (out.bias) join_parts(nullptr, 0, false, cats, 1, Finish(), out.bias, bias.type, cats, stream);
    return;
  }
  if (given_in.slots && (!given_in.p || !d_grad_logp)) fail(PCM_ERR_ARG, "gradient of linear scores: given categories and their derivatives go together");
  if (!w.p || !f.p || !d_log_sum) fail(PCM_ERR_ARG, "gradient of linear scores: a pointer is null");
  const Plan plan(f, w, out.features, out.weight, out.bias);
  check_workspace(d_work, work_bytes, plan.bytes, "gradient of linear scores");
  char* const work = static_cast<char*>(d_work);
  GivenRef given = given_in;
  given.vars = f.vars;
  float* const of_p = reinterpret_cast<float*>(work + plan.of_p);
  int *const expo = reinterpret_cast<int*>(work + plan.expo), *const most = reinterpret_cast<int*>(work + plan.most);
  hipLaunchKernelGGL(row_terms_kernel, dim3(kMostBlocks), dim3(256), 0, stream, given, d_grad_logp, d_grad_log_sum, d_log_sum, rows, cats, of_p, expo, most);
  const bool of_float = plan.of_float, of_half = f.type == PCM_F16;
  const int size = of_float ? 4 : 2;
  int* const skip = of_float && out.features && bias.p ? reinterpret_cast<int*>(work + plan.skip) : nullptr;
  if (skip) hipLaunchKernelGGL(masked_kernel, dim3((unsigned)((cats + 255) / 256)), dim3(256), 0, stream, bias, cats, skip);
  char* at = work + plan.f;
  const Operand features = of_float || plan.few ? Operand{} : operand_of(f, at, stream);
  LayOut scaled;
  scaled.expo = expo;
  if (of_half) scaled.most = most;
  if (out.weight && !of_float) lay_out(f, 0, rows, true, scaled, work + plan.f_turned, stream);
  LayOut masked;
  masked.mask = bias;
  const int64_t all_turned = laid_length(rows), index_bytes = given.type == PCM_U8 ? 1 : given.type == PCM_I32 ? 4 : 8;
  for (int64_t first = 0; first < cats; first += plan.piece) {
    const int64_t count = std::min(plan.piece, cats - first), laid = laid_length(count), pitch = of_float ? round_up(count, 4) : laid;
    Matrix2 of_piece = w;
    of_piece.p = static_cast<const char*>(w.p) + first * w.stride_ex * size;
    of_piece.examples = count;
    GradientTask t{};
    if (!plan.few && of_float) {
      t.fw = float_operand(of_piece, false);
      t.fk = f.length;
    } else if (plan.lay_w) {
      lay_out(w, first, count, false, LayOut(), work + plan.w, stream);
      t.w = {work + plan.w, laid_length(w.length) * 2, 0};
    } else if (!plan.few) {
      t.w = {of_piece.p, w.stride_ex * 2, 0};
    }
    t.cats = count;
    t.steps = {(int)(laid_length(f.length) * 2 / kKBytes), kOnePlane, 1};
    t.bias = bias;
    if (t.bias.p) t.bias.p = static_cast<const char*>(bias.p) + first * (bias.type == PCM_F32 ? 4 : 2);
    t.given = given;
    t.first_cat = first;
    t.pitch_row = pitch;
    if (of_float) t.dx = out.features || out.weight ? reinterpret_cast<float*>(work + plan.by_row) : nullptr;
    else t.by_row = out.features ? reinterpret_cast<uint16_t*>(work + plan.by_row) : nullptr;
    t.by_cat = out.weight && !of_float ? reinterpret_cast<uint16_t*>(work + plan.by_cat) : nullptr;
    int64_t bias_tiles = 0;
    for (int64_t row = 0; row < rows; row += plan.part) {
      const int64_t n = std::min(plan.part, rows - row), example = row / f.vars, turned = laid_length(n);
      Matrix2 of_rows = f;
      of_rows.p = static_cast<const char*>(f.p) + example * f.stride_ex * size;
      of_rows.examples = n / f.vars;
      if (!plan.few && of_float) t.ff = float_operand(of_rows, false);
      t.f = features;
      if (features.p) t.f.p = static_cast<const char*>(features.p) + row * features.pitch;
      t.rows = n;
      if (given.p) t.given.p = static_cast<const char*>(given.p) + example * given.stride_ex * index_bytes;
      t.grad_logp = d_grad_logp + row * given.slots;
      t.log_sum = d_log_sum + row;
      t.of_p = of_p + row;
      t.expo = expo + row;
      t.pitch_cat = turned;
      t.plane_row = n * laid;
      t.plane_cat = count * turned;
      t.bias_parts = out.bias ? reinterpret_cast<float*>(work + plan.bias) + bias_tiles * count : nullptr;
      if (plan.few) {
        const FewOperand fw = few_operand(of_piece), ff = few_operand(of_rows);
        if (of_float) launch_few<float>(t, fw, ff, f.length, stream);
        else if (f.type == PCM_BF16) launch_few<bf16>(t, fw, ff, f.length, stream);
        else launch_few<f16>(t, fw, ff, f.length, stream);
      } else if (of_float) launch<float, FloatTile, 1>(t, stream);
      else if (f.type == PCM_BF16) plan.dx_planes == 2 ? launch<bf16, 2>(t, stream) : launch<bf16, 1>(t, stream);
      else plan.dx_planes == 2 ? launch<f16, 2>(t, stream) : launch<f16, 1>(t, stream);
      const int64_t bias_rows = plan.few ? kFewRowsMost : tile_rows(count, n, t.steps.count, of_float);
      bias_tiles += (n + bias_rows - 1) / bias_rows;
      const Matrix2 dx{t.dx, PCM_F32, pitch, 0, 1, n, 1, (int32_t)count};
      if (out.features) {
        OutTask o{};
        if (of_float) {
          o.fa = float_operand(of_piece, true, skip ? skip + first : nullptr);
          o.fb = float_operand(dx, false);
          o.fk = count;
        } else {
          if (!row) lay_out(w, first, count, true, masked, work + plan.w_turned, stream);
          o.a = {work + plan.w_turned, laid * 2, 0};
          o.b = {t.by_row, laid * 2, t.plane_row * 2};
          if (of_half) o.finish.expo = t.expo;
        }
        o.m = f.length;
        o.n = n;
        o.steps = {(int)(laid * 2 / kKBytes), plan.dx_pairs, (int)std::min(plan.steps_of(count), (int64_t)plan.features_parts)};
        o.out = plan.features_direct ? static_cast<char*>(out.features) + row * f.length * size : work + plan.features + plan.features_parts * row * f.length * 4;
        o.type = plan.features_direct ? f.type : kRawSums;
        o.pitch = f.length;
        o.add = first > 0;
        o.finish.dead = t.expo;
        short_sums(f.type, o) ? product_short(f.type, o, stream) : product_out(f.type, o, stream);
      }
      if (out.weight) {
        OutTask o{};
        if (of_float) {
          o.fa = float_operand(of_rows, true, t.expo);
          o.fb = float_operand(dx, true);
          o.fk = n;
        } else {
          o.a = {work + plan.f_turned + row * 2, all_turned * 2, 0};
          o.b = {t.by_cat, turned * 2, t.plane_cat * 2};
          if (of_half) o.finish.most = most;
        }
        o.m = f.length;
        o.n = count;
        o.steps = {(int)(turned * 2 / kKBytes), plan.dx_pairs, (int)std::min(plan.steps_of(n), (int64_t)plan.weight_parts)};
        o.pitch = f.length;
        char* const to = static_cast<char*>(out.weight) + first * f.length * size;
        o.out = plan.weight_direct ? to : work + plan.weight;
        o.type = plan.weight_direct ? f.type : kRawSums;
        o.add = row > 0;
        short_sums(f.type, o) ? product_short(f.type, o, stream) : product_out(f.type, o, stream);
        // (a last part of fewer steps than parts of the sum leaves some of them as the rows before it did; so does a last piece below)
        if (!plan.weight_direct && row + n == rows) join_parts(o.out, plan.weight_parts, false, o.m, o.n, o.finish, to, f.type, f.length, stream);
      }
    }
    if (out.bias)
      hipLaunchKernelGGL(join_bias_kernel, dim3((unsigned)((count + 31) / 32)), dim3(256), 0, stream, reinterpret_cast<float*>(work + plan.bias), bias_tiles,
                         count, out.bias, bias.type, first);
  }
  if (out.features && !plan.features_direct)
    for (int64_t row = 0; row < rows; row += plan.part) {
      Finish finish;
      finish.dead = expo + row;
      if (of_half) finish.expo = expo + row;
      join_parts(work + plan.features + plan.features_parts * row * f.length * 4, plan.features_parts, false, f.length, std::min(plan.part, rows - row), finish,
                 static_cast<char*>(out.features) + row * f.length * size, f.type, f.length, stream);
    }
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) fail(PCM_ERR_HIP, "launch of linear_scores_backward failed: %s", hipGetErrorString(e));
}

}  // namespace pcm
