// Log-sums and log-probabilities of categories whose scores are products of features and weights, without keeping the scores.
//
//   x[n][c] = f[n] . w[c] + b[c],  Z[n] = log sum_c exp x[n][c],  logp[n][j] = x[n][g_j] - Z[n]
// Categories are the rows of a, so that a lane's sums are of one row of features: it takes their maximum and the sum of
// exponentials in registers, the tile's waves join theirs in LDS, and a pair of numbers per row and tile of categories is all that
// is written; a second launch joins those.  The score of a given category is written by the lane that has it.
//
// Bound by the matrix cores (4096 x 50304 of length 4096 bf16: 1.37 ms, 1.23 PFLOP/s at the clock that the card's power leaves; 2048 x 131072 in 8
// bits: 0.95 ms, 2.3 POP/s), few rows by reading the weights (1 x 131072 of length 4096 bf16: 193 us, 5.6 TB/s).  Kept scores would
// be 824 MB in the first, written once and read once.
#include "few_rows.hip.hpp"

namespace pcm {

namespace {
struct Part {            // of a row's sum: sum exp(x - base)
  float base, sum;
};
__device__ __forceinline__ Part join(Part a, Part b) {
  const float base = fmaxf(a.base, b.base), to = base == -INFINITY ? 0.f : base;
  // a part of nothing has base -inf and sum 0; NaN and +inf come through as NaN
  return {base, a.sum * expf(a.base - to) + b.sum * expf(b.base - to)};
}

struct ScoreTask : ScoreInputs {
  float* logp;           // [rows][slots]: the given categories' scores, for the joining launch
  Part* parts;           // [tile of categories][row]
};

template <typename T, typename S>
__device__ __forceinline__ void score_tile(const ScoreTask& t) {
  __shared__ __attribute__((aligned(16))) float bias[S::BM], scale[S::BM];
  tile_constants<S>(t, bias, scale);
  score_sums<T, S>(t, [&](auto& sums, int64_t m, int64_t n, char* lds) {
    const int lane = threadIdx.x & 63, half = lane >> 5, wave = threadIdx.x / 64, wm = wave % S::waves_m * S::WM;
    Part* const joined = reinterpret_cast<Part*>(lds);                      // [waves_m][BN]
    static_assert(S::waves_m * S::BN * sizeof(Part) <= S::stage);
    __syncthreads();
#pragma unroll
    for (int j = 0; j < S::FN; ++j) {
      __builtin_amdgcn_sched_barrier(0);   // one j at a time: registers are full
      const int64_t row = n + 32 * j + (lane & 31);
      const bool valid = row < t.rows;
      float x[S::FM][16];
      scores_of<S>(sums, j, t.scale.n ? t.scale.n[valid ? row : t.rows - 1] : 1.f, bias + wm, scale + wm, half, x);
      float largest = -INFINITY;
#pragma unroll
      for (int i = 0; i < S::FM; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) largest = fmaxf(largest, x[i][r]);
      const float base = largest == -INFINITY ? 0.f : largest;
      float sum = 0.f;
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < S::FM; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) sum += __builtin_amdgcn_exp2f((x[i][r] - base) * kLog2e);
      // (NaN beside no other category: the sum has it, with base 0)
      Part p{sum == 0.f ? largest : base, sum};
      p = join(p, {__shfl_xor(p.base, 32), __shfl_xor(p.sum, 32)});
      if (half == 0) joined[wave % S::waves_m * S::BN + (int)(n % S::BN) + 32 * j + lane] = p;
      if (valid && t.given.slots) {
        const int64_t e = row / t.given.vars, v = row % t.given.vars;
        for (int s = 0; s < t.given.slots; ++s) {
          const int64_t g = given_at(t.given, e, v, s) - m;
          if (g < 0 || g >= S::WM || (g >> 2 & 1) != half) continue;
          float found = 0.f;
#pragma unroll
          for (int i = 0; i < S::FM; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r)
              found = (int)g == 32 * i + 8 * (r / 4) + 4 * half + r % 4 ? x[i][r] : found;
          t.logp[row * t.given.slots + s] = found;
        }
      }
    }
    __syncthreads();
    const int64_t n0 = n / S::BN * S::BN, tile = m / S::BM;
    for (int i = threadIdx.x; i < S::BN; i += S::threads) {
      Part p = joined[i];
#pragma unroll
      for (int w = 1; w < S::waves_m; ++w) p = join(p, joined[w * S::BN + i]);
      if (n0 + i < t.rows) t.parts[tile * t.rows + n0 + i] = p;
    }
  });
}
template <typename T, typename S>
__global__ __launch_bounds__(S::threads, 2) void score_kernel(ScoreTask t) {
  score_tile<T, S>(t);
}

// Few rows: a thread has some of the tile's categories, of one row.  Three workgroups of four waves a compute unit, or two of eight (LDS has
// room for no more with 17 rows and more; 48 x 1001 x 50021 f16: 50 us, 57 with the registers of two; the gradient's kernel would not keep its sums in so few)
template <typename T, int kGroups>
__global__ __launch_bounds__(FewTile<kGroups>::threads, kGroups == 4 ? 3 : 4) void score_few_kernel(ScoreTask t, FewOperand w, FewOperand f, int length) {
  typedef FewTile<kGroups> S;
  __shared__ __attribute__((aligned(16))) char lds[S::lds];
  __shared__ Part joined[S::threads];
  const float* const sums = few_sums<T, kGroups>(w, f, t.cats, t.rows, length, 1, lds);
  constexpr int kLanes = S::threads / S::rows, kOwn = S::longs / kLanes;   // lanes to a row, and categories of each
  const int in = threadIdx.x % S::rows, lane = threadIdx.x / S::rows;
  const int64_t c0 = (int64_t)blockIdx.x * S::longs, n = (int64_t)blockIdx.z * S::rows + in;
  const float sn = t.scale.n && n < t.rows ? t.scale.n[n] : 1.f;
  float x[kOwn], base = -INFINITY, sum = 0.f;
#pragma unroll
  for (int i = 0; i < kOwn; ++i) {
    const int at = lane + i * kLanes;
    const int64_t c = c0 + at;
    float v = sums[at * S::pitch + in];
    if constexpr (sizeof(T) == 1) v = (float)__builtin_bit_cast(int, v) * sn * (c < t.cats ? t.scale.m[c] : 1.f);
    x[i] = score_of(v, bias_at(t.bias, c, t.cats));
    base = fmaxf(base, x[i]);
  }
  const float to = base == -INFINITY ? 0.f : base;
#pragma unroll
  for (int i = 0; i < kOwn; ++i) sum += __builtin_amdgcn_exp2f((x[i] - to) * kLog2e);
  joined[threadIdx.x] = {sum == 0.f ? base : to, sum};
  if (n < t.rows)
    for (int s = 0; s < t.given.slots; ++s) {
      const int64_t g = given_at(t.given, n / t.given.vars, n % t.given.vars, s) - t.first_cat - c0;
#pragma unroll
      for (int i = 0; i < kOwn; ++i)
        if (g == lane + i * kLanes) t.logp[n * t.given.slots + s] = x[i];
    }
  __syncthreads();
#pragma unroll
  for (int s = kLanes / 2; s; s /= 2) {
    if (lane < s) joined[threadIdx.x] = join(joined[threadIdx.x], joined[threadIdx.x + s * S::rows]);
    __syncthreads();
  }
  if (lane == 0 && n < t.rows) t.parts[blockIdx.x * t.rows + n] = joined[in];
}

// Joins the tiles' parts: `per` rows a workgroup, 256 / per lanes to each
__global__ __launch_bounds__(256) void join_scores_kernel(const Part* parts, int64_t tiles, int64_t rows, int per, GivenRef given, int64_t cats,
                                                          float* logp, float* log_sum) {
  __shared__ Part sub[256];
  const int in = threadIdx.x % per, lane = threadIdx.x / per, lanes = 256 / per;
  const int64_t n = (int64_t)blockIdx.x * per + in;
  Part p{-INFINITY, 0.f};
  if (n < rows) {
    float base = -INFINITY;
    for (int64_t i = lane; i < tiles; i += lanes) base = fmaxf(base, parts[i * rows + n].base);
    const float to = base == -INFINITY ? 0.f : base;
    float sum = 0.f;
    for (int64_t i = lane; i < tiles; i += lanes) {
      const Part q = parts[i * rows + n];
      sum += q.sum * expf(q.base - to);
    }
    p = {base, sum};
  }
  sub[threadIdx.x] = p;
  __syncthreads();
  for (int s = lanes / 2; s; s /= 2) {
    if (lane < s) sub[threadIdx.x] = join(sub[threadIdx.x], sub[threadIdx.x + s * per]);
    __syncthreads();
  }
  if (n >= rows) return;
  p = sub[in];
  const float z = p.base + logf(p.sum);            // no category: -inf + -inf
  if (lane == 0 && log_sum) log_sum[n] = z;
  for (int s = lane; s < given.slots; s += lanes) {
    const int64_t g = given_at(given, n / given.vars, n % given.vars, s);
    float& to = logp[n * given.slots + s];
    to = g < 0 ? 0.f : g >= cats ? __builtin_nanf("") : z == -INFINITY ? z : to - z;
  }
}

typedef TileSizes<256, 256, 128, 64> Wide;
typedef TileSizes<128, 128, 64, 64> Middle;
typedef TileSizes<128, 64, 64, 32> Slim;
typedef TileSizes<128, 32, 32, 32> Narrow;
enum { kWide, kMiddle, kSlim, kNarrow };

int tiles_for(int64_t m, int64_t n, int64_t steps, bool of_float) {
  if (of_float) return kMiddle;
  if (n <= 64) return n <= 32 ? kNarrow : kSlim;
  return wide_tiles(m, n, steps) ? kWide : kMiddle;
}
template <typename T, typename S>
void launch(const ScoreTask& t, hipStream_t stream) {
  const int64_t tiles_m = (t.cats + S::BM - 1) / S::BM, tiles_n = (t.rows + S::BN - 1) / S::BN, most = units_a_launch(tiles_m, S::threads);
  ScoreTask of_launch = t;
  for (int64_t first = 0; first < tiles_n; first += most) {
    of_launch.first_row = first * S::BN;
    hipLaunchKernelGGL((score_kernel<T, S>), dim3((unsigned)(tiles_m * std::min(most, tiles_n - first))), dim3(S::threads), 0, stream, of_launch);
  }
}
template <typename T>
void launch(const ScoreTask& t, hipStream_t stream) {
  const int size = tiles_for(t.cats, t.rows, t.steps.count, false);
  if (size == kWide) launch<T, Wide>(t, stream);
  else if (size == kMiddle) launch<T, Middle>(t, stream);
  else if (size == kSlim) launch<T, Slim>(t, stream);
  else launch<T, Narrow>(t, stream);
}
template <typename T>
void launch_few(const ScoreTask& t, const FewOperand& w, const FewOperand& f, int length, hipStream_t stream) {
  const int64_t tiles = (t.cats + kFewTile - 1) / kFewTile;
  const int threads = t.rows > 32 ? 256 : 512;
  const int64_t most = units_a_launch(1, threads);
  ScoreTask of_launch = t;
  FewOperand of_w = w;
  for (int64_t first = 0; first < tiles; first += most) {
    const int64_t cat = first * kFewTile;
    of_launch.first_cat = cat;
    of_launch.cats = std::min(most * kFewTile, t.cats - cat);
    of_w.p = static_cast<const char*>(w.p) + cat * w.stride_ex * (int64_t)sizeof(T);
    if (t.bias.p) of_launch.bias.p = static_cast<const char*>(t.bias.p) + cat * (t.bias.type == PCM_F32 ? 4 : 2);
    if (t.scale.m) of_launch.scale.m = t.scale.m + cat;
    of_launch.parts = t.parts + first * t.rows;
    const dim3 grid((unsigned)std::min(most, tiles - first), 1, (unsigned)((t.rows + kFewRowsMost - 1) / kFewRowsMost)), block(threads);
    if (t.rows <= 16) hipLaunchKernelGGL((score_few_kernel<T, 1>), grid, block, 0, stream, of_launch, of_w, f, length);
    else if (t.rows <= 32) hipLaunchKernelGGL((score_few_kernel<T, 2>), grid, block, 0, stream, of_launch, of_w, f, length);
    else hipLaunchKernelGGL((score_few_kernel<T, 4>), grid, block, 0, stream, of_launch, of_w, f, length);
  }
}
int64_t tiles_of_cats(int64_t cats, int64_t rows, int64_t steps, bool of_float, bool few) {
  const int64_t each = few ? kFewTile : tiles_for(cats, rows, steps, of_float) == kWide ? 256 : 128;
  return (cats + each - 1) / each;
}
int64_t parts_bytes(int64_t cats, int64_t rows, int64_t steps, bool of_float, bool few) {
  return round_up(tiles_of_cats(cats, rows, steps, of_float, few) * rows * (int64_t)sizeof(Part), 256);
}

void join_launch(const ScoreTask& t, bool few, float* d_log_sum, hipStream_t stream) {
  // few rows: all lanes of a workgroup to one, many: neighbouring rows side by side
  const int per = t.rows >= 4096 ? 16 : t.rows >= 512 ? 4 : 1;
  hipLaunchKernelGGL(join_scores_kernel, dim3((unsigned)((t.rows + per - 1) / per)), dim3(256), 0, stream, t.parts,
                     tiles_of_cats(t.cats, t.rows, t.steps.count, t.fw.p, few), t.rows, per, t.given, t.cats, t.logp, d_log_sum);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) fail(PCM_ERR_HIP, "launch of linear_scores failed: %s", hipGetErrorString(e));
}
}  // namespace

void check_linear(const Matrix2& f, const Matrix2& w, const BiasRef& bias, const GivenRef& given, const char* what) {
  if (f.type < PCM_F32 || f.type > PCM_F16 || w.type != f.type) fail(PCM_ERR_ARG, "%s: types %d and %d: both PCM_F32, PCM_BF16 or PCM_F16", what, f.type, w.type);
  if (bias.type < PCM_F32 || bias.type > PCM_F16) fail(PCM_ERR_ARG, "%s: type %d of the bias", what, bias.type);
  if (f.examples < 0 || f.vars < 1 || f.length < 1 || w.examples < 1)
    fail(PCM_ERR_SHAPE, "%s: %lld examples, %d variables, %lld categories of length %d", what, (long long)f.examples, f.vars, (long long)w.examples, f.length);
  if (f.examples > kMaxLinearRows || f.rows() > kMaxLinearRows || f.length > kMaxLength || w.examples > 1 << 30)
    fail(PCM_ERR_UNSUPPORTED, "%s: more than 2^22 rows, 2^30 categories or entries of length 2^20", what);
  check_given(given);
}

namespace {
bool few_tiles(int64_t rows, int64_t cats, int64_t length) {
  return rows <= 512 && length >= 512 && ((rows + 127) / 128) * ((cats + 127) / 128) <= 32;
}
}  // namespace
bool takes_few(const Matrix2& f, const Matrix2& w) {
  if (f.stride != 1 || w.stride != 1) return false;
  return (f.rows() <= kFewRowsMost && (f.type == PCM_F32 || !readable(f) || !readable(w) || w.examples < many_cats(f.rows(), 2 * f.length))) ||
         few_tiles(f.rows(), w.examples, f.length);
}
bool takes_few8(int64_t rows, int64_t cats, int64_t length) {
  return (rows <= kFewRowsMost && cats < many_cats(rows, length)) || few_tiles(rows, cats, length);
}
FewOperand few_operand(const Matrix2& x) { return {x.p, x.stride_ex, x.stride_var, x.vars}; }

int64_t linear_scores_workspace(const Matrix2& f, const Matrix2& w) {
  if (takes_few(f, w)) return parts_bytes(w.examples, f.rows(), 0, false, true);
  return (readable(f) ? 0 : laid_bytes(f.rows(), f.length, 1)) + (readable(w) ? 0 : laid_bytes(w.rows(), w.length, 1)) +
         parts_bytes(w.examples, f.rows(), laid_length(f.length) * 2 / kKBytes, f.type == PCM_F32, false);
}

void check_workspace(const void* d_work, int64_t work_bytes, int64_t need, const char* what) {
  if (need && (!d_work || work_bytes < need)) fail(PCM_ERR_ARG, "%s: workspace of %lld bytes, %lld needed", what, (long long)work_bytes, (long long)need);
  if ((uintptr_t)d_work & 15) fail(PCM_ERR_ARG, "%s: the workspace must be 16-byte aligned", what);
}

FloatOperand float_operand(const Matrix2& x, bool turned, const int* skip) {
  FloatOperand o{static_cast<const float*>(x.p), x.stride_ex, x.stride_var, x.stride, x.vars, turned, skip};
  if (x.vars > 1 && (x.examples == 1 || x.stride_ex == x.vars * x.stride_var)) {   // one axis of rows
    o.stride_ex = x.stride_var;
    o.vars = 1;
  }
  if (o.vars == 1 && o.stride != 1 && o.stride_ex == 1 && !skip) {                 // neighbours along the other axis
    std::swap(o.stride, o.stride_ex);
    o.turned = !turned;
  }
  return o;
}

// a matrix of 16-bit entries as a product reads it: where it is, or laid out at `work`, which then moves on
Operand operand_of(const Matrix2& x, char*& work, hipStream_t stream) {
  if (readable(x)) return {x.p, (x.vars == 1 ? x.stride_ex : x.stride_var) * 2, 0};
  lay_out(x, 0, x.rows(), false, LayOut(), work, stream);
  const Operand o{work, laid_length(x.length) * 2, 0};
  work += laid_bytes(x.rows(), x.length, 1);
  return o;
}

void linear_scores(const Matrix2& f, const Matrix2& w, const BiasRef& bias, const GivenRef& given, float* d_logp, float* d_log_sum, void* d_work,
                   int64_t work_bytes, hipStream_t stream) {
  check_linear(f, w, bias, given, "linear scores");
  if (!f.rows()) return;
  if (!f.p || !w.p || (given.slots && (!given.p || !d_logp))) fail(PCM_ERR_ARG, "linear scores: a pointer is null");
  check_workspace(d_work, work_bytes, linear_scores_workspace(f, w), "linear scores");
  ScoreTask t{};
  char* work = static_cast<char*>(d_work);
  const bool few = takes_few(f, w);
  if (!few && f.type == PCM_F32) {
    t.ff = float_operand(f, false);
    t.fw = float_operand(w, false);
    t.fk = f.length;
  } else if (!few) {
    t.f = operand_of(f, work, stream);
    t.w = operand_of(w, work, stream);
  }
  t.cats = w.examples;
  t.rows = f.rows();
  t.steps = {(int)(laid_length(f.length) * 2 / kKBytes), kOnePlane, 1};
  t.bias = bias;
  t.given = given;
  t.given.vars = f.vars;
  t.logp = d_logp;
  t.parts = reinterpret_cast<Part*>(work);
  if (few) {
    const FewOperand fw = few_operand(w), ff = few_operand(f);
    if (f.type == PCM_F32) launch_few<float>(t, fw, ff, f.length, stream);
    else if (f.type == PCM_F16) launch_few<f16>(t, fw, ff, f.length, stream);
    else launch_few<bf16>(t, fw, ff, f.length, stream);
  } else if (f.type == PCM_F32) {
    launch<float, FloatTile>(t, stream);
  } else if (f.type == PCM_F16) {
    launch<f16>(t, stream);
  } else {
    launch<bf16>(t, stream);
  }
  join_launch(t, few, d_log_sum, stream);
}

int64_t linear_scores8_workspace(int64_t rows, int64_t cats, int32_t length) {
  return rows < 1 || cats < 1 ? 0 : parts_bytes(cats, rows, round_up(length, kKBytes) / kKBytes, false, takes_few8(rows, cats, length));
}

void linear_scores8(const int8_t* f, const float* f_scales, int64_t examples, int32_t vars, const int8_t* w, const float* w_scales, int32_t cats,
                    int32_t length, const BiasRef& bias, const GivenRef& given, float* d_logp, float* d_log_sum, void* d_work, int64_t work_bytes,
                    hipStream_t stream) {
  Matrix2 shape{f, PCM_F32, 0, 0, 1, examples, vars, length}, weight{w, PCM_F32, 0, 0, 1, cats, 1, length};
  check_linear(shape, weight, bias, given, "linear scores of 8-bit rows");
  if (length > kMaxLength8) fail(PCM_ERR_UNSUPPORTED, "8-bit rows of length %d: a sum of more than 131071 products may pass 32 bits", length);
  if (!shape.rows()) return;
  if (!f || !f_scales || !w || !w_scales || (given.slots && (!given.p || !d_logp))) fail(PCM_ERR_ARG, "linear scores of 8-bit rows: a pointer is null");
  if (((uintptr_t)f | (uintptr_t)w) & 15) fail(PCM_ERR_ARG, "linear scores of 8-bit rows: codes must be 16-byte aligned");
  check_workspace(d_work, work_bytes, linear_scores8_workspace(shape.rows(), cats, length), "linear scores of 8-bit rows");
  ScoreTask t{};
  const int64_t pitch = round_up(length, kKBytes);
  t.f = {f, pitch, 0};
  t.w = {w, pitch, 0};
  t.cats = cats;
  t.rows = shape.rows();
  t.steps = {(int)(pitch / kKBytes), kOnePlane, 1};
  t.bias = bias;
  t.scale = {f_scales, w_scales};
  t.given = given;
  t.given.vars = vars;
  t.logp = d_logp;
  t.parts = static_cast<Part*>(d_work);
  const bool few = takes_few8(t.rows, cats, length);
  if (few) launch_few<int8_t>(t, FewOperand{w, pitch, 0, 1}, FewOperand{f, pitch, 0, 1}, (int)pitch, stream);
  else launch<int8_t>(t, stream);
  join_launch(t, few, d_log_sum, stream);
}

}  // namespace pcm
