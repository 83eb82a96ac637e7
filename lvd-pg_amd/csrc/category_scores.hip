// Log-probabilities of given categories, entropy and likeliest categories of rows of scores.
#include "category_rows.hpp"

namespace pcm {

void check_rows(const RowsRef& x, const RowsShape& shape, const char* what) {
  if (shape.examples < 0 || shape.vars < 1 || shape.cats < 1)
    fail(PCM_ERR_SHAPE, "%s: %lld examples, %d variables, %d categories", what, (long long)shape.examples, shape.vars, shape.cats);
  if (shape.examples > INT64_C(0x7fffffff) / shape.vars) fail(PCM_ERR_UNSUPPORTED, "%s: at most 2^31 - 1 rows", what);
  if (x.dtype != PCM_F32 && x.dtype != PCM_BF16 && x.dtype != PCM_F16) fail(PCM_ERR_ARG, "%s: type %d is none of PCM_F32, PCM_BF16, PCM_F16", what, x.dtype);
}

void check_given(const GivenRef& g) {
  if (g.slots < 0 || g.slots > kMaxSlots) fail(PCM_ERR_UNSUPPORTED, "0 to %d given categories per row, got %d", kMaxSlots, g.slots);
  if (g.slots && !g.p) fail(PCM_ERR_ARG, "given categories: the pointer is null");
  if (g.slots && g.type != PCM_U8 && g.type != PCM_I32 && g.type != PCM_I64)
    fail(PCM_ERR_ARG, "given categories: type %d is none of PCM_U8, PCM_I32, PCM_I64", g.type);
}

namespace {
struct ScoreOut {
  float *logp, *log_sum, *entropy, *top_logp;
  int32_t* top;
};

__device__ __forceinline__ float block_max(float v, float* sh) {
  for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
  __syncthreads();
  return fmaxf(fmaxf(sh[0], sh[1]), fmaxf(sh[2], sh[3]));
}
__device__ __forceinline__ float block_sum(float v, float* sh) {
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
  __syncthreads();
  return (sh[0] + sh[1]) + (sh[2] + sh[3]);
}

// One workgroup per row, three kinds of passes over it: maximum, sums, and one search per likeliest category.
template <typename T>
__global__ __launch_bounds__(256) void score_rows_kernel(RowsRef x, RowsShape shape, GivenRef given, int top, ScoreOut out) {
  __shared__ float sh[4];
  __shared__ uint64_t best_sh[4];
  const int64_t rows = shape.rows();
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const int64_t e = r / shape.vars, v = r % shape.vars;
    const T* row = static_cast<const T*>(x.p) + e * x.stride_ex + v * x.stride_var;
    float m = -3.4028235e38f;
    for (int c = threadIdx.x; c < shape.cats; c += 256) m = fmaxf(m, seen(row[c * x.stride_cat]));
    m = block_max(m, sh);
    float s = 0.f, t = 0.f;
    for (int c = threadIdx.x; c < shape.cats; c += 256) {
      const float d = seen(row[c * x.stride_cat]) - m, p = expf(d);
      s += p;
      if (p > 0.f) t += p * d;
    }
    s = block_sum(s, sh);
    t = block_sum(t, sh);
    const float ls = logf(s), z = m + ls;   // (no category at all: s = 0, z = -inf)
    const bool nan = !(z < INFINITY), none = s == 0.f;
    if (threadIdx.x == 0) {
      if (out.log_sum) out.log_sum[r] = nan ? NAN : none ? -INFINITY : z;
      if (out.entropy) out.entropy[r] = nan ? NAN : none ? 0.f : ls - t / s;
      for (int j = 0; j < given.slots; ++j) {
        const int64_t g = given_at(given, e, v, j);
        float lp = NAN;
        if (g < 0) lp = 0.f;
        else if (g < shape.cats && !nan) lp = none ? -INFINITY : seen(row[g * x.stride_cat]) - m - ls;
        out.logp[r * given.slots + j] = lp;
      }
    }
    uint64_t last = ~0ull;
    for (int j = 0; j < top; ++j) {
      uint64_t best = 0;
      for (int c = threadIdx.x; c < shape.cats; c += 256) {
        const float y = seen(row[c * x.stride_cat]);
        const uint64_t k = y > -INFINITY ? entry_key(y, c) : 0;
        if (k < last && k > best) best = k;
      }
      for (int o = 32; o > 0; o >>= 1) {
        const uint64_t k = __shfl_xor((unsigned long long)best, o);
        best = k > best ? k : best;
      }
      __syncthreads();
      if ((threadIdx.x & 63) == 0) best_sh[threadIdx.x >> 6] = best;
      __syncthreads();
      for (int q = 0; q < 4; ++q) best = best_sh[q] > best ? best_sh[q] : best;
      if (threadIdx.x == 0) {
        out.top[r * top + j] = nan || !best ? -1 : key_index(best);
        out.top_logp[r * top + j] = nan ? NAN : !best ? -INFINITY : key_value(best) - m - ls;
      }
      last = best ? best : 1;
    }
  }
}
}  // namespace

int64_t category_scores_workspace(const RowsShape&, int) { return 0; }

void category_scores(const RowsRef& x, const RowsShape& shape, const GivenRef& given, int top, float* d_logp, float* d_log_sum,
                     float* d_entropy, float* d_top_logp, int32_t* d_top, const CkptRef& ckpt, void*, int64_t, hipStream_t stream) {
  check_rows(x, shape, "scores");
  check_given(given);
  if (top < 0 || top > kMaxSlots) fail(PCM_ERR_UNSUPPORTED, "0 to %d likeliest categories, got %d", kMaxSlots, top);
  if (!ckpt.codes != !ckpt.scales) fail(PCM_ERR_ARG, "a checkpoint needs both its codes and its scales");
  if (!shape.examples) return;
  if (!x.p || (given.slots && !d_logp) || (top && (!d_top || !d_top_logp))) fail(PCM_ERR_ARG, "scores: a pointer is null");
  const ScoreOut out{d_logp, d_log_sum, d_entropy, d_top_logp, d_top};
  const dim3 grid((unsigned)std::min<int64_t>(shape.rows(), 1 << 20));
  if (x.dtype == PCM_F32) hipLaunchKernelGGL((score_rows_kernel<float>), grid, dim3(256), 0, stream, x, shape, given, top, out);
  else if (x.dtype == PCM_BF16) hipLaunchKernelGGL((score_rows_kernel<bf16>), grid, dim3(256), 0, stream, x, shape, given, top, out);
  else hipLaunchKernelGGL((score_rows_kernel<f16>), grid, dim3(256), 0, stream, x, shape, given, top, out);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) fail(PCM_ERR_HIP, "launch of category_scores failed: %s", hipGetErrorString(e));
  if (ckpt.codes) checkpoint_rows(x, shape, ckpt, stream);
}

}  // namespace pcm
