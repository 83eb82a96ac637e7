// Gradient of log-probabilities, entropy and likeliest categories with respect to the rows of scores.
#include "category_rows.hpp"

namespace pcm {

namespace {
struct GradIn {
  GivenRef given;
  const float* grad_logp;
  int top;
  const int32_t* top_index;
  const float *grad_top, *log_sum, *entropy, *grad_entropy;
};

// dx[c] = sum of the slots' gradients at c - p (G + gh (log p + H)), G the sum of all slots' gradients; one workgroup per row
template <typename T, bool kCkpt>
__global__ __launch_bounds__(256) void grad_rows_kernel(RowsRef x, CkptRef ckpt, RowsShape shape, GradIn in, RowsRef out) {
  __shared__ int64_t at[2 * kMaxSlots];
  __shared__ float by[2 * kMaxSlots];
  const int64_t rows = shape.rows();
  const int slots = in.given.slots + in.top;
  const int64_t pitch = (shape.cats + 15) / 16 * 16, blocks = (shape.cats + kCkptBlock - 1) / kCkptBlock;
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const int64_t e = r / shape.vars, v = r % shape.vars;
    const T* row = static_cast<const T*>(x.p) + e * x.stride_ex + v * x.stride_var;
    T* dst = static_cast<T*>(const_cast<void*>(out.p)) + e * out.stride_ex + v * out.stride_var;
    __syncthreads();
    if (threadIdx.x < slots) {
      const int j = threadIdx.x;
      const bool g = j < in.given.slots;
      at[j] = g ? given_at(in.given, e, v, j) : in.top_index[r * in.top + j - in.given.slots];
      by[j] = g ? in.grad_logp[r * in.given.slots + j] : in.grad_top[r * in.top + j - in.given.slots];
    }
    __syncthreads();
    const float z = in.log_sum[r], gh = in.grad_entropy ? in.grad_entropy[r] : 0.f, h = in.grad_entropy ? in.entropy[r] : 0.f;
    float total = 0.f;
    for (int j = 0; j < slots; ++j)
      if (at[j] >= 0) total += at[j] < shape.cats ? by[j] : NAN;
    for (int c = threadIdx.x; c < shape.cats; c += 256) {
      const float y = kCkpt ? block_entry(block_unit(ckpt.scales[r * blocks + c / kCkptBlock]), ckpt.codes[r * pitch + c])
                            : seen(row[c * x.stride_cat]);
      const float d = y - z, p = expf(d);
      float g = -p * total;
      if (p != 0.f) g -= gh * p * (d + h);
      for (int j = 0; j < slots; ++j)
        if (at[j] == c) g += by[j];
      if (z == -INFINITY) g = 0.f;
      dst[c * out.stride_cat] = from_float<T>(g);
    }
  }
}
}  // namespace

void category_scores_backward(const RowsRef& x, const CkptRef& ckpt, const RowsShape& shape, const GivenRef& given,
                              const float* d_grad_logp, int top, const int32_t* d_top, const float* d_grad_top,
                              const float* d_log_sum, const float* d_entropy, const float* d_grad_entropy, const RowsRef& out,
                              hipStream_t stream) {
  check_rows(out, shape, "gradient of scores");
  check_given(given);
  if (top < 0 || top > kMaxSlots) fail(PCM_ERR_UNSUPPORTED, "0 to %d likeliest categories, got %d", kMaxSlots, top);
  if (!ckpt.codes != !ckpt.scales) fail(PCM_ERR_ARG, "a checkpoint needs both its codes and its scales");
  if (!ckpt.codes == !x.p && shape.examples) fail(PCM_ERR_ARG, "gradient of scores: either the scores or their checkpoint");
  if (x.p && x.dtype != out.dtype) fail(PCM_ERR_ARG, "gradient of scores: type %d for scores of type %d", out.dtype, x.dtype);
  if (!shape.examples) return;
  if (!out.p || !d_log_sum || (given.slots && !d_grad_logp) || (top && (!d_top || !d_grad_top)) || (d_grad_entropy && !d_entropy))
    fail(PCM_ERR_ARG, "gradient of scores: a pointer is null");
  const GradIn in{given, d_grad_logp, top, d_top, d_grad_top, d_log_sum, d_entropy, d_grad_entropy};
  const dim3 grid((unsigned)std::min<int64_t>(shape.rows(), 1 << 20));
  auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(256), 0, stream, x, ckpt, shape, in, out); };
  const bool k = ckpt.codes != nullptr;
  if (out.dtype == PCM_F32) k ? launch(grad_rows_kernel<float, true>) : launch(grad_rows_kernel<float, false>);
  else if (out.dtype == PCM_BF16) k ? launch(grad_rows_kernel<bf16, true>) : launch(grad_rows_kernel<bf16, false>);
  else k ? launch(grad_rows_kernel<f16, true>) : launch(grad_rows_kernel<f16, false>);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) fail(PCM_ERR_HIP, "launch of category_scores_backward failed: %s", hipGetErrorString(e));
}

}  // namespace pcm
