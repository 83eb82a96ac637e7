// Checkpoints of rows in 8 bits, and the rows back from them.
#include "category_rows.hpp"

namespace pcm {

namespace {
// one wave per block of 64 entries
template <typename T>
__global__ __launch_bounds__(256) void checkpoint_kernel(RowsRef x, RowsShape shape, CkptRef ckpt) {
  const int lane = threadIdx.x & 63;
  const int64_t pitch = (shape.cats + 15) / 16 * 16, blocks = (shape.cats + kCkptBlock - 1) / kCkptBlock, all = shape.rows() * blocks;
  for (int64_t b = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); b < all; b += (int64_t)gridDim.x * 4) {
    const int64_t r = b / blocks, e = r / shape.vars, v = r % shape.vars;
    const int c = (int)(b % blocks) * kCkptBlock + lane;
    const T* row = static_cast<const T*>(x.p) + e * x.stride_ex + v * x.stride_var;
    const bool in = c < shape.cats;
    const float y = in ? to_float(row[c * x.stride_cat]) : -INFINITY;
    const bool off = y <= masked_from<T>();
    float hi = off ? -INFINITY : y, lo = off ? INFINITY : y;
    for (int o = 32; o > 0; o >>= 1) {
      hi = fmaxf(hi, __shfl_xor(hi, o));
      lo = fminf(lo, __shfl_xor(lo, o));
    }
    const BlockScale s = block_scale(hi, lo, __any(!(y < INFINITY)));
    if (c < pitch) ckpt.codes[r * pitch + c] = (uint8_t)block_code(s, y, off);
    if (lane == 0) ckpt.scales[b] = s.word;
  }
}

template <typename T>
__global__ __launch_bounds__(256) void restore_kernel(CkptRef ckpt, RowsShape shape, RowsRef out) {
  const int64_t pitch = (shape.cats + 15) / 16 * 16, blocks = (shape.cats + kCkptBlock - 1) / kCkptBlock, all = shape.rows() * shape.cats;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < all; i += (int64_t)gridDim.x * 256) {
    const int64_t r = i / shape.cats, c = i % shape.cats, e = r / shape.vars, v = r % shape.vars;
    const float y = block_entry(block_unit(ckpt.scales[r * blocks + c / kCkptBlock]), ckpt.codes[r * pitch + c]);
    static_cast<T*>(const_cast<void*>(out.p))[e * out.stride_ex + v * out.stride_var + c * out.stride_cat] =
        from_float<T>(y > type_max<T>() ? type_max<T>() : y);
  }
}
}  // namespace

void checkpoint_rows(const RowsRef& x, const RowsShape& shape, const CkptRef& ckpt, hipStream_t stream) {
  check_rows(x, shape, "checkpoint");
  if (!shape.examples) return;
  if (!x.p || !ckpt.codes || !ckpt.scales) fail(PCM_ERR_ARG, "checkpoint: a pointer is null");
  const dim3 grid((unsigned)std::min<int64_t>((shape.rows() * ckpt_blocks(shape.cats) + 3) / 4, 1 << 20));
  auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(256), 0, stream, x, shape, ckpt); };
  if (x.dtype == PCM_F32) launch(checkpoint_kernel<float>);
  else if (x.dtype == PCM_BF16) launch(checkpoint_kernel<bf16>);
  else launch(checkpoint_kernel<f16>);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) fail(PCM_ERR_HIP, "launch of checkpoint_rows failed: %s", hipGetErrorString(e));
}

void restore_rows(const CkptRef& ckpt, const RowsShape& shape, const RowsRef& out, hipStream_t stream) {
  check_rows(out, shape, "restored rows");
  if (!shape.examples) return;
  if (!out.p || !ckpt.codes || !ckpt.scales) fail(PCM_ERR_ARG, "restored rows: a pointer is null");
  const dim3 grid((unsigned)std::min<int64_t>((shape.rows() * shape.cats + 255) / 256, 1 << 20));
  auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(256), 0, stream, ckpt, shape, out); };
  if (out.dtype == PCM_F32) launch(restore_kernel<float>);
  else if (out.dtype == PCM_BF16) launch(restore_kernel<bf16>);
  else launch(restore_kernel<f16>);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) fail(PCM_ERR_HIP, "launch of restore_rows failed: %s", hipGetErrorString(e));
}

}  // namespace pcm
