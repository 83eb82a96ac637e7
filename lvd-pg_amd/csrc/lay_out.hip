// Rows of 16-bit types laid out for the products: in rows of multiples of 128 bytes, as they lie or turned.
//
// Bound by the bytes moved: 64 x 64 tiles by way of LDS, read along whichever axis has neighbours.
#include <algorithm>

#include "linear_scores.hpp"

namespace pcm {

namespace {
constexpr int kTile = 64;

template <typename T>
__device__ __forceinline__ T scaled(T v, int by) { return by == 0 ? v : (T)ldexpf((float)v, by); }

template <typename T>
__global__ __launch_bounds__(256) void lay_out_kernel(Matrix2 x, int64_t first, int64_t count, bool turned, bool along_rows, LayOut with, uint16_t* to,
                                                      int64_t pitch) {
  __shared__ T tile[kTile][kTile + 1];                  // [row][entry]
  __shared__ int by[kTile];                             // of a row: power of two, or kDeadRow
  const int64_t r0 = (int64_t)blockIdx.x * kTile;
  const int c0 = blockIdx.y * kTile;
  const int t = threadIdx.x;
  const int largest = with.expo ? largest_exponent(with.most) : 0;
  if (t < kTile) {
    int e = 0;
    if (r0 + t < count) {
      if (with.expo) {
        e = with.expo[first + r0 + t];
        if (e != kDeadRow) e = max(e - largest, -300);
      }
      if (with.mask.p && bias_at(with.mask, first + r0 + t, x.examples) == -INFINITY) e = kDeadRow;
    }
    by[t] = e;
  }
  const T* const from = static_cast<const T*>(x.p);
#pragma unroll
  for (int i = 0; i < kTile * kTile / 256; ++i) {
    const int at = i * 256 + t, r = along_rows ? at % kTile : at / kTile, c = along_rows ? at / kTile : at % kTile;
    T v = (T)0.f;
    if (r0 + r < count && c0 + c < x.length) {
      const int64_t row = first + r0 + r;
      v = from[row / x.vars * x.stride_ex + row % x.vars * x.stride_var + (int64_t)(c0 + c) * x.stride];
    }
    tile[r][c] = v;
  }
  __syncthreads();
  // groups of four neighbours of the result, sixteen to a row of the tile
  const int64_t rows = turned ? x.length : count;
#pragma unroll
  for (int i = 0; i < kTile * kTile / 1024; ++i) {
    const int at = i * 256 + t, out = at / 16, k = at % 16 * 4;
    const int64_t row = (turned ? c0 : r0) + out, entry = (turned ? r0 : c0) + k;
    if (row >= rows || entry >= pitch) continue;
    uint16_t h[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      T v = turned ? tile[k + j][out] : tile[out][k + j];
      const int e = by[turned ? k + j : out];
      v = e == kDeadRow ? (T)0.f : scaled(v, e);
      h[j] = __builtin_bit_cast(uint16_t, v);
    }
    uint16_t* const p = to + row * pitch + entry;
    *reinterpret_cast<uint2*>(p) = make_uint2(h[0] | (uint32_t)h[1] << 16, h[2] | (uint32_t)h[3] << 16);
  }
}
}  // namespace

// (float is read whatever its strides)
bool readable(const Matrix2& x) {
  if (x.type == PCM_F32) return true;
  const bool one_axis = x.vars == 1 || x.stride_ex == x.vars * x.stride_var;
  const int64_t pitch = x.vars == 1 ? x.stride_ex : x.stride_var;
  return x.length % (kKBytes / 2) == 0 && (x.stride == 1) && ((uintptr_t)x.p & 15) == 0 &&
         (x.rows() <= 1 || (one_axis && pitch % 8 == 0 && pitch > 0 && pitch <= kMaxLength * 4));
}

void lay_out(const Matrix2& x, int64_t first, int64_t count, bool turned, const LayOut& with, void* d_to, hipStream_t stream) {
  const int64_t pitch = laid_length(turned ? count : x.length);
  const dim3 grid((unsigned)((count + kTile - 1) / kTile), (unsigned)((x.length + kTile - 1) / kTile));
  const bool along_rows = x.vars == 1 && x.stride != 1 && (x.stride_ex == 1 || x.stride_ex == -1);
  uint16_t* const to = static_cast<uint16_t*>(d_to);
  if (x.type == PCM_BF16) hipLaunchKernelGGL((lay_out_kernel<bf16>), grid, dim3(256), 0, stream, x, first, count, turned, along_rows, with, to, pitch);
  else hipLaunchKernelGGL((lay_out_kernel<f16>), grid, dim3(256), 0, stream, x, first, count, turned, along_rows, with, to, pitch);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) fail(PCM_ERR_HIP, "launch of lay_out failed: %s", hipGetErrorString(e));
}

}  // namespace pcm
