// Rows of 16-bit types laid out for the products: in rows of multiples of 128 bytes, as they lie or turned.
//
// Bound by the bytes moved.  Rows of neighbours are copied 16 bytes a lane, or turned in tiles of 64 x 64: 4 x 4 entries in a lane's registers, the
// tile's rows put together in LDS (50000 x 4096 bf16: 170 us, 430 entry by entry); other strides go entry by entry.
#include "linear_plan.hpp"
#include "linear_scores.hpp"

namespace pcm {

namespace {
constexpr int kTile = 64;

template <typename T>
__device__ __forceinline__ T scaled(T v, int by) { return by == 0 ? v : (T)ldexpf((float)v, by); }

// what a row is multiplied by: a power of two, or kDeadRow
__device__ __forceinline__ int row_scale(const LayOut& with, const Matrix2& x, int64_t row, int largest) {
  if (with.mask.p && bias_at(with.mask, row, x.examples) == -INFINITY) return kDeadRow;
  if (!with.expo) return 0;
  const int e = with.expo[row];
  return e == kDeadRow ? e : with.most ? max(e - largest, -300) : 0;
}
template <typename T>
__device__ __forceinline__ uint32_t scaled_pair(uint32_t v, int by) {
  if (by == 0) return v;
  if (by == kDeadRow) return 0;
  const T a = __builtin_bit_cast(T, (uint16_t)(v & 0xffffu)), b = __builtin_bit_cast(T, (uint16_t)(v >> 16));
  return pair_of<T>(ldexpf((float)a, by), ldexpf((float)b, by));
}

// rows of neighbours, as they lie: eight entries a lane
template <typename T>
__global__ __launch_bounds__(256) void copy_rows_kernel(Matrix2 x, int64_t first, int64_t count, uint16_t* to, int64_t pitch) {
  const int c = (blockIdx.y * 8 + threadIdx.x % 8) * 8;
  if (c >= pitch) return;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int64_t r = (int64_t)blockIdx.x * 64 + i * 32 + threadIdx.x / 8;
    if (r >= count) return;
    const int64_t row = first + r;
    const T* const from = static_cast<const T*>(x.p) + row / x.vars * x.stride_ex + row % x.vars * x.stride_var + c;
    raw4 v = {0, 0, 0, 0};
    if (c + 8 <= x.length) {
      v = load16(from);
    } else {
      T e[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) e[k] = c + k < x.length ? from[k] : (T)0.f;
      v = __builtin_bit_cast(raw4, e);
    }
    *reinterpret_cast<raw4*>(to + r * pitch + c) = v;
  }
}

// ... turned
template <typename T>
__global__ __launch_bounds__(256) void turn_rows_kernel(Matrix2 x, int64_t first, int64_t count, LayOut with, uint16_t* to, int64_t pitch) {
  typedef uint32_t two __attribute__((ext_vector_type(2)));
  typedef two two_by2 __attribute__((aligned(2)));
  constexpr int kPitch = 136;                           // bytes: rows of LDS 34 banks apart
  __shared__ __attribute__((aligned(8))) char tile[kTile * kPitch];   // [entry][row]
  const int64_t r0 = (int64_t)blockIdx.x * kTile;
  const int c0 = blockIdx.y * kTile, block = threadIdx.x / 16 * 4, c = c0 + threadIdx.x % 16 * 4;
  const int largest = with.most ? largest_exponent(with.most) : 0;
  uint32_t a[4], b[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t r = r0 + block + i, row = first + min(r, count - 1);
    const T* const from = static_cast<const T*>(x.p) + row / x.vars * x.stride_ex + row % x.vars * x.stride_var + c;
    two v = {0, 0};
    if (c + 4 <= x.length) {
      v = *reinterpret_cast<const two_by2*>(from);
    } else {
      T e[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) e[k] = c + k < x.length ? from[k] : (T)0.f;
      v = __builtin_bit_cast(two, e);
    }
    const int by = r < count ? row_scale(with, x, row, largest) : kDeadRow;
    a[i] = scaled_pair<T>(v[0], by);
    b[i] = scaled_pair<T>(v[1], by);
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const uint32_t* const v = e < 2 ? a : b;
    const uint32_t order = e & 1 ? 0x07060302u : 0x05040100u;
    *reinterpret_cast<uint2*>(tile + (c - c0 + e) * kPitch + block * 2) =
        make_uint2(__builtin_amdgcn_perm(v[1], v[0], order), __builtin_amdgcn_perm(v[3], v[2], order));
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int at = i * 32 + threadIdx.x / 8, k = threadIdx.x % 8;
    if (c0 + at >= x.length) return;
    const uint2 lo = *reinterpret_cast<const uint2*>(tile + at * kPitch + k * 16), hi = *reinterpret_cast<const uint2*>(tile + at * kPitch + k * 16 + 8);
    *reinterpret_cast<uint4*>(to + (int64_t)(c0 + at) * pitch + r0 + k * 8) = make_uint4(lo.x, lo.y, hi.x, hi.y);
  }
}

template <typename T>
__global__ __launch_bounds__(256) void lay_out_kernel(Matrix2 x, int64_t first, int64_t count, bool turned, bool along_rows, LayOut with, uint16_t* to,
                                                      int64_t pitch) {
  __shared__ T tile[kTile][kTile + 1];                  // [row][entry]
  __shared__ int by[kTile];                             // of a row: power of two, or kDeadRow
  const int64_t r0 = (int64_t)blockIdx.x * kTile;
  const int c0 = blockIdx.y * kTile;
  const int t = threadIdx.x;
  const int largest = with.most ? largest_exponent(with.most) : 0;
  if (t < kTile) by[t] = r0 + t < count ? row_scale(with, x, first + r0 + t, largest) : 0;
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

namespace {
template <typename T>
void launch(const Matrix2& x, int64_t first, int64_t count, bool turned, const LayOut& with, void* d_to, hipStream_t stream) {
  const int64_t pitch = laid_length(turned ? count : x.length);
  const dim3 grid((unsigned)((count + kTile - 1) / kTile), (unsigned)((x.length + kTile - 1) / kTile));
  uint16_t* const to = static_cast<uint16_t*>(d_to);
  if (x.stride == 1 && turned) {
    hipLaunchKernelGGL((turn_rows_kernel<T>), grid, dim3(256), 0, stream, x, first, count, with, to, pitch);
  } else if (x.stride == 1) {
    hipLaunchKernelGGL((copy_rows_kernel<T>), grid, dim3(256), 0, stream, x, first, count, to, pitch);
  } else {
    const bool along_rows = x.vars == 1 && (x.stride_ex == 1 || x.stride_ex == -1);
    hipLaunchKernelGGL((lay_out_kernel<T>), grid, dim3(256), 0, stream, x, first, count, turned, along_rows, with, to, pitch);
  }
}
}  // namespace

void lay_out(const Matrix2& x, int64_t first, int64_t count, bool turned, const LayOut& with, void* d_to, hipStream_t stream) {
  // (turned rows are those of features or of a piece of the categories, which a launch takes at once)
  const int64_t most = units_a_launch(1, 256) * kTile, pitch = laid_length(x.length);
  for (int64_t at = 0; at < count; at += most) {
    uint16_t* const to = static_cast<uint16_t*>(d_to) + at * pitch;
    const int64_t n = std::min(most, count - at);
    if (x.type == PCM_BF16) launch<bf16>(x, first + at, n, turned, with, to, stream);
    else launch<f16>(x, first + at, n, turned, with, to, stream);
  }
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) fail(PCM_ERR_HIP, "launch of lay_out failed: %s", hipGetErrorString(e));
}

}  // namespace pcm
