// Rows in 8-bit integers with a scale each, and their products.  Rows are bound by memory: 8192 x 4096 bf16, which lie in the caches, 29 us.
#include "product_out.hip.hpp"

namespace pcm {

namespace {
// A workgroup per row: the largest |x| first, then code = rint(x (127 / largest)), scale = largest / 127.  A row with NaN or an infinity gets scale
// NaN; one whose largest |x| is below 2^-119 counts as zeros (127 / largest would pass the range).
struct RowScale {
  float by, scale;
  bool bad;
  __device__ __forceinline__ RowScale(float largest, float (&sub)[4]) {
    largest = over_lanes<64>(largest, LargerOrNan());
    __syncthreads();
    if (threadIdx.x % 64 == 0) sub[threadIdx.x / 64] = largest;
    __syncthreads();
    largest = __builtin_elementwise_maximum(__builtin_elementwise_maximum(sub[0], sub[1]), __builtin_elementwise_maximum(sub[2], sub[3]));
    bad = !(largest < INFINITY);
    const bool none = largest < 0x1p-119f;
    by = bad || none ? 0.f : 127.f / largest;
    scale = bad ? __builtin_nanf("") : none ? 0.f : largest / 127.f;
  }
  __device__ __forceinline__ uint32_t code(float x) const { return bad ? 0u : (uint32_t)(uint8_t)(int8_t)(int)rintf(x * by); }
};
// Rows of neighbours of up to 8192 entries stay in registers, eight to a lane at a time; any others are read twice, entry by entry
template <typename T>
__global__ __launch_bounds__(256) void rows8_kernel(Matrix2 x, int64_t pitch, int8_t* codes, float* scales) {
  __shared__ float sub[4];
  for (int64_t r = blockIdx.x; r < x.rows(); r += gridDim.x) {
    const T* const from = static_cast<const T*>(x.p) + r / x.vars * x.stride_ex + r % x.vars * x.stride_var;
    int8_t* const to = codes + r * pitch;
    float largest = 0.f;
    if (x.stride == 1 && x.length <= 8192) {
      float v[4][8];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int c = (i * 256 + threadIdx.x) * 8;
        if (c + 8 <= x.length) {
          if constexpr (sizeof(T) == 4) {
            const raw4 a = load16(from + c), b = load16(from + c + 4);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              v[i][k] = as_float(a[k]);
              v[i][4 + k] = as_float(b[k]);
            }
          } else {
            const raw4 a = load16(from + c);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const uint32_t w = a[k];
              v[i][2 * k] = (float)__builtin_bit_cast(T, (uint16_t)(w & 0xffffu));
              v[i][2 * k + 1] = (float)__builtin_bit_cast(T, (uint16_t)(w >> 16));
            }
          }
        } else {
#pragma unroll
          for (int k = 0; k < 8; ++k) v[i][k] = c + k < x.length ? (float)from[c + k] : 0.f;
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int k = 0; k < 8; ++k) largest = __builtin_elementwise_maximum(largest, fabsf(v[i][k]));
      const RowScale s(largest, sub);
      if (threadIdx.x == 0) scales[r] = s.scale;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int c = (i * 256 + threadIdx.x) * 8;
        if (c >= pitch) break;
        uint32_t w[2];
#pragma unroll
        for (int h = 0; h < 2; ++h)
          w[h] = s.code(v[i][4 * h]) | s.code(v[i][4 * h + 1]) << 8 | s.code(v[i][4 * h + 2]) << 16 | s.code(v[i][4 * h + 3]) << 24;
        *reinterpret_cast<uint2*>(to + c) = make_uint2(w[0], w[1]);
      }
      continue;
    }
    for (int i = threadIdx.x; i < x.length; i += 256) largest = __builtin_elementwise_maximum(largest, fabsf((float)from[i * x.stride]));
    const RowScale s(largest, sub);
    if (threadIdx.x == 0) scales[r] = s.scale;
    for (int i = threadIdx.x * 4; i < pitch; i += 1024) {
      uint32_t w = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) w |= (i + e < x.length ? s.code((float)from[(i + e) * x.stride]) : 0u) << 8 * e;
      *reinterpret_cast<uint32_t*>(to + i) = w;
    }
  }
}
}  // namespace

void rows8(const Matrix2& x, int8_t* d_codes, float* d_scales, hipStream_t stream) {
  if (x.type < PCM_F32 || x.type > PCM_F16) fail(PCM_ERR_ARG, "8-bit rows: type %d: PCM_F32, PCM_BF16 or PCM_F16", x.type);
  if (x.examples < 0 || x.vars < 1 || x.length < 1) fail(PCM_ERR_SHAPE, "8-bit rows: %lld examples, %d variables, length %d", (long long)x.examples, x.vars, x.length);
  if (x.examples > 0x7fffffff || x.rows() > 0x7fffffff || x.length > kMaxLength8)
    fail(PCM_ERR_UNSUPPORTED, "8-bit rows: more than 2^31 - 1 rows or 131071 entries");
  if (!x.rows()) return;
  if (!x.p || !d_codes || !d_scales) fail(PCM_ERR_ARG, "8-bit rows: a pointer is null");
  if ((uintptr_t)d_codes & 15) fail(PCM_ERR_ARG, "8-bit rows: codes must be 16-byte aligned");
  const dim3 grid((unsigned)std::min<int64_t>(x.rows(), 1 << 20));
  const int64_t pitch = round_up(x.length, kKBytes);
  if (x.type == PCM_F32) hipLaunchKernelGGL((rows8_kernel<float>), grid, dim3(256), 0, stream, x, pitch, d_codes, d_scales);
  else if (x.type == PCM_BF16) hipLaunchKernelGGL((rows8_kernel<bf16>), grid, dim3(256), 0, stream, x, pitch, d_codes, d_scales);
  else hipLaunchKernelGGL((rows8_kernel<f16>), grid, dim3(256), 0, stream, x, pitch, d_codes, d_scales);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) fail(PCM_ERR_HIP, "launch of rows8 failed: %s", hipGetErrorString(e));
}

namespace {
// Few rows, unless tiles of 128 channels fill the compute units (16 and 64 rows of 4096, 25000 channels: 22.3 us by tiles, 21.2 by few rows; 27.7,
// 29.9.  15000: 19.2, 13.5; 26.8, 18.3)
bool few8(int64_t rows, int64_t cats) { return rows <= kFewRowsMost && cats < (rows <= 32 ? 32768 : 20000); }
}  // namespace

int64_t product8_workspace(int64_t rows, int64_t cats, int32_t length) {
  if (rows < 1 || cats < 1 || length < 1 || length > kMaxLength8 || rows > 0x7fffffff || cats > 0x7fffffff) return 0;
  const int steps = (int)(round_up(length, kKBytes) / kKBytes);
  const int parts = few8(rows, cats) ? parts_for_few(cats, steps) : parts_for(cats, rows, steps);
  return parts > 1 ? round_up(parts * rows * cats * 4, 256) : 0;
}

void product8(const int8_t* a, const float* a_scales, int64_t rows, const int8_t* b, const float* b_scales, int64_t cats, int32_t length,
              const BiasRef& bias, void* d_out, int type, int64_t pitch, void* d_work, int64_t work_bytes, hipStream_t stream) {
  if (type < PCM_F32 || type > PCM_F16 || (bias.p && (bias.type < PCM_F32 || bias.type > PCM_F16)))
    fail(PCM_ERR_ARG, "8-bit product: type %d or %d: PCM_F32, PCM_BF16 or PCM_F16", type, bias.type);
  if (rows < 0 || cats < 1 || length < 1 || pitch < cats) fail(PCM_ERR_SHAPE, "8-bit product: %lld rows, %lld channels, length %d, pitch %lld", (long long)rows, (long long)cats, length, (long long)pitch);
  if (rows > 0x7fffffff || cats > 0x7fffffff || length > kMaxLength8)
    fail(PCM_ERR_UNSUPPORTED, "8-bit product: more than 2^31 - 1 rows or channels, or a length of which a sum may pass 32 bits (131071)");
  if (!rows) return;
  if (!a || !a_scales || !b || !b_scales || !d_out) fail(PCM_ERR_ARG, "8-bit product: a pointer is null");
  if (((uintptr_t)a | (uintptr_t)b) & 15) fail(PCM_ERR_ARG, "8-bit product: codes must be 16-byte aligned");
  check_workspace(d_work, work_bytes, product8_workspace(rows, cats, length), "8-bit product");
  const int64_t codes = round_up(length, kKBytes);
  const int steps = (int)(codes / kKBytes);
  const bool few = few8(rows, cats);
  const int parts = few ? parts_for_few(cats, steps) : parts_for(cats, rows, steps);
  OutTask t{};
  t.a = {b, codes, 0};
  t.b = {a, codes, 0};
  t.m = cats;
  t.n = rows;
  t.steps = {steps, kOnePlane, parts};
  t.finish.scale = {a_scales, b_scales};
  t.finish.bias = bias;
  if (parts == 1) {
    t.out = d_out;
    t.type = type;
    t.pitch = pitch;
    few ? product_few(t, stream) : product_out(PCM_U8, t, stream);
    return;
  }
  t.out = d_work;
  t.type = kRawSums;
  t.pitch = cats;
  few ? product_few(t, stream) : product_out(PCM_U8, t, stream);
  join_parts(d_work, parts, true, cats, rows, t.finish, d_out, type, pitch, stream);
}

}  // namespace pcm
