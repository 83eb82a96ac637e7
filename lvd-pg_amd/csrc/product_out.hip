// Products that are written out: gradients of features and weights, and products of 8-bit rows.
#include "product_out.hip.hpp"

namespace pcm {

namespace {
template <typename T, typename S>
__device__ __forceinline__ void out_tile(const OutTask& t, bool fours) {
  __shared__ __attribute__((aligned(16))) float bias[S::BM], scale[S::BM];
  const bool raw = t.type == kRawSums;
  const int most = t.finish.most ? largest_exponent(t.finish.most) : 0;
  const int64_t m0 = tile_at<S>(t.m, t.n).m0;
  for (int i = threadIdx.x; i < S::BM; i += S::threads) {
    bias[i] = m0 + i < t.m ? bias_of(t.finish.bias, m0 + i) : 0.f;
    scale[i] = t.finish.scale.m && m0 + i < t.m ? t.finish.scale.m[m0 + i] : 1.f;
  }
  auto done = [&](auto& sums, int64_t m, int64_t n, char* lds) {
    const int lane = threadIdx.x & 63, half = lane >> 5, wm = threadIdx.x / 64 % S::waves_m * S::WM;
    __syncthreads();
    if (raw) {
#pragma unroll
      for (int j = 0; j < S::FN; ++j) {
        const int64_t row = n + 32 * j + (lane & 31);
        if (row >= t.n) continue;
#pragma unroll
        for (int i = 0; i < S::FM; ++i)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const int64_t col = m + 32 * i + 8 * q + 4 * half;
            uint32_t* const to = static_cast<uint32_t*>(t.out) + ((int64_t)blockIdx.y * t.n + row) * t.pitch + col;
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (col + e < t.m) {
                auto v = sums[i][j][4 * q + e];
                if constexpr (!__is_same(T, int8_t)) {
                  if (t.add) v += __builtin_bit_cast(float, to[e]);
                }
                to[e] = __builtin_bit_cast(uint32_t, v);
              }
          }
      }
      return;
    }
    // eight rows of a wave's result at a time by way of its own LDS, so that they go out in whole lines
    constexpr int kPitch = S::WM + 4;                                              // floats
    float* const mine = reinterpret_cast<float*>(lds) + threadIdx.x / 64 * 8 * kPitch;
    static_assert(S::waves * 8 * kPitch * sizeof(float) <= S::stage);
#pragma unroll
    for (int j = 0; j < S::FN; ++j) {
      const int64_t row = n + 32 * j + (lane & 31);
      const FinishAt finish(t.finish, row < t.n ? row : t.n - 1, most);
      __builtin_amdgcn_sched_barrier(0);
      float4 v[S::FM][4];
#pragma unroll
      for (int i = 0; i < S::FM; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int in = wm + 32 * i + 8 * q + 4 * half;
          const float4 b = *reinterpret_cast<const float4*>(bias + in), s = *reinterpret_cast<const float4*>(scale + in);
#pragma unroll
          for (int e = 0; e < 4; ++e) (&v[i][q].x)[e] = finish((float)sums[i][j][4 * q + e], (&s.x)[e], (&b.x)[e]);
        }
#pragma unroll
      for (int eight = 0; eight < 4; ++eight) {
        if ((lane & 31) / 8 == eight)
#pragma unroll
          for (int i = 0; i < S::FM; ++i)
#pragma unroll
            for (int q = 0; q < 4; ++q) *reinterpret_cast<float4*>(mine + lane % 8 * kPitch + 32 * i + 8 * q + 4 * half) = v[i][q];
        __builtin_amdgcn_wave_barrier();
        constexpr int kLanes = S::WM / 4;                                          // of four columns to a row
#pragma unroll
        for (int r = 0; r < 8; r += 64 / kLanes) {
          const int in = r + lane / kLanes, at = lane % kLanes * 4;
          const int64_t to = n + 32 * j + 8 * eight + in, col = m + at;
          if (in < 8 && to < t.n) {
            const float4 w = *reinterpret_cast<const float4*>(mine + in * kPitch + at);
            const float v[4] = {w.x, w.y, w.z, w.w};
            if (fours && col + 4 <= t.m) store_four(t.out, t.type, to * t.pitch + col, v);
            else
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if (col + e < t.m) store_as(t.out, t.type, to * t.pitch + col + e, v[e]);
          }
        }
        __builtin_amdgcn_wave_barrier();
      }
    }
  };
  if constexpr (__is_same(T, float)) float_tile(t.fa, t.fb, t.m, t.n, t.fk, t.steps.parts, done);
  else product_tile<T, S>(t.a, t.b, t.m, t.n, t.steps, done);
}
template <typename T, typename S>
__global__ __launch_bounds__(S::threads, 2) void out_kernel(OutTask t, bool fours) {
  out_tile<T, S>(t, fours);
}

template <int kGroups>
__global__ __launch_bounds__(FewTile<kGroups>::threads) void out_few_kernel(OutTask t) {
  typedef FewTile<kGroups> S;
  __shared__ __attribute__((aligned(16))) char lds[S::lds];
  const float* const sums = few_sums<int8_t, kGroups>(FewOperand{t.a.p, t.a.pitch, 0, 1}, FewOperand{t.b.p, t.b.pitch, 0, 1}, t.m, t.n,
                                                      t.steps.count * kKBytes, t.steps.parts, lds);
  const int at = threadIdx.x % S::longs;
  const int64_t m = (int64_t)blockIdx.x * S::longs + at;
  if (m >= t.m) return;
  const float scale = t.finish.scale.m[m], bias = bias_of(t.finish.bias, m);
  for (int n = threadIdx.x / S::longs; n < t.n; n += S::threads / S::longs) {
    const float bits = sums[at * S::pitch + n];
    const int sum = __builtin_bit_cast(int, bits);
    if (t.type == kRawSums) static_cast<int*>(t.out)[((int64_t)blockIdx.y * t.n + n) * t.pitch + m] = sum;
    else store_as(t.out, t.type, n * t.pitch + m, FinishAt(t.finish, n, 0)((float)sum, scale, bias));
  }
}

__global__ __launch_bounds__(256) void join_parts_kernel(const uint32_t* parts, int count, bool whole, int64_t m, int64_t n, Finish finish, void* out,
                                                         int type, int64_t pitch) {
  const int most = finish.most ? largest_exponent(finish.most) : 0;
  const int64_t all = n * m;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < all; i += (int64_t)gridDim.x * 256) {
    const int64_t row = i / m, col = i % m;
    float sum = 0.f;
    if (whole) {
      int s = 0;
#pragma unroll 8
      for (int p = 0; p < count; ++p) s += (int)parts[p * all + i];
      sum = (float)s;
    } else {
#pragma unroll 8
      for (int p = 0; p < count; ++p) sum += __builtin_bit_cast(float, parts[p * all + i]);
    }
    const FinishAt f(finish, row, most);
    store_as(out, type, row * pitch + col, f(sum, finish.scale.m ? finish.scale.m[col] : 1.f, bias_of(finish.bias, col)));
  }
}

typedef TileSizes<256, 256, 128, 64> Wide;
typedef TileSizes<128, 128, 64, 64> Middle;
typedef TileSizes<128, 64, 64, 32> Slim;
typedef TileSizes<128, 32, 32, 32> Narrow;

template <typename T, typename S>
void launch(const OutTask& t, hipStream_t stream) {
  const int64_t tiles = ((t.m + S::BM - 1) / S::BM) * ((t.n + S::BN - 1) / S::BN);
  if (tiles > 0x7fffffff) fail(PCM_ERR_UNSUPPORTED, "product: %lld tiles", (long long)tiles);
  const int size = t.type == PCM_F32 ? 4 : 2;
  const bool fours = t.type != kRawSums && t.pitch % 4 == 0 && (uintptr_t)t.out % (4 * size) == 0;
  hipLaunchKernelGGL((out_kernel<T, S>), dim3((unsigned)tiles, (unsigned)t.steps.parts), dim3(S::threads), 0, stream, t, fours);
}
template <typename T>
void launch(const OutTask& t, hipStream_t stream) {
  if (t.n <= 32) launch<T, Narrow>(t, stream);
  else if (t.n <= 64) launch<T, Slim>(t, stream);
  else if (wide_tiles(t.m, t.n, t.steps.count * t.steps.pairs.count / t.steps.parts)) launch<T, Wide>(t, stream);
  else launch<T, Middle>(t, stream);
}
}  // namespace

int parts_for(int64_t m, int64_t n, int64_t steps, bool of_float) {
  if (!of_float && wide_tiles(m, n, steps)) return 1;
  const int64_t each = of_float || n > 64 ? 128 : n > 32 ? 64 : 32, tiles = ((m + 127) / 128) * ((n + each - 1) / each);
  // as many parts as leave two workgroups a compute unit at most (one, where the sums are short and joining them would cost more), each of four
  // steps or more
  return (int)std::max<int64_t>(1, std::min<int64_t>({(steps < 64 ? 256 : 512) / tiles, steps / 4, 64}));
}
int parts_for_few(int64_t m, int64_t steps) {
  // a workgroup's waves take a step each at a time: parts of four rounds or more, as many as give every compute unit two workgroups
  return (int)std::max<int64_t>(1, std::min<int64_t>({(512 * kFewTile + m - 1) / m, steps / 32, 16}));
}
void product_few(const OutTask& t, hipStream_t stream) {
  const int each = kFewTile;
  const dim3 grid((unsigned)((t.m + each - 1) / each), (unsigned)t.steps.parts), block(t.n > 32 ? 256 : 512);
  if (t.n <= 16) hipLaunchKernelGGL(out_few_kernel<1>, grid, block, 0, stream, t);
  else if (t.n <= 32) hipLaunchKernelGGL(out_few_kernel<2>, grid, block, 0, stream, t);
  else hipLaunchKernelGGL(out_few_kernel<4>, grid, block, 0, stream, t);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) fail(PCM_ERR_HIP, "launch of a product failed: %s", hipGetErrorString(e));
}

void product_out(int operands, const OutTask& t, hipStream_t stream) {
  if (operands == PCM_F32) launch<float, FloatTile>(t, stream);
  else if (operands == PCM_BF16) launch<bf16>(t, stream);
  else if (operands == PCM_F16) launch<f16>(t, stream);
  else launch<int8_t>(t, stream);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) fail(PCM_ERR_HIP, "launch of a product failed: %s", hipGetErrorString(e));
}

void join_parts(const void* parts, int count, bool whole, int64_t m, int64_t n, const Finish& finish, void* out, int type, int64_t pitch, hipStream_t stream) {
  hipLaunchKernelGGL(join_parts_kernel, dim3((unsigned)std::min<int64_t>((n * m + 255) / 256, 1 << 14)), dim3(256), 0, stream,
                     static_cast<const uint32_t*>(parts), count, whole, m, n, finish, out, type, pitch);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) fail(PCM_ERR_HIP, "launch of join_parts failed: %s", hipGetErrorString(e));
}

}  // namespace pcm
