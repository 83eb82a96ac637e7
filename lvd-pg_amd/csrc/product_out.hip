// Products that are written out: gradients of features and weights, and products of 8-bit rows.
//
// Long sums are bound by the matrix cores: 8192 x 16384 over 4096 in 8 bits 550 us (2.0 POP/s), 4096 x 4096 over 16384 bf16 460 us (1.19
// PFLOP/s).  Results go out by way of LDS, since a lane's four neighbours alone fill an eighth of a line.
#include "product_out.hip.hpp"

namespace pcm {

namespace {
template <typename T, typename S>
__device__ __forceinline__ void out_tile(const OutTask& t, bool fours) {
  __shared__ __attribute__((aligned(16))) float bias[S::BM], scale[S::BM];
  const bool raw = t.type == kRawSums;
  const int most = t.finish.most ? largest_exponent(t.finish.most) : 0;
  const int64_t m0 = tile_at<S>(t.m, 0).m0;
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
  if constexpr (__is_same(T, float)) float_tile(t.fa, t.fb, t.m, t.n, 0, t.fk, t.steps.parts, done);
  else product_tile<T, S>(t.a, t.b, t.m, t.n, 0, t.steps, done);
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

// Short sums (kSteps of 128 bytes), b in one part or two: bound by writing the result.  A wave keeps the operands of 32 rows of b in registers and
// goes over the columns, 64 at a time, whose operands come from the caches; nothing waits in LDS or at a barrier, as a tile's one or two steps
// do.  30000 x 4096 bf16 from 64 rows: 148 us by tiles, 90 so (2.7 TB/s; 130 with every wave at the same columns and straight from
// registers); 30001 x 1001 f16 from 50: 61, 38; 40000 x 1001 bf16 from 60 categories: 75, 46; 32768 x 768 f16 from 128: 34, 32.
template <typename T, int kSteps, int kPlanes>
__device__ __forceinline__ void short_rows(const OutTask& t, int chunks) {
  constexpr int kPitch = 144;                // bytes: 64 columns of a row and a gap
  __shared__ __attribute__((aligned(16))) char lds[4 * 32 * kPitch];
  const int lane = threadIdx.x & 63, half = lane >> 5, wave = threadIdx.x / 64;
  const int64_t n0 = ((int64_t)blockIdx.x * 4 + wave) * 32, n = n0 + (lane & 31);
  if (n0 >= t.n) return;
  char* const mine = lds + wave * 32 * kPitch;
  const FinishAt finish(t.finish, min(n, t.n - 1), t.finish.most ? largest_exponent(t.finish.most) : 0);
  const float by = ldexpf(1.f, finish.expo);   // (exponents lie within float's)
  const char* const b = static_cast<const char*>(t.b.p) + min(n, t.n - 1) * t.b.pitch + half * 16;
  v4i fb[kPlanes][4 * kSteps];
#pragma unroll
  for (int p = 0; p < kPlanes; ++p)
#pragma unroll
    for (int s = 0; s < 4 * kSteps; ++s) fb[p][s] = *reinterpret_cast<const v4i*>(b + p * t.b.plane + s * 32);
  for (int chunk = 0; chunk < chunks; ++chunk) {
    // (each workgroup begins elsewhere: rows of a power of two bytes would otherwise keep all at a few of the memory's channels)
    const int64_t m = ((int64_t)blockIdx.y * chunks + (chunk + blockIdx.x) % chunks) * 64;
    if (m >= t.m) continue;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const char* const a = static_cast<const char*>(t.a.p) + min(m + 32 * i + (lane & 31), t.m - 1) * t.a.pitch + half * 16;
      v4i fa[4 * kSteps];
#pragma unroll
      for (int s = 0; s < 4 * kSteps; ++s) fa[s] = *reinterpret_cast<const v4i*>(a + s * 32);
      v16f sums = {};
#pragma unroll
      for (int p = kPlanes - 1; p >= 0; --p)   // the smaller part first
#pragma unroll
        for (int s = 0; s < 4 * kSteps; ++s) sums = Cores<T>::mma(fa[s], fb[p][s], sums);
#pragma unroll
      for (int q = 0; q < 4; q += 2) {       // eight neighbouring columns a lane, from both halves' four
        uint32_t code[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float u = sums[4 * q + 2 * k], v = sums[4 * q + 2 * k + 1];
          code[k] = finish.dead ? 0u : pair_of<T>(u * by, v * by);
        }
        const auto lo = __builtin_amdgcn_permlane32_swap(code[0], code[2], false, false);
        const auto hi = __builtin_amdgcn_permlane32_swap(code[1], code[3], false, false);
        *reinterpret_cast<uint4*>(mine + (lane & 31) * kPitch + (32 * i + 8 * q + 8 * half) * 2) = make_uint4(lo[0], hi[0], lo[1], hi[1]);
      }
    }
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int r = 0; r < 32; r += 8) {        // eight rows' 128 bytes at a time
      const int in = r + lane / 8;
      const int64_t to_n = n0 + in, col = m + lane % 8 * 8;
      if (to_n >= t.n) continue;
      const char* const from = mine + in * kPitch + lane % 8 * 16;
      const raw4 v = *reinterpret_cast<const raw4*>(from);
      uint16_t* const to = static_cast<uint16_t*>(t.out) + to_n * t.pitch + col;
      // rows that begin inside a word: a lane's seven last entries and the next lane's first one, whole words
      const bool odd = (uintptr_t)to & 2;
      if (!odd && col + 8 <= t.m) {
        *reinterpret_cast<raw4_by4*>(to) = v;
      } else if (odd && lane % 8 < 7 && col + 9 <= t.m) {
        const uint32_t next = *reinterpret_cast<const uint32_t*>(from + 16);
        raw4 w;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t hi = k < 3 ? v[k < 3 ? k + 1 : 3] : next, lo = v[k];
          w[k] = __builtin_amdgcn_alignbit(hi, lo, 16);
        }
        *reinterpret_cast<raw4_by4*>(to + 1) = w;
        if (lane % 8 == 0) to[0] = (uint16_t)v[0];
      } else {
        const int e0 = odd && lane % 8 ? 1 : 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const uint32_t w = v[e / 2];
          if (e >= e0 && col + e < t.m) to[e] = (uint16_t)(w >> 16 * (e % 2));
        }
      }
    }
    __builtin_amdgcn_wave_barrier();
  }
}
template <typename T, int kSteps, int kPlanes>
__global__ __launch_bounds__(256) void out_short_kernel(OutTask t, int chunks) {   // chunks of 64 columns
  short_rows<T, kSteps, kPlanes>(t, chunks);
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
  if (tiles > most_blocks(S::threads)) fail(PCM_ERR_UNSUPPORTED, "product: %lld tiles", (long long)tiles);
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

namespace {
template <typename T>
void launch_short(const OutTask& t, hipStream_t stream) {
  // up to 16 chunks of columns a workgroup, as many as leave two workgroups a compute unit
  const int64_t rows = (t.n + 127) / 128, all = (t.m + 63) / 64;
  const int chunks = (int)std::max<int64_t>(1, std::min<int64_t>(16, all * rows / 512));
  const dim3 grid((unsigned)rows, (unsigned)((all + chunks - 1) / chunks));
  const bool one = t.steps.pairs.count == 1;
  if (t.steps.count == 1 && one) hipLaunchKernelGGL((out_short_kernel<T, 1, 1>), grid, dim3(256), 0, stream, t, chunks);
  else if (t.steps.count == 1) hipLaunchKernelGGL((out_short_kernel<T, 1, 2>), grid, dim3(256), 0, stream, t, chunks);
  else if (one) hipLaunchKernelGGL((out_short_kernel<T, 2, 1>), grid, dim3(256), 0, stream, t, chunks);
  else hipLaunchKernelGGL((out_short_kernel<T, 2, 2>), grid, dim3(256), 0, stream, t, chunks);
}
}  // namespace
void product_short(int operands, const OutTask& t, hipStream_t stream) {
  if (operands == PCM_BF16) launch_short<bf16>(t, stream);
  else launch_short<f16>(t, stream);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) fail(PCM_ERR_HIP, "launch of a product failed: %s", hipGetErrorString(e));
}

bool short_sums(int operands, const OutTask& t) {
  return operands != PCM_F32 && t.type == operands && t.steps.count <= 2 && t.steps.parts == 1 && !t.add;
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
