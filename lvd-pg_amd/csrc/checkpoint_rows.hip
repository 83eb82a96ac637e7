// Checkpoints of rows in 8 bits, and the rows back from them.  Both stream: bound by the bytes of rows and codes.
#include "category_tiles.hip.hpp"

namespace pcm {

namespace {
// Rows of neighbouring entries: the 64 of a block lie in 64 / kVec neighbouring lanes, which find the range with three or four steps.
// 100 rows of 3342336 f32: 320 us, 5.3 TB/s (a copy of the rows: 5.0); 333 of 10007 bf16: 7 us.
template <typename T>
__global__ __launch_bounds__(kTileThreads) void checkpoint_tile_kernel(RowsRef x, RowsShape shape, CkptRef ckpt, Tiles tiles) {
  constexpr int kVec = 16 / (int)sizeof(T);
  const int64_t rows = shape.rows();
  const int64_t pitch = (shape.cats + 15) / 16 * 16, blocks = (shape.cats + kCkptBlock - 1) / kCkptBlock;
  for (int64_t job = blockIdx.x; job < tiles.jobs; job += gridDim.x) {
    const TileAt tile = tile_at(tiles, job);
    const bool mine = tile.row < rows;
    const uint32_t r = (uint32_t)(mine ? tile.row : rows - 1);
    const int64_t e = shape.vars == 1 ? r : r / (uint32_t)shape.vars, v = shape.vars == 1 ? 0 : r % (uint32_t)shape.vars;
    const T* const row = static_cast<const T*>(x.p) + e * x.stride_ex + v * x.stride_var;
    raw4 raw[kTileGroups];
#pragma unroll
    for (int u = 0; u < kTileGroups; ++u) raw[u] = load_group(row, (int64_t)(tile.first + u * tile.step) * kVec, shape.cats);
#pragma unroll
    for (int u = 0; u < kTileGroups; ++u) {
      const int64_t c = (int64_t)(tile.first + u * tile.step) * kVec;
      float y[kVec];
      unpack(raw[u], y, T());
      const BlockCodes<kVec> k = encode_block<T>(y);
      if (mine) store_codes(ckpt, k, r, c, shape.cats, pitch, blocks);
    }
  }
}

// Rows that lie side by side: a lane per row, which holds the 64 entries of a block and finds their range alone; two blocks at a time,
// so that whole lines of codes are written.  65536 rows of 256, f32, the call: 22 us, 89 with a wave per block (17 for rows of
// neighbours); from 64 rows on, so that no lanes idle.
template <typename T>
__global__ __launch_bounds__(256) void checkpoint_column_kernel(RowsRef x, RowsShape shape, CkptRef ckpt, bool examples_first) {
  const int64_t rows = shape.rows(), pitch = (shape.cats + 15) / 16 * 16, blocks = (shape.cats + kCkptBlock - 1) / kCkptBlock;
  const int64_t sets = (rows + 63) / 64, jobs = sets * ((blocks + 1) / 2);
  for (int64_t job = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); job < jobs; job += (int64_t)gridDim.x * 4) {
    const int64_t pair = job / sets, at = (job - pair * sets) * 64 + (threadIdx.x & 63);
    if (at >= rows) continue;
    const RowAt n = row_at(shape, (uint32_t)at, examples_first);
    const T* const row = static_cast<const T*>(x.p) + n.e * x.stride_ex + n.v * x.stride_var;
    for (int64_t b = 2 * pair; b < min(2 * pair + 2, blocks); ++b) {
      const int c0 = (int)(b * kCkptBlock);
      float y[kCkptBlock], hi = -INFINITY, lo = INFINITY, kept = INFINITY;
#pragma unroll
      for (int i = 0; i < kCkptBlock; ++i) y[i] = c0 + i < shape.cats ? to_float(row[(int64_t)(c0 + i) * x.stride_cat]) : -INFINITY;
#pragma unroll
      for (int i = 0; i < kCkptBlock; ++i) {
        hi = __builtin_elementwise_maximum(hi, y[i]);
        lo = fminf(lo, y[i]);
        kept = fminf(kept, y[i] > masked_from<T>() ? y[i] : INFINITY);
      }
      const BlockScale s = block_scale(hi > masked_from<T>() ? hi : -INFINITY, kept, lo <= masked_from<T>(), !(hi < INFINITY));
      uint8_t* const to = ckpt.codes + n.r * pitch + c0;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        raw4 w = {0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float z = y[16 * q + i];
          w[i / 4] |= (z <= masked_from<T>() ? (uint32_t)kCkptMasked : block_code(s, z) & 0xffu) << (8 * (i % 4));
        }
        if (c0 + 16 * q < pitch) *reinterpret_cast<raw4*>(to + 16 * q) = w;
      }
      ckpt.scales[n.r * blocks + b] = s.word;
    }
  }
}

// Any strides: a wave per block of 64 entries
template <typename T>
__global__ __launch_bounds__(256) void checkpoint_kernel(RowsRef x, RowsShape shape, CkptRef ckpt) {
  const int lane = threadIdx.x & 63;
  const int64_t pitch = (shape.cats + 15) / 16 * 16, blocks = (shape.cats + kCkptBlock - 1) / kCkptBlock, all = shape.rows() * blocks;
  for (int64_t b = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); b < all; b += (int64_t)gridDim.x * 4) {
    const int64_t r = b / blocks, e = r / shape.vars, v = r % shape.vars;
    const int64_t c = (b % blocks) * kCkptBlock + lane;
    const T* row = static_cast<const T*>(x.p) + e * x.stride_ex + v * x.stride_var;
    const float y = c < shape.cats ? to_float(row[c * x.stride_cat]) : -INFINITY;
    const bool off = y <= masked_from<T>();
    const float hi = over_lanes<64>(off ? -INFINITY : y, LargerOrNan()), lo = over_lanes<64>(off ? INFINITY : y, Smaller());
    const BlockScale s = block_scale(hi > masked_from<T>() ? hi : -INFINITY, lo, __any(off), !(hi < INFINITY));
    if (c < pitch) ckpt.codes[r * pitch + c] = off ? (uint8_t)kCkptMasked : (uint8_t)block_code(s, y);
    if (lane == 0) ckpt.scales[b] = s.word;
  }
}

// (a value may have been rounded up past the largest of the type; NaN stays)
template <typename T>
__device__ __forceinline__ T restored(float y) { return from_float<T>(__builtin_elementwise_minimum(y, type_max<T>())); }

// 100 rows of 3342336 f32: 345 us, 4.9 TB/s
template <typename T>
__global__ __launch_bounds__(kTileThreads) void restore_tile_kernel(CkptRef ckpt, RowsShape shape, RowsRef out, Tiles tiles) {
  constexpr int kVec = 16 / (int)sizeof(T);
  const int64_t pitch = (shape.cats + 15) / 16 * 16, blocks = (shape.cats + kCkptBlock - 1) / kCkptBlock;
  for (int64_t job = blockIdx.x; job < tiles.jobs; job += gridDim.x) {
    const TileAt tile = tile_at(tiles, job);
    if (tile.row >= shape.rows()) continue;
    const uint32_t r = (uint32_t)tile.row;
    const int64_t e = shape.vars == 1 ? r : r / (uint32_t)shape.vars, v = shape.vars == 1 ? 0 : r % (uint32_t)shape.vars;
    T* const dst = static_cast<T*>(const_cast<void*>(out.p)) + e * out.stride_ex + v * out.stride_var;
    Codes<kVec> code[kTileGroups];
    uint32_t word[kTileGroups];
#pragma unroll
    for (int u = 0; u < kTileGroups; ++u) {
      const int64_t c = (int64_t)(tile.first + u * tile.step) * kVec;
      if (c >= shape.cats) continue;
      code[u] = load_codes<kVec>(ckpt.codes + r * pitch + c);
      word[u] = ckpt.scales[r * blocks + c / kCkptBlock];
    }
#pragma unroll
    for (int u = 0; u < kTileGroups; ++u) {
      const int64_t c = (int64_t)(tile.first + u * tile.step) * kVec;
      if (c >= shape.cats) continue;
      const BlockUnit unit = block_unit(word[u]);
      T w[kVec];
      float y[kVec];
      decode(code[u], unit, y);
#pragma unroll
      for (int i = 0; i < kVec; ++i) w[i] = restored<T>(y[i]);
      store_group(dst, c, shape.cats, w);
    }
  }
}

// ... into rows that lie side by side, a lane per row: 65536 of 256, f32, the call: 16 us, 125 entry by entry (15 into neighbours)
template <typename T>
__global__ __launch_bounds__(256) void restore_column_kernel(CkptRef ckpt, RowsShape shape, RowsRef out, bool examples_first) {
  const int64_t rows = shape.rows(), pitch = (shape.cats + 15) / 16 * 16, blocks = (shape.cats + kCkptBlock - 1) / kCkptBlock;
  const int64_t sets = (rows + 63) / 64, jobs = sets * blocks;
  for (int64_t job = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); job < jobs; job += (int64_t)gridDim.x * 4) {
    const int64_t set = job / blocks, b = job - set * blocks, at = set * 64 + (threadIdx.x & 63);
    if (at >= rows) continue;
    const RowAt n = row_at(shape, (uint32_t)at, examples_first);
    T* const dst = static_cast<T*>(const_cast<void*>(out.p)) + n.e * out.stride_ex + n.v * out.stride_var;
    const int c0 = (int)(b * kCkptBlock);
    const uint8_t* const from = ckpt.codes + n.r * pitch + c0;
    const BlockUnit unit = block_unit(ckpt.scales[n.r * blocks + b]);
    raw4 w[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) w[q] = c0 + 16 * q < pitch ? *reinterpret_cast<const raw4*>(from + 16 * q) : raw4{0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < kCkptBlock; ++i)
      if (c0 + i < shape.cats)
        dst[(int64_t)(c0 + i) * out.stride_cat] = restored<T>(block_entry_or_mask(unit, (float)(w[i / 16][i / 4 % 4] >> (8 * (i % 4)) & 0xffu)));
  }
}

template <typename T>
__global__ __launch_bounds__(256) void restore_kernel(CkptRef ckpt, RowsShape shape, RowsRef out) {
  const int64_t pitch = (shape.cats + 15) / 16 * 16, blocks = (shape.cats + kCkptBlock - 1) / kCkptBlock, all = shape.rows() * shape.cats;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < all; i += (int64_t)gridDim.x * 256) {
    const int64_t r = i / shape.cats, c = i % shape.cats, e = r / shape.vars, v = r % shape.vars;
    const float y = block_entry_or_mask(block_unit(ckpt.scales[r * blocks + c / kCkptBlock]), ckpt.codes[r * pitch + c]);
    static_cast<T*>(const_cast<void*>(out.p))[e * out.stride_ex + v * out.stride_var + c * out.stride_cat] = restored<T>(y);
  }
}

template <typename T>
void launch_checkpoint(const RowsRef& x, const RowsShape& shape, const CkptRef& ckpt, hipStream_t stream) {
  if (x.stride_cat == 1) {
    const Tiles t = tiles_of(shape, 16 / (int)sizeof(T), kCkptBlock * (int)sizeof(T) / 16);
    hipLaunchKernelGGL((checkpoint_tile_kernel<T>), tile_grid(t), dim3(kTileThreads), 0, stream, x, shape, ckpt, t);
  } else if (side_by_side(x, shape) && shape.rows() >= 64) {
    const int64_t jobs = (shape.rows() + 63) / 64 * ((ckpt_blocks(shape.cats) + 1) / 2);
    hipLaunchKernelGGL((checkpoint_column_kernel<T>), dim3((unsigned)std::min<int64_t>((jobs + 3) / 4, 1 << 20)), dim3(256), 0, stream, x, shape, ckpt,
                       examples_side_by_side(x, shape));
  } else {
    const dim3 grid((unsigned)std::min<int64_t>((shape.rows() * ckpt_blocks(shape.cats) + 3) / 4, 1 << 20));
    hipLaunchKernelGGL((checkpoint_kernel<T>), grid, dim3(256), 0, stream, x, shape, ckpt);
  }
}
template <typename T>
void launch_restore(const CkptRef& ckpt, const RowsShape& shape, const RowsRef& out, hipStream_t stream) {
  if (out.stride_cat == 1) {
    const Tiles t = tiles_of(shape, 16 / (int)sizeof(T), 1);
    hipLaunchKernelGGL((restore_tile_kernel<T>), tile_grid(t), dim3(kTileThreads), 0, stream, ckpt, shape, out, t);
  } else if (side_by_side(out, shape) && shape.rows() >= 64) {
    const int64_t jobs = (shape.rows() + 63) / 64 * ckpt_blocks(shape.cats);
    hipLaunchKernelGGL((restore_column_kernel<T>), dim3((unsigned)std::min<int64_t>((jobs + 3) / 4, 1 << 20)), dim3(256), 0, stream, ckpt, shape, out,
                       examples_side_by_side(out, shape));
  } else {
    const dim3 grid((unsigned)std::min<int64_t>((shape.rows() * shape.cats + 255) / 256, 1 << 20));
    hipLaunchKernelGGL((restore_kernel<T>), grid, dim3(256), 0, stream, ckpt, shape, out);
  }
}
}  // namespace

void checkpoint_rows(const RowsRef& x_in, const RowsShape& shape, const CkptRef& ckpt, hipStream_t stream) {
  RowsRef x = x_in;
  check_rows(x, shape, "checkpoint");
  if (!shape.examples) return;
  if (!x.p || !ckpt.codes || !ckpt.scales) fail(PCM_ERR_ARG, "checkpoint: a pointer is null");
  if ((uintptr_t)ckpt.codes & 15) fail(PCM_ERR_ARG, "checkpoint: codes must be 16-byte aligned");
  if (shape.cats == 1) x.stride_cat = 1;
  if (x.dtype == PCM_F32) launch_checkpoint<float>(x, shape, ckpt, stream);
  else if (x.dtype == PCM_BF16) launch_checkpoint<bf16>(x, shape, ckpt, stream);
  else launch_checkpoint<f16>(x, shape, ckpt, stream);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) fail(PCM_ERR_HIP, "launch of checkpoint_rows failed: %s", hipGetErrorString(e));
}

void restore_rows(const CkptRef& ckpt, const RowsShape& shape, const RowsRef& out_in, hipStream_t stream) {
  RowsRef out = out_in;
  check_rows(out, shape, "restored rows");
  if (!shape.examples) return;
  if (!out.p || !ckpt.codes || !ckpt.scales) fail(PCM_ERR_ARG, "restored rows: a pointer is null");
  if ((uintptr_t)ckpt.codes & 15) fail(PCM_ERR_ARG, "restored rows: codes must be 16-byte aligned");
  if (shape.cats == 1) out.stride_cat = 1;
  if (out.dtype == PCM_F32) launch_restore<float>(ckpt, shape, out, stream);
  else if (out.dtype == PCM_BF16) launch_restore<bf16>(ckpt, shape, out, stream);
  else launch_restore<f16>(ckpt, shape, out, stream);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) fail(PCM_ERR_HIP, "launch of restore_rows failed: %s", hipGetErrorString(e));
}

}  // namespace pcm
