// Gradient of log-probabilities, entropy and likeliest categories with respect to the rows of scores.
//
//   dx[c] = sum of the slots' gradients at c - p (G + gh (log p + H)),  p = exp(x[c] - log Z), G the sum of all slots' gradients:
// an exponential and four products an entry, so a kernel that streams: bound by the bytes of scores (or codes) and gradient.
#include "category_tiles.hip.hpp"

namespace pcm {

namespace {
constexpr int kStaged = 2048;   // slots of all rows of a workgroup, in LDS
// Most slots that every lane of a row of several per workgroup looks through; more are added in LDS by one lane of the row, where the row
// has more than kLdsCats f32 entries.  Looked through / in LDS, us: 65536 rows of 128 with 8 slots 21.8 / 19.3, 24 40 / 28, 64 95 / 58; 16384 of
// 500 with 24 31 / 23; 347990 of 22 with 24 69 / 78, 64 201 / 253; 16384 of 900 f16 with 24 36 / 36.
constexpr int kFewSlots = 6, kLdsCats = 64;

struct GradIn {
  GivenRef given;
  const float* grad_logp;
  int top;
  const int32_t* top_index;
  const float *grad_top, *log_sum, *entropy, *grad_entropy;
};
struct GradSlot {
  int at;      // category; -1: adds nothing
  float by;
};
__device__ __forceinline__ GradSlot grad_slot(const GradIn& in, int64_t r, int64_t e, int64_t v, int j, int cats, bool& past) {
  const bool g = j < in.given.slots;
  const int64_t at = g ? given_at(in.given, e, v, j) : in.top_index[r * in.top + j - in.given.slots];
  const float by = g ? in.grad_logp[r * in.given.slots + j] : in.grad_top[r * in.top + j - in.given.slots];
  past = at >= cats;
  return {at < 0 || past ? -1 : (int)at, by};
}
struct GradRow {
  float z, total, gh, h;
  // total: of the slots' gradients.  A row that has no category gets p = 0 everywhere.
  __device__ __forceinline__ GradRow(const GradIn& in, int64_t r, float sum) {
    z = in.log_sum[r];
    total = sum;
    gh = in.grad_entropy ? in.grad_entropy[r] : 0.f;
    h = in.grad_entropy ? in.entropy[r] : 0.f;
    if (z == -INFINITY) {
      z = INFINITY;
      total = gh = h = 0.f;
    }
  }
  __device__ __forceinline__ bool none() const { return z == INFINITY; }
  template <bool kEnt>
  __device__ __forceinline__ float at(float x) const {
    const float d = x - z, p = __builtin_amdgcn_exp2f(d * kLog2e);
    return kEnt ? -p * fmaf(gh, fmaxf(d, -200.f) + h, total) : -p * total;   // (p is 0 where d is below, and may be -inf)
  }
};

// Rows of neighbouring categories in and out (kUnit), or of any others, entry by entry.  Where a wave holds one row (64 lanes a row or more), its slots wait in the wave's lanes, and a
// group of the row asks once which of them it holds: none, mostly.  Slots of shorter rows wait in LDS.  Either way they are added in
// their order, so that sums come out the same every time.  512 x 784 rows of 256 f16 (kUnit): 98 us, 4.2 TB/s of scores and
// gradient; 65536 rows of 256 f32 of every second category, entry by entry: 71 us, 265 with a lane per row.
template <typename T, bool kCkpt, bool kEnt, bool kUnit, bool kInLds>
__global__ __launch_bounds__(kTileThreads) void grad_tile_kernel(RowsRef x, CkptRef ckpt, RowsShape shape, GradIn in, RowsRef out, Tiles tiles) {
  constexpr int kVec = 16 / (int)sizeof(T);
  __shared__ GradSlot slot_lds[kStaged];
  extern __shared__ float grad_lds[];   // kInLds (one turn): the rows' gradients, [per][width]
  const int slots = in.given.slots + in.top, per = kTileThreads >> tiles.lanes_log2, of = threadIdx.x >> tiles.lanes_log2, lane = threadIdx.x & 63;
  const int width = (kTileGroups * kVec) << tiles.lanes_log2;
  const int64_t rows = shape.rows();
  const int64_t pitch = (shape.cats + 15) / 16 * 16, blocks = (shape.cats + kCkptBlock - 1) / kCkptBlock;
  for (int64_t job = blockIdx.x; job < tiles.jobs; job += gridDim.x) {
    TileAt tile = tile_at(tiles, job);
    const bool mine = tile.row < rows;
    const uint32_t r = (uint32_t)(mine ? tile.row : rows - 1);
    const int64_t e = shape.vars == 1 ? r : r / (uint32_t)shape.vars, v = shape.vars == 1 ? 0 : r % (uint32_t)shape.vars;
    const T* const row = static_cast<const T*>(x.p) + e * x.stride_ex + v * x.stride_var;
    T* const dst = static_cast<T*>(const_cast<void*>(out.p)) + e * out.stride_ex + v * out.stride_var;

    raw4 raw[kCkpt ? 1 : kTileGroups];
    Codes<kVec> code[kCkpt ? kTileGroups : 1];
    uint32_t unit[kCkpt ? kTileGroups : 1];
    auto request = [&] {
#pragma unroll
      for (int u = 0; u < kTileGroups; ++u) {
        const int64_t c = (int64_t)(tile.first + u * tile.step) * kVec;
        if (c >= shape.cats) continue;
        if constexpr (kCkpt) {
          code[u] = load_codes<kVec>(ckpt.codes + r * pitch + c);
          unit[u] = ckpt.scales[r * blocks + c / kCkptBlock];
        } else if constexpr (kUnit) raw[u] = load_group(row, c, shape.cats);
        else raw[u] = gather_group(row, c, shape.cats, x.stride_cat);
      }
    };
    request();

    float total = 0.f;
    GradSlot own[2] = {{-1, 0.f}, {-1, 0.f}};   // slots lane and 64 + lane
    if (slots && per <= 4) {
      float sum = 0.f;
#pragma unroll
      for (int h = 0; h < 2; ++h)
        if (64 * h + lane < slots) {
          bool past;
          own[h] = grad_slot(in, r, e, v, 64 * h + lane, shape.cats, past);
          sum += past ? NAN : own[h].at >= 0 ? own[h].by : 0.f;
        }
      total = over_lanes<64>(sum, Sum());
    } else if (slots) {
      const int64_t r0 = job * per;   // (one segment a row)
      for (int i = threadIdx.x; i < per * slots; i += kTileThreads) {
        const int64_t q = r0 + i / slots;
        GradSlot s{-1, 0.f};
        if (q < rows) {
          bool past;
          const int64_t qe = shape.vars == 1 ? q : (uint32_t)q / (uint32_t)shape.vars;
          s = grad_slot(in, q, qe, q - qe * shape.vars, i % slots, shape.cats, past);
          if (past) s = {-2, 0.f};
        }
        slot_lds[i] = s;
      }
      __syncthreads();
      for (int j = 0; j < slots; ++j) {
        const GradSlot s = slot_lds[of * slots + j];
        total += s.at >= 0 ? s.by : s.at == -2 ? NAN : 0.f;
      }
    }
    const GradRow grad(in, r, total);
    const bool add = slots && !grad.none();
    for (int turn = 0;; ++turn) {
#pragma unroll
      for (int u = 0; u < kTileGroups; ++u) {
        const int64_t c = (int64_t)(tile.first + u * tile.step) * kVec;
        uint64_t here[2] = {0, 0};     // slots in the wave's part of the row (asked by all of its lanes)
        if (add && per <= 4) {
          const uint32_t c0 = (uint32_t)__builtin_amdgcn_readfirstlane((int)c);
#pragma unroll
          for (int h = 0; h < 2; ++h) here[h] = __ballot((uint32_t)own[h].at - c0 < (uint32_t)(64 * kVec));
        }
        if (c >= shape.cats) continue;
        float y[kVec];
        if constexpr (kCkpt) decode(code[u], block_unit(unit[u]), y);
        else unpack(raw[u], y, T());
#pragma unroll
        for (int i = 0; i < kVec; ++i) y[i] = grad.template at<kEnt>(y[i]);
        auto add_slot = [&](int at, float by) {
          const uint32_t i = (uint32_t)at - (uint32_t)c;
          if (i < (uint32_t)kVec)
#pragma unroll
            for (int k = 0; k < kVec; ++k) y[k] += i == (uint32_t)k ? by : 0.f;
        };
        if constexpr (kInLds) {
#pragma unroll
          for (int i = 0; i < kVec; ++i) grad_lds[of * width + (int)c + i] = y[i];
          continue;
        }
        if (per <= 4) {
#pragma unroll
          for (int h = 0; h < 2; ++h)
            for (uint64_t left = here[h]; left; left &= left - 1) {
              const int j = __builtin_ctzll(left);
              add_slot(__builtin_amdgcn_readlane(own[h].at, j), as_float(__builtin_amdgcn_readlane(__builtin_bit_cast(int, own[h].by), j)));
            }
        } else if (add)
          for (int j = 0; j < slots; ++j) add_slot(slot_lds[of * slots + j].at, slot_lds[of * slots + j].by);
        T w[kVec];
#pragma unroll
        for (int i = 0; i < kVec; ++i) w[i] = from_float<T>(y[i]);
        if (mine) {
          if constexpr (kUnit) store_group(dst, c, shape.cats, w);
          else scatter_group(dst, c, shape.cats, out.stride_cat, w);
        }
      }
      if constexpr (kInLds) {
        __syncthreads();
        if (add && (threadIdx.x & ((1 << tiles.lanes_log2) - 1)) == 0)
          for (int j = 0; j < slots; ++j) {
            const GradSlot s = slot_lds[of * slots + j];
            if (s.at >= 0) grad_lds[of * width + s.at] += s.by;
          }
        __syncthreads();
#pragma unroll
        for (int u = 0; u < kTileGroups; ++u) {
          const int64_t c = (int64_t)(tile.first + u * tile.step) * kVec;
          if (c >= shape.cats || !mine) continue;
          T w[kVec];
#pragma unroll
          for (int i = 0; i < kVec; ++i) w[i] = from_float<T>(grad_lds[of * width + (int)c + i]);
          if constexpr (kUnit) store_group(dst, c, shape.cats, w);
          else scatter_group(dst, c, shape.cats, out.stride_cat, w);
        }
      }
      if (turn + 1 == tiles.turns) break;
      tile.first += kTileGroups * tile.step;
      request();
    }
    if (slots && per > 4) __syncthreads();   // (the next rows' slots go where these are read)
  }
}

// Rows that lie side by side, in or out, a lane per row: 64 of them a wave, the categories cut among waves.  Slots are looked up per entry,
// the first four from registers.  65536 rows of 256 f32: 33 us from scores, 22 from codes (26 and 21 as rows of neighbours).
template <typename T, bool kCkpt>
__global__ __launch_bounds__(256) void grad_column_kernel(RowsRef x, CkptRef ckpt, RowsShape shape, GradIn in, RowsRef out, int parts, int len,
                                                          bool examples_first) {
  constexpr int kNear = 4, kStep = 8;
  const int lane = threadIdx.x & 63;
  const int64_t rows = shape.rows(), jobs = (rows + 63) / 64 * parts;
  const int slots = in.given.slots + in.top;
  const int64_t pitch = (shape.cats + 15) / 16 * 16, blocks = (shape.cats + kCkptBlock - 1) / kCkptBlock;
  for (int64_t job = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); job < jobs; job += (int64_t)gridDim.x * 4) {
    const int64_t set = job / parts;
    const int first = (int)(job - set * parts) * len, end = min(first + len, shape.cats);
    const int64_t at = set * 64 + lane;
    if (at >= rows) continue;
    const RowAt n = row_at(shape, (uint32_t)at, examples_first);
    const int64_t e = n.e, v = n.v, r = n.r;
    const T* const row = static_cast<const T*>(x.p) + e * x.stride_ex + v * x.stride_var;
    T* const dst = static_cast<T*>(const_cast<void*>(out.p)) + e * out.stride_ex + v * out.stride_var;
    GradSlot near[kNear];
    float total = 0.f;
#pragma unroll
    for (int j = 0; j < kNear; ++j) near[j] = {-1, 0.f};
    for (int j = 0; j < slots; ++j) {
      bool past;
      const GradSlot s = grad_slot(in, r, e, v, j, shape.cats, past);
      total += past ? NAN : s.at >= 0 ? s.by : 0.f;
#pragma unroll
      for (int k = 0; k < kNear; ++k)
        if (j == k) near[k] = s;
    }
    const GradRow grad(in, r, total);
    for (int c0 = first; c0 < end; c0 += kStep) {
      float y[kStep];
      if constexpr (kCkpt) {             // (c0 is a multiple of 8, the codes' pitch of 16)
        const Codes<kStep> code = load_codes<kStep>(ckpt.codes + r * pitch + c0);
        const BlockUnit unit = block_unit(ckpt.scales[r * blocks + c0 / kCkptBlock]);
#pragma unroll
        for (int i = 0; i < kStep; ++i) y[i] = block_entry_or_mask(unit, code[i]);
      } else {
#pragma unroll
        for (int i = 0; i < kStep; ++i) y[i] = c0 + i < end ? seen(row[(int64_t)(c0 + i) * x.stride_cat]) : -INFINITY;
      }
#pragma unroll
      for (int i = 0; i < kStep; ++i) {
        const int c = c0 + i;
        if (c >= end) break;
        float g = grad.template at<true>(y[i]);
        if (!grad.none()) {
#pragma unroll
          for (int j = 0; j < kNear; ++j) g += near[j].at == c ? near[j].by : 0.f;
          for (int j = kNear; j < slots; ++j) {
            bool past;
            const GradSlot s = grad_slot(in, r, e, v, j, shape.cats, past);
            g += s.at == c ? s.by : 0.f;
          }
        }
        dst[(int64_t)c * out.stride_cat] = from_float<T>(g);
      }
    }
  }
}

template <typename T>
void launch_grad(const RowsRef& x, const CkptRef& ckpt, const RowsShape& shape, const GradIn& in, const RowsRef& out, hipStream_t stream) {
  const int slots = in.given.slots + in.top;
  const bool unit = out.stride_cat == 1 && (ckpt.codes || x.stride_cat == 1);
  if (unit || !(side_by_side(out, shape) || (!ckpt.codes && side_by_side(x, shape)))) {
    const Tiles t = tiles_of(shape, 16 / (int)sizeof(T), (slots * kTileThreads + kStaged - 1) / kStaged, 8192);
    const bool in_lds = sizeof(T) == 4 && t.lanes_log2 < 6 && shape.cats > kLdsCats && slots > kFewSlots, ent = in.grad_entropy != nullptr;
    const int lds = in_lds ? kTileThreads * kTileGroups * (16 / (int)sizeof(T)) * 4 : 0;
    auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, tile_grid(t), dim3(kTileThreads), lds, stream, x, ckpt, shape, in, out, t); };
    auto choose = [&](auto keep) {
      constexpr bool kCkpt = decltype(keep)::value;
      if constexpr (sizeof(T) == 4)
        if (in_lds) return unit ? launch(grad_tile_kernel<T, kCkpt, true, true, true>) : launch(grad_tile_kernel<T, kCkpt, true, false, true>);
      if (!unit) launch(grad_tile_kernel<T, kCkpt, true, false, false>);
      else ent ? launch(grad_tile_kernel<T, kCkpt, true, true, false>) : launch(grad_tile_kernel<T, kCkpt, false, true, false>);
    };
    ckpt.codes ? choose(std::true_type()) : choose(std::false_type());
    return;
  }
  const int64_t sets = (shape.rows() + 63) / 64;
  const bool examples_first = examples_side_by_side(out, shape);
  int64_t parts = std::max<int64_t>(1, std::min<int64_t>((shape.cats + 31) / 32, (8192 + sets - 1) / sets));
  const int len = (int)(((shape.cats + parts - 1) / parts + 7) / 8 * 8);
  parts = (shape.cats + len - 1) / len;
  const dim3 grid((unsigned)std::min<int64_t>((sets * parts + 3) / 4, 1 << 22));
  auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(256), 0, stream, x, ckpt, shape, in, out, (int)parts, len, examples_first); };
  ckpt.codes ? launch(grad_column_kernel<T, true>) : launch(grad_column_kernel<T, false>);
}
}  // namespace

void category_scores_backward(const RowsRef& x_in, const CkptRef& ckpt, const RowsShape& shape, const GivenRef& given,
                              const float* d_grad_logp, int top, const int32_t* d_top, const float* d_grad_top,
                              const float* d_log_sum, const float* d_entropy, const float* d_grad_entropy, const RowsRef& out_in,
                              hipStream_t stream) {
  RowsRef x = x_in, out = out_in;
  check_rows(out, shape, "gradient of scores");
  check_given(given);
  if (top < 0 || top > kMaxSlots) fail(PCM_ERR_UNSUPPORTED, "0 to %d likeliest categories, got %d", kMaxSlots, top);
  if (!ckpt.codes != !ckpt.scales) fail(PCM_ERR_ARG, "a checkpoint needs both its codes and its scales");
  if (!ckpt.codes == !x.p && shape.examples) fail(PCM_ERR_ARG, "gradient of scores: either the scores or their checkpoint");
  if (x.p && x.dtype != out.dtype) fail(PCM_ERR_ARG, "gradient of scores: type %d for scores of type %d", out.dtype, x.dtype);
  if (!shape.examples) return;
  if (!out.p || !d_log_sum || (given.slots && !d_grad_logp) || (top && (!d_top || !d_grad_top)) || (d_grad_entropy && !d_entropy))
    fail(PCM_ERR_ARG, "gradient of scores: a pointer is null");
  if ((uintptr_t)ckpt.codes & 15) fail(PCM_ERR_ARG, "gradient of scores: codes must be 16-byte aligned");
  if (shape.cats == 1) x.stride_cat = out.stride_cat = 1;
  const GradIn in{given, d_grad_logp, top, d_top, d_grad_top, d_log_sum, d_entropy, d_grad_entropy};
  if (out.dtype == PCM_F32) launch_grad<float>(x, ckpt, shape, in, out, stream);
  else if (out.dtype == PCM_BF16) launch_grad<bf16>(x, ckpt, shape, in, out, stream);
  else launch_grad<f16>(x, ckpt, shape, in, out, stream);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) fail(PCM_ERR_HIP, "launch of category_scores_backward failed: %s", hipGetErrorString(e));
}

}  // namespace pcm
