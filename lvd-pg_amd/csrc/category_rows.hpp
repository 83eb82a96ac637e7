// Rows of category scores: what the kernels of category_scores.hip, category_grad.hip and checkpoint_rows.hip share.
//
// A row is the scores x[0..C) of C categories; rows are addressed as [example][variable] with element strides.  Types:
// float, bfloat16, half (PCM_F32, PCM_BF16, PCM_F16); every sum is held in float.
#pragma once

#include "common.hpp"

namespace pcm {

constexpr int kMaxSlots = 64;         // most given categories, and most likeliest ones, of a row
constexpr int kCkptBlock = 64;        // neighbours of a row that share a scale
constexpr int kCkptMasked = 255;      // the code of an entry of -inf

struct RowsRef {                      // rows of scores (or of a gradient) in device memory
  const void* p;
  int dtype;
  int64_t stride_ex, stride_var, stride_cat;
};
struct RowsShape {
  int64_t examples;
  int32_t vars, cats;
  __host__ __device__ int64_t rows() const { return examples * vars; }
};
struct GivenRef {                     // categories per row, [example][variable][slot]
  const void* p;
  int type;                           // PCM_U8, PCM_I32, PCM_I64
  int64_t stride_ex, stride_var, stride_slot;
  int32_t slots;
  int32_t vars = 1;                   // for a kernel that takes examples and variables as one axis: the latter's number
};
struct CkptRef {                      // codes [rows][pitch], scales [rows][blocks]
  uint8_t* codes;
  uint32_t* scales;
};
// Rows that lie side by side: one entry apart from example to example or from variable to variable
inline bool examples_side_by_side(const RowsRef& x, const RowsShape& shape) { return shape.vars > 1 && (x.stride_ex == 1 || x.stride_ex == -1); }
inline bool side_by_side(const RowsRef& x, const RowsShape& shape) {
  return examples_side_by_side(x, shape) || (shape.examples > 1 && (x.stride_ex == 1 || x.stride_ex == -1)) ||
         (shape.vars > 1 && (x.stride_var == 1 || x.stride_var == -1));
}
inline int64_t ckpt_blocks(int64_t cats) { return (cats + kCkptBlock - 1) / kCkptBlock; }

int64_t category_scores_workspace(const RowsShape& shape, int top);
void category_scores(const RowsRef& x, const RowsShape& shape, const GivenRef& given, int top, float* d_logp, float* d_log_sum,
                     float* d_entropy, float* d_top_logp, int32_t* d_top, const CkptRef& ckpt, void* d_work, int64_t work_bytes,
                     hipStream_t stream);
void category_scores_backward(const RowsRef& x, const CkptRef& ckpt, const RowsShape& shape, const GivenRef& given,
                              const float* d_grad_logp, int top, const int32_t* d_top, const float* d_grad_top,
                              const float* d_log_sum, const float* d_entropy, const float* d_grad_entropy, const RowsRef& out,
                              hipStream_t stream);
void checkpoint_rows(const RowsRef& x, const RowsShape& shape, const CkptRef& ckpt, hipStream_t stream);
void restore_rows(const CkptRef& ckpt, const RowsShape& shape, const RowsRef& out, hipStream_t stream);
// refusals that the four share
void check_rows(const RowsRef& x, const RowsShape& shape, const char* what);
void check_given(const GivenRef& given);

#ifdef __HIPCC__
// ---- device side ------------------------------------------------------------------------------------------------

// (by value: a bit cast of a vector's element takes the vector's first one)
__device__ __forceinline__ float as_float(uint32_t v) { return __builtin_bit_cast(float, v); }
template <typename T>
__device__ __forceinline__ float to_float(T v) { return (float)v; }
template <typename T>
__device__ __forceinline__ T from_float(float v) { return (T)v; }   // round to nearest, ties to even

typedef __bf16 bf16;
typedef _Float16 f16;
typedef uint32_t raw4 __attribute__((ext_vector_type(4)));

// 16 bytes of a row at an address that is aligned to its entries only
typedef raw4 raw4_by4 __attribute__((aligned(4)));
typedef raw4 raw4_by2 __attribute__((aligned(2)));
template <typename T>
__device__ __forceinline__ raw4 load16(const T* p) {
  if constexpr (sizeof(T) == 4) return *reinterpret_cast<const raw4_by4*>(p);
  else return *reinterpret_cast<const raw4_by2*>(p);
}
template <typename T>
__device__ __forceinline__ void store16(T* p, raw4 v) {
  if constexpr (sizeof(T) == 4) *reinterpret_cast<raw4_by4*>(p) = v;
  else *reinterpret_cast<raw4_by2*>(p) = v;
}

// Entry `slot` of a row's given categories, whatever their type; negative: not observed.
__device__ __forceinline__ int64_t given_at(const GivenRef& g, int64_t e, int64_t v, int slot) {
  const int64_t at = e * g.stride_ex + v * g.stride_var + slot * g.stride_slot;
  if (g.type == PCM_U8) return static_cast<const uint8_t*>(g.p)[at];
  if (g.type == PCM_I32) return static_cast<const int32_t*>(g.p)[at];
  return static_cast<const int64_t*>(g.p)[at];
}

// Order of floats as whole numbers (NaN aside), and back
__device__ __forceinline__ uint32_t float_order(float x) {
  const uint32_t b = __builtin_bit_cast(uint32_t, x);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float order_float(uint32_t o) {
  return __builtin_bit_cast(float, o & 0x80000000u ? o & 0x7fffffffu : ~o);
}

// Order of entries, likeliest first: larger value, then smaller index (the two zeros are one value).  0 is below them all.
__device__ __forceinline__ uint64_t entry_key(float x, uint32_t index) {
  return (uint64_t)float_order(x + 0.f) << 32 | (uint32_t)~index;
}
__device__ __forceinline__ float key_value(uint64_t k) {
  return order_float((uint32_t)(k >> 32));
}
__device__ __forceinline__ int32_t key_index(uint64_t k) { return (int32_t) ~(uint32_t)k; }

// ---- lanes of a wave --------------------------------------------------------------------------------------------
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

template <int kCtrl>
__device__ __forceinline__ float dpp(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), kCtrl, 0xf, 0xf, false));
}
// f over the lanes of groups of N (4, 8, 16 or 64) neighbours, in all of them; every lane is active
template <int N, typename F>
__device__ __forceinline__ float over_lanes(float v, F f) {
  v = f(v, dpp<0xB1>(v));                       // the neighbour
  v = f(v, dpp<0x4E>(v));                       // the next pair
  if (N >= 8) v = f(v, dpp<0x141>(v));          // mirrored in eight
  if (N >= 16) v = f(v, dpp<0x140>(v));         // mirrored in sixteen
  if (N >= 64) {
    auto h = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(uint32_t, v), __builtin_bit_cast(uint32_t, v), false, false);
    v = f(as_float(h[0]), as_float(h[1]));
    auto w = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, v), __builtin_bit_cast(uint32_t, v), false, false);
    v = f(as_float(w[0]), as_float(w[1]));
  }
  return v;
}
struct Larger { __device__ float operator()(float a, float b) const { return fmaxf(a, b); } };
struct Smaller { __device__ float operator()(float a, float b) const { return fminf(a, b); } };
struct LargerOrNan { __device__ float operator()(float a, float b) const { return __builtin_elementwise_maximum(a, b); } };
struct SmallerOrNan { __device__ float operator()(float a, float b) const { return __builtin_elementwise_minimum(a, b); } };
struct Sum { __device__ float operator()(float a, float b) const { return a + b; } };

// the value of lane ^ J
template <int J>
__device__ __forceinline__ uint32_t lane_xor(uint32_t v) {
  const int b = (int)v;
  if (J == 1) return __builtin_amdgcn_mov_dpp(b, 0xB1, 0xf, 0xf, false);
  if (J == 2) return __builtin_amdgcn_mov_dpp(b, 0x4E, 0xf, 0xf, false);
  if (J == 4)                                    // four up for the even quads, four down for the odd ones
    return __builtin_amdgcn_update_dpp(__builtin_amdgcn_update_dpp(b, b, 0x104, 0xf, 0x5, false), b, 0x114, 0xf, 0xa, false);
  if (J == 8) return __builtin_amdgcn_mov_dpp(b, 0x128, 0xf, 0xf, false);
  const bool low = !((threadIdx.x & 63) & J);
  if (J == 16) {
    auto h = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return low ? h[1] : h[0];
  }
  auto h = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return low ? h[1] : h[0];
}
template <int J>
__device__ __forceinline__ uint64_t lane_xor(uint64_t v) {
  return (uint64_t)lane_xor<J>((uint32_t)(v >> 32)) << 32 | lane_xor<J>((uint32_t)v);
}

// Bitonic sorts of groups of N neighbouring lanes: the step of merge size S whose pairs lie J apart.  Which lanes keep the larger
// value is a constant of the step, a mask that needs no comparison.
constexpr uint64_t larger_lanes(int N, int S, int J, bool falling) {
  uint64_t mask = 0;
  for (int lane = 0; lane < 64; ++lane) {
    bool f = falling;
    for (int n = N; n > S; n /= 2) f = !(lane & (n / 2)) == f;   // the two halves of a sort run against each other
    if (f == !(lane & J)) mask |= 1ull << lane;
  }
  return mask;
}
template <int N, int S, int J, bool kFalling, typename K>
__device__ __forceinline__ K sort_step(K v) {
  constexpr uint64_t larger = larger_lanes(N, S, J, kFalling);
  const K o = lane_xor<J>(v);
  return (v > o) == __builtin_amdgcn_inverse_ballot_w64(larger) ? v : o;
}
template <int N, int S, int J, bool kFalling, typename K>
__device__ __forceinline__ K sort_merge_steps(K v) {
  v = sort_step<N, S, J, kFalling>(v);
  if constexpr (J > 1) v = sort_merge_steps<N, S, J / 2, kFalling>(v);
  return v;
}
template <int N, int S, bool kFalling, typename K>
__device__ __forceinline__ K sort_sizes(K v) {
  if constexpr (S > 2) v = sort_sizes<N, S / 2, kFalling>(v);
  return sort_merge_steps<N, S, S / 2, kFalling>(v);
}
template <int N, bool kFalling, typename K>
__device__ __forceinline__ K sort_lanes(K v) { return sort_sizes<N, N, kFalling>(v); }
// the same of lanes that rise and then fall, or fall and then rise
template <int N, bool kFalling, typename K>
__device__ __forceinline__ K sort_merge(K v) { return sort_merge_steps<N, N, N / 2, kFalling>(v); }

// The largest entry that counts as masked: half of the type's lowest value (what adding a mask of the lowest value leaves).
template <typename T>
__device__ __forceinline__ float masked_from() { return -1.7014117e38f; }
template <>
__device__ __forceinline__ float masked_from<bf16>() { return -1.6947657e38f; }
template <>
__device__ __forceinline__ float masked_from<f16>() { return -32752.f; }
// a score with masks at -inf
template <typename T>
__device__ __forceinline__ float seen(T v) {
  const float x = to_float(v);
  return x <= masked_from<T>() ? -INFINITY : x;
}
// the entries of 16 bytes, scores with masks at -inf (f16: its masks lie within the range of the exponential)
__device__ __forceinline__ void unpack(raw4 r, float (&x)[4], float) {
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = as_float(r[i]);
}
__device__ __forceinline__ void unpack(raw4 r, float (&x)[8], bf16) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = as_float(r[i] << 16);
    x[2 * i + 1] = as_float(r[i] & 0xffff0000u);
  }
}
__device__ __forceinline__ void unpack(raw4 r, float (&x)[8], f16) {
  typedef f16 pair __attribute__((ext_vector_type(2)));
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t w = r[i];
    const pair h = __builtin_bit_cast(pair, w);
    x[2 * i] = seen(h[0]);
    x[2 * i + 1] = seen(h[1]);
  }
}
template <typename T>
__device__ __forceinline__ float type_max() { return 3.4028235e38f; }
template <>
__device__ __forceinline__ float type_max<bf16>() { return 3.3895314e38f; }
template <>
__device__ __forceinline__ float type_max<f16>() { return 65504.f; }

// The scale of a block of 64: entry = (base - code) 2^e, code 0..254.  e is the smallest exponent with 253 steps (254 between
// rounded ends) over the block's range where the range's mantissa allows, and with the largest entry within 2^14 steps, so that
// base fits 16 bits.  A power of two makes x 2^-e, its rounding and the product back exact: an entry is off by half a step
// at most, whoever computes it.  Word: base in bits 0..15, e + 127 in bits 16..23 (255 there: a block with NaN or +inf), bit 24: some
// code is 255, so that a block without it can be read without looking for them.
struct BlockScale {
  float inv, base;   // 2^-e, rint(max 2^-e)
  uint32_t word;
};
__device__ __forceinline__ BlockScale block_scale(float hi, float lo, bool masks, bool bad) {   // (hi < lo: no entry but masked ones)
  if (hi < lo) hi = lo = 0.f;
  const float r = 0.5f * hi - 0.5f * lo;   // halves: the difference itself may pass the range of float
  const float a = fmaxf(fabsf(hi), fabsf(lo));
  int e = -126;
  if (r > 0.f) e = max(e, __builtin_amdgcn_frexp_expf(r) - (__builtin_amdgcn_frexp_mantf(r) > 253.f / 256.f ? 6 : 7));
  if (a > 0.f) e = max(e, __builtin_amdgcn_frexp_expf(a) - 14);
  BlockScale s;
  s.inv = __builtin_bit_cast(float, (uint32_t)(127 - e) << 23);
  s.base = rintf(hi * s.inv);
  s.word = bad ? 0xff0000u : (uint32_t)(127 + e) << 16 | ((uint32_t)(int)s.base & 0xffffu) | (masks ? 1u << 24 : 0u);
  return s;
}
// base - rint(x 2^-e): adding 1.5 2^23 rounds the product, which is exact and below 2^14, to a whole number in the low bits
__device__ __forceinline__ uint32_t block_code(const BlockScale& s, float x) {
  return 0x4b400000u + (uint32_t)(int)s.base - __builtin_bit_cast(uint32_t, fmaf(x, s.inv, 12582912.f));
}
// Codes of the N entries that a lane holds of a block, which lies in 64 / N neighbouring lanes; every lane of the wave is active.
template <int N>
struct BlockCodes {
  uint32_t code[N / 4], word;
};
template <typename T, int N>
__device__ __forceinline__ BlockCodes<N> encode_block(const float (&y)[N]) {
  float hi = y[0], lo = y[0];
#pragma unroll
  for (int i = 1; i < N; ++i) {
    hi = __builtin_elementwise_maximum(hi, y[i]);
    lo = __builtin_elementwise_minimum(lo, y[i]);
  }
  hi = over_lanes<kCkptBlock / N>(hi, LargerOrNan());
  lo = over_lanes<kCkptBlock / N>(lo, SmallerOrNan());
  BlockCodes<N> out;
  if (!__any(!(lo > masked_from<T>() && hi < INFINITY))) {   // nothing masked, no NaN in any of the wave's blocks
    const BlockScale s = block_scale(hi, lo, false, false);
    out.word = s.word;
#pragma unroll
    for (int i = 0; i < N / 4; ++i)
      out.code[i] = block_code(s, y[4 * i]) | block_code(s, y[4 * i + 1]) << 8 | block_code(s, y[4 * i + 2]) << 16 | block_code(s, y[4 * i + 3]) << 24;
    return out;
  }
  float kept = INFINITY;
#pragma unroll
  for (int i = 0; i < N; ++i) kept = fminf(kept, y[i] > masked_from<T>() ? y[i] : INFINITY);
  kept = over_lanes<kCkptBlock / N>(kept, Smaller());
  const BlockScale s = block_scale(hi > masked_from<T>() ? hi : -INFINITY, kept, lo <= masked_from<T>(), !(hi < INFINITY));
  out.word = s.word;
#pragma unroll
  for (int i = 0; i < N / 4; ++i) out.code[i] = 0;
#pragma unroll
  for (int i = 0; i < N; ++i)
    out.code[i / 4] |= (y[i] <= masked_from<T>() ? (uint32_t)kCkptMasked : block_code(s, y[i]) & 0xffu) << (8 * (i % 4));
  return out;
}
// ... and where they go, for a lane whose entries begin at c of row r
template <int N>
__device__ __forceinline__ void store_codes(const CkptRef& ckpt, const BlockCodes<N>& k, int64_t r, int64_t c, int cats, int64_t pitch, int64_t blocks) {
  if (c >= pitch) return;
  uint8_t* const to = ckpt.codes + r * pitch + c;
  if constexpr (N == 4) *reinterpret_cast<uint32_t*>(to) = k.code[0];
  else *reinterpret_cast<uint2*>(to) = make_uint2(k.code[0], k.code[1]);
  if (c % kCkptBlock == 0 && c < cats) ckpt.scales[r * blocks + c / kCkptBlock] = k.word;
}

struct BlockUnit {
  float step, base;   // an entry is (base - code) step
  bool masks;
};
__device__ __forceinline__ BlockUnit block_unit(uint32_t word) {
  const uint32_t e = word >> 16 & 0xffu;
  const float step = e == 0xffu ? __builtin_nanf("") : __builtin_bit_cast(float, e << 23);
  return {step, (float)(int16_t)(word & 0xffffu), (word >> 24 & 1u) != 0};
}
// (base step alone may pass the range, an entry only by rounding the largest up)
__device__ __forceinline__ float block_entry(const BlockUnit& u, float code) { return (u.base - code) * u.step; }
__device__ __forceinline__ float block_entry_or_mask(const BlockUnit& u, float code) {
  return u.masks && code == (float)kCkptMasked ? -INFINITY : block_entry(u, code);
}
#endif

}  // namespace pcm
