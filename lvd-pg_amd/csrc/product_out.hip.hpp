// Products that are written out: the sums of a tile, finished and rounded to the result's type, or as they are into parts that a
// second launch joins.
#pragma once

#include "few_rows.hip.hpp"

namespace pcm {

enum { kRawSums = -1 };   // the type of parts: the sums themselves, 32 bits each

// What becomes of a sum of row m of a and row n of b
struct Finish {
  const int* dead = nullptr;     // 0 where it is kDeadRow (gradient of features)
  const int* expo = nullptr;     // 2^(expo[n] - 15) (gradient of features)
  const int* most = nullptr;     // 2^(the largest of most - 15) (gradient of weights)
  ScaleRef scale{nullptr, nullptr};
  BiasRef bias{nullptr, 0};      // of m
};
struct OutTask {
  Operand a, b;
  FloatOperand fa, fb;           // ... of float, of fk entries
  int64_t fk;
  int64_t m, n;
  Steps steps;
  void* out;                     // [n][pitch], entries of `type`; kRawSums: [part][n][pitch]
  int type;
  int64_t pitch;
  bool add;                      // to what the parts hold already
  Finish finish;
};

// launches of any size
void product_out(int operands, const OutTask& t, hipStream_t stream);   // operands: PCM_F32, PCM_BF16, PCM_F16, PCM_U8 (whole numbers)
// ... of 8-bit rows, a few of b (kFewRowsMost): t.a, t.b and t.steps as for product_out
void product_few(const OutTask& t, hipStream_t stream);
// ... of 16-bit types over one or two steps, in that type (short_sums), finished without scales and bias
bool short_sums(int operands, const OutTask& t);
void product_short(int operands, const OutTask& t, hipStream_t stream);
// out = the finished sums of parts [parts][n][m] floats (or whole numbers)
void join_parts(const void* parts, int count, bool whole, int64_t m, int64_t n, const Finish& finish, void* out, int type, int64_t pitch, hipStream_t stream);
// how many parts the summed axis of a product is best cut into
int parts_for(int64_t m, int64_t n, int64_t steps, bool of_float = false);
int parts_for_few(int64_t m, int64_t steps);   // ... of product_few

#ifdef __HIPCC__
struct FinishAt {                // of one n
  float scale;
  int expo;
  bool dead;
  __device__ __forceinline__ FinishAt(const Finish& f, int64_t n, int most) {
    expo = f.most ? most - 15 : f.expo ? f.expo[n] - 15 : 0;
    dead = f.dead && f.dead[n] == kDeadRow;
    scale = f.scale.n ? f.scale.n[n] : 1.f;
  }
  // scale_m, bias_m: of m
  __device__ __forceinline__ float operator()(float sum, float scale_m, float bias_m) const { return dead ? 0.f : ldexpf(sum * scale * scale_m, expo) + bias_m; }
};
__device__ __forceinline__ float bias_of(const BiasRef& b, int64_t m) {   // (a product's bias masks nothing)
  if (!b.p) return 0.f;
  return b.type == PCM_F32 ? static_cast<const float*>(b.p)[m] : b.type == PCM_BF16 ? (float)static_cast<const bf16*>(b.p)[m] : (float)static_cast<const f16*>(b.p)[m];
}
__device__ __forceinline__ void store_as(void* out, int type, int64_t at, float v) {
  if (type == PCM_F32) static_cast<float*>(out)[at] = v;
  else if (type == PCM_BF16) static_cast<bf16*>(out)[at] = (bf16)v;
  else static_cast<f16*>(out)[at] = (f16)v;
}
// four neighbours, the address a multiple of their size
__device__ __forceinline__ void store_four(void* out, int type, int64_t at, const float (&v)[4]) {
  if (type == PCM_F32) *reinterpret_cast<float4*>(static_cast<float*>(out) + at) = make_float4(v[0], v[1], v[2], v[3]);
  else if (type == PCM_BF16) *reinterpret_cast<uint2*>(static_cast<bf16*>(out) + at) = make_uint2(pair_of<bf16>(v[0], v[1]), pair_of<bf16>(v[2], v[3]));
  else *reinterpret_cast<uint2*>(static_cast<f16*>(out) + at) = make_uint2(pair_of<f16>(v[0], v[1]), pair_of<f16>(v[2], v[3]));
}
#endif

}  // namespace pcm
