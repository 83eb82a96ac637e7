// Scores of categories that are products of features and weights, x[n][c] = f[n] . w[c] + b[c]: what the kernels of linear_scores.hip,
// linear_gradient.hip, product8.hip and lay_out.hip share.
//
// Products of 16-bit types and of 8-bit codes run over rows that are neighbours along the summed axis, in pieces of 128 bytes
// (product_tiles.hip.hpp); rows that do not lie so (odd lengths, other strides, or summed along the other axis) are laid out in the
// workspace first (lay_out.hip).  Float is read where it is, as three bfloat16 parts (float_tiles.hip.hpp).
#pragma once

#include "category_rows.hpp"

namespace pcm {

constexpr int64_t kMaxLength = 1 << 20;      // entries of a row of features or weights
constexpr int64_t kMaxLinearRows = 1 << 22;  // rows of features (tokens)
constexpr int64_t kMaxLength8 = 131071;      // of 8-bit rows: so many products of -128 and -128 stay within 32 bits
constexpr int kKBytes = 128;                 // bytes of a row that a step of a product takes
constexpr int kDeadRow = -100000;            // the exponent of a row whose gradient is nothing

struct Matrix2 {                             // rows of a matrix in device memory, [example][variable][entry] (weights: vars = 1)
  const void* p;
  int type;                                  // PCM_F32, PCM_BF16, PCM_F16
  int64_t stride_ex, stride_var, stride;
  int64_t examples;
  int32_t vars, length;
  __host__ __device__ int64_t rows() const { return examples * vars; }
};
struct Operand {                             // rows that a product can read: 16-byte aligned, multiples of 128 bytes, zeros behind the end
  const void* p;
  int64_t pitch, plane;                      // bytes from row to row, and from plane to plane (numbers in two parts)
};
struct BiasRef {                             // a number per category; null: zeros
  const void* p;
  int type;
};
struct ScaleRef {                            // of 8-bit rows: scales of b's rows (n) and of a's rows (m); null: none
  const float *n, *m;
};

inline int64_t round_up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }
// entries of a laid out row: a multiple of 128 bytes of 16-bit entries
inline int64_t laid_length(int64_t length) { return round_up(length, kKBytes / 2); }
inline int64_t laid_bytes(int64_t rows, int64_t length, int planes) { return round_up(rows * laid_length(length) * 2 * planes, 256); }

// What laying out changes on the way: rows are scaled by powers of two (float exponents `expo` relative to the largest of `most`, if given;
// nothing of a row at kDeadRow), categories that the bias masks become zeros.
struct LayOut {
  const int* expo = nullptr;
  const int* most = nullptr;                 // 256 candidates of the largest exponent
  BiasRef mask{nullptr, 0};
};
// rows [first, first + count) of x, of a 16-bit type, as [row][laid_length(length)], or with `turned` as [entry][laid_length(count)]
void lay_out(const Matrix2& x, int64_t first, int64_t count, bool turned, const LayOut& with, void* d_to, hipStream_t stream);
// whether a product can read the rows where they are
bool readable(const Matrix2& x);

// what the entry points share
void check_linear(const Matrix2& f, const Matrix2& w, const BiasRef& bias, const GivenRef& given, const char* what);
void check_workspace(const void* d_work, int64_t work_bytes, int64_t need, const char* what);
Operand operand_of(const Matrix2& x, char*& work, hipStream_t stream);

int64_t linear_scores_workspace(const Matrix2& f, const Matrix2& w);
void linear_scores(const Matrix2& f, const Matrix2& w, const BiasRef& bias, const GivenRef& given, float* d_logp, float* d_log_sum,
                   void* d_work, int64_t work_bytes, hipStream_t stream);
int64_t linear_scores8_workspace(int64_t rows, int64_t cats, int32_t length);
void linear_scores8(const int8_t* f, const float* f_scales, int64_t examples, int32_t vars, const int8_t* w, const float* w_scales, int32_t cats,
                    int32_t length, const BiasRef& bias, const GivenRef& given, float* d_logp, float* d_log_sum, void* d_work, int64_t work_bytes,
                    hipStream_t stream);
struct LinearGradients {                     // results, each may be null
  void *features, *weight;                   // [rows][length], [cats][length], of the features' type
  void* bias;                                // [cats], of the bias's type
};
int64_t linear_scores_backward_workspace(const Matrix2& f, const Matrix2& w, bool of_features, bool of_weight, bool of_bias);
void linear_scores_backward(const Matrix2& f, const Matrix2& w, const BiasRef& bias, const GivenRef& given, const float* d_grad_logp,
                            const float* d_grad_log_sum, const float* d_log_sum, const LinearGradients& out, void* d_work, int64_t work_bytes,
                            hipStream_t stream);
void rows8(const Matrix2& x, int8_t* d_codes, float* d_scales, hipStream_t stream);
int64_t product8_workspace(int64_t rows, int64_t cats, int32_t length);
void product8(const int8_t* a, const float* a_scales, int64_t rows, const int8_t* b, const float* b_scales, int64_t cats, int32_t length,
              const BiasRef& bias, void* d_out, int type, int64_t pitch, void* d_work, int64_t work_bytes, hipStream_t stream);

#ifdef __HIPCC__
// The bias of category m with what masks it at -inf, and everything behind the last category
__device__ __forceinline__ float bias_at(const BiasRef& b, int64_t m, int64_t cats) {
  if (m >= cats) return -INFINITY;
  if (!b.p) return 0.f;
  if (b.type == PCM_F32) return seen(static_cast<const float*>(b.p)[m]);
  if (b.type == PCM_BF16) return seen(static_cast<const bf16*>(b.p)[m]);
  return seen(static_cast<const f16*>(b.p)[m]);
}
// a score: the product and the bias, -inf where the bias masks the category, whatever the product
__device__ __forceinline__ float score_of(float product, float bias) {
  return bias == -INFINITY ? -INFINITY : product + bias;
}
__device__ __forceinline__ int largest_exponent(const int* most) {   // by every lane of a wave
  const int lane = threadIdx.x & 63;
  int e = max(max(most[lane], most[lane + 64]), max(most[lane + 128], most[lane + 192]));
#pragma unroll
  for (int s = 32; s; s /= 2) e = max(e, __shfl_xor(e, s));
  return e;
}
template <typename T>
__device__ __forceinline__ uint32_t pair_of(float a, float b) {   // two of 16 bits
  typedef float two __attribute__((ext_vector_type(2)));
  typedef T pair __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((two{a, b}), pair));
}
#endif

}  // namespace pcm
