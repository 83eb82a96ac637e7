// How the work of linear_scores.hip, linear_gradient.hip, product_out.hip and lay_out.hip is cut: rules on sizes alone, without HIP.
#pragma once

#include <algorithm>
#include <cstdint>

namespace pcm {

// Whether a product is best cut into tiles of 256 x 256, a workgroup's work a compute unit: enough of them, and long enough sums.  Short ones wait for
// their first fragments and for their stores one after the other, which two workgroups of 128 x 128 do in turns (32768 x 768 over 128 f16: 42 us, 35).
inline bool wide_tiles(int64_t m, int64_t n, int64_t steps) {
  return n > 64 && steps >= 12 && ((m + 255) / 256) * ((n + 255) / 256) >= 192;
}

// HIP takes fewer than 2^32 threads along an axis of a grid
inline int64_t most_blocks(int threads) { return (((int64_t)1 << 32) - 1) / threads; }
// How many units of `blocks` workgroups each one launch takes: further ones go into launches of their own
inline int64_t units_a_launch(int64_t blocks, int threads) { return most_blocks(threads) / blocks; }

// Gradients go in pieces of the categories, and many rows in parts, so that the workspace does not grow with either: a part's derivatives of a
// piece take up to kMostDerivatives entries, the piece's weights that are laid out up to 2^30, and those whose sums wait for further parts 2^28.
// What smaller ones cost: 40 x 16384 x 140000 bf16 in pieces of 2^28 weights 8.4 ms, at once 7.0; 100000 x 256 x 8192 f16 in two parts 3.7
// ms, at once 3.5.
constexpr int64_t kMostDerivatives = (int64_t)1 << 29, kLeastPiece = 4096;
// The most categories of a piece: 2^26 derivatives or so, kLeastPiece categories at least and 2^20 at most, but no more than the weights say (256 at least).
// laid: the piece's weights are laid out
inline int64_t most_piece(int64_t rows, int64_t length, bool laid) {
  const int64_t most = std::min<int64_t>((int64_t)1 << 20, std::max<int64_t>(kLeastPiece, ((int64_t)1 << 26) / rows / 256 * 256));
  const bool waits = rows > kMostDerivatives / kLeastPiece;
  return waits || laid ? std::min(most, std::max<int64_t>(256, ((int64_t)1 << (waits ? 28 : 30)) / length / 256 * 256)) : most;
}
// Rows of a part, whole examples of `vars` rows: all of them, or as many as there is room for, in multiples of 64
inline int64_t part_rows(int64_t rows, int64_t vars, int64_t piece) {
  if (rows * piece <= kMostDerivatives) return rows;
  int64_t each = vars;
  while (each % 64) each *= 2;
  return std::min(rows, std::max(each, kMostDerivatives / piece / each * each));
}

}  // namespace pcm
