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

}  // namespace pcm
