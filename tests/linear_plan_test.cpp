// Host test of csrc/linear_plan.hpp: how the work of scores from features and weights is cut.  Prints one line per case: "<name> <value>".
#include <cstdio>

#include "linear_plan.hpp"

using namespace pcm;

int main() {
  // launches over rows of tiles, and over tiles of 32 categories, at the largest sizes that the entry points take and at powers of two below
  const struct { int64_t bm, bn; int threads; } tiles[] = {{256, 256, 512}, {128, 128, 256}, {128, 64, 256}, {128, 32, 256}};
  int none = 0, past = 0, several = 0;
  for (const auto& t : tiles)
    for (int64_t cats = (int64_t)1 << 30; cats; cats /= 2)
      for (int64_t rows = (int64_t)1 << 22; rows; rows /= 2) {
        const int64_t tiles_m = (cats + t.bm - 1) / t.bm, tiles_n = (rows + t.bn - 1) / t.bn, most = units_a_launch(tiles_m, t.threads);
        none += most < 1;
        past += std::min(most, tiles_n) * tiles_m * t.threads >= (int64_t)1 << 32;
        several += most < tiles_n;
      }
  std::printf("tiles_none %d\ntiles_past %d\ntiles_several %d\n", none, past, several);
  std::printf("few_512 %lld\nfew_256 %lld\n", (long long)units_a_launch(1, 512), (long long)units_a_launch(1, 256));
  std::printf("few_past %d\n", units_a_launch(1, 512) * 512 >= (int64_t)1 << 32 || units_a_launch(1, 256) * 256 >= (int64_t)1 << 32);
}
