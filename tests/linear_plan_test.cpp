// Host test of csrc/linear_plan.hpp: how the work of scores from features and weights is cut.  Prints one line per case: "<name> <value>".
// With arguments m n steps: whether such a product goes by tiles of 256 x 256.  With rows length: the most categories of a piece.
#include <cstdio>
#include <cstdlib>

#include "linear_plan.hpp"

using namespace pcm;

int main(int argc, char** argv) {
  if (argc == 4) return std::printf("wide %d\n", wide_tiles(std::atoll(argv[1]), std::atoll(argv[2]), std::atoll(argv[3]))), 0;
  if (argc == 3) return std::printf("piece %lld\n", (long long)most_piece(std::atoll(argv[1]), std::atoll(argv[2]), true)), 0;
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
  // pieces of the categories and parts of the rows
  int uneven = 0, large = 0, many = 0;
  for (int64_t rows = 1; rows <= (int64_t)1 << 22; rows += rows < 100 ? 1 : rows / 3)
    for (int64_t vars : {1, 3, 64, 100, 1000})
      for (int64_t length = 1; length <= (int64_t)1 << 20; length *= 4)
        for (bool laid : {false, true}) {
          if (rows % vars) continue;
          const int64_t piece = most_piece(rows, length, laid), part = part_rows(rows, vars, piece);
          uneven += piece < 256 || piece % 256 || part < 1 || part > rows || part % vars || (part < rows && part % 64);
          large += part * piece > kMostDerivatives && part > 64 * vars;
          large += laid && piece * length > (int64_t)1 << 30 && piece > 256;
          large += part < rows && piece * length > (int64_t)1 << 28 && piece > 256;
          many += part < rows;
        }
  std::printf("pieces_uneven %d\npieces_large %d\npieces_parts %d\n", uneven, large, many);
  std::printf("few_past %d\n", units_a_launch(1, 512) * 512 >= (int64_t)1 << 32 || units_a_launch(1, 256) * 256 >= (int64_t)1 << 32);
}
