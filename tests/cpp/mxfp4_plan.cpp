// Prints which forms products over 4-bit weights and gated blocks run in, for calls read from stdin, one a line.
//   0 rows columns reduction kind weights pieces direct: the row kernels; row tile, column tiles, workgroups that share a reduction
//   1 rows columns reduction gated: the dense product, with the columns of one weight and the steps of all operand pairs; tile's rows, tile's columns, workgroups
#include "caifx_rows_plan.hpp"
#include "caifx_wide_plan.hpp"

#include <cstdio>

using namespace caifx;

int main()
{
  int which;
  while (std::scanf("%d", &which) == 1) {
    long long M, C, R;
    if (std::scanf("%lld %lld %lld", &M, &C, &R) != 3) return 1;
    if (which == 0) {
      int kind, weights, pieces, direct;
      if (std::scanf("%d %d %d %d", &kind, &weights, &pieces, &direct) != 4) return 1;
      const long long blocks = (R + 31) / 32;
      const RowsPlan p = rows_plan_of(kind, weights, pieces, direct != 0, M, C, R, blocks, kind == ROWS_DENSE ? 2 * R : 16 * blocks);
      std::printf("%d %d %d\n", rows_tile(M, pieces), rows_column_tiles(p.span, weights), p.splits);
    } else {
      int gated;
      if (std::scanf("%d", &gated) != 1) return 1;
      const int parts = gated ? 1 : wide_parts(M, C, R).parts, tile = best_tile(M, gated ? 2 * C : C, 0, parts);
      std::printf("%d %d %d\n", tile == TILE_256 ? 256 : 128, tile == TILE_128 ? 128 : 256, parts);
    }
  }
  return 0;
}
