// How the row kernels (caifx_rows.hpp) cut a call up (host only).
#pragma once

#include <cstdint>

namespace caifx {

enum { ROWS_MX = 0, ROWS_DENSE = 1, ROWS_BOTH = 2 };      // ROWS_BOTH: weight and activations in microscaled 4 bits

// How a launch is cut up: columns of a workgroup, workgroups that share a reduction.
struct RowsPlan {
  int span, splits;
};
// Rows of a workgroup's tile.
inline int rows_tile(int64_t M, int pieces) { return M <= 16 ? 16 : M <= 32 || pieces == 3 ? 32 : 64; }
// The time of a launch in us, fitted to 60 calls (1 to 64 rows, 1024 x 4096 to 8192 x 28672 and 14336 x 4096): a start, the rounds that a
// wave's units take, a compute unit's share of the weight at 20.7 KB a us (5.3 TB/s in all) and of the activations, which its caches
// serve, at 80; a shared reduction costs a second launch and the sums' way there and back.
inline double rows_us(double rows, double columns, double span, double splits, double units, double weight_row, double x_tile, double result)
{
  double rounds = rows * columns * splits / 256;
  rounds = rounds < 1 ? 1 : rounds;
  double turns = units / splits / 8;
  turns = turns < 1 ? 1 : turns;
  return 2.4 + rounds * (0.55 * turns + span * weight_row / splits / 20700 + x_tile / splits / 80000) + (splits > 1 ? 3.3 + splits * result * 8 / 4.0e6 : 0.0);
}
// A compute unit has some 100 lines on their way at a time whatever it asks for, so the launch is as fast as its fullest compute unit: the
// columns are cut into a multiple of 256 parts, as large as the column tiles allow.  Where that leaves a workgroup few columns, so that
// the activations are most of what it reads, 2 to 8 workgroups share a reduction of wider parts (N = 4096, K = 14336, 32 rows: 18 us in four,
// 20 in one; the estimates say where).  x_tile: bytes of the activations that a workgroup reads.
inline RowsPlan rows_plan(int64_t M, int64_t N, int64_t R, int weights, int pieces, double weight_row, double x_tile)
{
  const int tile = rows_tile(M, pieces);
  const int64_t rows = (M + tile - 1) / tile, most = (pieces == 3 && tile == 32 ? 32 : 64) / weights;      // (three pieces of 32 rows: two column tiles)
  const double units = static_cast<double>((R + 511) / 512);
  RowsPlan best{};
  double best_us = 0;
  for (int splits = 1; splits <= 8; splits *= 2) {
    if (splits > 1 && (weights > 1 || units < 4 * splits || rows * splits > 256)) break;
    // rounds of workgroups, as few as leave the columns in parts of at most `most`
    const int64_t least = (N + most - 1) / most, rounds = (least * rows * splits + 255) / 256;
    const int64_t parts = 256 * rounds / (rows * splits), span = (N + parts - 1) / parts;
    const double us = rows_us(static_cast<double>(rows), static_cast<double>((N + span - 1) / span), static_cast<double>(span), splits, units, weight_row, x_tile,
                              static_cast<double>(M) * static_cast<double>(N));
    if (splits == 1 || us < best_us) {
      best = RowsPlan{static_cast<int>(span), splits};
      best_us = us;
    }
  }
  return best;
}
// The same from what a weight row is: in 4 bits `blocks` blocks with their scales, dense w_pitch bytes.  direct: activations are read where they are, 16-bit
// ones or fp32 ones that a workgroup takes apart, otherwise packed in `pieces` pieces; up to four rows are not filled up to a tile then.
inline RowsPlan rows_plan_of(int kind, int weights, int pieces, bool direct, int64_t M, int64_t N, int64_t R, int64_t blocks, int64_t w_pitch)
{
  const double row = kind == ROWS_DENSE ? static_cast<double>(w_pitch) : 17.0 * static_cast<double>(blocks);
  const double x_row = kind == ROWS_BOTH ? row : (direct ? 2.0 + (pieces > 1 ? 2.0 : 0.0) : 2.0 * pieces) * static_cast<double>(R);
  return rows_plan(M, N, R, weights, pieces, row, x_row * (M <= 4 && (direct || pieces == 1) ? 4 : rows_tile(M, pieces)));
}
// Column tiles of the kernel that takes `span` columns of each weight: 1, 2 or 4 in all
inline int rows_column_tiles(int span, int weights)
{
  const int tiles = weights * ((span + 15) / 16);
  return tiles > 2 ? 4 : tiles;
}

}  // namespace caifx
