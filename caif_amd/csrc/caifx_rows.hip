// Products of caifx_rows.hpp in bf16, also on the three bf16 pieces of fp32 activations, and of two operands in 4 bits.
#include "caifx_rows.hpp"

namespace caifx {

int rows_bf16(const RowsArgs &g, int weight, int weights, int pieces, bool direct, hipStream_t s)
{
  if (weight == ROWS_MX) return weights == 2 ? rows_pick<bf16_t, ROWS_MX, 2>(g, pieces, direct, s) : rows_pick<bf16_t, ROWS_MX, 1>(g, pieces, direct, s);
  return weights == 2 ? rows_pick<bf16_t, ROWS_DENSE, 2>(g, pieces, direct, s) : rows_pick<bf16_t, ROWS_DENSE, 1>(g, pieces, direct, s);
}

int rows_both(const RowsArgs &g, hipStream_t s)
{
  switch (rows_tile(g.M, 1)) {
    case 16: return rows_pick_columns<bf16_t, 1, ROWS_BOTH, 1, 1, 0>(g, s);
    case 32: return rows_pick_columns<bf16_t, 1, ROWS_BOTH, 1, 2, 0>(g, s);
    default: return rows_pick_columns<bf16_t, 1, ROWS_BOTH, 1, 4, 0>(g, s);
  }
}

}  // namespace caifx
