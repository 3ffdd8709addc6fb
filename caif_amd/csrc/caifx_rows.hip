// Products of caifx_rows.hpp in bf16, also on the three bf16 pieces of fp32 activations.
#include "caifx_rows.hpp"

namespace caifx {

int rows_bf16(const RowsArgs &g, int weight, int weights, int pieces, bool direct, hipStream_t s)
{
  if (weight == ROWS_MX) return weights == 2 ? rows_pick<bf16_t, ROWS_MX, 2>(g, pieces, direct, s) : rows_pick<bf16_t, ROWS_MX, 1>(g, pieces, direct, s);
  return weights == 2 ? rows_pick<bf16_t, ROWS_DENSE, 2>(g, pieces, direct, s) : rows_pick<bf16_t, ROWS_DENSE, 1>(g, pieces, direct, s);
}

}  // namespace caifx
