// Products of caifx_rows.hpp in fp16.
#include "caifx_rows.hpp"

namespace caifx {

int rows_f16(const RowsArgs &g, int weight, int weights, bool direct, hipStream_t s)
{
  if (weight == ROWS_MX) return weights == 2 ? rows_pick<f16_t, ROWS_MX, 2>(g, 1, direct, s) : rows_pick<f16_t, ROWS_MX, 1>(g, 1, direct, s);
  return weights == 2 ? rows_pick<f16_t, ROWS_DENSE, 2>(g, 1, direct, s) : rows_pick<f16_t, ROWS_DENSE, 1>(g, 1, direct, s);
}

}  // namespace caifx
