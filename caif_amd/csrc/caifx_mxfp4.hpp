// Operands laid out for the products over microscaled 4-bit weights: dense copies of a weight, activations in the row kernels' order.
#pragma once

#include "caifx_rows.hpp"

namespace caifx {

// what a source holds: a caifx_dtype, or codes and scales
enum { OPERAND_MX = 100 };

// [rows, cols] as dense values of `to` (16-bit), row n at out + n * stride + first, zeros from column cols to pitch (a multiple of 8, as are
// stride and first)
int operand_dense(const void *p, const void *scales, int kind, int64_t rows, int64_t cols, int to, void *out, int64_t pitch, int64_t stride, int64_t first,
                  hipStream_t s);
// transposed: value (n, k) at out[k * stride + first + n], zeros for n from rows to pitch (a multiple of 64)
int operand_transposed(const void *p, const void *scales, int kind, int64_t rows, int64_t cols, int to, void *out, int64_t pitch, int64_t stride, int64_t first,
                       hipStream_t s);
// activations for rows_bf16 / rows_f16 with packed operands, `to` CAIFX_F32: three bf16 pieces (kind CAIFX_F32 or CAIFX_F16 then); chunk0: where the
// source's chunks begin among `chunks`
int operand_rows(const void *p, int kind, int64_t rows, int64_t cols, int to, void *out, int chunk0, int chunks, hipStream_t s);

// y[M, C] = A B^T of two operands in microscaled 4 bits with `blocks` blocks a row, in tiles for the matrix cores.  The workspace is for the
// scales in another order.
bool mx_gemm_takes(int64_t M, int64_t C, int64_t blocks);
double mx_gemm_us(int64_t M, int64_t C, int64_t blocks);      // an estimate
size_t mx_gemm_workspace_bytes(int64_t M, int64_t C, int64_t blocks);
int mx_gemm(int64_t M, int64_t C, int64_t blocks, const void *a, const void *sa, const void *b, const void *sb, void *d, int d_dtype, void *workspace, hipStream_t s);

int gating_backward(const void *grad, const void *gate, const void *up, void *grad_gate, void *grad_up, int64_t n, int dtype, hipStream_t s);

}  // namespace caifx
