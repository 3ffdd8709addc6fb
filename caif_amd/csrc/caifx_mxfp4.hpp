// Operands laid out for the products over microscaled 4-bit weights: dense copies of a weight, activations in the row kernels' order.
#pragma once

#include "caifx_rows.hpp"

namespace caifx {

// what a source holds: a caifx_dtype, or codes and scales
enum { OPERAND_MX = 100 };

// one or two matrices [rows, cols] of one kind
struct Operand {
  const void *p[2];
  const void *scales[2];      // OPERAND_MX
  int count, kind;
  int64_t rows, cols;
};

// as dense rows of `to` (16-bit), `pitch` (a multiple of 8) long with zeros from column cols on; the second one's rows behind the first's
int operand_dense(const Operand &a, int to, void *out, int64_t pitch, hipStream_t s);
// transposed: value (n, k) at out[k * stride + n], zeros for n from rows to pitch (a multiple of 64); the second one's `second` values on
int operand_transposed(const Operand &a, int to, void *out, int64_t pitch, int64_t stride, int64_t second, hipStream_t s);
// activations of fp32 or fp16 as three dense bf16 matrices [rows, pitch] that add up to them, the second one's three behind the first's
int operand_pieces(const Operand &a, void *out, int64_t pitch, hipStream_t s);
// activations for rows_bf16 / rows_f16 with packed operands of `chunks` chunks, the second one's behind the first's; `to` CAIFX_F32: three
// bf16 pieces (kind CAIFX_F32 or CAIFX_F16 then)
int operand_rows(const Operand &a, int to, void *out, int chunks, hipStream_t s);

// y[M, K] = sum over one or two weights [N, K] of x_i w_i, the weights as they are stored (caifx_mxfp4_dx.hip)
struct DxProduct {
  int64_t M, N, K;
  int count;
  const void *w[2], *s[2];
  bool mx;
  const void *x[2];          // direct: [M, N] of the compute type (fp32 too), N at least 8, at any address; otherwise x[0] packed by operand_rows
  bool direct;
  int compute_dtype;         // CAIFX_F32: three bf16 pieces (mx only)
  void *y;
  int y_dtype;
  const void *addend;
};
bool dx_takes(const DxProduct &p);
bool dx_reads(const DxProduct &p);      // whether activations that can be direct should be
double dx_us(const DxProduct &p);      // an estimate
size_t dx_partial_bytes(const DxProduct &p);
int dx_product(const DxProduct &p, void *partial, hipStream_t s);

// y[M, C] = A B^T of two operands in microscaled 4 bits with `blocks` blocks a row, in tiles for the matrix cores.  The workspace is for the
// scales in another order.
bool mx_gemm_takes(int64_t M, int64_t C, int64_t blocks);
double mx_gemm_us(int64_t M, int64_t C, int64_t blocks);      // an estimate
size_t mx_gemm_workspace_bytes(int64_t M, int64_t C, int64_t blocks);
int mx_gemm(int64_t M, int64_t C, int64_t blocks, const void *a, const void *sa, const void *b, const void *sb, void *d, int d_dtype, void *workspace, hipStream_t s);

// y = the sum of `parts` fp32 arrays of n values in order, and the addend: sums of a shared reduction
int join_sums(const float *partial, int parts, int64_t n, void *y, int y_dtype, const void *addend, hipStream_t s);

int gating_backward(const void *grad, const void *gate, const void *up, void *grad_gate, void *grad_up, int64_t n, int dtype, hipStream_t s);

}  // namespace caifx
