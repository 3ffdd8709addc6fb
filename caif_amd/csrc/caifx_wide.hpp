// The dense product of caifx_gemm_wide.hip on operands that are there already, and its two forms over a pair of weights.
#pragma once

#include "caifx_internal.hpp"

namespace caifx {

enum {
  WIDE_PLAIN = 0,      // d = a[0] b[0]^T
  WIDE_GATED = 1,      // d = silu(a[0] b[0]^T) * (a[0] b[1]^T), the two products kept in gate and up unless those are null; no addend
  WIDE_CHAIN = 2       // d = a[0] b[0]^T + a[1] b[1]^T, one sum
};

struct WideProduct {
  int form;
  const void *a[2];       // [M, R] of the compute type
  const void *b[2];       // [C, R] of the compute type
  void *d, *gate, *up;    // [M, C] of d_dtype (gated: the compute type)
  const void *addend;     // d = T(float(T(sum)) + float(addend))
  int64_t M, C, R;
  int compute_dtype, d_dtype;
};

// silu in fp32 from 1 / (1 + exp(-g)) with the exponential of -|g|, whose inverse stays in (0.5, 1]
__device__ __forceinline__ float gate_act(float g)
{
  const float e = expf(-fabsf(g)), high = __builtin_amdgcn_rcpf(1.0f + e);
  return g * (g < 0.0f ? e * high : high);
}

// whether the kernel takes these sizes; every pointer has to be aligned to 16 bytes
bool wide_takes(int64_t M, int64_t C, int64_t R);
int wide_product(const WideProduct &p, hipStream_t s);
// what a product takes, in us, estimated; gated: C of both weights together, chained: R of both pairs
double wide_product_us(int64_t M, int64_t C, int64_t R);

}  // namespace caifx
