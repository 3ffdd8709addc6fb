// The dense product of caifx_gemm_wide.hip on operands that are there already, and its two forms over a pair of weights.
#pragma once

#include "caifx_internal.hpp"
#include "caifx_wide_plan.hpp"

namespace caifx {

// what the kernel's forms combine
enum { WIDE_PLAIN = 0, WIDE_GATED = 1, WIDE_CHAIN = 2, WIDE_RAGGED = 4 };

struct WideProduct {
  // d = sum over the pairs i of A_i B_i^T: A_i behind `a` by i a_stride bytes, B_i behind b[0] by (i / b_every) b_stride bytes
  const void *a;          // [M, R] each, of the compute type
  const void *b[2];       // [C, R] each
  int64_t a_stride, b_stride;
  int pairs, b_every;
  int parts;              // workgroups that share a tile's steps; more than one: d holds `parts` fp32 results one behind the other, not gated, no addend
  // gated: d = silu(that) * (the same with b[1]), and the two kept in gate and up unless those are null; no addend.  d is of the compute
  // type, or with several pairs fp32.
  bool gated;
  void *d, *gate, *up;    // [M, C] of d_dtype
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

// whether the kernel takes these sizes; the operands have to be aligned to 16 bytes
bool wide_takes(int64_t M, int64_t C, int64_t R);
int wide_product(const WideProduct &p, hipStream_t s);

}  // namespace caifx
