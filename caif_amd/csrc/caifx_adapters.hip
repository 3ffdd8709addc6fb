// Low-rank adapters beside a frozen projection: the branch of every row's own adapter added to the projection's result, and the
// branch's gradients.  Row m uses adapter l = ids[m] (none where ids[m] is outside [0, L)):
//
//   forward    h[m] = x[m] A[l]^T                  y[m]  = T(base[m] + scaling[l] h[m] B[l]^T)
//   backward   g[m] = scaling[l] dy[m] B[l]        dx[m] = T(base[m] + g[m] A[l])
//              dA[l] = T(sum over m of l of g[m]^T x[m])      dB[l] = T(sum over m of l of scaling[l] dy[m]^T h[m])
//
// with x [M,K], A [L,r,K], B [L,N,r], h and g [M,r] in fp32.  All sums are fp32 and of a fixed order.
#include "caifx_common.hpp"

namespace caifx {
namespace {

constexpr int kThreads = 256;

struct Problem {
  int64_t M, N, K;
  int r, L;
  const int32_t *ids;
  const void *a, *b;
  const float *scaling;
};

__device__ __forceinline__ int adapter_of(const Problem &p, int64_t m)
{
  const int l = p.ids[m];
  return l >= 0 && l < p.L ? l : -1;
}

__device__ __forceinline__ float wave_sum(float v)
{
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

// out[m][j] = scale * sum_c z[m][c] f[l][j * js + c * cs]: one wave per row and rank index
template <typename T>
__global__ __launch_bounds__(kThreads) void shrink_kernel(Problem p, const T *z, int64_t C, const T *f, int64_t js, int64_t cs, bool scaled, float *out)
{
  const int lane = threadIdx.x & 63;
  const int64_t w = (static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x) >> 6;
  const int64_t m = w / p.r;
  const int j = static_cast<int>(w - m * p.r);
  if (m >= p.M) return;
  const int l = adapter_of(p, m);
  float sum = 0.0f;
  if (l >= 0) {
    const T *row = f + static_cast<int64_t>(l) * p.r * C + j * js;
    for (int64_t c = lane; c < C; c += 64) sum += to_f32<T>(z[m * C + c]) * to_f32<T>(row[c * cs]);
    sum = wave_sum(sum);
    if (scaled) sum *= p.scaling[l];
  }
  if (lane == 0) out[m * p.r + j] = sum;
}

// out[m][c] = T(base[m][c] + scale * sum_j u[m][j] f[l][j * js + c * cs])
template <typename T>
__global__ __launch_bounds__(kThreads) void expand_kernel(Problem p, const float *u, int64_t C, const T *f, int64_t js, int64_t cs, bool scaled,
                                                          const T *base, T *out)
{
  const int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  if (i >= p.M * C) return;
  const int64_t m = i / C, c = i - m * C;
  const int l = adapter_of(p, m);
  float sum = 0.0f;
  if (l >= 0) {
    const T *col = f + static_cast<int64_t>(l) * p.r * C + c * cs;
    for (int j = 0; j < p.r; ++j) sum += u[m * p.r + j] * to_f32<T>(col[j * js]);
    if (scaled) sum *= p.scaling[l];
  }
  if (base) sum = l >= 0 ? to_f32<T>(base[i]) + sum : to_f32<T>(base[i]);
  out[i] = from_f32<T>(sum);
}

// grad[l][j * js + c * cs] = T(scale * sum over the rows m of l of u[m][j] z[m][c])
template <typename T, typename Z>
__global__ __launch_bounds__(kThreads) void outer_kernel(Problem p, const float *u, const Z *z, const float *z_scales, int64_t C, int64_t js, int64_t cs,
                                                         bool scaled, T *grad)
{
  const int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  const int64_t lj = i / C, c = i - lj * C;
  const int l = static_cast<int>(lj / p.r), j = static_cast<int>(lj - static_cast<int64_t>(l) * p.r);
  if (l >= p.L) return;
  const int64_t groups = (C + CAIFX_CHECKPOINT_GROUP - 1) / CAIFX_CHECKPOINT_GROUP;
  float sum = 0.0f;
  for (int64_t m = 0; m < p.M; ++m) {
    if (p.ids[m] != l) continue;
    float v = static_cast<float>(z[m * C + c]);
    if (z_scales) v *= z_scales[m * groups + c / CAIFX_CHECKPOINT_GROUP];
    sum += u[m * p.r + j] * v;
  }
  if (scaled) sum *= p.scaling[l];
  grad[static_cast<int64_t>(l) * p.r * C + j * js + c * cs] = from_f32<T>(sum);
}

unsigned blocks(int64_t threads) { return static_cast<unsigned>((threads + kThreads - 1) / kThreads); }

template <typename T> int forward(const Problem &p, const void *x, const void *base, void *y, float *h, hipStream_t s)
{
  hipLaunchKernelGGL(shrink_kernel<T>, dim3(blocks(p.M * p.r * 64)), dim3(kThreads), 0, s, p, static_cast<const T *>(x), p.K, static_cast<const T *>(p.a),
                     p.K, int64_t{1}, false, h);
  hipLaunchKernelGGL(expand_kernel<T>, dim3(blocks(p.M * p.N)), dim3(kThreads), 0, s, p, h, p.N, static_cast<const T *>(p.b), int64_t{1},
                     static_cast<int64_t>(p.r), true, static_cast<const T *>(base), static_cast<T *>(y));
  return launch_status();
}

template <typename T>
int backward(const Problem &p, const void *dy, const void *x, const float *x_scales, const float *hidden, const void *base, void *dx, void *ga, void *gb,
             float *g, hipStream_t s)
{
  const int64_t each = static_cast<int64_t>(p.L) * p.r;
  if (p.M > 0 && (dx || ga))
    hipLaunchKernelGGL(shrink_kernel<T>, dim3(blocks(p.M * p.r * 64)), dim3(kThreads), 0, s, p, static_cast<const T *>(dy), p.N,
                       static_cast<const T *>(p.b), int64_t{1}, static_cast<int64_t>(p.r), true, g);
  if (p.M > 0 && dx)
    hipLaunchKernelGGL(expand_kernel<T>, dim3(blocks(p.M * p.K)), dim3(kThreads), 0, s, p, g, p.K, static_cast<const T *>(p.a), p.K, int64_t{1}, false,
                       static_cast<const T *>(base), static_cast<T *>(dx));
  if (ga && x_scales)
    hipLaunchKernelGGL((outer_kernel<T, int8_t>), dim3(blocks(each * p.K)), dim3(kThreads), 0, s, p, g, static_cast<const int8_t *>(x), x_scales, p.K, p.K,
                       int64_t{1}, false, static_cast<T *>(ga));
  else if (ga)
    hipLaunchKernelGGL((outer_kernel<T, T>), dim3(blocks(each * p.K)), dim3(kThreads), 0, s, p, g, static_cast<const T *>(x), x_scales, p.K, p.K, int64_t{1},
                       false, static_cast<T *>(ga));
  if (gb)
    hipLaunchKernelGGL((outer_kernel<T, T>), dim3(blocks(each * p.N)), dim3(kThreads), 0, s, p, hidden, static_cast<const T *>(dy), nullptr, p.N, int64_t{1},
                       static_cast<int64_t>(p.r), true, static_cast<T *>(gb));
  return launch_status();
}

size_t workspace_bytes(int64_t M, int rank) { return static_cast<size_t>(M) * rank * 4; }

int check(int64_t M, int64_t N, int64_t K, int rank, int num_adapters, int dtype)
{
  if (!valid_dtype(dtype) || M < 0 || N <= 0 || K <= 0 || rank <= 0 || num_adapters <= 0) return CAIFX_ERR_INVALID_ARGUMENT;
  constexpr int64_t kMost = int64_t{1} << 30;
  if (rank > CAIFX_ADAPTER_RANK_MAX || M > kMost || N > kMost || K > kMost) return CAIFX_ERR_UNSUPPORTED;
  return CAIFX_OK;
}

}  // namespace
}  // namespace caifx

using namespace caifx;

extern "C" {

size_t caifx_adapters_workspace_bytes(int64_t M, int64_t N, int64_t K, int rank, int num_adapters, int dtype, int backward)
{
  (void)backward;
  if (check(M, N, K, rank, num_adapters, dtype) != CAIFX_OK) return 0;
  return workspace_bytes(M, rank);
}

int caifx_adapters_forward(int64_t M, int64_t N, int64_t K, int rank, int num_adapters, const void *x, const int32_t *ids, const void *a, const void *b,
                           const float *scaling, const void *base, void *y, float *hidden, int dtype, void *workspace, size_t workspace_size,
                           caifx_stream_t stream)
{
  const int st = check(M, N, K, rank, num_adapters, dtype);
  if (st != CAIFX_OK || M == 0) return st;
  if (!x || !ids || !a || !b || !scaling || !y) return CAIFX_ERR_INVALID_ARGUMENT;
  const size_t es = dtype_size(dtype);
  if (!aligned_to(x, es) || !aligned_to(a, es) || !aligned_to(b, es) || !aligned_to(base, es) || !aligned_to(y, es) || !aligned_to(ids, 4) ||
      !aligned_to(scaling, 4) || !aligned_to(hidden, 4) || !aligned_to(workspace, 4))
    return CAIFX_ERR_MISALIGNED;
  if (!workspace || workspace_size < workspace_bytes(M, rank)) return CAIFX_ERR_WORKSPACE_TOO_SMALL;
  const Problem p{M, N, K, rank, num_adapters, ids, a, b, scaling};
  float *h = hidden ? hidden : static_cast<float *>(workspace);
  hipStream_t s = as_stream(stream);
  switch (dtype) {
    case CAIFX_F32: return forward<float>(p, x, base, y, h, s);
    case CAIFX_F16: return forward<f16_t>(p, x, base, y, h, s);
    default: return forward<bf16_t>(p, x, base, y, h, s);
  }
}

int caifx_adapters_backward(int64_t M, int64_t N, int64_t K, int rank, int num_adapters, const void *dy, const void *x, const float *x_scales,
                            const float *hidden, const int32_t *ids, const void *a, const void *b, const float *scaling, const void *base, void *dx,
                            void *grad_a, void *grad_b, int dtype, void *workspace, size_t workspace_size, caifx_stream_t stream)
{
  const int st = check(M, N, K, rank, num_adapters, dtype);
  if (st != CAIFX_OK || ((M == 0 || !dx) && !grad_a && !grad_b)) return st;
  if (M > 0 && (!dy || !ids || !scaling || (dx && !a) || ((dx || grad_a) && !b) || (grad_a && !x) || (grad_b && !hidden))) return CAIFX_ERR_INVALID_ARGUMENT;
  const size_t es = dtype_size(dtype);
  if (!aligned_to(dy, es) || (!x_scales && !aligned_to(x, es)) || !aligned_to(x_scales, 4) || !aligned_to(hidden, 4) || !aligned_to(ids, 4) ||
      !aligned_to(a, es) || !aligned_to(b, es) || !aligned_to(scaling, 4) || !aligned_to(base, es) || !aligned_to(dx, es) || !aligned_to(grad_a, es) ||
      !aligned_to(grad_b, es) || !aligned_to(workspace, 4))
    return CAIFX_ERR_MISALIGNED;
  if (M > 0 && (!workspace || workspace_size < workspace_bytes(M, rank))) return CAIFX_ERR_WORKSPACE_TOO_SMALL;
  const Problem p{M, N, K, rank, num_adapters, ids, a, b, scaling};
  float *g = static_cast<float *>(workspace);
  hipStream_t s = as_stream(stream);
  switch (dtype) {
    case CAIFX_F32: return backward<float>(p, dy, x, x_scales, hidden, base, dx, grad_a, grad_b, g, s);
    case CAIFX_F16: return backward<f16_t>(p, dy, x, x_scales, hidden, base, dx, grad_a, grad_b, g, s);
    default: return backward<bf16_t>(p, dy, x, x_scales, hidden, base, dx, grad_a, grad_b, g, s);
  }
}

}  // extern "C"
