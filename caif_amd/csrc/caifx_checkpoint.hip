// Activation checkpoints in 8 bits: an activation of the forward pass kept as one int8 code per value and one fp32 scale per
// 128 neighbouring values of a row, and the gating of a feed-forward block that writes and reads such checkpoints.
//
//   scale = fl32(max|x| * fl32(1 / 127)), 1 where that is zero, NaN where the group holds an infinity or a NaN
//   code  = clamp(rint(fl32(x / scale)), -127, 127)            value = code * scale
//
// Everything here is bound by memory.  Sixteen lanes take a group, eight values each, so that a lane's part is one 16-byte
// access of a 16-bit type; rows of any length and alignment take the same path (the hardware splits an access that straddles
// a line), only a row's last values are moved one by one.
#include "caifx_common.hpp"

#pragma clang fp contract(off)

namespace caifx {
namespace {

constexpr int kGroup = CAIFX_CHECKPOINT_GROUP;
constexpr int kPer = 8;                               // values of a lane
constexpr int kLanes = kGroup / kPer;                 // lanes of a group
constexpr int kThreads = 256;
constexpr int kUnits = kThreads / kLanes;             // groups of a workgroup

template <typename T> struct Eight { T v[kPer]; };

// eight values from p, `have` of them in the row (zeros for the others)
template <typename T> __device__ __forceinline__ Eight<T> load8(const T *p, int have)
{
  Eight<T> e;
  if (have >= kPer) {
    __builtin_memcpy(&e, p, sizeof e);
  } else {
#pragma unroll
    for (int i = 0; i < kPer; ++i) e.v[i] = i < have ? p[i] : T(0);
  }
  return e;
}
template <typename T> __device__ __forceinline__ void store8(T *p, const Eight<T> &e, int have)
{
  if (have >= kPer) {
    __builtin_memcpy(p, &e, sizeof e);
  } else {
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      if (i < have) p[i] = e.v[i];
  }
}

// The place of a lane: its group (row, column of the group) and its eight values in it.
struct Place {
  int64_t at;                                         // flat index of the lane's first value
  int64_t scale_at;                                   // flat index of the group's scale
  int have;                                           // values of the lane inside the row, 0 past the last group
};
__device__ __forceinline__ Place place(int64_t rows, int64_t cols, int64_t groups)
{
  const int64_t first = static_cast<int64_t>(blockIdx.x) * kUnits;             // the workgroup's first group, the same for all lanes
  const int64_t row0 = first / groups;
  const uint32_t in_row = static_cast<uint32_t>(first - row0 * groups) + threadIdx.x / kLanes;
  const uint32_t down = in_row / static_cast<uint32_t>(groups);
  const int64_t row = row0 + down;
  const int64_t col = static_cast<int64_t>(in_row - down * static_cast<uint32_t>(groups)) * kGroup + (threadIdx.x % kLanes) * kPer;
  const int64_t left = row < rows ? cols - col : 0;
  return {row * cols + col, first + threadIdx.x / kLanes, left >= kPer ? kPer : (left > 0 ? static_cast<int>(left) : 0)};
}

// maximum over the sixteen lanes of a group
__device__ __forceinline__ uint32_t group_max(uint32_t v)
{
#pragma unroll
  for (int o = kLanes / 2; o > 0; o >>= 1) {
    const uint32_t w = __shfl_xor(v, o, kLanes);
    v = v > w ? v : w;
  }
  return v;
}

// Codes of a lane's eight values, and the group's scale.  The magnitudes are compared as bit patterns: an infinity is larger
// than any number and a NaN larger than that, so one comparison at the end tells whether the group holds either.
template <typename T> __device__ __forceinline__ Eight<int8_t> quantise(const Eight<T> &x, float &scale)
{
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const uint32_t b = __builtin_bit_cast(uint32_t, to_f32<T>(x.v[i])) & 0x7FFFFFFFu;
    top = top > b ? top : b;
  }
  top = group_max(top);
  const bool finite = top < 0x7F800000u;
  scale = finite ? __builtin_bit_cast(float, top) * (1.0f / 127.0f) : __builtin_nanf("");
  if (scale == 0.0f) scale = 1.0f;
  Eight<int8_t> q;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const float n = fminf(fmaxf(rintf(to_f32<T>(x.v[i]) / scale), -127.0f), 127.0f);
    q.v[i] = static_cast<int8_t>(finite ? static_cast<int>(n) : 0);
  }
  return q;
}

template <typename T>
__global__ __launch_bounds__(kThreads) void pack_kernel(const T *__restrict__ x, int8_t *__restrict__ codes, float *__restrict__ scales, int64_t rows,
                                                        int64_t cols, int64_t groups)
{
  const Place p = place(rows, cols, groups);
  const Eight<T> v = load8(x + p.at, p.have);
  float scale;
  const Eight<int8_t> q = quantise(v, scale);
  store8(codes + p.at, q, p.have);
  if (threadIdx.x % kLanes == 0 && p.have > 0) scales[p.scale_at] = scale;
}

template <typename T>
__global__ __launch_bounds__(kThreads) void unpack_kernel(const int8_t *__restrict__ codes, const float *__restrict__ scales, T *__restrict__ out,
                                                          int64_t rows, int64_t cols, int64_t groups)
{
  const Place p = place(rows, cols, groups);
  if (p.have == 0) return;
  const Eight<int8_t> q = load8(codes + p.at, p.have);
  const float scale = scales[p.scale_at];
  Eight<T> v;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    float value = static_cast<float>(q.v[i]) * scale;
    // the product is an fp32 number first: fused with the conversion to fp16 it would be rounded once, to another value in places
    asm("" : "+v"(value));
    v.v[i] = from_f32<T>(value);
  }
  store8(out + p.at, v, p.have);
}

// hidden = silu_multiply(gate, up), bit for bit (silu(gate) is rounded to T first), and both inputs' checkpoints
template <typename T>
__global__ __launch_bounds__(kThreads) void gate_kernel(const T *__restrict__ gate, const T *__restrict__ up, T *__restrict__ hidden,
                                                        int8_t *__restrict__ gate_codes, float *__restrict__ gate_scales, int8_t *__restrict__ up_codes,
                                                        float *__restrict__ up_scales, int64_t rows, int64_t cols, int64_t groups)
{
  const Place p = place(rows, cols, groups);
  const Eight<T> g = load8(gate + p.at, p.have), u = load8(up + p.at, p.have);
  Eight<T> h;
#pragma unroll
  for (int i = 0; i < kPer; ++i) h.v[i] = swiglu_fwd_one<T>(g.v[i], u.v[i]);
  store8(hidden + p.at, h, p.have);
  float gs, us;
  const Eight<int8_t> gq = quantise(g, gs), uq = quantise(u, us);
  store8(gate_codes + p.at, gq, p.have);
  store8(up_codes + p.at, uq, p.have);
  if (threadIdx.x % kLanes == 0 && p.have > 0) {
    gate_scales[p.scale_at] = gs;
    up_scales[p.scale_at] = us;
  }
}

// g, u = the checkpoints' values in fp32; grad_up = T(d silu(g)), grad_gate = T(d u silu'(g)) and, where it is asked for,
// hidden = T(silu(g) u): each result is rounded once.
template <typename T, bool kHidden>
__global__ __launch_bounds__(kThreads) void gate_bwd_kernel(const int8_t *__restrict__ gate_codes, const float *__restrict__ gate_scales,
                                                            const int8_t *__restrict__ up_codes, const float *__restrict__ up_scales,
                                                            const T *__restrict__ grad, T *__restrict__ grad_gate, T *__restrict__ grad_up,
                                                            T *__restrict__ hidden, int64_t rows, int64_t cols, int64_t groups)
{
  const Place p = place(rows, cols, groups);
  if (p.have == 0) return;
  const Eight<int8_t> gq = load8(gate_codes + p.at, p.have), uq = load8(up_codes + p.at, p.have);
  const Eight<T> d = load8(grad + p.at, p.have);
  const float gs = gate_scales[p.scale_at], us = up_scales[p.scale_at];
  Eight<T> og, ou, oh;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const float g = static_cast<float>(gq.v[i]) * gs, u = static_cast<float>(uq.v[i]) * us, grad_h = to_f32<T>(d.v[i]);
    const float s = 1.0f / (1.0f + expf(-g)), act = g * s;
    ou.v[i] = from_f32<T>(grad_h * act);
    og.v[i] = from_f32<T>(grad_h * u * (s * __builtin_fmaf(g, 1.0f - s, 1.0f)));
    if constexpr (kHidden) oh.v[i] = from_f32<T>(act * u);
  }
  store8(grad_gate + p.at, og, p.have);
  store8(grad_up + p.at, ou, p.have);
  if constexpr (kHidden) store8(hidden + p.at, oh, p.have);
}

// CAIFX_OK and `go` for a launch that has work; blocks of the launch
int check(int64_t rows, int64_t cols, int dtype, bool missing, bool misaligned, bool &go, dim3 &grid, int64_t &groups)
{
  go = false;
  if (!valid_dtype(dtype) || rows < 0 || cols < 0) return CAIFX_ERR_INVALID_ARGUMENT;
  if (rows == 0 || cols == 0) return CAIFX_OK;
  if (missing) return CAIFX_ERR_INVALID_ARGUMENT;
  if (misaligned) return CAIFX_ERR_MISALIGNED;
  groups = (cols + kGroup - 1) / kGroup;
  // a grid has fewer than 2^32 threads, and a row's groups fit 31 bits
  if (groups > INT32_MAX / 2 || rows > (int64_t{1} << 30) || groups > ((int64_t{1} << 24) - 1) * kUnits / rows) return CAIFX_ERR_UNSUPPORTED;
  grid = dim3(static_cast<unsigned>((rows * groups + kUnits - 1) / kUnits));
  go = true;
  return CAIFX_OK;
}

}  // namespace
}  // namespace caifx

using namespace caifx;

// one launch for the element type of `dtype`
#define CAIFX_BY_TYPE(go)                       \
  switch (dtype) {                              \
    case CAIFX_F32: { typedef float T; go; break; }   \
    case CAIFX_F16: { typedef f16_t T; go; break; }   \
    default: { typedef bf16_t T; go; break; }         \
  }

extern "C" {

int caifx_checkpoint_pack(const void *input, void *codes, float *scales, int64_t rows, int64_t cols, int dtype, caifx_stream_t stream)
{
  bool go;
  dim3 grid;
  int64_t groups;
  const int st = check(rows, cols, dtype, !input || !codes || !scales, !aligned_to(input, dtype_size(dtype)) || !aligned_to(scales, 4), go, grid, groups);
  if (!go) return st;
  CAIFX_BY_TYPE(hipLaunchKernelGGL(pack_kernel<T>, grid, dim3(kThreads), 0, as_stream(stream), static_cast<const T *>(input),
                                   static_cast<int8_t *>(codes), scales, rows, cols, groups));
  return launch_status();
}

int caifx_checkpoint_unpack(const void *codes, const float *scales, void *output, int64_t rows, int64_t cols, int dtype, caifx_stream_t stream)
{
  bool go;
  dim3 grid;
  int64_t groups;
  const int st = check(rows, cols, dtype, !output || !codes || !scales, !aligned_to(output, dtype_size(dtype)) || !aligned_to(scales, 4), go, grid, groups);
  if (!go) return st;
  CAIFX_BY_TYPE(hipLaunchKernelGGL(unpack_kernel<T>, grid, dim3(kThreads), 0, as_stream(stream), static_cast<const int8_t *>(codes), scales,
                                   static_cast<T *>(output), rows, cols, groups));
  return launch_status();
}

int caifx_silu_multiply_checkpoint(const void *gate, const void *up, void *hidden, void *gate_codes, float *gate_scales, void *up_codes,
                                   float *up_scales, int64_t rows, int64_t cols, int dtype, caifx_stream_t stream)
{
  bool go;
  dim3 grid;
  int64_t groups;
  const size_t es = dtype_size(dtype);
  const int st = check(rows, cols, dtype, !gate || !up || !hidden || !gate_codes || !gate_scales || !up_codes || !up_scales,
                       !aligned_to(gate, es) || !aligned_to(up, es) || !aligned_to(hidden, es) || !aligned_to(gate_scales, 4) || !aligned_to(up_scales, 4),
                       go, grid, groups);
  if (!go) return st;
  CAIFX_BY_TYPE(hipLaunchKernelGGL(gate_kernel<T>, grid, dim3(kThreads), 0, as_stream(stream), static_cast<const T *>(gate), static_cast<const T *>(up),
                                   static_cast<T *>(hidden), static_cast<int8_t *>(gate_codes), gate_scales, static_cast<int8_t *>(up_codes), up_scales,
                                   rows, cols, groups));
  return launch_status();
}

int caifx_swiglu_backward_checkpoint(const void *gate_codes, const float *gate_scales, const void *up_codes, const float *up_scales,
                                     const void *grad_hidden, void *grad_gate, void *grad_up, void *hidden, int64_t rows, int64_t cols, int dtype,
                                     caifx_stream_t stream)
{
  bool go;
  dim3 grid;
  int64_t groups;
  const size_t es = dtype_size(dtype);
  const int st = check(rows, cols, dtype, !gate_codes || !gate_scales || !up_codes || !up_scales || !grad_hidden || !grad_gate || !grad_up,
                       !aligned_to(gate_scales, 4) || !aligned_to(up_scales, 4) || !aligned_to(grad_hidden, es) || !aligned_to(grad_gate, es) ||
                           !aligned_to(grad_up, es) || !aligned_to(hidden, es), go, grid, groups);
  if (!go) return st;
  hipStream_t s = as_stream(stream);
#define CAIFX_GO(kHidden)                                                                                                                          \
  hipLaunchKernelGGL((gate_bwd_kernel<T, kHidden>), grid, dim3(kThreads), 0, s, static_cast<const int8_t *>(gate_codes), gate_scales,              \
                     static_cast<const int8_t *>(up_codes), up_scales, static_cast<const T *>(grad_hidden), static_cast<T *>(grad_gate),           \
                     static_cast<T *>(grad_up), static_cast<T *>(hidden), rows, cols, groups)
  if (hidden) {
    CAIFX_BY_TYPE(CAIFX_GO(true));
  } else {
    CAIFX_BY_TYPE(CAIFX_GO(false));
  }
#undef CAIFX_GO
  return launch_status();
}

}  // extern "C"
