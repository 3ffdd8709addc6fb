// Activation checkpoints in 8 bits: an activation of the forward pass kept as one int8 code per value and one fp32 scale per
// 128 neighbouring values of a row, and the gating of a feed-forward block that writes and reads such checkpoints.
//
//   scale = fl32(max|x| * fl32(1 / 127)), 1 where that is zero, NaN where the group holds an infinity or a NaN
//   code  = clamp(rint(fl32(x / scale)), -127, 127)            value = code * scale
//
// Everything here is bound by memory, if the arithmetic is kept short: 45 M values through silu and two divisions each are as long a way
// for the vector units as their 360 MB for the memory.  Sixteen lanes take a group, eight values each, so that a lane's part is one
// 16-byte access of a 16-bit type; rows of any length and alignment take the same path (the hardware splits an access that straddles
// a line), only a row's last values are moved one by one.  Measured in bf16, three sets of tensors in turn: 16384 x 4096 packed in 34 us and unpacked in
// 32 (6.0 and 6.4 TB/s, in part from the memory-side cache; with divisions and shuffles 64 and 42), 4096 x 11008 gated in 88 us, three
// quarters of it vector instructions (silu's exponential and division are a third of the 54 for a pair of values), its backward in 71
// (5.1 TB/s).
#include "caifx_common.hpp"

#pragma clang fp contract(off)

namespace caifx {
namespace {

constexpr int kGroup = CAIFX_CHECKPOINT_GROUP;
constexpr int kPer = 8;                               // values of a lane
constexpr int kLanes = kGroup / kPer;                 // lanes of a group
constexpr int kThreads = 256;
constexpr int kTurns = 2;                             // groups of a lane, both asked for before the first is used
constexpr int kUnits = kTurns * kThreads / kLanes;    // groups of a workgroup

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

// rows x cols in groups of a row.  Rows of whole groups need no row: their groups stand in one line.
struct Shape {
  uint32_t units, groups, magic;                      // groups in all, of a row, floor(2^32 / groups) or 2^32 - 1
  int64_t cols;
};
// The place of a lane: its eight values in a group.
struct Place {
  int64_t at;                                         // flat index of the first
  uint32_t unit;                                      // flat index of the group
  int have;                                           // values inside the row, 0 past the last group
};
template <bool kWhole> __device__ __forceinline__ Place place(const Shape &s, int turn)
{
  const uint32_t unit = (blockIdx.x * kTurns + turn) * (kThreads / kLanes) + threadIdx.x / kLanes, in = (threadIdx.x % kLanes) * kPer;
  if constexpr (kWhole) {
    return {static_cast<int64_t>(unit) * kGroup + in, unit, unit < s.units ? kPer : 0};
  } else {
    uint32_t row = __umulhi(unit, s.magic);           // the quotient or one less
    if (unit - row * s.groups >= s.groups) ++row;
    const int64_t col = static_cast<int64_t>(unit - row * s.groups) * kGroup + in, left = unit < s.units ? s.cols - col : 0;
    return {row * s.cols + col, unit, left >= kPer ? kPer : (left > 0 ? static_cast<int>(left) : 0)};
  }
}

// Maximum over the sixteen lanes of a group, which are a row of the wave's data-parallel moves: neighbours, pairs, mirrored halves.
__device__ __forceinline__ uint32_t group_max(uint32_t v)
{
  auto with = [&](uint32_t w) { v = v > w ? v : w; };
  with(__builtin_amdgcn_mov_dpp(v, 0xB1, 0xF, 0xF, true));              // lanes 1 0 3 2
  with(__builtin_amdgcn_mov_dpp(v, 0x4E, 0xF, 0xF, true));              // lanes 2 3 0 1
  with(__builtin_amdgcn_mov_dpp(v, 0x141, 0xF, 0xF, true));             // eight lanes backwards
  with(__builtin_amdgcn_mov_dpp(v, 0x140, 0xF, 0xF, true));             // sixteen lanes backwards
  return v;
}

typedef uint16_t u16x2_t __attribute__((ext_vector_type(2)));

// The largest magnitude of a group, as the bits of an fp32 number.  Magnitudes are compared as bit patterns: an infinity is larger than
// any number and a NaN larger than that, so one comparison tells whether the group holds either.
template <typename T> __device__ __forceinline__ uint32_t group_top(const Eight<T> &x)
{
  if constexpr (sizeof(T) == 4) {
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const uint32_t b = __builtin_bit_cast(uint32_t, x.v[i]) & 0x7FFFFFFFu;
      top = top > b ? top : b;
    }
    return group_max(top);
  } else {
    struct Words { uint32_t w[kPer / 2]; };
    const Words words = __builtin_bit_cast(Words, x);
    u16x2_t top = __builtin_bit_cast(u16x2_t, words.w[0] & 0x7FFF7FFFu);
#pragma unroll
    for (int i = 1; i < kPer / 2; ++i) top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x2_t, words.w[i] & 0x7FFF7FFFu));
    const uint32_t most = group_max(top[0] > top[1] ? top[0] : top[1]);
    const float value = to_f32<T>(__builtin_bit_cast(T, static_cast<uint16_t>(most)));
    return __builtin_bit_cast(uint32_t, value);
  }
}

// Codes of a lane's eight values, and the group's scale.  The quotient is rounded as a division rounds it without being one: with the
// rounded inverse y of the scale, q = x y is at most 1.5 steps off, q + (x - q s) y within a step, and the same once more is the rounded
// quotient (Markstein: a quotient within a step, corrected by its exact remainder times the rounded inverse).  For 16-bit values one
// correction gives the same codes: all pairs of a maximum's and a value's 11 bits were compared.  Adding 1.5 2^23 rounds the quotient to
// an integer, ties to even, and leaves the integer in the low byte.  Scales below 2^-100, where the remainders would underflow, divide.
template <typename T> __device__ __forceinline__ Eight<int8_t> quantise(const Eight<T> &x, float &scale)
{
  const uint32_t top = group_top(x);
  const bool finite = top < 0x7F800000u;
  scale = finite ? __builtin_bit_cast(float, top) * (1.0f / 127.0f) : __builtin_nanf("");
  if (scale == 0.0f) scale = 1.0f;
  uint32_t bits[kPer];
  if (scale < 0x1p-100f) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const float n = fminf(fmaxf(rintf(to_f32<T>(x.v[i]) / scale), -127.0f), 127.0f);
      bits[i] = static_cast<uint32_t>(static_cast<int>(n));
    }
  } else {
    const float y = 1.0f / scale;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const float v = to_f32<T>(x.v[i]);
      float q = v * y;
      q = __builtin_fmaf(__builtin_fmaf(-q, scale, v), y, q);
      if constexpr (sizeof(T) == 4) q = __builtin_fmaf(__builtin_fmaf(-q, scale, v), y, q);
      bits[i] = __builtin_bit_cast(uint32_t, q + 12582912.0f);
    }
  }
  struct Words { uint32_t w[2]; } words;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const uint32_t lo = __builtin_amdgcn_perm(bits[4 * h + 1], bits[4 * h], 0x0C0C0400u), hi = __builtin_amdgcn_perm(bits[4 * h + 3], bits[4 * h + 2], 0x04000C0Cu);
    words.w[h] = finite ? lo | hi : 0u;
  }
  return __builtin_bit_cast(Eight<int8_t>, words);
}

template <typename T, bool kWhole>
__global__ __launch_bounds__(kThreads) void pack_kernel(const T *__restrict__ x, int8_t *__restrict__ codes, float *__restrict__ scales, Shape s)
{
  Place p[kTurns];
  Eight<T> v[kTurns];
#pragma unroll
  for (int k = 0; k < kTurns; ++k) {
    p[k] = place<kWhole>(s, k);
    v[k] = load8(x + p[k].at, p[k].have);
  }
#pragma unroll
  for (int k = 0; k < kTurns; ++k) {
    float scale;
    const Eight<int8_t> q = quantise(v[k], scale);
    store8(codes + p[k].at, q, p[k].have);
    if (threadIdx.x % kLanes == 0 && p[k].have > 0) scales[p[k].unit] = scale;
  }
}

template <typename T, bool kWhole>
__global__ __launch_bounds__(kThreads) void unpack_kernel(const int8_t *__restrict__ codes, const float *__restrict__ scales, T *__restrict__ out, Shape s)
{
  Place p[kTurns];
  Eight<int8_t> q[kTurns];
  float scale[kTurns];
#pragma unroll
  for (int k = 0; k < kTurns; ++k) {
    p[k] = place<kWhole>(s, k);
    q[k] = load8(codes + p[k].at, p[k].have);
    scale[k] = p[k].have > 0 ? scales[p[k].unit] : 0.0f;
  }
#pragma unroll
  for (int k = 0; k < kTurns; ++k) {
    Eight<T> v;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      float value = static_cast<float>(q[k].v[i]) * scale[k];
      // the product is an fp32 number first: fused with the conversion to fp16 it would be rounded once, to another value in places
      asm("" : "+v"(value));
      v.v[i] = from_f32<T>(value);
    }
    store8(out + p[k].at, v, p[k].have);
  }
}

// hidden = silu_multiply(gate, up), bit for bit (silu(gate) is rounded to T first), and both inputs' checkpoints
template <typename T, bool kWhole>
__global__ __launch_bounds__(kThreads) void gate_kernel(const T *__restrict__ gate, const T *__restrict__ up, T *__restrict__ hidden,
                                                        int8_t *__restrict__ gate_codes, float *__restrict__ gate_scales, int8_t *__restrict__ up_codes,
                                                        float *__restrict__ up_scales, Shape s)
{
  Place p[kTurns];
  Eight<T> g[kTurns], u[kTurns];
#pragma unroll
  for (int k = 0; k < kTurns; ++k) {
    p[k] = place<kWhole>(s, k);
    g[k] = load8(gate + p[k].at, p[k].have);
    u[k] = load8(up + p[k].at, p[k].have);
  }
#pragma unroll
  for (int k = 0; k < kTurns; ++k) {
    Eight<T> h;
#pragma unroll
    for (int i = 0; i < kPer; ++i) h.v[i] = swiglu_fwd_one<T>(g[k].v[i], u[k].v[i]);
    store8(hidden + p[k].at, h, p[k].have);
    float gs, us;
    const Eight<int8_t> gq = quantise(g[k], gs), uq = quantise(u[k], us);
    store8(gate_codes + p[k].at, gq, p[k].have);
    store8(up_codes + p[k].at, uq, p[k].have);
    if (threadIdx.x % kLanes == 0 && p[k].have > 0) {
      gate_scales[p[k].unit] = gs;
      up_scales[p[k].unit] = us;
    }
  }
}

// g, u = the checkpoints' values in fp32; grad_up = T(d silu(g)), grad_gate = T(d u silu'(g)) and, where it is asked for,
// hidden = T(silu(g) u): each result is rounded once.  The logistic function's inverse is the instruction's, within a step.
template <typename T, bool kHidden, bool kWhole>
__global__ __launch_bounds__(kThreads) void gate_bwd_kernel(const int8_t *__restrict__ gate_codes, const float *__restrict__ gate_scales,
                                                            const int8_t *__restrict__ up_codes, const float *__restrict__ up_scales,
                                                            const T *__restrict__ grad, T *__restrict__ grad_gate, T *__restrict__ grad_up,
                                                            T *__restrict__ hidden, Shape s)
{
  Place p[kTurns];
  Eight<int8_t> gq[kTurns], uq[kTurns];
  Eight<T> d[kTurns];
  float gs[kTurns], us[kTurns];
#pragma unroll
  for (int k = 0; k < kTurns; ++k) {
    p[k] = place<kWhole>(s, k);
    gq[k] = load8(gate_codes + p[k].at, p[k].have);
    uq[k] = load8(up_codes + p[k].at, p[k].have);
    d[k] = load8(grad + p[k].at, p[k].have);
    gs[k] = p[k].have > 0 ? gate_scales[p[k].unit] : 0.0f;
    us[k] = p[k].have > 0 ? up_scales[p[k].unit] : 0.0f;
  }
#pragma unroll
  for (int k = 0; k < kTurns; ++k) {
    Eight<T> og, ou, oh;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const float g = static_cast<float>(gq[k].v[i]) * gs[k], u = static_cast<float>(uq[k].v[i]) * us[k], grad_h = to_f32<T>(d[k].v[i]);
      // e / (1 + e) and 1 / (1 + e) with e = exp(-|g|): the inverse stays in (0.5, 1], where exp(-g) would take it below the normal numbers
      const float e = expf(-fabsf(g)), high = __builtin_amdgcn_rcpf(1.0f + e), low = e * high;
      const float sg = g < 0.0f ? low : high, rest = g < 0.0f ? high : low, act = g * sg;
      ou.v[i] = from_f32<T>(grad_h * act);
      og.v[i] = from_f32<T>(grad_h * u * (sg * __builtin_fmaf(g, rest, 1.0f)));
      if constexpr (kHidden) oh.v[i] = from_f32<T>(act * u);
    }
    store8(grad_gate + p[k].at, og, p[k].have);
    store8(grad_up + p[k].at, ou, p[k].have);
    if constexpr (kHidden) store8(hidden + p[k].at, oh, p[k].have);
  }
}

// CAIFX_OK and `go` for a launch that has work, its shape and workgroups
int check(int64_t rows, int64_t cols, int dtype, bool missing, bool misaligned, bool &go, dim3 &grid, Shape &shape)
{
  go = false;
  if (!valid_dtype(dtype) || rows < 0 || cols < 0) return CAIFX_ERR_INVALID_ARGUMENT;
  if (rows == 0 || cols == 0) return CAIFX_OK;
  if (missing) return CAIFX_ERR_INVALID_ARGUMENT;
  if (misaligned) return CAIFX_ERR_MISALIGNED;
  const int64_t groups = (cols + kGroup - 1) / kGroup;
  // a grid has fewer than 2^32 threads
  if (rows > INT32_MAX || groups > INT32_MAX || groups > ((int64_t{1} << 24) - 1) * kUnits / rows) return CAIFX_ERR_UNSUPPORTED;
  const uint32_t g = static_cast<uint32_t>(groups);
  shape = Shape{static_cast<uint32_t>(rows * groups), g, g == 1 ? UINT32_MAX : static_cast<uint32_t>((uint64_t{1} << 32) / g), cols};
  grid = dim3(static_cast<unsigned>((rows * groups + kUnits - 1) / kUnits));
  go = true;
  return CAIFX_OK;
}

}  // namespace
}  // namespace caifx

using namespace caifx;

// one launch for the element type of `dtype`, and for rows of whole groups or others
#define CAIFX_BY_WIDTH(...)                                                 \
  if (cols % kGroup == 0) { constexpr bool kWhole = true; __VA_ARGS__; }            \
  else { constexpr bool kWhole = false; __VA_ARGS__; }
#define CAIFX_BY_TYPE(...)                                                  \
  switch (dtype) {                                                         \
    case CAIFX_F32: { typedef float T; CAIFX_BY_WIDTH(__VA_ARGS__) break; }         \
    case CAIFX_F16: { typedef f16_t T; CAIFX_BY_WIDTH(__VA_ARGS__) break; }         \
    default: { typedef bf16_t T; CAIFX_BY_WIDTH(__VA_ARGS__) break; }               \
  }

extern "C" {

int caifx_checkpoint_pack(const void *input, void *codes, float *scales, int64_t rows, int64_t cols, int dtype, caifx_stream_t stream)
{
  bool go;
  dim3 grid;
  Shape shape;
  const int st = check(rows, cols, dtype, !input || !codes || !scales, !aligned_to(input, dtype_size(dtype)) || !aligned_to(scales, 4), go, grid, shape);
  if (!go) return st;
  CAIFX_BY_TYPE(hipLaunchKernelGGL((pack_kernel<T, kWhole>), grid, dim3(kThreads), 0, as_stream(stream), static_cast<const T *>(input),
                                   static_cast<int8_t *>(codes), scales, shape));
  return launch_status();
}

int caifx_checkpoint_unpack(const void *codes, const float *scales, void *output, int64_t rows, int64_t cols, int dtype, caifx_stream_t stream)
{
  bool go;
  dim3 grid;
  Shape shape;
  const int st = check(rows, cols, dtype, !output || !codes || !scales, !aligned_to(output, dtype_size(dtype)) || !aligned_to(scales, 4), go, grid, shape);
  if (!go) return st;
  CAIFX_BY_TYPE(hipLaunchKernelGGL((unpack_kernel<T, kWhole>), grid, dim3(kThreads), 0, as_stream(stream), static_cast<const int8_t *>(codes), scales,
                                   static_cast<T *>(output), shape));
  return launch_status();
}

int caifx_silu_multiply_checkpoint(const void *gate, const void *up, void *hidden, void *gate_codes, float *gate_scales, void *up_codes,
                                   float *up_scales, int64_t rows, int64_t cols, int dtype, caifx_stream_t stream)
{
  bool go;
  dim3 grid;
  Shape shape;
  const size_t es = dtype_size(dtype);
  const int st = check(rows, cols, dtype, !gate || !up || !hidden || !gate_codes || !gate_scales || !up_codes || !up_scales,
                       !aligned_to(gate, es) || !aligned_to(up, es) || !aligned_to(hidden, es) || !aligned_to(gate_scales, 4) || !aligned_to(up_scales, 4),
                       go, grid, shape);
  if (!go) return st;
  CAIFX_BY_TYPE(hipLaunchKernelGGL((gate_kernel<T, kWhole>), grid, dim3(kThreads), 0, as_stream(stream), static_cast<const T *>(gate), static_cast<const T *>(up),
                                   static_cast<T *>(hidden), static_cast<int8_t *>(gate_codes), gate_scales, static_cast<int8_t *>(up_codes), up_scales,
                                   shape));
  return launch_status();
}

int caifx_swiglu_backward_checkpoint(const void *gate_codes, const float *gate_scales, const void *up_codes, const float *up_scales,
                                     const void *grad_hidden, void *grad_gate, void *grad_up, void *hidden, int64_t rows, int64_t cols, int dtype,
                                     caifx_stream_t stream)
{
  bool go;
  dim3 grid;
  Shape shape;
  const size_t es = dtype_size(dtype);
  const int st = check(rows, cols, dtype, !gate_codes || !gate_scales || !up_codes || !up_scales || !grad_hidden || !grad_gate || !grad_up,
                       !aligned_to(gate_scales, 4) || !aligned_to(up_scales, 4) || !aligned_to(grad_hidden, es) || !aligned_to(grad_gate, es) ||
                           !aligned_to(grad_up, es) || !aligned_to(hidden, es), go, grid, shape);
  if (!go) return st;
  hipStream_t s = as_stream(stream);
#define CAIFX_GO(kHidden)                                                                                                                          \
  hipLaunchKernelGGL((gate_bwd_kernel<T, kHidden, kWhole>), grid, dim3(kThreads), 0, s, static_cast<const int8_t *>(gate_codes), gate_scales,              \
                     static_cast<const int8_t *>(up_codes), up_scales, static_cast<const T *>(grad_hidden), static_cast<T *>(grad_gate),           \
                     static_cast<T *>(grad_up), static_cast<T *>(hidden), shape)
  if (hidden) {
    CAIFX_BY_TYPE(CAIFX_GO(true));
  } else {
    CAIFX_BY_TYPE(CAIFX_GO(false));
  }
#undef CAIFX_GO
  return launch_status();
}

}  // extern "C"
