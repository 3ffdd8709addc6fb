// Microscaled 4-bit floating point: a tensor put into codes and scales, brought back, and laid out for the products that take it.
//
//   byte = clamp(floor(log2 max|x|) - 2, -127, 127) + 127, the exponent field of the largest magnitude less two (0 for a block of zeros)
//   code = the nearest of 0, 1/2, 1, 3/2, 2, 3, 4, 6 to |x| 2^(127 - byte), ties to the even mantissa, and the sign
//
// The conversions are gfx950's own (v_cvt_scalef32_pk_fp4_f32 and back), which round and saturate exactly so for every scale.  Bound by
// memory: four lanes take a block, eight values each, so that a lane's part is one 16-byte access of a 16-bit type (14336 x 4096 in bf16:
// quantised in 25.5 us and brought back in 22.4, 5.8 and 6.6 TB/s, in part from the memory-side cache).
#include "caifx_mxfp4.hpp"

#include <type_traits>

namespace caifx {
namespace {

constexpr int kBlock = CAIFX_MXFP4_BLOCK;
constexpr int kPer = 8;                               // values of a lane
constexpr int kLanes = kBlock / kPer;                 // lanes of a block
constexpr int kThreads = 256;
constexpr int kUnits = kThreads / kLanes;             // blocks of a workgroup

template <typename T> struct Eight { T v[kPer]; };
// the same as whole 16-byte accesses at any address (as eight values the compiler may pull one out of them, two accesses then)
template <typename T> struct Pieces {
  typedef uint32_t piece_t __attribute__((ext_vector_type(4), aligned(2), may_alias));
  piece_t p[sizeof(Eight<T>) / 16];
};

// eight values from p, `have` of them in the row (zeros for the others); any alignment of T
template <typename T> __device__ __forceinline__ Eight<T> load8(const T *p, int have)
{
  Eight<T> e;
  if (have >= kPer) {
    const Pieces<T> pieces = *reinterpret_cast<const Pieces<T> *>(p);
    __builtin_memcpy(&e, &pieces, sizeof e);
  } else {
#pragma unroll
    for (int i = 0; i < kPer; ++i) e.v[i] = i < have ? p[i] : T(0);
  }
  return e;
}
template <typename T> __device__ __forceinline__ void store8(T *p, const Eight<T> &e, int have)
{
  if (have >= kPer) {
    Pieces<T> pieces;
    __builtin_memcpy(&pieces, &e, sizeof e);
    *reinterpret_cast<Pieces<T> *>(p) = pieces;
  } else {
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      if (i < have) p[i] = e.v[i];
  }
}

// rows x cols in blocks of a row.  Rows of whole blocks need no row: their blocks stand in one line.
struct Shape {
  uint32_t units, blocks, magic;                      // blocks in all, of a row, floor(2^32 / blocks) or 2^32 - 1
  int64_t cols;
};
struct Place {
  int64_t at;                                         // flat index of a lane's first value
  uint32_t unit;                                      // flat index of its block
  int have;                                           // values inside the row, 0 past the last block
};
template <bool kWhole> __device__ __forceinline__ Place place(const Shape &s)
{
  const uint32_t unit = blockIdx.x * kUnits + threadIdx.x / kLanes, in = (threadIdx.x % kLanes) * kPer;
  if constexpr (kWhole) {
    return {static_cast<int64_t>(unit) * kBlock + in, unit, unit < s.units ? kPer : 0};
  } else {
    uint32_t row = __umulhi(unit, s.magic);           // the quotient or one less
    if (unit - row * s.blocks >= s.blocks) ++row;
    const int64_t col = static_cast<int64_t>(unit - row * s.blocks) * kBlock + in, left = unit < s.units ? s.cols - col : 0;
    return {row * s.cols + col, unit, left >= kPer ? kPer : (left > 0 ? static_cast<int>(left) : 0)};
  }
}

// (One block for four lanes: four of them, asked for together, are slower at every size, bf16, 28672 x 8192 115 us instead of 105, 512 x 4096 3.9
// instead of 3.1.)
template <typename T, bool kWhole>
__global__ __launch_bounds__(kThreads) void quantize_kernel(const T *__restrict__ x, uint32_t *__restrict__ codes, uint8_t *__restrict__ scales, Shape s)
{
  const Place p = place<kWhole>(s);
  const Eight<T> v = load8(x + p.at, p.have);
  float f[kPer];
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    f[i] = to_f32<T>(v.v[i]);
    const uint32_t b = __builtin_bit_cast(uint32_t, f[i]) & 0x7FFFFFFFu;      // magnitudes in the order of their bits
    top = top > b ? top : b;
  }
  auto with = [&](uint32_t w) { top = top > w ? top : w; };
  with(__builtin_amdgcn_mov_dpp(top, 0xB1, 0xF, 0xF, true));            // lanes 1 0 3 2
  with(__builtin_amdgcn_mov_dpp(top, 0x4E, 0xF, 0xF, true));            // lanes 2 3 0 1
  const uint32_t exponent = top >> 23;
  const bool finite = exponent < 255;
  const uint32_t byte = finite ? (exponent > 2 ? exponent - 2 : 0) : 255;
  const float scale = mxfp4_scale(byte);
  uint32_t c = 0;
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, f[0], f[1], scale, 0);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, f[2], f[3], scale, 1);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, f[4], f[5], scale, 2);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, f[6], f[7], scale, 3);
  if (p.unit < s.units) {
    codes[static_cast<int64_t>(p.unit) * kLanes + threadIdx.x % kLanes] = finite ? c : 0u;
    if (threadIdx.x % kLanes == 0) scales[p.unit] = static_cast<uint8_t>(byte);
  }
}

template <typename T> __device__ __forceinline__ Eight<T> values8(uint32_t codes, float scale)
{
  if constexpr (sizeof(T) == 2) {
    return __builtin_bit_cast(Eight<T>, mxfp4_eight<T>(codes, scale));
  } else {
    typedef float pair_t __attribute__((ext_vector_type(2)));
    Eight<T> e;
    const pair_t a = __builtin_bit_cast(pair_t, __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, scale, 0)),
                 b = __builtin_bit_cast(pair_t, __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, scale, 1)),
                 c = __builtin_bit_cast(pair_t, __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, scale, 2)),
                 d = __builtin_bit_cast(pair_t, __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, scale, 3));
    e.v[0] = a[0], e.v[1] = a[1], e.v[2] = b[0], e.v[3] = b[1], e.v[4] = c[0], e.v[5] = c[1], e.v[6] = d[0], e.v[7] = d[1];
    return e;
  }
}

template <typename T, bool kWhole>
__global__ __launch_bounds__(kThreads) void dequantize_kernel(const uint32_t *__restrict__ codes, const uint8_t *__restrict__ scales, T *__restrict__ out, Shape s)
{
  const Place p = place<kWhole>(s);
  const uint32_t unit = p.unit < s.units ? p.unit : s.units - 1;      // (nothing of it is stored)
  const uint32_t c = codes[static_cast<int64_t>(unit) * kLanes + threadIdx.x % kLanes], byte = scales[unit];
  store8(out + p.at, values8<T>(c, mxfp4_scale(byte)), p.have);
}

// ------------------------------------------------------------------ operands laid out for the products
struct Source {
  const void *p;             // MX codes, or values of a float type
  const uint8_t *scales;
  int64_t rows, cols, blocks;
};
struct Mx {};                // a source in microscaled 4 bits
struct Sources {             // one or two of one shape, a launch's last extent
  Source g[2];
};

// eight values (n, k .. k + 7) of a source in CT, zeros outside; k is a multiple of 8.  kInside: all eight are inside, nothing is tested (behind
// a test the compiler waits for one access before it asks for the next).
template <typename S, typename CT, bool kInside = false> __device__ __forceinline__ u32x4_t source8(const Source &g, int64_t n, int64_t k)
{
  if (!kInside && (n >= g.rows || k >= g.cols)) return u32x4_t{0, 0, 0, 0};
  const int64_t left = kInside ? kPer : g.cols - k;
  if constexpr (sizeof(S) == 1) {
    const int64_t block = n * g.blocks + (k >> 5);
    uint32_t c = *reinterpret_cast<const uint32_t *>(static_cast<const uint8_t *>(g.p) + block * 16 + ((k & 31) >> 1));
    if (left < kPer) c &= (1u << (4 * static_cast<int>(left))) - 1u;      // (codes behind the last column count for nothing)
    u32x4_t v = mxfp4_eight<CT>(c, mxfp4_scale(g.scales[block]));
    if (left < kPer) {
      // under a scale of NaN also a code of zero is a NaN
      Eight<uint16_t> e = __builtin_bit_cast(Eight<uint16_t>, v);
#pragma unroll
      for (int i = 0; i < kPer; ++i)
        if (i >= left) e.v[i] = 0;
      v = __builtin_bit_cast(u32x4_t, e);
    }
    return v;
  } else {
    const Eight<S> e = load8(static_cast<const S *>(g.p) + n * g.cols + k, left < kPer ? static_cast<int>(left) : kPer);
    if constexpr (__is_same(S, CT)) {
      return __builtin_bit_cast(u32x4_t, e);
    } else {
      u32x4_t v;
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = pack2<CT>(to_f32<S>(e.v[2 * i]), to_f32<S>(e.v[2 * i + 1]));
      return v;
    }
  }
}

// [rows, cols] as dense rows of CT, `pitch` long with zeros behind the last column; the second source's rows behind the first's (codes of 11008 x 4096:
// 25 us, 4.5 TB/s)
template <typename S, typename CT>
__global__ __launch_bounds__(kThreads) void dense_kernel(Sources two, CT *__restrict__ out, int64_t pitch)
{
  const Source g = two.g[blockIdx.z];
  out += blockIdx.z * g.rows * pitch;
  const int64_t p = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  if (p * kPer >= pitch) return;
  for (int64_t n = blockIdx.y; n < g.rows; n += gridDim.y) *reinterpret_cast<u32x4_t *>(out + n * pitch + p * kPer) = source8<S, CT>(g, n, p * kPer);
}

// the same transposed: [cols] rows `stride` long with the rows' values, zeros up to a multiple of 64; the second source's `second` values on.
// A workgroup takes 64 rows x 256 columns: a thread reads eight columns of eight rows and lays them out in LDS as rows of 64 n, which
// are then written in whole 128-byte lines; workgroups that run together take neighbouring rows, lines beside each other (codes of 11008 x 4096: 25 us,
// 4.5 TB/s).  The piece position is rotated by the thread's columns so that the eight lanes of a group use different banks.
template <typename S, typename CT>
__global__ __launch_bounds__(kThreads) void dense_transposed_kernel(Sources two, CT *__restrict__ out, int64_t stride, int64_t second)
{
  const Source g = two.g[blockIdx.z];
  out += blockIdx.z * second;
  __shared__ __attribute__((aligned(16))) unsigned char tile[256 * 128];
  const int kl = threadIdx.x & 31, ng = threadIdx.x >> 5;
  const int64_t n0 = static_cast<int64_t>(blockIdx.x) * 64, k0 = static_cast<int64_t>(blockIdx.y) * 256;
  Eight<uint16_t> e[8];
  if (n0 + 64 <= g.rows && k0 + 256 <= g.cols) {
#pragma unroll
    for (int r = 0; r < 8; ++r) e[r] = __builtin_bit_cast(Eight<uint16_t>, source8<S, CT, true>(g, n0 + 8 * ng + r, k0 + 8 * kl));
  } else {
#pragma unroll
    for (int r = 0; r < 8; ++r) e[r] = __builtin_bit_cast(Eight<uint16_t>, source8<S, CT>(g, n0 + 8 * ng + r, k0 + 8 * kl));
  }
#pragma unroll
  for (int c = 0; c < 8; ++c) {
    Eight<uint16_t> t;
#pragma unroll
    for (int r = 0; r < 8; ++r) t.v[r] = e[r].v[c];
    *reinterpret_cast<u32x4_t *>(tile + (8 * kl + c) * 128 + (((ng + kl) & 7) << 4)) = __builtin_bit_cast(u32x4_t, t);
  }
  __syncthreads();
  const int piece = threadIdx.x & 7;
#pragma unroll
  for (int it = 0; it < 8; ++it) {
    const int k = it * 32 + (threadIdx.x >> 3);
    if (k0 + k >= g.cols) continue;
    const u32x4_t v = *reinterpret_cast<const u32x4_t *>(tile + k * 128 + (((piece + (k >> 3)) & 7) << 4));
    *reinterpret_cast<u32x4_t *>(out + (k0 + k) * stride + n0 + 8 * piece) = v;
  }
}

// Eight values (m, k .. k + 7) of activations as three bf16 pieces each.  Zeros outside.
template <typename S> __device__ __forceinline__ void pieces8(const Source &g, int64_t m, int64_t k, Eight<uint16_t> (&piece)[3])
{
  const int64_t left = m < g.rows ? g.cols - k : 0;
  const Eight<S> e = load8(static_cast<const S *>(g.p) + m * g.cols + k, left > 0 ? (left < kPer ? static_cast<int>(left) : kPer) : 0);
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    uint32_t bits[3];
    pieces_of_f32(to_f32<S>(e.v[i]), bits);
#pragma unroll
    for (int p = 0; p < 3; ++p) piece[p].v[i] = static_cast<uint16_t>(bits[p] >> 16);
  }
}

// The pieces of fp32 activations as three dense matrices [rows, pitch], one behind the other, zeros behind the last column; the second
// source's behind the first's.
template <typename S>
__global__ __launch_bounds__(kThreads) void pieces_kernel(Sources two, uint16_t *__restrict__ out, int64_t pitch)
{
  const Source g = two.g[blockIdx.z];
  const int64_t piece_size = g.rows * pitch, p = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  out += blockIdx.z * 3 * piece_size;
  if (p * kPer >= pitch) return;
  for (int64_t m = blockIdx.y; m < g.rows; m += gridDim.y) {
    Eight<uint16_t> piece[3];
    pieces8<S>(g, m, p * kPer, piece);
#pragma unroll
    for (int i = 0; i < 3; ++i) *reinterpret_cast<u32x4_t *>(out + i * piece_size + m * pitch + p * kPer) = __builtin_bit_cast(u32x4_t, piece[i]);
  }
}

// Activations in the order in which the row kernels read them: for each tile of 16 rows, chunk of 256 reduction elements and piece, eight
// kilobytes of which the u-th holds every lane's operand of instruction u.  fp32 in P = 3 pieces.
template <typename S, typename CT, int P>
__global__ __launch_bounds__(kThreads) void pack_rows_kernel(Sources two, unsigned char *__restrict__ out, int own, int chunks)
{
  const Source g = two.g[blockIdx.z];
  const int c = static_cast<int>(blockIdx.x >> 1), chunk0 = static_cast<int>(blockIdx.z) * own;
  for (int64_t tile = blockIdx.y; tile * 16 < g.rows; tile += gridDim.y) {
    unsigned char *to = out + (tile * chunks + chunk0 + c) * (P * 8 * 1024);
    const int at = static_cast<int>(blockIdx.x & 1) * kThreads + threadIdx.x, lane = at & 63, u = at >> 6;
    const int64_t m = tile * 16 + (lane & 15), k = static_cast<int64_t>(c) * kRowsChunk + 32 * u + 8 * (lane >> 4);
    if constexpr (P == 1) {
      *reinterpret_cast<u32x4_t *>(to + at * 16) = source8<S, CT>(g, m, k);
    } else {
      Eight<uint16_t> piece[3];
      pieces8<S>(g, m, k, piece);
#pragma unroll
      for (int p = 0; p < 3; ++p) *reinterpret_cast<u32x4_t *>(to + p * 8192 + at * 16) = __builtin_bit_cast(u32x4_t, piece[p]);
    }
  }
}

// The gating's backward: grad_up = T(d g s), grad_gate = T(d u s (1 + g (1 - s))), s = 1 / (1 + exp(-g)).  Bound by memory: five tensors
// (bf16, 2048 x 11008 42 us, 5.3 TB/s).  The results are rounded before the products that they go into: dx is the product of the gradients that
// the caller gets, as where the projections' gradients are taken one after the other.  In bf16 dx is 2.35e-3 from 64 bits so (2-norm; 2048 rows, N =
// 11008, K = 4096), 1.66e-3, its own rounding alone, with unrounded factors; those would be two bf16 pieces each, twice the matrix
// instructions, 245 us more on 360.
template <typename T>
__global__ __launch_bounds__(kThreads) void gating_backward_kernel(const T *__restrict__ grad, const T *__restrict__ gate, const T *__restrict__ up,
                                                                   T *__restrict__ grad_gate, T *__restrict__ grad_up, int64_t n)
{
  for (int64_t at = (static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x) * kPer; at < n; at += static_cast<int64_t>(gridDim.x) * (kThreads * kPer)) {
    const int have = n - at < kPer ? static_cast<int>(n - at) : kPer;
    const Eight<T> d = load8(grad + at, have), gt = load8(gate + at, have), ut = load8(up + at, have);
    Eight<T> og, ou;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const float g = to_f32<T>(gt.v[i]), u = to_f32<T>(ut.v[i]), h = to_f32<T>(d.v[i]);
      // e / (1 + e) and 1 / (1 + e) with e = exp(-|g|): the inverse stays in (0.5, 1], where exp(-g) would take it below the normal numbers
      const float e = expf(-fabsf(g)), high = __builtin_amdgcn_rcpf(1.0f + e), low = e * high;
      const float s = g < 0.0f ? low : high, rest = g < 0.0f ? high : low;
      ou.v[i] = from_f32<T>(h * (g * s));
      og.v[i] = from_f32<T>(h * u * (s * __builtin_fmaf(g, rest, 1.0f)));
    }
    store8(grad_gate + at, og, have);
    store8(grad_up + at, ou, have);
  }
}

Sources sources(const Operand &a)
{
  const int64_t blocks = (a.cols + kBlock - 1) / kBlock;
  return Sources{{Source{a.p[0], static_cast<const uint8_t *>(a.scales[0]), a.rows, a.cols, blocks}, Source{a.p[1], static_cast<const uint8_t *>(a.scales[1]), a.rows, a.cols, blocks}}};
}
unsigned rows_grid(int64_t rows) { return static_cast<unsigned>(rows < 65535 ? rows : 65535); }

}  // namespace

// one call for the source's and the target's type
#define CAIFX_BY_SOURCE(...)                                                    \
  switch (a.kind) {                                                             \
    case OPERAND_MX: { typedef Mx S; __VA_ARGS__; break; }                      \
    case CAIFX_F32: { typedef float S; __VA_ARGS__; break; }                    \
    case CAIFX_F16: { typedef f16_t S; __VA_ARGS__; break; }                    \
    default: { typedef bf16_t S; __VA_ARGS__; break; }                          \
  }
#define CAIFX_BY_TARGET(...)                                                    \
  if (to == CAIFX_BF16) { typedef bf16_t CT; CAIFX_BY_SOURCE(__VA_ARGS__) }     \
  else { typedef f16_t CT; CAIFX_BY_SOURCE(__VA_ARGS__) }

int operand_dense(const Operand &a, int to, void *out, int64_t pitch, hipStream_t s)
{
  const dim3 grid(static_cast<unsigned>((pitch / kPer + kThreads - 1) / kThreads), rows_grid(a.rows), static_cast<unsigned>(a.count));
  CAIFX_BY_TARGET(hipLaunchKernelGGL((dense_kernel<S, CT>), grid, dim3(kThreads), 0, s, sources(a), static_cast<CT *>(out), pitch))
  return launch_status();
}

int operand_transposed(const Operand &a, int to, void *out, int64_t pitch, int64_t stride, int64_t second, hipStream_t s)
{
  const dim3 grid(static_cast<unsigned>(pitch / 64), static_cast<unsigned>((a.cols + 255) / 256), static_cast<unsigned>(a.count));
  CAIFX_BY_TARGET(hipLaunchKernelGGL((dense_transposed_kernel<S, CT>), grid, dim3(kThreads), 0, s, sources(a), static_cast<CT *>(out), stride, second))
  return launch_status();
}

int operand_pieces(const Operand &a, void *out, int64_t pitch, hipStream_t s)
{
  const dim3 grid(static_cast<unsigned>((pitch / kPer + kThreads - 1) / kThreads), rows_grid(a.rows), static_cast<unsigned>(a.count));
  if (a.kind == CAIFX_F32) hipLaunchKernelGGL((pieces_kernel<float>), grid, dim3(kThreads), 0, s, sources(a), static_cast<uint16_t *>(out), pitch);
  else hipLaunchKernelGGL((pieces_kernel<f16_t>), grid, dim3(kThreads), 0, s, sources(a), static_cast<uint16_t *>(out), pitch);
  return launch_status();
}

int operand_rows(const Operand &a, int to, void *out, int chunks, hipStream_t s)
{
  const int own = static_cast<int>((a.cols + kRowsChunk - 1) / kRowsChunk);
  const dim3 grid(static_cast<unsigned>(2 * own), rows_grid((a.rows + 15) / 16), static_cast<unsigned>(a.count));
  unsigned char *o = static_cast<unsigned char *>(out);
  if (to == CAIFX_F32) {
    if (a.kind == CAIFX_F32) hipLaunchKernelGGL((pack_rows_kernel<float, bf16_t, 3>), grid, dim3(kThreads), 0, s, sources(a), o, own, chunks);
    else hipLaunchKernelGGL((pack_rows_kernel<f16_t, bf16_t, 3>), grid, dim3(kThreads), 0, s, sources(a), o, own, chunks);
  } else {
    CAIFX_BY_TARGET(hipLaunchKernelGGL((pack_rows_kernel<S, CT, 1>), grid, dim3(kThreads), 0, s, sources(a), o, own, chunks))
  }
  return launch_status();
}

int gating_backward(const void *grad, const void *gate, const void *up, void *grad_gate, void *grad_up, int64_t n, int dtype, hipStream_t s)
{
  const int64_t groups = (n + kThreads * kPer - 1) / (kThreads * kPer);
  const dim3 grid(static_cast<unsigned>(groups < (1 << 22) ? groups : (1 << 22)));
  const auto go = [&](auto type_) {
    typedef decltype(type_) T;
    hipLaunchKernelGGL((gating_backward_kernel<T>), grid, dim3(kThreads), 0, s, static_cast<const T *>(grad), static_cast<const T *>(gate),
                       static_cast<const T *>(up), static_cast<T *>(grad_gate), static_cast<T *>(grad_up), n);
  };
  if (dtype == CAIFX_BF16) go(bf16_t{});
  else if (dtype == CAIFX_F16) go(f16_t{});
  else go(float{});
  return launch_status();
}

namespace {

// Sums of a shared reduction.  Few values and many parts: a wave of its own for 64 lanes' values, sixteen parts on their way at once.
template <typename T, int V> __global__ __launch_bounds__(256) void join_kernel(const float *__restrict__ partial, int parts, int64_t n, T *y, const T *addend)
{
  constexpr int kTogether = 16;
  struct alignas(V * sizeof(float)) Sums { float e[V]; };
  struct alignas(V * sizeof(T)) Values { T e[V]; };
  const int64_t i = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) * V;
  if (i >= n) return;
  Sums sum{};
  for (int from = 0; from < parts; from += kTogether) {
    Sums part[kTogether];
#pragma unroll
    for (int p = 0; p < kTogether; ++p) part[p] = *reinterpret_cast<const Sums *>(partial + (from + p < parts ? from + p : parts - 1) * n + i);
#pragma unroll
    for (int p = 0; p < kTogether; ++p)
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (from + p < parts) sum.e[e] = from + p == 0 ? part[p].e[e] : sum.e[e] + part[p].e[e];
  }
  Values out;
  if (addend) {
    const Values add = *reinterpret_cast<const Values *>(addend + i);
#pragma unroll
    for (int e = 0; e < V; ++e) out.e[e] = from_f32<T>(to_f32<T>(from_f32<T>(sum.e[e])) + to_f32<T>(add.e[e]));
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e) out.e[e] = from_f32<T>(sum.e[e]);
  }
  *reinterpret_cast<Values *>(y + i) = out;
}

template <typename T> int join(const float *partial, int parts, int64_t n, void *y_, const void *addend_, hipStream_t s)
{
  T *y = static_cast<T *>(y_);
  const T *addend = static_cast<const T *>(addend_);
  const bool four = n % 4 == 0 && aligned_to(y, 4 * sizeof(T)) && aligned_to(addend, 4 * sizeof(T));
  const int64_t lanes = four ? n / 4 : n;
  const int block = lanes < 65536 ? 64 : 256;
  const dim3 grid(static_cast<unsigned>((lanes + block - 1) / block));
  if (four) hipLaunchKernelGGL((join_kernel<T, 4>), grid, dim3(block), 0, s, partial, parts, n, y, addend);
  else hipLaunchKernelGGL((join_kernel<T, 1>), grid, dim3(block), 0, s, partial, parts, n, y, addend);
  return launch_status();
}

// CAIFX_OK and `go` for a launch that has work, its shape and workgroups
int check(int64_t rows, int64_t cols, int dtype, bool missing, bool misaligned, bool &go, dim3 &grid, Shape &shape)
{
  go = false;
  if (!valid_dtype(dtype) || rows < 0 || cols < 0) return CAIFX_ERR_INVALID_ARGUMENT;
  if (rows == 0 || cols == 0) return CAIFX_OK;
  if (missing) return CAIFX_ERR_INVALID_ARGUMENT;
  if (misaligned) return CAIFX_ERR_MISALIGNED;
  const int64_t blocks = cols / kBlock + (cols % kBlock != 0);
  if (rows > (1 << 29) || blocks > (1 << 29) || rows * blocks > (1 << 29)) return CAIFX_ERR_UNSUPPORTED;
  const uint32_t b = static_cast<uint32_t>(blocks);
  shape = Shape{static_cast<uint32_t>(rows * blocks), b, b == 1 ? UINT32_MAX : static_cast<uint32_t>((uint64_t{1} << 32) / b), cols};
  grid = dim3(static_cast<unsigned>((rows * blocks + kUnits - 1) / kUnits));
  go = true;
  return CAIFX_OK;
}

}  // namespace

int join_sums(const float *partial, int parts, int64_t n, void *y, int y_dtype, const void *addend, hipStream_t s)
{
  if (y_dtype == CAIFX_F32) return join<float>(partial, parts, n, y, addend, s);
  if (y_dtype == CAIFX_F16) return join<f16_t>(partial, parts, n, y, addend, s);
  return join<bf16_t>(partial, parts, n, y, addend, s);
}

}  // namespace caifx

using namespace caifx;

// one launch for the element type of `dtype`, and for rows of whole blocks or others
#define CAIFX_BY_WIDTH(...)                                                         \
  if (cols % kBlock == 0) { constexpr bool kWhole = true; __VA_ARGS__; }            \
  else { constexpr bool kWhole = false; __VA_ARGS__; }
#define CAIFX_BY_TYPE(...)                                                          \
  switch (dtype) {                                                                  \
    case CAIFX_F32: { typedef float T; CAIFX_BY_WIDTH(__VA_ARGS__) break; }         \
    case CAIFX_F16: { typedef f16_t T; CAIFX_BY_WIDTH(__VA_ARGS__) break; }         \
    default: { typedef bf16_t T; CAIFX_BY_WIDTH(__VA_ARGS__) break; }               \
  }

extern "C" {

int caifx_mxfp4_quantize(const void *input, void *codes, void *scales, int64_t rows, int64_t cols, int dtype, caifx_stream_t stream)
{
  bool go;
  dim3 grid;
  Shape shape;
  const int st = check(rows, cols, dtype, !input || !codes || !scales, !aligned_to(input, dtype_size(dtype)) || !aligned_to(codes, 16), go, grid, shape);
  if (!go) return st;
  CAIFX_BY_TYPE(hipLaunchKernelGGL((quantize_kernel<T, kWhole>), grid, dim3(kThreads), 0, as_stream(stream), static_cast<const T *>(input),
                                   static_cast<uint32_t *>(codes), static_cast<uint8_t *>(scales), shape));
  return launch_status();
}

int caifx_mxfp4_dequantize(const void *codes, const void *scales, void *output, int64_t rows, int64_t cols, int dtype, caifx_stream_t stream)
{
  bool go;
  dim3 grid;
  Shape shape;
  const int st = check(rows, cols, dtype, !output || !codes || !scales, !aligned_to(output, dtype_size(dtype)) || !aligned_to(codes, 16), go, grid, shape);
  if (!go) return st;
  CAIFX_BY_TYPE(hipLaunchKernelGGL((dequantize_kernel<T, kWhole>), grid, dim3(kThreads), 0, as_stream(stream), static_cast<const uint32_t *>(codes),
                                   static_cast<const uint8_t *>(scales), static_cast<T *>(output), shape));
  return launch_status();
}

}  // extern "C"
