// Products with up to some hundred rows of activations and a weight in microscaled 4 bits, or dense in the 16-bit compute type:
//   y[m, n] = sum_k x[m, k] w[n, k]       and, over two weights (gate and up) at once, hidden = silu(x w0^T) * (x w1^T).
//
// Bound by memory with few rows (the weight's bytes), by the L1 from some dozens on.  A workgroup of eight waves owns 16 MT rows and
// 16 NT weight rows of the result; the waves take the chunks of 256 reduction elements in turn and their sums meet in LDS at the end.
// So every wave streams its part of the weight rows straight into matrix-core operands, no wave waits for another in between, and a
// launch of a usual weight has all of it on its way at once.  The reduction indices inside a chunk are permuted such that a lane's 16
// bytes of codes are one block of 32 values of one weight row: lane (j, q) of v_mfma_f32_16x16x32 holds block q (then q + 4) of row j,
// instruction i takes its values 8 i .. 8 i + 7, and the activations follow that order.  The codes become operands by
// v_cvt_scalef32_pk_{bf16,f16}_fp4 with the block's scale: exact in bf16, in fp16 rounded like any weight that is cast to it.  Where the
// activations have 4 bits too, the same blocks go into v_mfma_scale_f32_16x16x128_f8f6f4 as they are.
#pragma once

#include "caifx_wide.hpp"

namespace caifx {

constexpr int kRowsChunk = 256;              // reduction elements of a chunk: 128 bytes of codes of a weight row
constexpr int kRowsWaves = 8;

struct RowsArgs {
  const void *x;          // direct: [M, x_pitch] of the compute type; packed: see pack_rows_kernel
  int64_t x_pitch;
  const void *w[2];       // MX codes or dense rows of the compute type
  const uint8_t *s[2];    // MX scales
  const uint8_t *xs;      // both in 4 bits: scales of x, whose codes are rows of w_pitch bytes
  int64_t M, N, R;        // R: elements of the reduction (direct: a multiple of 8)
  int64_t blocks;         // MX blocks of a weight row
  int64_t w_pitch;        // bytes of a weight row
  int chunks, tiles;      // chunks of the reduction, row tiles of 16 in the packed activations
  void *y;                // [M, N] result, or hidden
  void *gate, *up;        // two weights: kept projections, or null
  const void *addend;     // one weight: y = T(float(T(acc)) + float(addend))
  int y_dtype;
};

enum { ROWS_MX = 0, ROWS_DENSE = 1, ROWS_BOTH = 2 };      // ROWS_BOTH: weight and activations in microscaled 4 bits
// first of the eight reduction elements that lane group q holds for instruction u (0 .. 7) of a chunk
template <int kWeight> __device__ __forceinline__ int rows_element(int u, int q)
{
  return kWeight == ROWS_MX ? 128 * (u >> 2) + 32 * q + 8 * (u & 3) : 32 * u + 8 * q;
}

// one block of 32 values of each of 16 rows and 16 columns per lane group, in 4 bits with their scales
__device__ __forceinline__ floatx4_t mfma_micro(u32x4_t a, u32x4_t b, floatx4_t c, uint32_t sa, uint32_t sb)
{
  typedef int eight_t __attribute__((ext_vector_type(8)));
  const eight_t va = {static_cast<int>(a[0]), static_cast<int>(a[1]), static_cast<int>(a[2]), static_cast<int>(a[3]), 0, 0, 0, 0},
                vb = {static_cast<int>(b[0]), static_cast<int>(b[1]), static_cast<int>(b[2]), static_cast<int>(b[3]), 0, 0, 0, 0};
  typedef float four_t __attribute__((ext_vector_type(4)));
  return __builtin_bit_cast(floatx4_t, __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(va, vb, __builtin_bit_cast(four_t, c), 4, 4, 0, static_cast<int>(sa), 0,
                                                                                       static_cast<int>(sb)));
}

template <typename CT> struct Mfma16;
template <> struct Mfma16<bf16_t> {
  static __device__ __forceinline__ floatx4_t run(u32x4_t a, u32x4_t b, floatx4_t c)
  {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
  }
};
template <> struct Mfma16<f16_t> {
  static __device__ __forceinline__ floatx4_t run(u32x4_t a, u32x4_t b, floatx4_t c)
  {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
  }
};

// P: pieces of an activation (3: fp32).  NW: weights (2: gate and up; the first half of the NT column tiles is gate's).
template <typename CT, int P, int kWeight, int NW, int MT, int NT, bool kDirect>
__global__ __launch_bounds__(kRowsWaves * 64) void rows_kernel(RowsArgs g)
{
  constexpr int NC = NT / NW;                // column tiles of one weight
  constexpr bool kMicro = kWeight != ROWS_DENSE, kBoth = kWeight == ROWS_BOTH;
  constexpr int WV = kMicro ? 1 : 4, XV = kBoth ? 1 : 4;      // 16-byte pieces of a column tile and of a row tile per half chunk
  static_assert(NT % NW == 0 && (P == 1 || !kDirect), "");
  __shared__ floatx4_t sums[kRowsWaves / 2][MT * NT][64];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int j = lane & 15, q = lane >> 4;
  const int64_t n0 = static_cast<int64_t>(blockIdx.x) * (16 * NC), m0 = static_cast<int64_t>(blockIdx.y) * (16 * MT);

  // what each lane reads from: rows past the end are the last one again, and are not stored
  const uint8_t *wp[NT];
  const uint8_t *sp[NT];
#pragma unroll
  for (int c = 0; c < NT; ++c) {
    const int v = c / NC;
    int64_t n = n0 + (c % NC) * 16 + j;
    n = n < g.N ? n : g.N - 1;
    wp[c] = static_cast<const uint8_t *>(g.w[v]) + n * g.w_pitch;
    if constexpr (kMicro) sp[c] = g.s[v] + n * g.blocks;
  }
  const uint8_t *xp[MT];
  const uint8_t *xsp[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) {
    if constexpr (kBoth) {
      int64_t m = m0 + t * 16 + j;
      m = m < g.M ? m : g.M - 1;
      xp[t] = static_cast<const uint8_t *>(g.x) + m * g.w_pitch;
      xsp[t] = g.xs + m * g.blocks;
    } else if constexpr (kDirect) {
      int64_t m = m0 + t * 16 + j;
      m = m < g.M ? m : g.M - 1;
      xp[t] = static_cast<const uint8_t *>(g.x) + m * g.x_pitch * 2;
    } else {
      int64_t tile = (m0 >> 4) + t;
      tile = tile < g.tiles ? tile : g.tiles - 1;
      xp[t] = static_cast<const uint8_t *>(g.x) + tile * g.chunks * (P * 8 * 1024) + lane * 16;
    }
  }

  // half chunk number `at` of this wave: chunk wave + 8 (at / 2), half at & 1
  struct Half {
    u32x4_t w[NT][WV];
    uint32_t scale[kMicro ? NT : 1];
    u32x4_t x[MT][P][XV];
    uint32_t x_scale[kBoth ? MT : 1];
  };
  const int mine = g.chunks > wave ? 2 * ((g.chunks - 1 - wave) / kRowsWaves + 1) : 0;
  auto load = [&](Half &b, int at) __attribute__((always_inline)) {
    const int use = at < mine ? at : (mine > 0 ? mine - 1 : 0);
    const int chunk = wave + kRowsWaves * (use >> 1), h = use & 1;
    const int64_t c = chunk < g.chunks ? chunk : g.chunks - 1;
    if constexpr (kMicro) {
      const int64_t block = c * 8 + h * 4 + q;
      const bool in = block < g.blocks;
      const int64_t safe = in ? block : g.blocks - 1;
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        b.w[t][0] = *reinterpret_cast<const u32x4_t *>(wp[t] + safe * 16);
        b.scale[t] = in ? sp[t][safe] : 0u;
        if (!in) b.w[t][0] = u32x4_t{0, 0, 0, 0};
      }
      if constexpr (kBoth) {
#pragma unroll
        for (int t = 0; t < MT; ++t) {
          b.x[t][0][0] = *reinterpret_cast<const u32x4_t *>(xp[t] + safe * 16);
          b.x_scale[t] = in ? xsp[t][safe] : 0u;
        }
        return;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int64_t k = c * kRowsChunk + rows_element<kWeight>(4 * h + i, q);
        const bool in = k < g.R;
        const int64_t safe = in ? k : 0;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          b.w[t][i] = *reinterpret_cast<const u32x4_t *>(wp[t] + safe * 2);
          if (!in) b.w[t][i] = u32x4_t{0, 0, 0, 0};
        }
      }
    }
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (kDirect) {
          const int64_t k = c * kRowsChunk + rows_element<kWeight>(4 * h + i, q);
          const bool in = k < g.R;
          b.x[t][0][i] = *reinterpret_cast<const u32x4_t *>(xp[t] + (in ? k : 0) * 2);
          if (!in) b.x[t][0][i] = u32x4_t{0, 0, 0, 0};
        } else {
#pragma unroll
          for (int p = 0; p < P; ++p) b.x[t][p][i] = *reinterpret_cast<const u32x4_t *>(xp[t] + ((c * P + p) * 8 + 4 * h + i) * 1024);
        }
      }
  };

  floatx4_t acc[MT][NT];
#pragma unroll
  for (int t = 0; t < MT; ++t)
#pragma unroll
    for (int c = 0; c < NT; ++c) acc[t][c] = floatx4_t{0.0f, 0.0f, 0.0f, 0.0f};
  auto compute = [&](const Half &b) __attribute__((always_inline)) {
#pragma unroll
    for (int c = 0; c < NT; ++c)
#pragma unroll
      for (int i = 0; i < XV; ++i) {
        if constexpr (kBoth) {
#pragma unroll
          for (int t = 0; t < MT; ++t) acc[t][c] = mfma_micro(b.x[t][0][0], b.w[c][0], acc[t][c], b.x_scale[t], b.scale[c]);
          continue;
        }
        u32x4_t w;
        if constexpr (kMicro) w = mxfp4_eight<CT>(b.w[c][0][i], mxfp4_scale(b.scale[c]));
        else w = b.w[c][i];
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
          for (int p = 0; p < P; ++p)
            if constexpr (!kBoth) acc[t][c] = Mfma16<CT>::run(b.x[t][p][i], w, acc[t][c]);
      }
  };
  Half even, odd;
  load(even, 0);
  for (int at = 0; at < mine; at += 2) {
    load(odd, at + 1);
    compute(even);
    load(even, at + 2);
    compute(odd);
  }

  // the eight waves' sums, in a fixed order: wave w + 4's into wave w's, then those four into the result
  constexpr int kHalf = kRowsWaves / 2;
  if (wave >= kHalf)
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int c = 0; c < NT; ++c) sums[wave - kHalf][t * NT + c][lane] = acc[t][c];
  __syncthreads();
  if (wave < kHalf)
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int c = 0; c < NT; ++c) sums[wave][t * NT + c][lane] += acc[t][c];
  __syncthreads();

  const float *flat = reinterpret_cast<const float *>(sums);
  auto total = [&](int tile, int row, int col) __attribute__((always_inline)) {       // row, col inside the 16 x 16 tile
    const int at = (tile * 64 + (row >> 2) * 16 + col) * 4 + (row & 3);
    float v = flat[at];
#pragma unroll
    for (int w = 1; w < kHalf; ++w) v += flat[w * (MT * NT * 256) + at];
    return v;
  };
  auto store = [&](auto type_) __attribute__((always_inline)) {
    typedef decltype(type_) T;
    for (int at = threadIdx.x; at < MT * NC * 256; at += kRowsWaves * 64) {
      const int col = at % (16 * NC), row = at / (16 * NC);
      const int64_t m = m0 + row, n = n0 + col;
      if (m >= g.M || n >= g.N) continue;
      const int tile = (row >> 4) * NT + (col >> 4);
      const float v = total(tile, row & 15, col & 15);
      const int64_t to = m * g.N + n;
      if constexpr (NW == 2) {
        const float u = total(tile + NC, row & 15, col & 15);
        static_cast<T *>(g.y)[to] = from_f32<T>(gate_act(v) * u);
        if (g.gate) {
          static_cast<T *>(g.gate)[to] = from_f32<T>(v);
          static_cast<T *>(g.up)[to] = from_f32<T>(u);
        }
      } else {
        T r = from_f32<T>(v);
        if (g.addend) r = from_f32<T>(to_f32<T>(r) + to_f32<T>(static_cast<const T *>(g.addend)[to]));
        static_cast<T *>(g.y)[to] = r;
      }
    }
  };
  if (g.y_dtype == CAIFX_BF16) store(bf16_t{});
  else if (g.y_dtype == CAIFX_F16) store(f16_t{});
  else store(float{});
}

template <typename CT, int P, int kWeight, int NW, int MT, int NT, bool kDirect>
int rows_launch(const RowsArgs &g, hipStream_t s)
{
  constexpr int NC = NT / NW;
  const int64_t rows = (g.M + 16 * MT - 1) / (16 * MT), cols = (g.N + 16 * NC - 1) / (16 * NC);
  // a grid's second extent has 65535 blocks: more rows than that go in several launches
  for (int64_t r = 0; r < rows; r += 65535) {
    RowsArgs part = g;
    const int64_t m0 = r * 16 * MT, es = static_cast<int64_t>(dtype_size(g.y_dtype));
    const auto forth = [&](const void *p, int64_t bytes) { return p ? const_cast<char *>(static_cast<const char *>(p)) + bytes : nullptr; };
    part.M = g.M - m0;
    part.tiles = g.tiles - static_cast<int>(m0 / 16);
    part.x = forth(g.x, kWeight == ROWS_BOTH ? m0 * g.w_pitch : kDirect ? m0 * g.x_pitch * 2 : m0 / 16 * g.chunks * (P * 8 * 1024));
    part.xs = g.xs ? g.xs + m0 * g.blocks : nullptr;
    part.y = forth(g.y, m0 * g.N * es);
    part.gate = forth(g.gate, m0 * g.N * es);
    part.up = forth(g.up, m0 * g.N * es);
    part.addend = forth(g.addend, m0 * g.N * es);
    const dim3 grid(static_cast<unsigned>(cols), static_cast<unsigned>(rows - r < 65535 ? rows - r : 65535));
    hipLaunchKernelGGL((rows_kernel<CT, P, kWeight, NW, MT, NT, kDirect>), grid, dim3(kRowsWaves * 64), 0, s, part);
  }
  return launch_status();
}

// Column tiles of a workgroup: as many as leave three quarters of the chip's 256 compute units a workgroup each.
inline int rows_column_tiles(const RowsArgs &g, int weights, int mt)
{
  const int64_t rows = (g.M + 16 * mt - 1) / (16 * mt);
  for (int nt = 4; nt > weights; nt /= 2)
    if (rows * ((g.N + 16 * (nt / weights) - 1) / (16 * (nt / weights))) >= 192) return nt;
  return weights;
}

template <typename CT, int P, int kWeight, int NW, int MT, bool kDirect>
int rows_pick_columns(const RowsArgs &g, hipStream_t s)
{
  switch (rows_column_tiles(g, NW, MT)) {
    case 4: return rows_launch<CT, P, kWeight, NW, MT, 4, kDirect>(g, s);
    case 2: return rows_launch<CT, P, kWeight, NW, MT, 2, kDirect>(g, s);
    default:
      if constexpr (NW == 1) return rows_launch<CT, P, kWeight, NW, MT, 1, kDirect>(g, s);
      else return rows_launch<CT, P, kWeight, NW, MT, 2, kDirect>(g, s);
  }
}
template <typename CT, int kWeight, int NW> int rows_pick(const RowsArgs &g, int pieces, bool direct, hipStream_t s)
{
  if constexpr (dtype_code<CT>::value == CAIFX_BF16) {
    if (pieces == 3) return rows_pick_columns<CT, 3, kWeight, NW, 1, false>(g, s);
  }
  if (direct) return g.M <= 16 ? rows_pick_columns<CT, 1, kWeight, NW, 1, true>(g, s) : rows_pick_columns<CT, 1, kWeight, NW, 2, true>(g, s);
  return g.M <= 32 ? rows_pick_columns<CT, 1, kWeight, NW, 2, false>(g, s) : rows_pick_columns<CT, 1, kWeight, NW, 4, false>(g, s);
}

int rows_both(const RowsArgs &g, hipStream_t s);
int rows_bf16(const RowsArgs &g, int weight, int weights, int pieces, bool direct, hipStream_t s);
int rows_f16(const RowsArgs &g, int weight, int weights, bool direct, hipStream_t s);

}  // namespace caifx
