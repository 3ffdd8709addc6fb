// Input gradient for up to some hundred rows, dX[m, k] = sum_n dY[m, n] W[n, k], and the sum of two such products, with the weights in
// microscaled 4 bits or stored in the 16-bit compute type, read once as they are.
//
// The reduction runs down the weight's rows, and a matrix-core operand holds eight of its elements, eight weight rows of one column, per
// lane.  So lane (j, q) of v_mfma_f32_16x16x32 reads sixteen neighbouring columns of the eight rows 8 q .. 8 q + 7 of a step of 32 (8 bytes of
// codes a row, 16 lanes together a line), turns them into pairs of columns in the compute type and those, with one byte permutation per
// two values, into pairs of rows: sixteen operands, of column c of every lane each.  Per 8192 codes of a wave 64 conversions, 64
// permutations and 16 matrix instructions for 16 rows of dY; the copy of the weight that larger calls transpose first would be written
// and read again, 4 bytes for half a byte of codes.
// A workgroup of eight waves owns 256 columns, its waves take steps in turn and meet in LDS; workgroups share a reduction, as many as the
// chip has room for, and a second launch adds their sums in a fixed order.
// N = 14336, K = 4096, bf16, 16 rows: 16 us (the weight's bytes alone 6.3), behind a transposed copy 57; 256 rows 66 us, 456 TFLOP/s, and 79.
#include "caifx_mxfp4.hpp"

#include <type_traits>

namespace caifx {
namespace {

constexpr int kColumns = 256;              // of a workgroup
constexpr int kSets = 16;                  // columns of a lane
constexpr int kWaves = 8;

struct DxArgs {
  const uint8_t *w[2], *s[2];       // one or two weights of N rows, `pitch` bytes long
  const uint8_t *x[2];              // direct: [M, N] of the compute type (P = 3: fp32); packed: x[0], see pack_rows_kernel, the second's chunks behind the first's
  int64_t M, N, K, blocks, pitch;
  int count, steps;                 // weights; steps of 32 rows of one weight
  int chunks, tiles;                // packed: chunks in all, row tiles of 16
  int splits;                       // workgroups that share a reduction: the z-th writes its sums to y + z M K (fp32)
  void *y;
  const void *addend;
  int y_dtype;
};

template <typename CT, int P, bool kMx, int MT, bool kDirect>
__global__ __launch_bounds__(kWaves * 64) void dx_kernel(DxArgs g)
{
  typedef u32x2_t codes_t __attribute__((aligned(8)));
  typedef u32x4_t anywhere_t __attribute__((aligned(2)));
  __shared__ floatx4_t sums[kWaves / 2][kSets][65];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int j = lane & 15, q = lane >> 4;
  const int64_t k0 = static_cast<int64_t>(blockIdx.x) * kColumns, m0 = static_cast<int64_t>(blockIdx.y) * (16 * MT);
  // a lane's first column: past the end of a row the last sixteen columns again (stored once)
  const int64_t width = kMx ? 32 * g.blocks : g.K;
  const auto first_column = [&](int lane_j) __attribute__((always_inline)) {
    const int64_t k = k0 + kSets * lane_j;
    return k + kSets <= width ? k : width - kSets;
  };
  const int64_t column = first_column(j);

  constexpr int XW = kDirect && P == 3 ? 2 : P;      // loads of eight activations: direct fp32 ones are taken apart once they are used
  struct Step {
    u32x4_t w[8][kMx ? 1 : 2];        // (codes: half of it)
    uint32_t scale[8];
    u32x4_t x[MT][XW];
  };
  auto load = [&](Step &b, int step) __attribute__((always_inline)) {
    const int second = step >= g.steps ? 1 : 0, at = step - second * g.steps;
    const uint8_t *w = g.w[0], *s = g.s[0], *x = g.x[0];
    if (second) {
      w = g.w[1];
      s = g.s[1];
      if constexpr (kDirect) x = g.x[1];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      // rows past the end: the last one again, against zeros
      const int64_t n = static_cast<int64_t>(at) * 32 + 8 * q + i, row = n < g.N ? n : g.N - 1;
      if constexpr (kMx) {
        const u32x2_t c = *reinterpret_cast<const codes_t *>(w + row * g.pitch + (column >> 1));
        b.w[i][0] = u32x4_t{c[0], c[1], 0, 0};
        b.scale[i] = s[row * g.blocks + (column >> 5)];
      } else {
        const uint8_t *from = w + row * g.pitch + column * 2;
        b.w[i][0] = *reinterpret_cast<const anywhere_t *>(from);
        b.w[i][1] = *reinterpret_cast<const anywhere_t *>(from + 16);
      }
    }
    if constexpr (kDirect) {
      // (eight elements that end past the row, or begin there: its last eight)
      const int64_t n = static_cast<int64_t>(at) * 32 + 8 * q, from_n = n + 8 <= g.N ? n : g.N - 8;
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        int64_t m = m0 + 16 * t + j;
        m = m < g.M ? m : g.M - 1;
        const uint8_t *from = x + (m * g.N + from_n) * (2 * XW);
#pragma unroll
        for (int i = 0; i < XW; ++i) b.x[t][i] = *reinterpret_cast<const anywhere_t *>(from + 16 * i);
      }
    } else {
      // steps of a weight fill whole chunks of eight in the packed order
      const int64_t chunk = (second ? g.chunks / 2 : 0) + (at >> 3);
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        int64_t tile = (m0 >> 4) + t;
        tile = tile < g.tiles ? tile : g.tiles - 1;
#pragma unroll
        for (int p = 0; p < P; ++p)
          b.x[t][p] = *reinterpret_cast<const u32x4_t *>(x + (((tile * g.chunks + chunk) * P + p) * 8 + (at & 7)) * 1024 + lane * 16);
      }
    }
  };

  floatx4_t acc[MT][kSets];
#pragma unroll
  for (int t = 0; t < MT; ++t)
#pragma unroll
    for (int c = 0; c < kSets; ++c) acc[t][c] = floatx4_t{0.0f, 0.0f, 0.0f, 0.0f};
  auto compute = [&](Step &b, int step) __attribute__((always_inline)) {
    // (an infinity of the last row against those zeros would be a NaN)
    const int n = (step >= g.steps ? step - g.steps : step) * 32;
    if (n + 32 > g.N) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (n + 8 * q + i >= g.N) b.w[i][0] = b.w[i][kMx ? 0 : 1] = u32x4_t{0, 0, 0, 0};
      if constexpr (kDirect) {
        const int past = n + 8 * q + 8 - static_cast<int>(g.N);
        if (past > 0)
#pragma unroll
          for (int t = 0; t < MT; ++t) drop_first<XW>(b.x[t], past);
      }
    }
    u32x4_t x[MT][P];
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      if constexpr (kDirect && P == 3) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const floatx4_t four = __builtin_bit_cast(floatx4_t, b.x[t][i >> 1]);
          uint32_t even[3], odd[3];
          pieces_of_f32(four[2 * (i & 1)], even);
          pieces_of_f32(four[2 * (i & 1) + 1], odd);
#pragma unroll
          for (int p = 0; p < 3; ++p) x[t][p][i] = __builtin_amdgcn_perm(odd[p], even[p], 0x07060302u);
        }
      } else {
#pragma unroll
        for (int p = 0; p < P; ++p) x[t][p] = b.x[t][p];
      }
    }
    // eight columns at a time
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      u32x4_t rows[8];                       // eight values of a row, in pairs of columns
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if constexpr (kMx) rows[i] = mxfp4_eight<CT>(b.w[i][0][half], mxfp4_scale(b.scale[i]));
        else rows[i] = b.w[i][half];
      }
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        u32x4_t w;                           // eight rows of a column
#pragma unroll
        for (int d = 0; d < 4; ++d) w[d] = __builtin_amdgcn_perm(rows[2 * d + 1][c >> 1], rows[2 * d][c >> 1], (c & 1) ? 0x07060302u : 0x05040100u);
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
          for (int p = 0; p < P; ++p) acc[t][half * 8 + c] = Mfma16<CT>::run(x[t][p], w, acc[t][half * 8 + c]);
      }
    }
  };
  const int total = g.count * g.steps, z = static_cast<int>(blockIdx.z);
  const int begin = static_cast<int>(static_cast<int64_t>(total) * z / g.splits), end = static_cast<int>(static_cast<int64_t>(total) * (z + 1) / g.splits);
  int at = begin + wave;
  if (at < end) {
    if constexpr (kMx || MT == 1) {
      Step now, next;
      load(now, at);
      for (; at + kWaves < end; at += kWaves) {
        load(next, at + kWaves);
        compute(now, at);
        now = next;
      }
      compute(now, at);
    } else {
      // (two steps of a stored weight and 32 rows' sums do not fit the registers)
      for (; at < end; at += kWaves) {
        Step now;
        load(now, at);
        compute(now, at);
      }
    }
  }

  // The waves' sums, in a fixed order, 16 rows at a time.  A thread takes four rows of one column at once: neighbouring threads read sets of
  // sums 1040 bytes apart, sixteen bytes each, and write neighbouring columns.
  constexpr int kHalf = kWaves / 2;
  auto store = [&](auto type_) __attribute__((always_inline)) {
    typedef decltype(type_) T;
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      if (t > 0) __syncthreads();
      if (wave >= kHalf)
#pragma unroll
        for (int c = 0; c < kSets; ++c) sums[wave - kHalf][c][lane] = acc[t][c];
      __syncthreads();
      if (wave < kHalf)
#pragma unroll
        for (int c = 0; c < kSets; ++c) sums[wave][c][lane] += acc[t][c];
      __syncthreads();
#pragma unroll
      for (int i = threadIdx.x; i < 4 * kColumns; i += kWaves * 64) {
        const int four = i / kColumns, within = i % kColumns;
        const int64_t m = m0 + 16 * t + 4 * four, k = first_column(within / kSets) + within % kSets;
        floatx4_t v = sums[0][within % kSets][four * 16 + within / kSets];
#pragma unroll
        for (int w = 1; w < kHalf; ++w) v += sums[w][within % kSets][four * 16 + within / kSets];
        if (k >= g.K || k < k0 + within / kSets * kSets) continue;      // (another lane's, where the end of a row moved this one's)
        const int64_t to = (z * g.M + m) * g.K + k;
#pragma unroll
        for (int row = 0; row < 4; ++row) {
          if (m + row >= g.M) break;
          const int64_t at_row = to + row * g.K;
          T r = from_f32<T>(v[row]);
          if (g.addend) r = from_f32<T>(to_f32<T>(r) + to_f32<T>(static_cast<const T *>(g.addend)[at_row]));
          static_cast<T *>(g.y)[at_row] = r;
        }
      }
    }
  };
  if (g.y_dtype == CAIFX_BF16) store(bf16_t{});
  else if (g.y_dtype == CAIFX_F16) store(f16_t{});
  else store(float{});
}

int tile_of(int64_t M) { return M <= 16 ? 16 : 32; }

// Workgroups that share a reduction: one for each compute unit in all, as many as the registers hold at once (N = 14336, K = 4096, 32 rows: 128
// workgroups 32 us, 256 26, 512 41), and each wave at least one step
int splits_of(const DxProduct &p)
{
  const int64_t total = p.count * ((p.N + 31) / 32), others = (p.K + kColumns - 1) / kColumns * ((p.M + tile_of(p.M) - 1) / tile_of(p.M));
  int64_t most = 256 / others;
  const int64_t steps = (total + kWaves - 1) / kWaves;
  most = most < steps ? most : steps;
  return static_cast<int>(most < 1 ? 1 : most);
}

template <typename CT, int P, bool kMx> int launch(const DxArgs &g, bool direct, hipStream_t s)
{
  const int tile = tile_of(g.M);
  const dim3 grid(static_cast<unsigned>((g.K + kColumns - 1) / kColumns), static_cast<unsigned>((g.M + tile - 1) / tile), static_cast<unsigned>(g.splits));
  const auto go = [&](auto mt_, auto direct_) {
    hipLaunchKernelGGL((dx_kernel<CT, P, kMx, decltype(mt_)::value, decltype(direct_)::value>), grid, dim3(kWaves * 64), 0, s, g);
  };
  const std::integral_constant<int, 1> one;
  const std::integral_constant<int, 2> two;
  if (direct) {
    if (tile == 16) go(one, std::true_type{});
    else go(two, std::true_type{});
    return launch_status();
  }
  if (tile == 16) go(one, std::false_type{});
  else go(two, std::false_type{});
  return launch_status();
}

}  // namespace

bool dx_takes(const DxProduct &p)
{
  // (a grid's second extent has 65535 blocks; sixteen columns at a time)
  return p.M <= 1024 && (p.mx || p.K >= kSets);
}

// steps that a wave of the last workgroup has taken
static int64_t turns_of(const DxProduct &p)
{
  const int splits = splits_of(p);
  const int64_t others = (p.K + kColumns - 1) / kColumns * ((p.M + tile_of(p.M) - 1) / tile_of(p.M));
  return (others * splits + 255) / 256 * ((p.count * ((p.N + 31) / 32) + kWaves * splits - 1) / (kWaves * splits));
}

bool dx_reads(const DxProduct &p)
{
  // fp32, us, packed / direct: one step N = 2048, K = 1403, 64 rows 17.2 / 14.7, three 333 rows 24.3 / 22.2, four N = K = 4096, 128 rows 26.6 / 26.6, seven
  // N = 14336, K = 4096, 64 rows 37.2 / 38.7; 16 rows 21.1 / 18.2
  return p.compute_dtype != CAIFX_F32 || p.M <= 16 || turns_of(p) <= 4;
}

double dx_us(const DxProduct &p)
{
  const int splits = splits_of(p);
  const double step = (p.compute_dtype == CAIFX_F32 ? 3.4 : 1.85) * (p.mx ? 1.0 : 1.2);
  const double join = splits > 1 ? 3.0 + 8e-7 * static_cast<double>(splits) * static_cast<double>(p.M) * static_cast<double>(p.K) : 0.0;
  return 5.0 + (p.direct ? 0.0 : 3.0) + join + step * static_cast<double>(turns_of(p));
}

size_t dx_partial_bytes(const DxProduct &p)
{
  const int splits = splits_of(p);
  return splits > 1 ? static_cast<size_t>(splits) * static_cast<size_t>(p.M) * static_cast<size_t>(p.K) * 4 : 0;
}

int dx_product(const DxProduct &p, void *partial, hipStream_t s)
{
  DxArgs g{};
  for (int i = 0; i < p.count; ++i) {
    g.w[i] = static_cast<const uint8_t *>(p.w[i]);
    g.s[i] = static_cast<const uint8_t *>(p.s[i]);
    g.x[i] = static_cast<const uint8_t *>(p.x[i]);
  }
  g.M = p.M;
  g.N = p.N;
  g.K = p.K;
  g.blocks = (p.K + CAIFX_MXFP4_BLOCK - 1) / CAIFX_MXFP4_BLOCK;
  g.pitch = p.mx ? 16 * g.blocks : 2 * p.K;
  g.count = p.count;
  g.steps = static_cast<int>((p.N + 31) / 32);
  g.chunks = p.count * static_cast<int>((p.N + kRowsChunk - 1) / kRowsChunk);
  g.tiles = static_cast<int>((p.M + 15) / 16);
  g.splits = splits_of(p);
  g.y = g.splits > 1 ? partial : p.y;
  g.y_dtype = g.splits > 1 ? static_cast<int>(CAIFX_F32) : p.y_dtype;
  g.addend = g.splits > 1 ? nullptr : p.addend;
  int st;
  if (p.compute_dtype == CAIFX_F32) st = launch<bf16_t, 3, true>(g, p.direct, s);
  else if (p.compute_dtype == CAIFX_F16) st = p.mx ? launch<f16_t, 1, true>(g, p.direct, s) : launch<f16_t, 1, false>(g, p.direct, s);
  else st = p.mx ? launch<bf16_t, 1, true>(g, p.direct, s) : launch<bf16_t, 1, false>(g, p.direct, s);
  if (st != CAIFX_OK || g.splits == 1) return st;
  return join_sums(static_cast<const float *>(partial), g.splits, p.M * p.K, p.y, p.y_dtype, p.addend, s);
}

}  // namespace caifx
