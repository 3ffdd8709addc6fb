// Products over frozen weights in microscaled 4 bits (forward, input gradient, both operands in 4 bits), and the gated feed-forward block
// over two such weights or two stored in the 16-bit type: which kernels run on what, and the operands that they need in the workspace.
#include "caifx_mxfp4.hpp"

namespace caifx {
namespace {

int64_t up_to(int64_t v, int64_t m) { return (v + m - 1) / m * m; }
int64_t chunks_of(int64_t reduction) { return (reduction + kRowsChunk - 1) / kRowsChunk; }

// A workspace handed out in pieces of whole 256 bytes; without memory only the sizes are added up.
struct Room {
  char *p = nullptr;
  size_t used = 0;
  void *take(size_t bytes)
  {
    void *at = p ? p + used : nullptr;
    used += (bytes + 255) / 256 * 256;
    return at;
  }
};

int pieces_of(int compute_dtype) { return compute_dtype == CAIFX_F32 ? 3 : 1; }
size_t packed_bytes(int64_t rows, int64_t chunks, int compute_dtype)
{
  return static_cast<size_t>((rows + 15) / 16) * static_cast<size_t>(chunks) * static_cast<size_t>(pieces_of(compute_dtype)) * 8192;
}
// fp32 products of bf16 activations: every factor is a bf16 number as it is
int computed_in(const GemmArgs &a) { return a.compute_dtype == CAIFX_F32 && a.x_dtype == CAIFX_BF16 ? CAIFX_BF16 : a.compute_dtype; }
int stored_as(int compute_dtype) { return compute_dtype == CAIFX_F16 ? CAIFX_F16 : CAIFX_BF16; }

// One weight of a product, in either form
struct Weight {
  const void *p;
  const void *scales;      // MX only
  bool mx;
};

// One or two products x w^T.  x [M, R] of x_dtype; w [N, R].
struct Product {
  int64_t M, N, R;
  const void *x;
  int x_dtype, compute_dtype;
  int weights;
  Weight w[2];
  void *y, *gate, *up;
  int y_dtype;
  const void *addend;
};

RowsArgs rows_args(const Product &p)
{
  RowsArgs g{};
  const int64_t blocks = (p.R + CAIFX_MXFP4_BLOCK - 1) / CAIFX_MXFP4_BLOCK;
  for (int i = 0; i < p.weights; ++i) {
    g.w[i] = p.w[i].p;
    g.s[i] = static_cast<const uint8_t *>(p.w[i].scales);
  }
  g.M = p.M;
  g.N = p.N;
  g.R = p.R;
  g.blocks = blocks;
  g.w_pitch = p.w[0].mx ? 16 * blocks : 2 * p.R;
  g.x_pitch = p.R;
  g.chunks = static_cast<int>(chunks_of(p.R));
  g.tiles = static_cast<int>((p.M + 15) / 16);
  g.y = p.y;
  g.gate = p.gate;
  g.up = p.up;
  g.addend = p.addend;
  g.y_dtype = p.y_dtype;
  return g;
}

// Runs the row kernels on laid out operands, or adds up what they need of the workspace: the sums of shared reductions.
int rows_run(RowsArgs g, int kind, int weights, int compute_dtype, bool direct, Room &room, bool only_size, hipStream_t s)
{
  const int pieces = pieces_of(compute_dtype);
  const RowsPlan plan = rows_plan_of(kind, weights, pieces, direct, g.M, g.N, g.R, g.blocks, g.w_pitch);
  void *partial = plan.splits > 1 ? room.take(static_cast<size_t>(plan.splits) * static_cast<size_t>(g.M) * static_cast<size_t>(g.N) * 4) : nullptr;
  if (only_size) return CAIFX_OK;
  g.span = plan.span;
  g.splits = plan.splits;
  const RowsArgs asked = g;
  if (plan.splits > 1) {
    g.y = partial;
    g.y_dtype = CAIFX_F32;
    g.addend = nullptr;
  }
  const int st = kind == ROWS_BOTH ? rows_both(g, s) : compute_dtype == CAIFX_F16 ? rows_f16(g, kind, weights, direct, s) : rows_bf16(g, kind, weights, pieces, direct, s);
  if (st != CAIFX_OK || plan.splits == 1) return st;
  return join_sums(static_cast<const float *>(partial), plan.splits, g.M * g.N, asked.y, asked.y_dtype, asked.addend, s);
}

// The dense product, in parts where that is faster, or the size of their sums.
int wide_run(WideProduct d, Room &room, bool only_size, hipStream_t s)
{
  d.parts = d.gated ? 1 : wide_parts(d.M, d.C, d.pairs * d.R).parts;
  if (d.parts == 1) return only_size ? CAIFX_OK : wide_product(d, s);
  void *partial = room.take(static_cast<size_t>(d.parts) * static_cast<size_t>(d.M) * static_cast<size_t>(d.C) * 4);
  if (only_size) return CAIFX_OK;
  const WideProduct asked = d;
  d.d = partial;
  d.d_dtype = CAIFX_F32;
  d.addend = nullptr;
  const int st = wide_product(d, s);
  return st != CAIFX_OK ? st : join_sums(static_cast<const float *>(partial), d.parts, d.M * d.C, asked.d, asked.d_dtype, asked.addend, s);
}

// Whether the row kernels read the activations where they are, each workgroup its rows, which pays for the launch that packs them while all
// workgroups run at once.  us, packed / direct, bf16: 64 rows, N = 14336, K = 4096 22.1 / 20.7; N = 4096, K = 14336 25.7 / 22.6; 2048 x 1408 8.0 / 7.6;
// 256 rows, N = K = 4096 19.9 / 16.3; two rounds, 96 rows, N = 11008, K = 2048 21.6 / 23.4.  fp32 ones are taken apart by every workgroup: for one
// group of four rows (N = K = 4096, 4 rows 10.8 / 6.8, 8 rows 10.9 / 11.9).
bool direct_rows(const Product &p)
{
  if (p.x_dtype != p.compute_dtype || p.R < 8) return false;
  if (p.compute_dtype == CAIFX_F32) return p.M <= 4;
  return p.M <= 32 || (p.M + 63) / 64 * ((p.weights * p.N + 63) / 64) <= 256;
}

// The weights of a product or the activations of a gradient, as a source of operands
Operand weights_of(const Weight (&w)[2], int count, int64_t rows, int64_t cols, int stored)
{
  Operand o{};
  for (int i = 0; i < count; ++i) {
    o.p[i] = w[i].p;
    o.scales[i] = w[i].scales;
  }
  o.count = count;
  o.kind = w[0].mx ? OPERAND_MX : stored;
  o.rows = rows;
  o.cols = cols;
  return o;
}
Operand activations_of(const void *x, const void *second, int kind, int64_t rows, int64_t cols)
{
  Operand o{};
  o.p[0] = x;
  o.p[1] = second;
  o.count = second ? 2 : 1;
  o.kind = kind;
  o.rows = rows;
  o.cols = cols;
  return o;
}

// Whether a product with this many rows runs on dense operands (caifx_gemm_wide.hip) instead of the row kernels.
bool wide_product_pays(const Product &p)
{
  const int64_t R = up_to(p.R, 64) < 128 ? 128 : up_to(p.R, 64);
  const int pieces = pieces_of(p.compute_dtype);
  if (p.M <= 64 || !wide_takes(p.M, p.N, R) || p.N * R >= (int64_t{1} << 32)) return false;
  if (!p.w[0].mx) return true;
  // A workgroup of the row kernels takes 64 x 64 results in 4.5 us and 1.3 for every 512 elements of the reduction, 256 of them at a time (few, a
  // third of that and up), on three pieces 32 x 32 in 2.2 and 1.3; the dense product is twice as fast and more, behind copies of the weights.
  // us, rows / dense, bf16: N = 14336, K = 4096, 256 rows 62 / 66, 384 rows 86 / 83; N = 11008 384 rows 72 / 70; N = K = 4096, 256 rows 20 / 41; N =
  // 4096, K = 14336, 512 rows 84 / 98; 5120 x 794, 512 rows 29 / 23.
  const double weights = p.weights, millions = 1e-6 * weights * static_cast<double>(p.N) * static_cast<double>(R);
  const int64_t tile = pieces == 3 ? 32 : 64, groups = (p.M + tile - 1) / tile * ((p.weights * p.N + tile - 1) / tile);
  const double rounds = static_cast<double>(groups / 256) + (groups % 256 == 0 ? 0.0 : 0.35 + 0.65 / 256 * static_cast<double>(groups % 256));
  const double rows = 5.0 + rounds * ((pieces == 3 ? 2.2 : 4.5) + 1.3 * static_cast<double>((R + 511) / 512));
  return (p.weights == 2 ? wide_us_of(p.M, 2 * p.N, pieces * R) : wide_parts(p.M, p.N, pieces * R).us) + (pieces == 3 ? 12.0 : 8.0) + 0.56 * millions < rows;
}

// Whether the dense product reads activations from a copy: of another type or length, or that no 16-byte access takes where they are.  us, 4096 rows, N =
// 11008, K = 4096, bf16, in place / copied / on the row kernels, which take any address: forward 302 / 300 / 596, gradient 263 / 297 / 953; 300 rows, N = 14336,
// K = 4096, gradient 72 / 78 / 138.  A size query, which has no address, counts the copy.
bool copied(int pieces, int x_dtype, int to, int64_t length, int64_t R, const void *x, const void *second)
{
  return pieces == 3 || x_dtype != to || length != R || !x || !aligned_to(x, 16) || !aligned_to(second, 16);
}

// The product on dense operands: the weights dequantised into the workspace, activations copied where they have to be.
int product_wide(const Product &p, Room &room, bool only_size, hipStream_t s)
{
  const int64_t R = up_to(p.R, 64) < 128 ? 128 : up_to(p.R, 64);
  const int to = stored_as(p.compute_dtype), pieces = pieces_of(p.compute_dtype);
  int st = CAIFX_OK;
  WideProduct d{};
  d.pairs = pieces;
  d.b_every = pieces;
  d.gated = p.weights == 2;
  d.b[0] = p.w[0].p;
  d.b[1] = p.w[1].p;
  if (p.w[0].mx || R != p.R) {
    const size_t one = static_cast<size_t>(p.N) * static_cast<size_t>(R) * 2;
    char *copy = static_cast<char *>(room.take(p.weights * one));
    d.b[0] = copy;
    d.b[1] = copy + (only_size ? 0 : one);
    if (!only_size) st = operand_dense(weights_of(p.w, p.weights, p.N, p.R, to), to, copy, R, s);
  }
  d.a = p.x;
  const Operand x = activations_of(p.x, nullptr, p.x_dtype, p.M, p.R);
  if (pieces == 3) {
    d.a_stride = p.M * R * 2;
    void *copy = room.take(static_cast<size_t>(p.M) * static_cast<size_t>(R) * 6);
    d.a = copy;
    if (!only_size && st == CAIFX_OK) st = operand_pieces(x, copy, R, s);
  } else if (copied(pieces, p.x_dtype, to, p.R, R, p.x, nullptr)) {
    void *copy = room.take(static_cast<size_t>(p.M) * static_cast<size_t>(R) * 2);
    d.a = copy;
    if (!only_size && st == CAIFX_OK) st = operand_dense(x, to, copy, R, s);
  }
  d.d = p.y;
  d.gate = p.gate;
  d.up = p.up;
  d.addend = p.addend;
  d.M = p.M;
  d.C = p.N;
  d.R = R;
  d.compute_dtype = to;
  d.d_dtype = p.y_dtype;
  return st != CAIFX_OK ? st : wide_run(d, room, only_size, s);
}

// The product on the row kernels, any sizes and types.
int product_rows(const Product &p, Room &room, bool only_size, hipStream_t s)
{
  Product d = p;
  const int to = stored_as(p.compute_dtype);
  const int64_t pitch = up_to(p.R, 8);
  // rows of a stored weight start at any multiple of two bytes where R is odd: the row kernels take them from a copy
  if (!p.w[0].mx && p.R != pitch) {
    const size_t one = static_cast<size_t>(p.N) * static_cast<size_t>(pitch) * 2;
    char *copy = static_cast<char *>(room.take(p.weights * one));
    d.w[0].p = copy;
    d.w[1].p = copy + (only_size ? 0 : one);
    if (!only_size) {
      const int st = operand_dense(weights_of(p.w, p.weights, p.N, p.R, to), to, copy, pitch, s);
      if (st != CAIFX_OK) return st;
    }
  }
  RowsArgs g = rows_args(d);
  if (!p.w[0].mx && p.R != pitch) {
    g.R = pitch;
    g.w_pitch = 2 * pitch;
  }
  const bool direct = direct_rows(p);
  if (!direct) {
    void *packed = room.take(packed_bytes(p.M, g.chunks, p.compute_dtype));
    if (!only_size) {
      const int st = operand_rows(activations_of(p.x, nullptr, p.x_dtype, p.M, p.R), p.compute_dtype, packed, g.chunks, s);
      if (st != CAIFX_OK) return st;
    }
    g.x = packed;
  } else {
    g.x = p.x;
  }
  return rows_run(g, p.w[0].mx ? ROWS_MX : ROWS_DENSE, p.weights, p.compute_dtype, direct, room, only_size, s);
}

// What one way of a product takes of the workspace
template <typename P> size_t room_of(int (*way)(const P &, Room &, bool, hipStream_t), const P &p)
{
  Room need;
  way(p, need, true, nullptr);
  return need.used;
}
// One way of a product, in room that is checked first to hold what it takes at these addresses
template <typename P> int run_in(int (*way)(const P &, Room &, bool, hipStream_t), const P &p, void *workspace, size_t bytes, hipStream_t s)
{
  Room room{static_cast<char *>(workspace), 0};
  return room_of(way, p) > bytes ? static_cast<int>(CAIFX_ERR_WORKSPACE_TOO_SMALL) : way(p, room, false, s);
}

size_t product_bytes(const Product &p, bool dense_copy = true)
{
  return room_of(dense_copy && wide_product_pays(p) ? product_wide : product_rows, p);
}
int product(const Product &p, void *workspace, size_t bytes, hipStream_t s)
{
  const bool wide = wide_product_pays(p) && bytes >= room_of(product_wide, p);
  return run_in(wide ? product_wide : product_rows, p, workspace, bytes, s);
}

// y[M,K] = sum over the weights of x[i][M,N] w[i][N,K], as one reduction over their rows
struct Gradient {
  int64_t M, N, K;
  const void *x[2];
  int x_dtype, compute_dtype;
  int weights;
  Weight w[2];
  void *y;
  int y_dtype;
  const void *addend;
};

int64_t reduction_of(const Gradient &p) { return up_to(p.N, 64) < 128 ? 128 : up_to(p.N, 64); }
// Whether a gradient can run on the dense product behind the transposed copies.
bool wide_gradient_takes(const Gradient &p) { return p.M > 32 && wide_takes(p.M, p.K, reduction_of(p)); }

int gradient_wide(const Gradient &p, Room &room, bool only_size, hipStream_t s)
{
  const int to = stored_as(p.compute_dtype), pieces = pieces_of(p.compute_dtype);
  const int64_t R = reduction_of(p);
  int st = CAIFX_OK;
  WideProduct d{};
  d.pairs = p.weights * pieces;
  d.b_every = pieces;
  d.b_stride = p.K * R * 2;
  void *copy = room.take(p.weights * static_cast<size_t>(p.K) * static_cast<size_t>(R) * 2);
  d.b[0] = copy;
  if (!only_size) st = operand_transposed(weights_of(p.w, p.weights, p.N, p.K, to), to, copy, R, R, p.K * R, s);
  const Operand x = activations_of(p.x[0], p.x[1], p.x_dtype, p.M, p.N);
  d.a = p.x[0];
  d.a_stride = static_cast<const char *>(p.x[1]) - static_cast<const char *>(p.x[0]);
  if (copied(pieces, p.x_dtype, to, p.N, R, p.x[0], p.x[1])) {
    const size_t one = static_cast<size_t>(p.M) * static_cast<size_t>(R) * 2;
    void *operand = room.take(d.pairs * one);
    d.a = operand;
    d.a_stride = static_cast<int64_t>(one);
    if (!only_size && st == CAIFX_OK) st = pieces == 3 ? operand_pieces(x, operand, R, s) : operand_dense(x, to, operand, R, s);
  }
  d.d = p.y;
  d.addend = p.addend;
  d.M = p.M;
  d.C = p.K;
  d.R = R;
  d.compute_dtype = to;
  d.d_dtype = p.y_dtype;
  return st != CAIFX_OK ? st : wide_run(d, room, only_size, s);
}

// The row kernels on the transposed copies: what neither of the others takes, weights of nearly 2^22 rows and stored ones of less than 16 columns.
int gradient_rows(const Gradient &p, Room &room, bool only_size, hipStream_t s)
{
  const int to = stored_as(p.compute_dtype);
  const int64_t pitch = up_to(p.N, kRowsChunk), stride = pitch * p.weights;       // whole chunks of each weight's rows
  const int chunks = static_cast<int>(stride / kRowsChunk);
  void *copy = room.take(static_cast<size_t>(p.K) * static_cast<size_t>(stride) * 2);
  void *packed = room.take(packed_bytes(p.M, chunks, p.compute_dtype));
  if (!only_size) {
    int st = operand_transposed(weights_of(p.w, p.weights, p.N, p.K, to), to, copy, pitch, stride, pitch, s);
    if (st == CAIFX_OK) st = operand_rows(activations_of(p.x[0], p.x[1], p.x_dtype, p.M, p.N), p.compute_dtype, packed, chunks, s);
    if (st != CAIFX_OK) return st;
  }
  RowsArgs g{};
  g.w[0] = copy;
  g.M = p.M;
  g.N = p.K;
  g.R = stride;
  g.w_pitch = 2 * stride;
  g.chunks = chunks;
  g.tiles = static_cast<int>((p.M + 15) / 16);
  g.x = packed;
  g.y = p.y;
  g.addend = p.addend;
  g.y_dtype = p.y_dtype;
  return rows_run(g, ROWS_DENSE, 1, p.compute_dtype, false, room, only_size, s);
}

// The gradient from the weights as they are stored.
DxProduct dx_of(const Gradient &p)
{
  DxProduct d{};
  d.M = p.M;
  d.N = p.N;
  d.K = p.K;
  d.count = p.weights;
  for (int i = 0; i < p.weights; ++i) {
    d.w[i] = p.w[i].p;
    d.s[i] = p.w[i].scales;
    d.x[i] = p.x[i];
  }
  d.mx = p.w[0].mx;
  d.compute_dtype = p.compute_dtype;
  d.y = p.y;
  d.y_dtype = p.y_dtype;
  d.addend = p.addend;
  d.direct = p.x_dtype == p.compute_dtype && p.N >= 8 && dx_reads(d);
  return d;
}

// The stored weights are turned around for every 32 rows again, the copies once: few rows run on dx, many on the copies.  Estimates in us of
// both.  Measured, copies / dx: N = 14336, K = 4096, bf16, 16 rows 57 / 16, 128 rows 61 / 39, 256 rows 79 / 66, 512 rows 96 / 116; N = 4096, K = 14336, 256 rows 66 / 73; N = K = 4096, 512 rows 38 / 36, in fp32 76 / 65, a gated block's
// gradient 69 / 78; 2048 x 1408, 512 rows 21 / 19.
bool dx_pays(const Gradient &p)
{
  const DxProduct d = dx_of(p);
  if (!dx_takes(d)) return false;
  if (!wide_gradient_takes(p)) return true;
  const int pieces = pieces_of(p.compute_dtype);
  const double values = p.weights * static_cast<double>(p.N) * static_cast<double>(p.K);
  const double far = values > 64e6 ? (values - 64e6) * 0.5e-6 : 0.0;      // (copies of more than half of the memory-side cache are read from further away)
  const double copies = 4.0 + values * (p.w[0].mx ? 2.53 : 4.0) / 4.4e6 + far + (pieces == 3 ? 19.0 : 0.0);
  return dx_us(d) < copies + wide_parts(p.M, p.K, p.weights * pieces * reduction_of(p)).us;
}

int gradient_dx(const Gradient &p, Room &room, bool only_size, hipStream_t s)
{
  DxProduct d = dx_of(p);
  void *partial = room.take(dx_partial_bytes(d));
  if (!d.direct) {
    const int chunks = p.weights * static_cast<int>(chunks_of(p.N));
    void *packed = room.take(packed_bytes(p.M, chunks, p.compute_dtype));
    if (only_size) return CAIFX_OK;
    const int st = operand_rows(activations_of(p.x[0], p.x[1], p.x_dtype, p.M, p.N), p.compute_dtype, packed, chunks, s);
    if (st != CAIFX_OK) return st;
    d.x[0] = packed;
  }
  return only_size ? CAIFX_OK : dx_product(d, partial, s);
}

int (*gradient_way(const Gradient &p))(const Gradient &, Room &, bool, hipStream_t)
{
  return dx_pays(p) ? gradient_dx : wide_gradient_takes(p) ? gradient_wide : gradient_rows;
}
size_t gradient_bytes(const Gradient &p) { return room_of(gradient_way(p), p); }
int gradient(const Gradient &p, void *workspace, size_t bytes, hipStream_t s) { return run_in(gradient_way(p), p, workspace, bytes, s); }

Product product_of(const GemmArgs &a)
{
  Product p{};
  p.M = a.M;
  p.N = a.N;
  p.R = a.K;
  p.x = a.x;
  p.x_dtype = a.x_dtype;
  p.compute_dtype = computed_in(a);
  p.weights = 1;
  p.w[0] = Weight{a.w.q, a.w.scales, true};
  p.y = a.y;
  p.y_dtype = a.y_dtype;
  p.addend = a.addend;
  return p;
}
Gradient gradient_of(const GemmArgs &a)
{
  Gradient p{};
  p.M = a.M;
  p.N = a.N;
  p.K = a.K;
  p.x[0] = a.x;
  p.x_dtype = a.x_dtype;
  p.compute_dtype = computed_in(a);
  p.weights = 1;
  p.w[0] = Weight{a.w.q, a.w.scales, true};
  p.y = a.y;
  p.y_dtype = a.y_dtype;
  p.addend = a.addend;
  return p;
}

// sizes that every launch here has a grid for
bool fits(int64_t M, int64_t N, int64_t K) { return M <= (1 << 30) && N < (1 << 22) && K < (1 << 22); }

}  // namespace

size_t mxfp4_workspace_bytes(const GemmArgs &a, bool backward, bool dense_copy)
{
  if (a.M <= 0 || a.N <= 0 || a.K <= 0 || !fits(a.M, a.N, a.K)) return 0;
  if (backward) return dense_copy ? gradient_bytes(gradient_of(a)) : 0;
  return product_bytes(product_of(a), dense_copy);
}

int mxfp4_linear(const GemmArgs &a, bool backward, hipStream_t s)
{
  if (!fits(a.M, a.N, a.K)) return CAIFX_ERR_UNSUPPORTED;
  const size_t need = mxfp4_workspace_bytes(a, backward, backward);
  if (need > 0 && (!a.workspace || a.workspace_bytes < need || !aligned_to(a.workspace, 16))) return CAIFX_ERR_UNSUPPORTED;
  if (backward) return gradient(gradient_of(a), a.workspace, a.workspace_bytes, s);
  return product(product_of(a), a.workspace, a.workspace && aligned_to(a.workspace, 16) ? a.workspace_bytes : 0, s);
}

}  // namespace caifx

using namespace caifx;

namespace {

int64_t blocks_of(int64_t columns) { return (columns + CAIFX_MXFP4_BLOCK - 1) / CAIFX_MXFP4_BLOCK; }
// whether a product of two operands in 4 bits runs in tiles rather than on the row kernels
bool tiles_pay(int64_t M, int64_t N, int64_t blocks)
{
  // A workgroup of the row kernels takes 64 x 64 results in 2.2 us and 1.1 for every 512 elements of the reduction, 256 of them at a time.  us, rows /
  // tiles, bf16: N = 14336, K = 4096, 96 rows 25 / 20; N = 4096, K = 14336, 96 rows 26 / 23, 256 rows 37 / 27; N = K = 4096, 256 rows 14 / 16, 512 rows
  // 26 / 17; 2048 x 1408, 512 rows 7 / 11.
  const int64_t groups = (M + 63) / 64 * ((N + 63) / 64);
  const double rounds = static_cast<double>(groups / 256) + (groups % 256 == 0 ? 0.0 : 0.35 + 0.65 / 256 * static_cast<double>(groups % 256));
  return M > 64 && mx_gemm_takes(M, N, blocks) && mx_gemm_us(M, N, blocks) < 3.5 + rounds * (2.2 + 1.1 * static_cast<double>((blocks + 15) / 16));
}

RowsArgs both_args(int64_t M, int64_t N, int64_t blocks)
{
  RowsArgs g{};
  g.M = M;
  g.N = N;
  g.R = 32 * blocks;
  g.blocks = blocks;
  g.w_pitch = 16 * blocks;
  g.chunks = static_cast<int>(chunks_of(g.R));
  return g;
}

// what both gated calls check; `go`: there is work
int gated_check(int64_t M, int64_t N, int64_t K, int w_kind, int dtype, bool &go)
{
  go = false;
  if (M < 0 || N <= 0 || K <= 0 || !valid_dtype(dtype)) return CAIFX_ERR_INVALID_ARGUMENT;
  if (w_kind < CAIFX_W_INT8 || (w_kind > CAIFX_W_BF16 && w_kind != CAIFX_W_MXFP4)) return CAIFX_ERR_INVALID_ARGUMENT;
  const bool stored = (w_kind == CAIFX_W_F16 && dtype == CAIFX_F16) || (w_kind == CAIFX_W_BF16 && dtype == CAIFX_BF16);
  if ((w_kind != CAIFX_W_MXFP4 && !stored) || !fits(M, N, K)) return CAIFX_ERR_UNSUPPORTED;
  go = M > 0;
  return CAIFX_OK;
}
Product gated_product(int64_t M, int64_t N, int64_t K, int w_kind, int dtype)
{
  Product p{};
  p.M = M;
  p.N = N;
  p.R = K;
  p.x_dtype = p.compute_dtype = p.y_dtype = dtype;
  p.weights = 2;
  p.w[0].mx = p.w[1].mx = w_kind == CAIFX_W_MXFP4;
  return p;
}
Gradient gated_gradient(int64_t M, int64_t N, int64_t K, int w_kind, int dtype)
{
  Gradient p{};
  p.M = M;
  p.N = N;
  p.K = K;
  p.x_dtype = p.compute_dtype = p.y_dtype = dtype;
  p.weights = 2;
  p.w[0].mx = p.w[1].mx = w_kind == CAIFX_W_MXFP4;
  return p;
}

}  // namespace

extern "C" {

size_t caifx_mxfp4_matmul_workspace_bytes(int64_t M, int64_t N, int64_t K)
{
  if (M <= 0 || N <= 0 || K <= 0 || !fits(M, N, K)) return 0;
  const int64_t blocks = blocks_of(K);
  Room room;
  rows_run(both_args(M, N, blocks), ROWS_BOTH, 1, CAIFX_BF16, true, room, true, nullptr);
  const size_t tiles = tiles_pay(M, N, blocks) ? mx_gemm_workspace_bytes(M, N, blocks) : 0;
  return tiles > room.used ? tiles : room.used;
}

int caifx_mxfp4_matmul(int64_t M, int64_t N, int64_t K, const void *a_codes, const void *a_scales, const void *b_codes, const void *b_scales, void *y,
                       int y_dtype, void *workspace, size_t workspace_bytes, caifx_stream_t stream)
{
  if (M < 0 || N < 0 || K <= 0 || !valid_dtype(y_dtype)) return CAIFX_ERR_INVALID_ARGUMENT;
  if (M == 0 || N == 0) return CAIFX_OK;
  if (!a_codes || !a_scales || !b_codes || !b_scales || !y) return CAIFX_ERR_INVALID_ARGUMENT;
  if (!fits(M, N, K)) return CAIFX_ERR_UNSUPPORTED;
  if (!aligned_to(a_codes, 16) || !aligned_to(b_codes, 16) || !aligned_to(y, dtype_size(y_dtype)) || !aligned_to(workspace, 16)) return CAIFX_ERR_MISALIGNED;
  const size_t need = caifx_mxfp4_matmul_workspace_bytes(M, N, K);
  if (need > 0 && (!workspace || workspace_bytes < need)) return CAIFX_ERR_WORKSPACE_TOO_SMALL;
  const int64_t blocks = blocks_of(K);
  if (tiles_pay(M, N, blocks))
    return mx_gemm(M, N, blocks, a_codes, a_scales, b_codes, b_scales, y, y_dtype, workspace, as_stream(stream));
  RowsArgs g = both_args(M, N, blocks);
  g.x = a_codes;
  g.xs = static_cast<const uint8_t *>(a_scales);
  g.w[0] = b_codes;
  g.s[0] = static_cast<const uint8_t *>(b_scales);
  g.y = y;
  g.y_dtype = y_dtype;
  Room room{static_cast<char *>(workspace), 0};
  return rows_run(g, ROWS_BOTH, 1, CAIFX_BF16, true, room, false, as_stream(stream));
}

size_t caifx_gated_workspace_bytes(int64_t M, int64_t N, int64_t K, int w_kind, int dtype, int backward)
{
  bool go;
  if (gated_check(M, N, K, w_kind, dtype, go) != CAIFX_OK || !go) return 0;
  if (backward) return gradient_bytes(gated_gradient(M, N, K, w_kind, dtype));
  return product_bytes(gated_product(M, N, K, w_kind, dtype));
}

int caifx_gated_forward(int64_t M, int64_t N, int64_t K, const void *x, const void *w_gate, const void *scales_gate, const void *w_up,
                        const void *scales_up, int w_kind, void *hidden, void *gate, void *up, int dtype, void *workspace, size_t workspace_bytes,
                        caifx_stream_t stream)
{
  bool go;
  const int st = gated_check(M, N, K, w_kind, dtype, go);
  if (!go) return st;
  const bool mx = w_kind == CAIFX_W_MXFP4;
  if (!x || !w_gate || !w_up || !hidden || (mx && (!scales_gate || !scales_up)) || (gate == nullptr) != (up == nullptr)) return CAIFX_ERR_INVALID_ARGUMENT;
  if (x == hidden || x == gate || x == up || hidden == gate || hidden == up || (gate && gate == up)) return CAIFX_ERR_INVALID_ARGUMENT;
  const size_t es = dtype_size(dtype);
  if (!aligned_to(x, es) || !aligned_to(hidden, es) || !aligned_to(gate, es) || !aligned_to(up, es) || !aligned_to(w_gate, 16) || !aligned_to(w_up, 16) ||
      !aligned_to(workspace, 16))
    return CAIFX_ERR_MISALIGNED;
  const size_t need = caifx_gated_workspace_bytes(M, N, K, w_kind, dtype, 0);
  if (need > 0 && (!workspace || workspace_bytes < need)) return CAIFX_ERR_WORKSPACE_TOO_SMALL;
  Product p = gated_product(M, N, K, w_kind, dtype);
  p.x = x;
  p.w[0].p = w_gate;
  p.w[0].scales = scales_gate;
  p.w[1].p = w_up;
  p.w[1].scales = scales_up;
  p.y = hidden;
  p.gate = gate;
  p.up = up;
  return product(p, workspace, workspace_bytes, as_stream(stream));
}

int caifx_gated_backward(int64_t M, int64_t N, int64_t K, const void *grad_hidden, const void *gate, const void *up, const void *w_gate,
                         const void *scales_gate, const void *w_up, const void *scales_up, int w_kind, void *grad_gate, void *grad_up, void *dx, int dtype,
                         void *workspace, size_t workspace_bytes, caifx_stream_t stream)
{
  bool go;
  int st = gated_check(M, N, K, w_kind, dtype, go);
  if (!go) return st;
  const bool mx = w_kind == CAIFX_W_MXFP4;
  if (!grad_hidden || !gate || !up || !grad_gate || !grad_up || (dx && (!w_gate || !w_up || (mx && (!scales_gate || !scales_up)))))
    return CAIFX_ERR_INVALID_ARGUMENT;
  const void *in[3] = {grad_hidden, gate, up};
  for (const void *i : in)
    if (i == grad_gate || i == grad_up || i == dx) return CAIFX_ERR_INVALID_ARGUMENT;
  if (grad_gate == grad_up || grad_gate == dx || grad_up == dx) return CAIFX_ERR_INVALID_ARGUMENT;
  const size_t es = dtype_size(dtype);
  if (!aligned_to(grad_hidden, es) || !aligned_to(gate, es) || !aligned_to(up, es) || !aligned_to(grad_gate, es) || !aligned_to(grad_up, es) ||
      !aligned_to(dx, es) || !aligned_to(w_gate, 16) || !aligned_to(w_up, 16) || !aligned_to(workspace, 16))
    return CAIFX_ERR_MISALIGNED;
  const size_t need = dx ? caifx_gated_workspace_bytes(M, N, K, w_kind, dtype, 1) : 0;
  if (need > 0 && (!workspace || workspace_bytes < need)) return CAIFX_ERR_WORKSPACE_TOO_SMALL;
  hipStream_t s = as_stream(stream);
  st = gating_backward(grad_hidden, gate, up, grad_gate, grad_up, M * N, dtype, s);
  if (st != CAIFX_OK || !dx) return st;
  Gradient p = gated_gradient(M, N, K, w_kind, dtype);
  p.x[0] = grad_gate;
  p.x[1] = grad_up;
  p.w[0].p = w_gate;
  p.w[0].scales = scales_gate;
  p.w[1].p = w_up;
  p.w[1].scales = scales_up;
  p.y = dx;
  return gradient(p, workspace, workspace_bytes, s);
}

}  // extern "C"
