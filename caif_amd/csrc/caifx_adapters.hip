// Low-rank adapters beside a frozen projection: the branch of every row's own adapter added to the projection's result, and the
// branch's gradients.  Row m uses adapter l = ids[m] (none where ids[m] is outside [0, L)):
//
//   forward    h[m] = x[m] A[l]^T                  y[m]  = T(base[m] + scaling[l] h[m] B[l]^T)
//   backward   g[m] = scaling[l] dy[m] B[l]        dx[m] = T(base[m] + g[m] A[l])
//              dA[l] = T(sum over m of l of g[m]^T x[m])      dB[l] = T(sum over m of l of scaling[l] dy[m]^T h[m])
//
// with x [M,K], A [L,r,K], B [L,N,r], h and g [M,r] in fp32.  A rank of 16 leaves 16 multiply-adds for a value read or written,
// so all of it is bound by memory: x, dy, base and the result pass once, the factors come from the caches, and the matrix cores
// keep the arithmetic out of the way.  Four kinds of product:
//
//   shrink   rows x factor over the long axis (h, g): a workgroup takes 16 rows, its waves share the axis
//   expand   rank -> long axis (y, dx): a wave takes 16 rows x 64 columns, adds base and rounds once
//   outer    sums over the rows of an adapter (dA, dB): a workgroup takes 128 columns of one adapter and lists its rows first
//   row      shrink and expand of one row in one launch, for decode steps
//
// Precision: products of two 16-bit values are exact in fp32 and summed in fp32.  h and g stay fp32; on the 16-bit matrix cores they
// are two bf16 pieces that add up to them but for 2^-17 (and an fp16 partner two bf16 pieces that add up to it exactly, so no value
// leaves the range of a piece), which is far below the one rounding of the result.  fp32 tensors use the fp32 instruction.
//
// Rows of different adapters never meet in a product: a tile with several adapters is multiplied by each of them and every row
// keeps the result of its own, so that an infinity in one adapter's factors stays out of the other rows.
#include "caifx_common.hpp"

#include <type_traits>

namespace caifx {
namespace {

struct Problem {
  int64_t M, N, K;
  int r, L;
  const int32_t *ids;
  const void *a, *b;
  const float *scaling;
};

// ------------------------------------------------------------------ operands
// Eight values of a lane: reduction elements 8 q .. + 7 of row (column) i, with i = lane % 16, q = lane / 16.  One step of every
// product below is 16 x 16 x 32.
typedef __attribute__((__vector_size__(8 * sizeof(float)))) float f32x8_t;
template <typename T> struct Vec8;
template <> struct Vec8<float> { typedef f32x8_t type; };
template <> struct Vec8<f16_t> { typedef f16x8_t type; };
template <> struct Vec8<bf16_t> { typedef bf16x8_t type; };
template <typename T> using vec8 = typename Vec8<T>::type;

template <typename V> __device__ __forceinline__ V zero8()
{
  V v;
  __builtin_memset(&v, 0, sizeof v);
  return v;
}
// eight values from p, of any alignment; `have` of them exist (zeros for the others, which are not read)
template <typename T> __device__ __forceinline__ vec8<T> load8(const T *p)
{
  vec8<T> v;
  __builtin_memcpy(&v, p, sizeof v);
  return v;
}
template <typename T> __device__ __forceinline__ vec8<T> load8(const T *p, int have)
{
  if (have >= 8) return load8<T>(p);
  vec8<T> v = zero8<vec8<T>>();
#pragma unroll
  for (int i = 0; i < 7; ++i)
    if (i < have) v[i] = p[i];
  return v;
}
__device__ __forceinline__ int clamp8(int64_t n) { return n >= 8 ? 8 : (n > 0 ? static_cast<int>(n) : 0); }

// acc[4 q + e][i] += a (row i) . b (column i)
__device__ __forceinline__ floatx4_t mma(bf16x8_t a, bf16x8_t b, floatx4_t acc) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, acc, 0, 0, 0); }
__device__ __forceinline__ floatx4_t mma(f16x8_t a, f16x8_t b, floatx4_t acc) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, acc, 0, 0, 0); }
__device__ __forceinline__ floatx4_t mma(f32x8_t a, f32x8_t b, floatx4_t acc)
{
#pragma unroll
  for (int e = 0; e < 8; ++e) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], b[e], acc, 0, 0, 0);
  return acc;
}

// fp32 values as two bf16 pieces
struct Pieces {
  bf16x8_t hi, lo;
};
__device__ __forceinline__ Pieces split(const f32x8_t &v)
{
  Pieces p;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    p.hi[e] = from_f32<bf16_t>(v[e]);
    p.lo[e] = from_f32<bf16_t>(v[e] - to_f32<bf16_t>(p.hi[e]));
  }
  return p;
}
// the fp32 side of a product with tensors of type T
template <typename T> struct Fine { typedef Pieces type; };
template <> struct Fine<float> { typedef f32x8_t type; };
template <typename T> __device__ __forceinline__ typename Fine<T>::type fine(const f32x8_t &v)
{
  if constexpr (sizeof(T) == 4) return v;
  else return split(v);
}
// the tensor's side: bf16 and fp32 as they are, fp16 as two pieces
__device__ __forceinline__ bf16x8_t whole(bf16x8_t v) { return v; }
__device__ __forceinline__ f32x8_t whole(f32x8_t v) { return v; }
__device__ __forceinline__ Pieces whole(f16x8_t v)
{
  f32x8_t w;
#pragma unroll
  for (int e = 0; e < 8; ++e) w[e] = to_f32<f16_t>(v[e]);
  return split(w);
}
__device__ __forceinline__ floatx4_t mma(const f32x8_t &w, const f32x8_t &u, floatx4_t acc, int) { return mma(w, u, acc); }
__device__ __forceinline__ floatx4_t mma(const bf16x8_t &w, const Pieces &u, floatx4_t acc, int) { return mma(w, u.lo, mma(w, u.hi, acc)); }
__device__ __forceinline__ floatx4_t mma(const Pieces &w, const Pieces &u, floatx4_t acc, int)
{
  return mma(w.lo, u.hi, mma(w.hi, u.lo, mma(w.hi, u.hi, acc)));
}
__device__ __forceinline__ floatx4_t mma(const Pieces &u, const bf16x8_t &w, floatx4_t acc, int) { return mma(u.lo, w, mma(u.hi, w, acc)); }

// Operand of a tile whose reduction runs down the rows of a matrix in LDS (row-major, `pitch` values a row): lane (i, q) gets rows
// 8 q .. + 7 of column column(i) = 4 (i / 4) columns apart by `spread`: i % 4 + spread * (i / 4).  The 16-bit form reads with the
// transposing instruction: of the sixteen lanes of a q, lane t asks for four neighbouring values of row t / 4, columns
// spread (t % 4) .. + 3, and receives column t of the four rows.
typedef __attribute__((__vector_size__(4 * sizeof(short)))) short s16x4_t;
template <typename T> __device__ __forceinline__ vec8<T> down(const T *m, int pitch, int spread, int lane)
{
  const int q = lane >> 4, t = lane & 15;
  if constexpr (sizeof(T) == 2) {
    typedef __attribute__((address_space(3))) s16x4_t lds_t;
    const T *p = m + (8 * q + (t >> 2)) * pitch + spread * (t & 3);
    struct { s16x4_t a, b; } v;
    v.a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_t *)(p));
    v.b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_t *)(p + 4 * pitch));
    return __builtin_bit_cast(vec8<T>, v);
  } else {
    vec8<T> v;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = m[(8 * q + e) * pitch + spread * (t >> 2) + (t & 3)];
    return v;
  }
}

// ------------------------------------------------------------------ adapters of a tile of rows
// Lane (i, q) holds row i's adapter, -1 for none.  next() goes through the adapters of the tile, each once.
struct TileIds {
  int mine;
  uint64_t pending;
  __device__ TileIds(const Problem &p, int64_t m)
  {
    mine = -1;
    if (m < p.M) {
      const int l = p.ids[m];
      if (l >= 0 && l < p.L) mine = l;
    }
    pending = __ballot(mine >= 0);
  }
  // the next adapter of the tile, the same for all lanes; -1 when there is none
  __device__ int next()
  {
    if (pending == 0) return -1;
    const int l = __builtin_amdgcn_readlane(mine, __builtin_ctzll(pending));
    pending &= ~__ballot(mine == l);
    return l;
  }
};

// ------------------------------------------------------------------ shrink
constexpr int kShrinkWaves = 8;
constexpr int kUnit = 64;                             // columns that a wave takes at a time: a line of a row in 16 bits

// out[slice][m][j] = scale sum over the slice's columns c of z[m][c] f[l][j][c] (kDown: f[l][c][j]), rows without adapter zero.
// The factor is the A operand (rows j), the rows are the B operand, so a lane's results belong to one row m = i.
template <typename T, int JT, bool kDown>
__global__ __launch_bounds__(64 * kShrinkWaves) void shrink_kernel(Problem p, const T *__restrict__ z, int64_t C, const T *__restrict__ f, int64_t per_slice,
                                                                   bool scaled, float *__restrict__ out)
{
  constexpr int R = 16 * JT;
  constexpr int kSteps = R * sizeof(T) >= (kDown ? 256 : 512) ? 1 : 2;       // of 32 columns, staged or loaded together
  constexpr int kCols = 32 * kSteps;
  constexpr int kStage = kDown ? kCols * R * sizeof(T) : 0;             // bytes of a wave's staged factor
  constexpr int kSums = 16 * R * 4;
  __shared__ __align__(32) unsigned char lds[kShrinkWaves * (kStage > kSums ? kStage : kSums)];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i = lane & 15, q = lane >> 4;
  const int64_t m = static_cast<int64_t>(blockIdx.x) * 16 + i;
  const int64_t lo = blockIdx.y * per_slice, hi = lo + per_slice < C ? lo + per_slice : C;
  TileIds ids(p, m);
  floatx4_t sum[JT];
#pragma unroll
  for (int j = 0; j < JT; ++j) sum[j] = floatx4_t{0, 0, 0, 0};
  const T *row = z + (m < p.M ? m : 0) * C;
  T *stage = reinterpret_cast<T *>(lds) + wave * (kStage / sizeof(T));
  for (int l = ids.next(); l >= 0; l = ids.next()) {
    const bool mine = ids.mine == l;
    const T *factor = f + static_cast<int64_t>(l) * p.r * C;
    floatx4_t acc[JT];
#pragma unroll
    for (int j = 0; j < JT; ++j) acc[j] = floatx4_t{0, 0, 0, 0};
    auto unit = [&](int64_t c0, auto is_full) {
      constexpr bool kFull = decltype(is_full)::value;
      vec8<T> zv[kSteps], fv[kSteps][JT];
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        const int64_t c = c0 + 32 * s + 8 * q;
        zv[s] = zero8<vec8<T>>();
        if (mine) zv[s] = kFull ? load8<T>(row + c) : load8<T>(row + c, clamp8(hi - c));
        if constexpr (!kDown) {
#pragma unroll
          for (int j = 0; j < JT; ++j) {
            const int at = 16 * j + i < p.r ? 16 * j + i : p.r - 1;         // rows past the rank repeat the last; their sums are not kept
            fv[s][j] = kFull ? load8<T>(factor + at * C + c) : load8<T>(factor + at * C + c, clamp8(hi - c));
          }
        }
      }
      if constexpr (kDown) {
        // the factor's rows c0 .. + kCols, eight ranks at a time, zeros past the rank and past the last column
        constexpr int kOct = R / 8;
        vec8<T> st[kCols * kOct / 64];
#pragma unroll
        for (int o = 0; o < kCols * kOct / 64; ++o) {
          const int at = o * 64 + lane, c = at / kOct, j = at % kOct * 8;
          st[o] = load8<T>(factor + (c0 + c) * p.r + j, kFull || c0 + c < hi ? clamp8(p.r - j) : 0);
        }
#pragma unroll
        for (int o = 0; o < kCols * kOct / 64; ++o) *reinterpret_cast<vec8<T> *>(stage + (o * 64 + lane) * 8) = st[o];
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int s = 0; s < kSteps; ++s)
#pragma unroll
          for (int j = 0; j < JT; ++j) fv[s][j] = down<T>(stage + 32 * s * R + 16 * j, R, 4, lane);
        __builtin_amdgcn_wave_barrier();
      }
#pragma unroll
      for (int s = 0; s < kSteps; ++s)
#pragma unroll
        for (int j = 0; j < JT; ++j) acc[j] = mma(fv[s][j], zv[s], acc[j]);
    };
    int64_t c0 = lo + wave * kCols;
    for (; c0 + kCols <= hi; c0 += kShrinkWaves * kCols) unit(c0, std::true_type{});
    if (c0 < hi) unit(c0, std::false_type{});
#pragma unroll
    for (int j = 0; j < JT; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) sum[j][e] = mine ? acc[j][e] : sum[j][e];
  }
  // the waves' shares, [wave][m][j], added in the waves' order
  __syncthreads();
  float *sums = reinterpret_cast<float *>(lds);
#pragma unroll
  for (int j = 0; j < JT; ++j) *reinterpret_cast<floatx4_t *>(sums + (wave * 16 + i) * R + 16 * j + 4 * q) = sum[j];
  __syncthreads();
  for (int o = threadIdx.x; o < 16 * R; o += 64 * kShrinkWaves) {
    const int64_t mm = static_cast<int64_t>(blockIdx.x) * 16 + o / R;
    const int j = o % R;
    if (mm >= p.M || j >= p.r) continue;
    float v = 0.0f;
#pragma unroll
    for (int w = 0; w < kShrinkWaves; ++w) v += sums[w * 16 * R + o];
    if (scaled) {
      const int l = p.ids[mm];
      v = l >= 0 && l < p.L ? v * p.scaling[l] : 0.0f;
    }
    out[(blockIdx.y * p.M + mm) * p.r + j] = v;
  }
}

// ------------------------------------------------------------------ the fp32 rows h and g
// [slices][M][r]; a row is the sum of its slices in order
struct Rows {
  const float *at;
  int slices;
};
// values j .. j + 7 of row m, zeros past the rank
__device__ __forceinline__ f32x8_t rank8(const Problem &p, const Rows &u, int64_t m, int j)
{
  const int have = clamp8(p.r - j);
  const float *at = u.at + m * p.r + j;
  f32x8_t v = load8<float>(at, have);
  for (int s = 1; s < u.slices; ++s) {
    const f32x8_t w = load8<float>(at + s * p.M * p.r, have);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] += w[e];
  }
  return v;
}

// ------------------------------------------------------------------ expand
constexpr int kExpandWaves = 4;
constexpr int kExpandCols = 64;                       // of a wave

// out[m][c] = T(base[m][c] + scale sum_j u[m][j] f[l][c][j])  (kDown: f[l][j][c]).  Of the 16 x 16 results of a product a lane holds
// four neighbouring columns of one row; two products whose columns alternate by fours give it eight, one 16-byte access.
// hidden: the rows themselves, written by the first columns' waves.
template <typename T, int RS, bool kDown>
__global__ __launch_bounds__(64 * kExpandWaves) void expand_kernel(Problem p, Rows u, int64_t C, int64_t col_tiles, const T *__restrict__ f, bool scaled,
                                                                   const T *base, T *out, float *__restrict__ hidden)
{
  constexpr int kPitch = kExpandCols + 8;
  __shared__ __align__(32) T lds[kDown ? kExpandWaves * 32 * kPitch : 1];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i = lane & 15, q = lane >> 4;
  const int64_t tile = static_cast<int64_t>(blockIdx.x) / col_tiles;
  const int64_t c0 = ((static_cast<int64_t>(blockIdx.x) - tile * col_tiles) * kExpandWaves + wave) * kExpandCols;
  if (c0 >= C) return;
  const int64_t m = tile * 16 + i;
  const bool in = m < p.M;
  vec8<T> old[2];
  int have[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int64_t c = c0 + 32 * h + 8 * q;
    have[h] = in ? clamp8(C - c) : 0;
    old[h] = zero8<vec8<T>>();
    if (base) old[h] = load8<T>(base + m * C + c, have[h]);
  }
  TileIds ids(p, m);
  typename Fine<T>::type uv[RS];
  const float scale = scaled && ids.mine >= 0 ? p.scaling[ids.mine] : 1.0f;
#pragma unroll
  for (int s = 0; s < RS; ++s) {
    f32x8_t v = zero8<f32x8_t>();
    if (in) v = rank8(p, u, m, 32 * s + 8 * q);
    if (hidden && c0 == 0 && in) {
      for (int e = 0; e < 8; ++e)
        if (32 * s + 8 * q + e < p.r) hidden[m * p.r + 32 * s + 8 * q + e] = v[e];
    }
    if (scaled) {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] *= scale;
    }
    uv[s] = fine<T>(v);
  }
  floatx4_t sum[4];
#pragma unroll
  for (int t = 0; t < 4; ++t) sum[t] = floatx4_t{0, 0, 0, 0};
  T *stage = lds + (kDown ? wave * 32 * kPitch : 0);
  for (int l = ids.next(); l >= 0; l = ids.next()) {
    const bool mine = ids.mine == l;
    const T *factor = f + static_cast<int64_t>(l) * p.r * C;
    floatx4_t acc[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) acc[t] = floatx4_t{0, 0, 0, 0};
#pragma unroll
    for (int s = 0; s < RS; ++s) {
      vec8<T> fv[4];
      if constexpr (kDown) {
        // ranks 32 s .. + 31 of the wave's columns, zeros past the rank and past the last column
        vec8<T> st[4];
#pragma unroll
        for (int o = 0; o < 4; ++o) {
          const int j = 32 * s + 8 * o + (lane >> 3);
          const int64_t c = c0 + 8 * (lane & 7);
          st[o] = load8<T>(factor + j * C + c, j < p.r ? clamp8(C - c) : 0);
        }
#pragma unroll
        for (int o = 0; o < 4; ++o) *reinterpret_cast<vec8<T> *>(stage + (8 * o + (lane >> 3)) * kPitch + 8 * (lane & 7)) = st[o];
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int t = 0; t < 4; ++t) fv[t] = down<T>(stage + 32 * (t >> 1) + 4 * (t & 1), kPitch, 8, lane);
        __builtin_amdgcn_wave_barrier();
      } else {
        const int j = 32 * s + 8 * q, hj = clamp8(p.r - j);
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          const int64_t c = c0 + 32 * (t >> 1) + 8 * (i >> 2) + 4 * (t & 1) + (i & 3);
          fv[t] = load8<T>(factor + c * p.r + j, c < C ? hj : 0);
        }
      }
#pragma unroll
      for (int t = 0; t < 4; ++t) acc[t] = mma(whole(fv[t]), uv[s], acc[t], 0);
    }
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) sum[t][e] = mine ? acc[t][e] : sum[t][e];
  }
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    // a row without adapter keeps its base bit for bit, also a NaN's
    if (ids.mine >= 0) {
#pragma unroll
      for (int e = 0; e < 8; ++e) old[h][e] = from_f32<T>(to_f32<T>(old[h][e]) + sum[2 * h + (e >> 2)][e & 3]);
    }
    T *to = out + m * C + c0 + 32 * h + 8 * q;
    if (have[h] == 8) {
      __builtin_memcpy(to, &old[h], sizeof old[h]);
    } else {
#pragma unroll
      for (int e = 0; e < 7; ++e)
        if (e < have[h]) to[e] = old[h][e];
    }
  }
}

// ------------------------------------------------------------------ one row, both products
constexpr int kRowWaves = 8;

// A workgroup takes one row and a part of the result's columns and forms the row's h itself: the other parts do the same from the
// caches, which costs less than a second launch.  Both products use one row (column) of sixteen; the matrix cores are not what
// bounds them.
template <typename T, int JT>
__global__ __launch_bounds__(64 * kRowWaves) void row_kernel(Problem p, const T *__restrict__ x, const T *__restrict__ a, const T *__restrict__ b,
                                                             int64_t per_block, const T *base, T *out, float *__restrict__ hidden)
{
  constexpr int R = 16 * JT, RS = (JT + 1) / 2;
  __shared__ float shares[kRowWaves][R], total[RS * 32];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i = lane & 15, q = lane >> 4;
  const int64_t m = blockIdx.y;
  const int64_t lo = blockIdx.x * per_block, hi = lo + per_block < p.N ? lo + per_block : p.N;
  const int l = p.ids[m];
  if (l < 0 || l >= p.L) {
    for (int64_t c = lo + threadIdx.x; c < hi; c += 64 * kRowWaves) out[m * p.N + c] = base ? base[m * p.N + c] : T(0.0f);
    if (hidden && blockIdx.x == 0 && threadIdx.x < static_cast<unsigned>(p.r)) hidden[m * p.r + threadIdx.x] = 0.0f;
    return;
  }
  const T *fa = a + static_cast<int64_t>(l) * p.r * p.K, *fb = b + static_cast<int64_t>(l) * p.N * p.r, *row = x + m * p.K;
  floatx4_t acc[JT];
#pragma unroll
  for (int j = 0; j < JT; ++j) acc[j] = floatx4_t{0, 0, 0, 0};
  for (int64_t c = wave * 32; c < p.K; c += 32 * kRowWaves) {
    const int64_t at = c + 8 * q;
    const int have = clamp8(p.K - at);
    const vec8<T> xv = load8<T>(row + at, have);
#pragma unroll
    for (int j = 0; j < JT; ++j) {
      const int64_t r = 16 * j + i < p.r ? 16 * j + i : p.r - 1;
      acc[j] = mma(load8<T>(fa + r * p.K + at, have), xv, acc[j]);
    }
  }
  if (i == 0) {
#pragma unroll
    for (int j = 0; j < JT; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) shares[wave][16 * j + 4 * q + e] = acc[j][e];
  }
  __syncthreads();
  if (threadIdx.x < RS * 32) {
    float v = 0.0f;
    if (threadIdx.x < static_cast<unsigned>(p.r)) {
#pragma unroll
      for (int w = 0; w < kRowWaves; ++w) v += shares[w][threadIdx.x];
      if (hidden && blockIdx.x == 0) hidden[m * p.r + threadIdx.x] = v;
    }
    total[threadIdx.x] = v * p.scaling[l];
  }
  __syncthreads();
  typename Fine<T>::type uv[RS];
#pragma unroll
  for (int s = 0; s < RS; ++s) {
    f32x8_t v;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = 32 * s + 8 * q + e < p.r ? total[32 * s + 8 * q + e] : 0.0f;
    uv[s] = fine<T>(v);
  }
  for (int64_t c0 = lo + wave * 64; c0 < hi; c0 += 64 * kRowWaves) {
    floatx4_t y[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) y[t] = floatx4_t{0, 0, 0, 0};
#pragma unroll
    for (int s = 0; s < RS; ++s) {
      const int j = 32 * s + 8 * q, hj = clamp8(p.r - j);
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const int64_t c = c0 + 16 * t + i;
        y[t] = mma(uv[s], whole(load8<T>(fb + c * p.r + j, c < hi ? hj : 0)), y[t], 0);
      }
    }
    // every row of a product is the same: the lanes of q keep column tile q
    const float v = q == 0 ? y[0][0] : q == 1 ? y[1][0] : q == 2 ? y[2][0] : y[3][0];
    const int64_t c = c0 + lane;
    if (c < hi) out[m * p.N + c] = from_f32<T>((base ? to_f32<T>(base[m * p.N + c]) : 0.0f) + v);
  }
}

// ------------------------------------------------------------------ outer
constexpr int kOuterThreads = 256;
constexpr int kOuterCols = 128;                       // of a workgroup, 32 of a wave; a checkpoint's group
constexpr int kOuterRows = 32;                        // of a step
constexpr int kOuterList = 1024;                      // rows looked through at a time

// what a tensor's values are in LDS: int8 codes are exact in bf16
template <typename Z, typename T> struct Staged { typedef Z type; };
template <typename T> struct Staged<int8_t, T> { typedef bf16_t type; };
template <> struct Staged<int8_t, float> { typedef float type; };
template <typename Z> __device__ __forceinline__ void load8_as(vec8<Z> &v, const Z *p, int have) { v = load8<Z>(p, have); }
template <typename V> __device__ __forceinline__ void load8_as(V &v, const int8_t *p, int have)
{
  int8_t c[8] = {0, 0, 0, 0, 0, 0, 0, 0};
  if (have >= 8) {
    __builtin_memcpy(c, p, 8);
  } else {
#pragma unroll
    for (int e = 0; e < 7; ++e)
      if (e < have) c[e] = p[e];
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = static_cast<float>(c[e]);
}

struct Outer {
  const void *z;                                      // [M, C], int8 codes with z_scales [M, groups]
  const float *z_scales;
  Rows u;
  int64_t C;
  bool scaled;
  int64_t js, cs;                                     // of the result: [l][j * js + c * cs]
  void *grad;                                         // T, or fp32 [splits] of it
  int splits;
  int64_t rows;                                       // of a split
};

// grad[l][c][j] = scale sum over the rows m of l of z[m][c] u[m][j]: both operands run down their rows, so both are staged in LDS as
// they lie in memory and read with the transposing instruction.  The rows of the adapter are listed first (in order: results repeat),
// so rows of other adapters cost nothing but their id.
template <typename Z, typename T, int JT, bool kPartial>
__global__ __launch_bounds__(kOuterThreads) void outer_kernel(Problem p, Outer o)
{
  typedef typename Staged<Z, T>::type S;
  constexpr int R = 16 * JT;
  constexpr int kZPitch = kOuterCols + 8, kUPitch = R + 8;
  constexpr bool k16 = sizeof(T) == 2;
  typedef typename std::conditional<k16, bf16_t, float>::type UT;
  __shared__ __align__(32) S zs[kOuterRows * kZPitch];
  __shared__ __align__(16) UT us[k16 ? 2 : 1][kOuterRows * kUPitch];
  __shared__ int32_t list[kOuterList];
  __shared__ int counts[kOuterThreads / 64];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, i = lane & 15, q = lane >> 4;
  const int64_t tiles = (o.C + kOuterCols - 1) / kOuterCols;
  int64_t at = blockIdx.x;
  const int64_t c0 = at % tiles * kOuterCols;
  at /= tiles;
  const int l = static_cast<int>(at % p.L);
  const int64_t split = at / p.L;
  const int64_t lo = split * o.rows, hi = lo + o.rows < p.M ? lo + o.rows : p.M;
  const Z *z = static_cast<const Z *>(o.z);
  const int64_t groups = (o.C + CAIFX_CHECKPOINT_GROUP - 1) / CAIFX_CHECKPOINT_GROUP, group = c0 / CAIFX_CHECKPOINT_GROUP;
  floatx4_t acc[2][JT];
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int j = 0; j < JT; ++j) acc[t][j] = floatx4_t{0, 0, 0, 0};

  bool any = false;
  for (int64_t base = lo; base < hi; base += kOuterList) {
    // rows base .. + 1023 of this adapter, in order: thread t looks at four neighbouring rows
    int mine[4], n = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int64_t m = base + tid * 4 + k;
      mine[k] = m < hi && p.ids[m] == l;
      n += mine[k];
    }
    int before = n;
#pragma unroll
    for (int s = 1; s < 64; s <<= 1) {
      const int up = __shfl_up(before, s, 64);
      if (lane >= s) before += up;
    }
    __syncthreads();                                  // the last window's list has been read
    if (lane == 63) counts[wave] = before;
    __syncthreads();
    int total = 0;
    before -= n;
#pragma unroll
    for (int w = 0; w < kOuterThreads / 64; ++w) {
      if (w < wave) before += counts[w];
      total += counts[w];
    }
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (mine[k]) list[before++] = tid * 4 + k;
    __syncthreads();

    // a step's values of a thread: two octets of z, 2 JT values of u
    vec8<S> zv[2];
    float uv[2 * JT];
    const int zrow = tid >> 4, zcol = (tid & 15) * 8, urow = tid >> 3, ucol = (tid & 7) * 2 * JT;
    auto fetch = [&](int s) {
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int e = s * kOuterRows + zrow + 16 * k;
        zv[k] = zero8<vec8<S>>();
        if (e < total) load8_as(zv[k], z + (base + list[e]) * o.C + c0 + zcol, clamp8(o.C - c0 - zcol));
      }
      const int e = s * kOuterRows + urow;
#pragma unroll
      for (int k = 0; k < 2 * JT; ++k) uv[k] = 0.0f;
      if (e < total) {
        const int64_t m = base + list[e];
        const float by = o.z_scales ? o.z_scales[m * groups + group] : 1.0f;
#pragma unroll
        for (int k = 0; k < 2 * JT; ++k) {
          if (ucol + k < p.r) {
            const float *from = o.u.at + m * p.r + ucol + k;
            float v = *from;
            for (int w = 1; w < o.u.slices; ++w) v += from[w * p.M * p.r];
            uv[k] = v * by;
          }
        }
      }
    };
    const int steps = (total + kOuterRows - 1) / kOuterRows;
    any |= steps > 0;
    if (steps > 0) fetch(0);
    for (int s = 0; s < steps; ++s) {
      if (s > 0) __syncthreads();                     // the step before has been read
#pragma unroll
      for (int k = 0; k < 2; ++k) *reinterpret_cast<vec8<S> *>(zs + (zrow + 16 * k) * kZPitch + zcol) = zv[k];
#pragma unroll
      for (int k = 0; k < 2 * JT; ++k) {
        if constexpr (k16) {
          const bf16_t top = from_f32<bf16_t>(uv[k]);
          us[0][urow * kUPitch + ucol + k] = top;
          us[1][urow * kUPitch + ucol + k] = from_f32<bf16_t>(uv[k] - to_f32<bf16_t>(top));
        } else {
          us[0][urow * kUPitch + ucol + k] = uv[k];
        }
      }
      __syncthreads();
      if (s + 1 < steps) fetch(s + 1);
      typename Fine<T>::type uf[JT];
#pragma unroll
      for (int j = 0; j < JT; ++j) {
        if constexpr (k16) {
          uf[j].hi = down<UT>(us[0] + 16 * j, kUPitch, 4, lane);
          uf[j].lo = down<UT>(us[1] + 16 * j, kUPitch, 4, lane);
        } else {
          uf[j] = down<UT>(us[0] + 16 * j, kUPitch, 4, lane);
        }
      }
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const auto w = whole(down<S>(zs + 32 * wave + 16 * t, kZPitch, 4, lane));
#pragma unroll
        for (int j = 0; j < JT; ++j) acc[t][j] = mma(w, uf[j], acc[t][j], 0);
      }
    }
  }
  // an adapter without rows has zero gradients whatever its scaling
  const float scale = o.scaled && any ? p.scaling[l] : 1.0f;
  const int64_t first = static_cast<int64_t>(l) * p.r * o.C;
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int j = 0; j < JT; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int64_t c = c0 + 32 * wave + 16 * t + 4 * q + e;
        const int jj = 16 * j + i;
        if (c >= o.C || jj >= p.r) continue;
        const int64_t to = first + jj * o.js + c * o.cs;
        const float v = acc[t][j][e] * scale;
        if constexpr (kPartial) static_cast<float *>(o.grad)[split * p.L * p.r * o.C + to] = v;
        else static_cast<T *>(o.grad)[to] = from_f32<T>(v);
      }
}

// both gradients' splits added in order
struct Join {
  const float *part;
  void *grad;
  int64_t n;
  int splits;
};
template <typename T> __global__ __launch_bounds__(256) void join_kernel(Join a, Join b)
{
  int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const bool second = i >= a.n;
  if (second) i -= a.n;
  const Join &j = second ? b : a;
  if (i >= j.n) return;
  float v = j.part[i];
  for (int s = 1; s < j.splits; ++s) v += j.part[s * j.n + i];
  static_cast<T *>(j.grad)[i] = from_f32<T>(v);
}

// ------------------------------------------------------------------ host
int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Workgroups of the shrinking product per 16 rows: enough that some 512 run, a slice no shorter than one unit for each wave.
struct Slices {
  int count;
  int64_t columns;
};
Slices plan_slices(int64_t M, int64_t C)
{
  const int64_t tiles = ceil_div(M, 16), whole = ceil_div(C, kShrinkWaves * kUnit);
  int64_t n = 512 / (tiles > 0 ? tiles : 1);
  n = n < 1 ? 1 : (n > 16 ? 16 : n);
  if (n > whole) n = whole;
  const int64_t columns = ceil_div(whole, n) * kShrinkWaves * kUnit;
  return {static_cast<int>(ceil_div(C, columns)), columns};
}

// Shares of the rows for the gradients of the factors: enough that some 512 workgroups run, none shorter than 128 rows.
int plan_splits(int64_t M, int64_t C, int L)
{
  const int64_t tiles = ceil_div(C, kOuterCols) * L;
  int64_t n = ceil_div(512, tiles);
  if (n > M / 128) n = M / 128;
  return static_cast<int>(n < 1 ? 1 : (n > 16 ? 16 : n));
}

// a decode step: the rows' factors are read from the caches for every part of the columns
bool row_at_a_time(int64_t M) { return M <= 64; }

size_t up16(size_t n) { return (n + 15) & ~static_cast<size_t>(15); }

struct Plan {
  Slices slices;
  int splits_a, splits_b;
  size_t rows, part_a, part_b, total;                 // bytes
};
Plan plan(int64_t M, int64_t N, int64_t K, int rank, int L, bool backward)
{
  Plan w{};
  w.slices = plan_slices(M, backward ? N : K);
  w.rows = up16(static_cast<size_t>(w.slices.count) * M * rank * 4);
  if (!backward && row_at_a_time(M)) w.rows = 0;
  if (backward) {
    w.splits_a = plan_splits(M, K, L);
    w.splits_b = plan_splits(M, N, L);
    w.part_a = w.splits_a > 1 ? up16(static_cast<size_t>(w.splits_a) * L * rank * K * 4) : 0;
    w.part_b = w.splits_b > 1 ? up16(static_cast<size_t>(w.splits_b) * L * rank * N * 4) : 0;
  }
  w.total = w.rows + w.part_a + w.part_b;
  return w;
}

template <typename T, bool kDown>
void shrink(const Problem &p, const Slices &sl, const void *z, int64_t C, const void *f, bool scaled, float *out, hipStream_t s)
{
  const dim3 grid(static_cast<unsigned>(ceil_div(p.M, 16)), sl.count), block(64 * kShrinkWaves);
  const T *zz = static_cast<const T *>(z), *ff = static_cast<const T *>(f);
  if (p.r <= 16) hipLaunchKernelGGL((shrink_kernel<T, 1, kDown>), grid, block, 0, s, p, zz, C, ff, sl.columns, scaled, out);
  else if (p.r <= 32) hipLaunchKernelGGL((shrink_kernel<T, 2, kDown>), grid, block, 0, s, p, zz, C, ff, sl.columns, scaled, out);
  else if (p.r <= 64) hipLaunchKernelGGL((shrink_kernel<T, 4, kDown>), grid, block, 0, s, p, zz, C, ff, sl.columns, scaled, out);
  else hipLaunchKernelGGL((shrink_kernel<T, 8, kDown>), grid, block, 0, s, p, zz, C, ff, sl.columns, scaled, out);
}

template <typename T, bool kDown>
void expand(const Problem &p, const Rows &u, int64_t C, const void *f, bool scaled, const void *base, void *out, float *hidden, hipStream_t s)
{
  const int64_t tiles = ceil_div(C, kExpandWaves * kExpandCols);
  const dim3 grid(static_cast<unsigned>(ceil_div(p.M, 16) * tiles)), block(64 * kExpandWaves);
  const T *ff = static_cast<const T *>(f), *bb = static_cast<const T *>(base);
  T *oo = static_cast<T *>(out);
  if (p.r <= 32) hipLaunchKernelGGL((expand_kernel<T, 1, kDown>), grid, block, 0, s, p, u, C, tiles, ff, scaled, bb, oo, hidden);
  else if (p.r <= 64) hipLaunchKernelGGL((expand_kernel<T, 2, kDown>), grid, block, 0, s, p, u, C, tiles, ff, scaled, bb, oo, hidden);
  else hipLaunchKernelGGL((expand_kernel<T, 4, kDown>), grid, block, 0, s, p, u, C, tiles, ff, scaled, bb, oo, hidden);
}

template <typename T> int forward(const Problem &p, const void *x, const void *base, void *y, float *hidden, void *workspace, hipStream_t s)
{
  if (row_at_a_time(p.M)) {
    const int64_t units = ceil_div(p.N, 64 * kRowWaves), parts = 256 / p.M < units ? 256 / p.M : units;
    const int64_t per = ceil_div(units, parts) * 64 * kRowWaves;
    const dim3 grid(static_cast<unsigned>(ceil_div(p.N, per)), static_cast<unsigned>(p.M)), block(64 * kRowWaves);
    const T *xx = static_cast<const T *>(x), *a = static_cast<const T *>(p.a), *b = static_cast<const T *>(p.b), *bb = static_cast<const T *>(base);
    T *yy = static_cast<T *>(y);
    if (p.r <= 16) hipLaunchKernelGGL((row_kernel<T, 1>), grid, block, 0, s, p, xx, a, b, per, bb, yy, hidden);
    else if (p.r <= 32) hipLaunchKernelGGL((row_kernel<T, 2>), grid, block, 0, s, p, xx, a, b, per, bb, yy, hidden);
    else if (p.r <= 64) hipLaunchKernelGGL((row_kernel<T, 4>), grid, block, 0, s, p, xx, a, b, per, bb, yy, hidden);
    else hipLaunchKernelGGL((row_kernel<T, 8>), grid, block, 0, s, p, xx, a, b, per, bb, yy, hidden);
    return launch_status();
  }
  const Plan w = plan(p.M, p.N, p.K, p.r, p.L, false);
  float *h = static_cast<float *>(workspace);
  if (hidden && w.slices.count == 1) h = hidden, hidden = nullptr;
  shrink<T, false>(p, w.slices, x, p.K, p.a, false, h, s);
  expand<T, false>(p, Rows{h, w.slices.count}, p.N, p.b, true, base, y, hidden, s);
  return launch_status();
}

template <typename Z, typename T> void outer(const Problem &p, const Outer &o, hipStream_t s)
{
  const dim3 grid(static_cast<unsigned>(ceil_div(o.C, kOuterCols) * p.L * o.splits)), block(kOuterThreads);
#define CAIFX_GO(JT)                                                                                   \
  if (o.splits > 1) hipLaunchKernelGGL((outer_kernel<Z, T, JT, true>), grid, block, 0, s, p, o);       \
  else hipLaunchKernelGGL((outer_kernel<Z, T, JT, false>), grid, block, 0, s, p, o)
  if (p.r <= 16) {
    CAIFX_GO(1);
  } else if (p.r <= 32) {
    CAIFX_GO(2);
  } else if (p.r <= 64) {
    CAIFX_GO(4);
  } else {
    CAIFX_GO(8);
  }
#undef CAIFX_GO
}

template <typename T>
int backward(const Problem &p, const void *dy, const void *x, const float *x_scales, const float *hidden, const void *base, void *dx, void *ga, void *gb,
             void *workspace, hipStream_t s)
{
  const Plan w = plan(p.M, p.N, p.K, p.r, p.L, true);
  unsigned char *at = static_cast<unsigned char *>(workspace);
  float *g = reinterpret_cast<float *>(at), *pa = reinterpret_cast<float *>(at + w.rows), *pb = reinterpret_cast<float *>(at + w.rows + w.part_a);
  const Rows rows{g, w.slices.count};
  if (p.M > 0 && (dx || ga)) shrink<T, true>(p, w.slices, dy, p.N, p.b, true, g, s);
  if (p.M > 0 && dx) expand<T, true>(p, rows, p.K, p.a, false, base, dx, nullptr, s);
  Join ja{nullptr, nullptr, 0, 0}, jb = ja;
  if (ga) {
    const bool many = w.splits_a > 1;
    const Outer o{x, x_scales, rows, p.K, false, p.K, 1, many ? pa : ga, w.splits_a, ceil_div(p.M, w.splits_a)};
    if (x_scales) outer<int8_t, T>(p, o, s);
    else outer<T, T>(p, o, s);
    if (many) ja = Join{pa, ga, static_cast<int64_t>(p.L) * p.r * p.K, w.splits_a};
  }
  if (gb) {
    const bool many = w.splits_b > 1;
    const Outer o{dy, nullptr, Rows{hidden, 1}, p.N, true, 1, p.r, many ? pb : gb, w.splits_b, ceil_div(p.M, w.splits_b)};
    outer<T, T>(p, o, s);
    if (many) jb = Join{pb, gb, static_cast<int64_t>(p.L) * p.r * p.N, w.splits_b};
  }
  if (ja.n + jb.n > 0) hipLaunchKernelGGL(join_kernel<T>, dim3(static_cast<unsigned>(ceil_div(ja.n + jb.n, 256))), dim3(256), 0, s, ja, jb);
  return launch_status();
}

int check(int64_t M, int64_t N, int64_t K, int rank, int num_adapters, int dtype)
{
  if (!valid_dtype(dtype) || M < 0 || N <= 0 || K <= 0 || rank <= 0 || num_adapters <= 0) return CAIFX_ERR_INVALID_ARGUMENT;
  constexpr int64_t kMost = int64_t{1} << 30;
  if (rank > CAIFX_ADAPTER_RANK_MAX || M > kMost || N > kMost || K > kMost) return CAIFX_ERR_UNSUPPORTED;
  // a grid has fewer than 2^32 threads
  const int64_t longest = N > K ? N : K, grid = (int64_t{1} << 24) - 1;
  if (ceil_div(M, 16) > grid / ceil_div(longest, kExpandWaves * kExpandCols) || num_adapters > grid / 16 / ceil_div(longest, kOuterCols) ||
      ceil_div(M, 16) > (int64_t{1} << 23) / 16)
    return CAIFX_ERR_UNSUPPORTED;
  return CAIFX_OK;
}

}  // namespace
}  // namespace caifx

using namespace caifx;

extern "C" {

size_t caifx_adapters_workspace_bytes(int64_t M, int64_t N, int64_t K, int rank, int num_adapters, int dtype, int backward)
{
  if (check(M, N, K, rank, num_adapters, dtype) != CAIFX_OK || M == 0) return 0;
  return plan(M, N, K, rank, num_adapters, backward != 0).total;
}

int caifx_adapters_forward(int64_t M, int64_t N, int64_t K, int rank, int num_adapters, const void *x, const int32_t *ids, const void *a, const void *b,
                           const float *scaling, const void *base, void *y, float *hidden, int dtype, void *workspace, size_t workspace_bytes,
                           caifx_stream_t stream)
{
  const int st = check(M, N, K, rank, num_adapters, dtype);
  if (st != CAIFX_OK || M == 0) return st;
  if (!x || !ids || !a || !b || !scaling || !y) return CAIFX_ERR_INVALID_ARGUMENT;
  const size_t es = dtype_size(dtype), need = plan(M, N, K, rank, num_adapters, false).total;
  if (!aligned_to(x, es) || !aligned_to(a, es) || !aligned_to(b, es) || !aligned_to(base, es) || !aligned_to(y, es) || !aligned_to(ids, 4) ||
      !aligned_to(scaling, 4) || !aligned_to(hidden, 4) || !aligned_to(workspace, 4))
    return CAIFX_ERR_MISALIGNED;
  if (need > 0 && (!workspace || workspace_bytes < need)) return CAIFX_ERR_WORKSPACE_TOO_SMALL;
  const Problem p{M, N, K, rank, num_adapters, ids, a, b, scaling};
  hipStream_t s = as_stream(stream);
  switch (dtype) {
    case CAIFX_F32: return forward<float>(p, x, base, y, hidden, workspace, s);
    case CAIFX_F16: return forward<f16_t>(p, x, base, y, hidden, workspace, s);
    default: return forward<bf16_t>(p, x, base, y, hidden, workspace, s);
  }
}

int caifx_adapters_backward(int64_t M, int64_t N, int64_t K, int rank, int num_adapters, const void *dy, const void *x, const float *x_scales,
                            const float *hidden, const int32_t *ids, const void *a, const void *b, const float *scaling, const void *base, void *dx,
                            void *grad_a, void *grad_b, int dtype, void *workspace, size_t workspace_bytes, caifx_stream_t stream)
{
  const int st = check(M, N, K, rank, num_adapters, dtype);
  if (st != CAIFX_OK || ((M == 0 || !dx) && !grad_a && !grad_b)) return st;
  if (M > 0 && (!dy || !ids || !scaling || (dx && !a) || ((dx || grad_a) && !b) || (grad_a && !x) || (grad_b && !hidden))) return CAIFX_ERR_INVALID_ARGUMENT;
  const size_t es = dtype_size(dtype), need = plan(M, N, K, rank, num_adapters, true).total;
  if (!aligned_to(dy, es) || (!x_scales && !aligned_to(x, es)) || !aligned_to(x_scales, 4) || !aligned_to(hidden, 4) || !aligned_to(ids, 4) ||
      !aligned_to(a, es) || !aligned_to(b, es) || !aligned_to(scaling, 4) || !aligned_to(base, es) || !aligned_to(dx, es) || !aligned_to(grad_a, es) ||
      !aligned_to(grad_b, es) || !aligned_to(workspace, 4))
    return CAIFX_ERR_MISALIGNED;
  if (M > 0 && (!workspace || workspace_bytes < need)) return CAIFX_ERR_WORKSPACE_TOO_SMALL;
  const Problem p{M, N, K, rank, num_adapters, ids, a, b, scaling};
  hipStream_t s = as_stream(stream);
  switch (dtype) {
    case CAIFX_F32: return backward<float>(p, dy, x, x_scales, hidden, base, dx, grad_a, grad_b, workspace, s);
    case CAIFX_F16: return backward<f16_t>(p, dy, x, x_scales, hidden, base, dx, grad_a, grad_b, workspace, s);
    default: return backward<bf16_t>(p, dy, x, x_scales, hidden, base, dx, grad_a, grad_b, workspace, s);
  }
}

}  // extern "C"
