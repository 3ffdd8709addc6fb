// Low-rank adapters beside a frozen projection: the branch of every row's own adapter added to the projection's result, and the
// branch's gradients.  Row m uses adapter l = ids[m] (none where ids[m] is outside [0, L)):
//
//   forward    h[m] = x[m] A[l]^T                  y[m]  = T(base[m] + scaling[l] h[m] B[l]^T)
//   backward   g[m] = scaling[l] dy[m] B[l]        dx[m] = T(base[m] + g[m] A[l])
//              dA[l] = T(sum over m of l of g[m]^T x[m])      dB[l] = T(sum over m of l of scaling[l] dy[m]^T h[m])
//
// with x [M,K], A [L,r,K], B [L,N,r], h and g [M,r] in fp32.  A rank of 16 leaves 16 multiply-adds for a value read or written,
// so all of it is bound by memory: x, dy (twice), base and the results pass, the factors come from the caches, and the matrix cores
// keep the arithmetic out of the way.  Four kinds of product:
//
//   shrink   rows x factor over the long axis (h, g): a workgroup takes 16 or 32 rows, its waves share the axis
//   expand   rank -> long axis (y, dx): a wave takes 16 rows x 256 columns (64 in small calls and in fp32 above rank 64), adds base and rounds once
//   outer    sums over the rows of an adapter (dA, dB): a workgroup takes 128 columns and a run of the adapter's rows
//   row      shrink and expand of one row in one launch, for decode steps
//
// The forward is row, or shrink and expand; the backward is shrink (with a workgroup that sorts the rows by adapter beside it), outer and
// expand in one launch, and the sum of an adapter's runs where it has several.  Measured on one MI355X against the copy of as many bytes (in
// three buffers in turn, 5.0 TB/s): y of 4096 x 11008 in bf16 45 us of 35, h of 4096 x 4096 12 of 8, g of 4096 x 11008 25 of 18 (rank 64:
// 51, where the factor's reads count), both gradients and dx of the two together 47 of 42.
//
// Precision: products of two 16-bit values are exact in fp32 and summed in fp32.  h and g stay fp32; on the 16-bit matrix cores they
// are two pieces that add up to them but for 2^-17 or less, which is far below the one rounding of the result.  fp32 tensors use the
// fp32 instruction.
//
// Rows of different adapters never meet in a product: a tile with several adapters is multiplied by each of them and every row
// keeps the result of its own, so that an infinity in one adapter's factors stays out of the other rows.  Within a row infinities give what the
// formulas give.
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
template <typename T> __device__ __forceinline__ vec8<T> down(const T *m, int pitch, int spread, int lane, int q)
{
  const int t = lane & 15;
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
// The adapters of ROWS rows from m0 on: lane l holds that of row l % ROWS, -1 for none.  next() goes through the adapters, each once.
// Where few rows run, several workgroups take a tile and share its adapters: `of` of them, this one the `turn`-th, in turn; a row belongs to
// its adapter's, a row without adapter to the first.  (32 rows of 32 adapters of rank 64 from 4096 to 14336 took 54 us with one workgroup
// for each tile, 29 with sixteen.)
template <int ROWS> struct TileIds {
  int mine;
  uint64_t pending, kept;
  bool owned;
  __device__ __forceinline__ TileIds(const Problem &p, int64_t m0, int turn, int of)
  {
    const int64_t m = m0 + (threadIdx.x & (ROWS - 1));
    mine = -1;
    if (m < p.M) {
      const int l = p.ids[m];
      if (l >= 0 && l < p.L) mine = l;
    }
    pending = __ballot(mine >= 0);
    kept = ~uint64_t{0};
    if (of > 1) {
      uint64_t all = pending;
      kept = turn == 0 ? __ballot(mine < 0) : 0;
      for (int k = 0; all != 0; ++k) {
        const int l = __builtin_amdgcn_readlane(mine, __builtin_ctzll(all));
        const uint64_t rows = __ballot(mine == l);
        all &= ~rows;
        if (k % of == turn) kept |= rows;
      }
      pending &= kept;
    }
    owned = owned_row(threadIdx.x & (ROWS - 1));
  }
  __device__ __forceinline__ int of_row(int row) const { return __shfl(mine, row, 64); }
  __device__ __forceinline__ bool owned_row(int row) const { return (kept >> row) & 1; }
  // the next adapter of the tile, the same for all lanes; -1 when there is none
  __device__ __forceinline__ int next()
  {
    if (pending == 0) return -1;
    const int l = __builtin_amdgcn_readlane(mine, __builtin_ctzll(pending));
    pending &= ~__ballot(mine == l);
    return l;
  }
};

// ------------------------------------------------------------------ rows sorted by adapter
// What the products over an adapter's rows are cut into: a slot is up to `chunk` of the rows of one adapter, as they stand in the list of
// rows sorted by adapter.  An adapter with one slot (also one without rows) writes its gradient, the slots of the others go to
// `part` and are added by join_kernel.
struct Slot {
  int32_t adapter, first, count, part;                // part -1: none
};
struct Multi {
  int32_t adapter, part, parts, unused;
};
struct Cut {
  int32_t *header;                                    // number of slots, number of entries in multi
  Slot *slots;
  Multi *multi;
  int32_t chunk;
};

constexpr int kSortThreads = 512;

struct Sort {
  int32_t *rows;                                      // [M]
  int32_t *spare;                                     // [adapters], where they do not fit LDS
  Cut a, b;
};

// number of lanes with the same adapter, and of those below this lane; `bits` of an adapter's number are looked at
__device__ __forceinline__ uint64_t same_lanes(int l, int bits)
{
  uint64_t same = __ballot(l >= 0);
  for (int k = 0; k < bits; ++k) {
    const bool one = l >= 0 && ((l >> k) & 1);
    const uint64_t with = __ballot(one);
    same &= one ? with : ~with;
  }
  return l >= 0 ? same : 0;
}

// One workgroup lists the rows of each adapter, in their order, and cuts the lists into slots.  The rows are shared among as many waves as
// have room for a counter for each adapter; counters first, their running sums next, then every wave places its rows in order.
__device__ __forceinline__ void sort_rows(const Problem &p, const Sort &o, int32_t *lds, int room)
{
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const bool inside = p.L <= room;
  int waves = inside ? room / p.L : 1;
  if (waves > kSortThreads / 64) waves = kSortThreads / 64;
  int32_t *counts = inside ? lds : o.spare;           // [waves][L]
  for (int k = threadIdx.x; k < waves * p.L; k += kSortThreads) counts[k] = 0;
  const int64_t share = ((p.M + waves - 1) / waves + 63) / 64 * 64, lo = wave * share, hi = lo + share < p.M ? lo + share : p.M;
  int32_t *mine = counts + wave * p.L;
  __syncthreads();
  if (wave < waves) {
    for (int64_t m = lo + lane; m < hi; m += 64) {
      const int l = p.ids[m];
      if (l >= 0 && l < p.L) atomicAdd(mine + l, 1);
    }
  }
  __threadfence_block();
  __syncthreads();
  if (wave == 0) {
    // running sums over the adapters: rows, slots and parts of either gradient, entries of the lists of those with several slots
    int32_t row0 = 0, slot0[2] = {0, 0}, part0[2] = {0, 0}, multi0[2] = {0, 0};
    for (int base = 0; base < p.L; base += 64) {
      const int l = base + lane;
      int n = 0;
      if (l < p.L) {
        for (int w = 0; w < waves; ++w) n += counts[w * p.L + l];
      }
      auto running = [&](int v, int32_t &carry) {     // the sum of the lanes before this one
        int up = v;
#pragma unroll
        for (int k = 1; k < 64; k <<= 1) {
          const int x = __shfl_up(up, k, 64);
          if (lane >= k) up += x;
        }
        const int before = carry + up - v;
        carry += __shfl(up, 63, 64);
        return before;
      };
      const int row = running(n, row0);
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        const Cut &cut = g ? o.b : o.a;
        const int slots = l >= p.L ? 0 : (n > cut.chunk ? (n + cut.chunk - 1) / cut.chunk : 1);
        const int slot = running(slots, slot0[g]), part = running(slots > 1 ? slots : 0, part0[g]), multi = running(slots > 1 ? 1 : 0, multi0[g]);
        for (int k = 0; k < slots; ++k) {
          const int left = n - k * cut.chunk;
          cut.slots[slot + k] = Slot{l, row + k * cut.chunk, left < cut.chunk ? left : cut.chunk, slots > 1 ? part + k : -1};
        }
        if (slots > 1) cut.multi[multi] = Multi{l, part, slots, 0};
      }
      if (l < p.L) {
        int at = row;
        for (int w = 0; w < waves; ++w) {
          const int c = counts[w * p.L + l];
          counts[w * p.L + l] = at;
          at += c;
        }
      }
    }
    if (lane == 0) {
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        const Cut &cut = g ? o.b : o.a;
        cut.header[0] = slot0[g];
        cut.header[1] = multi0[g];
      }
    }
  }
  __threadfence_block();
  __syncthreads();
  if (wave < waves) {
    const int bits = 32 - __builtin_clz(static_cast<unsigned>(p.L > 1 ? p.L - 1 : 1));
    for (int64_t base = lo; base < hi; base += 64) {
      const int64_t m = base + lane;
      int l = -1;
      if (m < hi) {
        const int id = p.ids[m];
        if (id >= 0 && id < p.L) l = id;
      }
      const uint64_t same = same_lanes(l, bits);
      const int below = __builtin_popcountll(same & ((uint64_t{1} << lane) - 1));
      if (l >= 0) {
        const int at = mine[l];
        o.rows[at + below] = static_cast<int32_t>(m);
        __builtin_amdgcn_wave_barrier();
        if (below == 0) mine[l] = at + __builtin_popcountll(same);
      }
      __threadfence_block();
    }
  }
}

// ------------------------------------------------------------------ shrink
constexpr int kShrinkWaves = 8;

constexpr int shrink_steps(int bytes, bool down) { return down ? (bytes >= 16 ? 1 : 2) : (bytes >= 32 ? 1 : bytes >= 8 ? 2 : 4); }
// Columns that a wave asks for at a time (as much as its registers hold, so that a memory round trip is paid for few times), and tiles of
// 16 rows of a workgroup.
template <typename T, int JT, bool kDown> struct ShrinkUnit {
  static constexpr int kBytes = JT * static_cast<int>(sizeof(T));       // 2 .. 32: registers of the factor grow with it
  static constexpr int kSteps = shrink_steps(kBytes, kDown);
  static constexpr int kCols = 32 * kSteps;
  // kDown stages the factor once for all rows of a workgroup
  static constexpr int kTiles = !kDown || kBytes >= 32 ? 1 : 2;
};

// out[slice][m][j] = scale sum over the slice's columns c of z[m][c] f[l][j][c] (kDown: f[l][c][j]), rows without adapter zero.
// The factor is the A operand (rows j), the rows are the B operand, so a lane's results belong to one row m = i.
template <typename T, int JT, bool kDown>
__global__ __launch_bounds__(64 * kShrinkWaves) void shrink_kernel(Problem p, const T *__restrict__ z, int64_t C, const T *__restrict__ f, int64_t per_slice,
                                                                   bool scaled, float *__restrict__ out, Sort sort)
{
  constexpr int R = 16 * JT;
  constexpr int kSteps = ShrinkUnit<T, JT, kDown>::kSteps, kCols = 32 * kSteps, MT = ShrinkUnit<T, JT, kDown>::kTiles;
  constexpr int kStage = kDown ? kCols * R * sizeof(T) : 0;             // bytes of a wave's staged factor
  constexpr int kSums = 16 * MT * R * 4;
  __shared__ __align__(32) unsigned char lds[kShrinkWaves * (kStage > kSums ? kStage : kSums)];
  __shared__ bool owned[16 * MT];
  if constexpr (kDown) {
    static_assert(64 * kShrinkWaves == kSortThreads);
    if (blockIdx.x == 0 && sort.rows != nullptr) {     // the gradients' list of rows, beside the others' work
      if (blockIdx.y == 0 && blockIdx.z == 0) sort_rows(p, sort, reinterpret_cast<int32_t *>(lds), static_cast<int>(sizeof lds / 4));
      return;
    }
  }
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i = lane & 15, q = lane >> 4;
  const int64_t m0 = (static_cast<int64_t>(blockIdx.x) - (kDown && sort.rows != nullptr ? 1 : 0)) * (16 * MT);
  const int64_t lo = blockIdx.y * per_slice, hi = lo + per_slice < C ? lo + per_slice : C;
  // lanes hold the rows m0 + lane for the list of adapters, and m0 + 16 t + i for the products
  TileIds<16 * MT> ids(p, m0, blockIdx.z, gridDim.z);
  if (__ballot(ids.owned) == 0) return;               // the same for all waves
  if (threadIdx.x < 16 * MT) owned[threadIdx.x] = ids.owned;
  int mine[MT];
  bool have_row[MT];
  const T *row[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) {
    mine[t] = ids.of_row(16 * t + i);
    have_row[t] = ids.owned_row(16 * t + i);
    const int64_t m = m0 + 16 * t + i;
    row[t] = z + (m < p.M ? m : p.M - 1) * C;
  }
  floatx4_t sum[MT][JT];
#pragma unroll
  for (int t = 0; t < MT; ++t)
#pragma unroll
    for (int j = 0; j < JT; ++j) sum[t][j] = floatx4_t{0, 0, 0, 0};
  T *stage = reinterpret_cast<T *>(lds) + wave * (kStage / sizeof(T));
  for (int l = ids.next(); l >= 0; l = ids.next()) {
    const T *factor = f + static_cast<int64_t>(l) * p.r * C;
    floatx4_t acc[MT][JT];
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int j = 0; j < JT; ++j) acc[t][j] = floatx4_t{0, 0, 0, 0};
    vec8<T> zv[MT][kSteps];
    auto fetch_rows = [&](int64_t c0, bool full) {
#pragma unroll
      for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
          const int64_t c = c0 + 32 * s + 8 * q;
          zv[t][s] = zero8<vec8<T>>();
          if (have_row[t]) zv[t][s] = full ? load8<T>(row[t] + c) : load8<T>(row[t] + c, clamp8(hi - c));
        }
    };
    int64_t c0 = lo + wave * kCols;
    if constexpr (!kDown) {
      auto unit = [&](bool full) {
        vec8<T> fv[kSteps][JT];
        fetch_rows(c0, full);
#pragma unroll
        for (int j = 0; j < JT; ++j) {
          const int at = 16 * j + i < p.r ? 16 * j + i : p.r - 1;           // rows past the rank repeat the last; their sums are not kept
          const T *from = factor + at * C + c0 + 8 * q;
#pragma unroll
          for (int s = 0; s < kSteps; ++s) fv[s][j] = full ? load8<T>(from + 32 * s) : load8<T>(from + 32 * s, clamp8(hi - c0 - 32 * s - 8 * q));
        }
#pragma unroll
        for (int s = 0; s < kSteps; ++s)
#pragma unroll
          for (int j = 0; j < JT; ++j)
#pragma unroll
            for (int t = 0; t < MT; ++t) acc[t][j] = mma(fv[s][j], zv[t][s], acc[t][j]);
      };
      for (; c0 + kCols <= hi; c0 += kShrinkWaves * kCols) unit(true);
      if (c0 < hi) unit(false);
    } else {
      // the factor's rows c0 .. + kCols, eight ranks at a time, zeros past the rank and past the last column; a unit's values are asked for
      // before the products of the unit in front
      constexpr int kOct = R / 8, kEach = kCols * kOct / 64;
      vec8<T> st[kEach];
      auto fetch = [&]() {
        const bool full = c0 + kCols <= hi;
        fetch_rows(c0, full);
#pragma unroll
        for (int o = 0; o < kEach; ++o) {
          const int at = o * 64 + lane, c = at / kOct, j = at % kOct * 8;
          st[o] = load8<T>(factor + (c0 + c) * p.r + j, full || c0 + c < hi ? clamp8(p.r - j) : 0);
        }
      };
      if (c0 < hi) fetch();
      while (c0 < hi) {
#pragma unroll
        for (int o = 0; o < kEach; ++o) *reinterpret_cast<vec8<T> *>(stage + (o * 64 + lane) * 8) = st[o];
        vec8<T> now[MT][kSteps];
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
          for (int s = 0; s < kSteps; ++s) now[t][s] = zv[t][s];
        __builtin_amdgcn_wave_barrier();
        c0 += kShrinkWaves * kCols;
        if (c0 < hi) fetch();
#pragma unroll
        for (int s = 0; s < kSteps; ++s)
#pragma unroll
          for (int j = 0; j < JT; ++j) {
            const vec8<T> fv = down<T>(stage + 32 * s * R + 16 * j, R, 4, lane, q);
#pragma unroll
            for (int t = 0; t < MT; ++t) acc[t][j] = mma(fv, now[t][s], acc[t][j]);
          }
        __builtin_amdgcn_wave_barrier();
      }
    }
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int j = 0; j < JT; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) sum[t][j][e] = mine[t] == l ? acc[t][j][e] : sum[t][j][e];
  }
  // the waves' shares, [wave][m][j], added in the waves' order
  __syncthreads();
  float *sums = reinterpret_cast<float *>(lds);
#pragma unroll
  for (int t = 0; t < MT; ++t)
#pragma unroll
    for (int j = 0; j < JT; ++j) *reinterpret_cast<floatx4_t *>(sums + ((wave * MT + t) * 16 + i) * R + 16 * j + 4 * q) = sum[t][j];
  __syncthreads();
  for (int o = threadIdx.x; o < 16 * MT * R; o += 64 * kShrinkWaves) {
    const int64_t mm = m0 + o / R;
    const int j = o % R;
    if (mm >= p.M || j >= p.r || !owned[o / R]) continue;
    float v = 0.0f;
#pragma unroll
    for (int w = 0; w < kShrinkWaves; ++w) v += sums[w * 16 * MT * R + o];
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
// values j .. j + 7 of row m, zeros past the rank; kMany: more than a few slices, asked for four at a time
template <bool kMany> __device__ __forceinline__ f32x8_t rank8(const Problem &p, const Rows &u, int64_t m, int j)
{
  const int have = clamp8(p.r - j);
  const float *at = u.at + m * p.r + j;
  f32x8_t v = load8<float>(at, have);
  const int64_t apart = p.M * p.r;
  int s = 1;
  for (; kMany && s + 4 <= u.slices; s += 4) {
    f32x8_t w[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) w[k] = load8<float>(at + (s + k) * apart, have);
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] += w[k][e];
  }
  for (; s < u.slices; ++s) {
    const f32x8_t w = load8<float>(at + s * apart, have);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] += w[e];
  }
  return v;
}

// value j of row m, its slices added in rank8's order
__device__ __forceinline__ float rank1(const Problem &p, const Rows &u, int64_t m, int j)
{
  const float *at = u.at + m * p.r + j;
  const int64_t apart = p.M * p.r;
  float v = at[0];
  for (int s = 1; s < u.slices; ++s) v += at[s * apart];
  return v;
}

// ------------------------------------------------------------------ infinities
// The matrix cores' sum is a NaN in places where the definition's is not: the pieces of an infinity, and of a number beyond the 16-bit type's
// range, are an infinity and a NaN or an infinity of the other sign; a zero piece or a spare rank's zero meets an infinite factor.  It is never a
// number where the definition's is not.  So every result that comes out as a NaN is formed again in fp32, value by value, up to
// the first NaN of the definition's own.  The test for it is within
// 1.5 % of a pass in every case (the largest: fp32 gradients, 2048 x 4096 x 4096 of rank 64, 104.6 -> 106.2 us).
__device__ __forceinline__ bool any_nan(const floatx4_t &v) { return __builtin_isunordered(v[0], v[1]) | __builtin_isunordered(v[2], v[3]); }

// ------------------------------------------------------------------ expand
// The fp32 side of the expanding products.  16-bit tensors are multiplied by the row in two pieces of their own type, hi + lo: bf16 has
// fp32's range, an fp16 row is first scaled by a power of two that brings its largest value to 2^14 (the pieces then add up to the value
// but for 2^-22 of it, down to 2^-28 of the largest), and the results are scaled back.
template <typename T> struct TwoPieces {
  vec8<T> hi, lo;
};
template <typename T> __device__ __forceinline__ TwoPieces<T> two_pieces(const f32x8_t &v)
{
  TwoPieces<T> p;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    p.hi[e] = from_f32<T>(v[e]);
    p.lo[e] = from_f32<T>(v[e] - to_f32<T>(p.hi[e]));
  }
  return p;
}
// A row's operand for one step.  kHalf: ranks up to 16, where the 32 elements of a step hold both pieces, hi in the lanes q = 0, 1 and lo in
// q = 2, 3, each beside the same sixteen values of the factor.
template <typename T, bool kHalf> struct RowOperand {
  TwoPieces<T> u;
  __device__ __forceinline__ void set(const f32x8_t &v, int) { u = two_pieces<T>(v); }
  __device__ __forceinline__ floatx4_t with(const vec8<T> &f, floatx4_t acc) const { return mma(f, u.lo, mma(f, u.hi, acc)); }
  __device__ __forceinline__ floatx4_t as_rows(const vec8<T> &f, floatx4_t acc) const { return mma(u.lo, f, mma(u.hi, f, acc)); }
};
template <typename T> struct RowOperand<T, true> {
  vec8<T> u;
  __device__ __forceinline__ void set(const f32x8_t &v, int q)
  {
    const TwoPieces<T> p = two_pieces<T>(v);
    u = q < 2 ? p.hi : p.lo;
  }
  __device__ __forceinline__ floatx4_t with(const vec8<T> &f, floatx4_t acc) const { return mma(f, u, acc); }
  __device__ __forceinline__ floatx4_t as_rows(const vec8<T> &f, floatx4_t acc) const { return mma(u, f, acc); }
};
struct RowOperandF32 {
  f32x8_t u;
  __device__ __forceinline__ void set(const f32x8_t &v, int) { u = v; }
  __device__ __forceinline__ floatx4_t with(const f32x8_t &f, floatx4_t acc) const { return mma(f, u, acc); }
  __device__ __forceinline__ floatx4_t as_rows(const f32x8_t &f, floatx4_t acc) const { return mma(u, f, acc); }
};
template <> struct RowOperand<float, true> : RowOperandF32 {};
template <> struct RowOperand<float, false> : RowOperandF32 {};
// the power of two that an fp16 row is multiplied by: its largest magnitude, a value of any lane i, q, comes to [2^14, 2^15); 1 for rows of
// zeros, infinities, NaN, and for the other types
template <typename T, int N> __device__ __forceinline__ float row_scale(const f32x8_t (&v)[N])
{
  if constexpr (dtype_code<T>::value != CAIFX_F16) return 1.0f;
  uint32_t top = 0;
#pragma unroll
  for (int s = 0; s < N; ++s)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float x = v[s][e];
      const uint32_t b = __builtin_bit_cast(uint32_t, x) & 0x7FFFFFFFu;
      top = top > b ? top : b;
    }
#pragma unroll
  for (int o = 16; o < 64; o <<= 1) {
    const uint32_t w = __shfl_xor(top, o, 64);
    top = top > w ? top : w;
  }
  const int exponent = static_cast<int>(top >> 23);                     // biased; the scale's own exponent stays in the normal range
  if (exponent == 0 || exponent == 255) return 1.0f;
  const int e = 127 + 14 + 127 - exponent;
  return __builtin_bit_cast(float, static_cast<uint32_t>(e > 253 ? 253 : (e < 1 ? 1 : e)) << 23);
}

constexpr int kExpandWaves = 4;                       // of 16 rows each
constexpr int kExpandCols = 64;                       // of a wave at a time

// out[m][c] = T(base[m][c] + scale sum_j u[m][j] f[l][c][j])  (kDown: f[l][j][c]).  The factor's columns are the A operand, the rows the B
// operand: of the 16 x 16 results of a product a lane holds four neighbouring columns of one row, and two products whose columns
// alternate by fours give it eight, one 16-byte access.  A wave keeps its rows' operands for all its columns: what is not
// a load, a store or a product costs as much as the memory otherwise (built for each 64 columns: 56 us for 4096 x 11008 in bf16).
// hidden: the rows themselves, written by the first columns' waves.
struct Expand {
  Rows u;
  int64_t C, col_tiles;
  const void *f;                                      // the factor, T
  bool scaled;
  const void *base;                                   // T, null for zero
  void *out;                                          // T, may be base
  float *hidden;                                      // null: not wanted
  unsigned turns, places;                             // workgroups of a tile, tiles: all tiles' first workgroups come first, so
                                                      // that those with work (often the first alone) spread over the XCDs
};
template <typename T, int RS> constexpr int expand_lds() { return kExpandWaves * (RS == 0 && sizeof(T) == 2 ? 16 : 32) * (kExpandCols + 8) * static_cast<int>(sizeof(T)); }
template <typename T, int RS, bool kDown, int G>
__device__ __forceinline__ void expand_block(const Problem &p, const Expand &o, unsigned block, T *lds)
{
  const Rows &u = o.u;
  const int64_t C = o.C;
  const T *__restrict__ f = static_cast<const T *>(o.f);
  const bool scaled = o.scaled;
  const T *base = static_cast<const T *>(o.base);
  T *out = static_cast<T *>(o.out);
  float *__restrict__ hidden = o.hidden;
  constexpr bool kHalf = RS == 0;
  constexpr int S = RS == 0 ? 1 : RS;
  constexpr bool kPieces = kHalf && sizeof(T) == 2;    // both pieces in one step
  constexpr int kStageRows = kPieces ? 16 : 32;
  constexpr int kPitch = kExpandCols + 8;
  constexpr bool kTurns = G == 1;                      // of the tiles' adapters, where few waves run
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i = lane & 15, q = lane >> 4;
  const unsigned turn = kTurns ? block / o.places : 0, place = kTurns ? block - turn * o.places : block;
  const unsigned tile = place / static_cast<unsigned>(o.col_tiles);
  const int64_t first = static_cast<int64_t>(place - tile * static_cast<unsigned>(o.col_tiles)) * (kExpandCols * G);
  const int64_t m = (static_cast<int64_t>(tile) * kExpandWaves + wave) * 16 + i;
  if (m - i >= p.M) return;
  const bool in = m < p.M;
  // a tile that is whole in every direction asks for all of its base at once
  const bool whole_tile = m - i + 16 <= p.M && p.r % 8 == 0 && first + G * kExpandCols <= C;
  vec8<T> early[G][2];
  auto ask = [&]() {
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
      for (int h = 0; h < 2; ++h) early[g][h] = base ? load8<T>(base + m * C + first + kExpandCols * g + 32 * h + 8 * q) : zero8<vec8<T>>();
  };
  if (whole_tile && !kTurns) ask();
  TileIds<16> ids(p, m - i, turn, kTurns ? o.turns : 1);
  if (__ballot(ids.owned) == 0) return;
  if (whole_tile && kTurns && ids.owned) ask();
  const int qj = kPieces ? q & 1 : q;                  // which eight ranks of a step
  f32x8_t v[S];
#pragma unroll
  for (int s = 0; s < S; ++s) {
    if constexpr (kTurns) {
      v[s] = zero8<f32x8_t>();
      if (in && ids.owned) v[s] = rank8<true>(p, u, m, 32 * s + 8 * qj);
    } else {
      v[s] = rank8<false>(p, u, in ? m : p.M - 1, 32 * s + 8 * qj);
    }
  }
  if (hidden && first == 0 && in && ids.owned && (!kPieces || q < 2)) {
#pragma unroll
    for (int s = 0; s < S; ++s)
      for (int e = 0; e < 8; ++e)
        if (32 * s + 8 * qj + e < p.r) hidden[m * p.r + 32 * s + 8 * qj + e] = v[s][e];
  }
  if (scaled) {
    const float scale = ids.mine >= 0 ? p.scaling[ids.mine] : 0.0f;
#pragma unroll
    for (int s = 0; s < S; ++s)
#pragma unroll
      for (int e = 0; e < 8; ++e) v[s][e] *= scale;
  }
  const float up = row_scale<T>(v);                    // a power of two, and its inverse
  const float back = __builtin_bit_cast(float, (254u << 23) - __builtin_bit_cast(uint32_t, up));
  RowOperand<T, kHalf> row[S];
#pragma unroll
  for (int s = 0; s < S; ++s) {
    if constexpr (dtype_code<T>::value == CAIFX_F16) {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[s][e] *= up;
    }
    row[s].set(v[s], q);
  }
  const uint64_t pending = ids.pending;
  T *stage = lds + (kDown ? wave * kStageRows * kPitch : 0);
  unsigned odd = 0;                                    // half groups where this lane's results have a NaN, the last in bit 0: not stored yet

  auto group = [&](int64_t c0, const vec8<T> (&early)[2], auto is_full) {
    constexpr bool kFull = decltype(is_full)::value;    // all 16 rows, all 64 columns, ranks in whole octets
    vec8<T> old[2];
    int have[2];
    T *to = out + m * C + c0 + 8 * q;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      have[h] = kFull ? 8 : (in && ids.owned ? clamp8(C - c0 - 32 * h - 8 * q) : 0);
      if (kFull) old[h] = early[h];
      else old[h] = base ? load8<T>(base + m * C + c0 + 8 * q + 32 * h, have[h]) : zero8<vec8<T>>();
    }
    floatx4_t sum[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) sum[k] = floatx4_t{0, 0, 0, 0};
    ids.pending = pending;
    bool again = false;
    for (int l = ids.next(); l >= 0; l = ids.next()) {
      const T *factor = f + static_cast<int64_t>(l) * p.r * C;
      floatx4_t acc[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) acc[k] = floatx4_t{0, 0, 0, 0};
#pragma unroll
      for (int s = 0; s < S; ++s) {
        vec8<T> fv[4];
        if constexpr (kDown) {
          // a step's ranks of the 64 columns, zeros past the rank and past the last column
          vec8<T> st[kStageRows / 8];
#pragma unroll
          for (int o = 0; o < kStageRows / 8; ++o) {
            const int j = 32 * s + 8 * o + (lane >> 3);
            const T *from = factor + j * C + c0 + 8 * (lane & 7);
            if (kFull) st[o] = j < p.r ? load8<T>(from) : zero8<vec8<T>>();
            else st[o] = load8<T>(from, j < p.r ? clamp8(C - c0 - 8 * (lane & 7)) : 0);
          }
#pragma unroll
          for (int o = 0; o < kStageRows / 8; ++o) *reinterpret_cast<vec8<T> *>(stage + (8 * o + (lane >> 3)) * kPitch + 8 * (lane & 7)) = st[o];
          __builtin_amdgcn_wave_barrier();
#pragma unroll
          for (int k = 0; k < 4; ++k) fv[k] = down<T>(stage + 32 * (k >> 1) + 4 * (k & 1), kPitch, 8, lane, qj);
          __builtin_amdgcn_wave_barrier();
        } else {
          const int j = 32 * s + 8 * qj;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int64_t c = c0 + 32 * (k >> 1) + 8 * (i >> 2) + 4 * (k & 1) + (i & 3);
            // past the rank (where the row's operand is zero) the factor's last values again: they are there, and of the same adapter
            if (kFull) fv[k] = load8<T>(factor + c * p.r + (j < p.r ? j : p.r - 8));
            else fv[k] = load8<T>(factor + c * p.r + j, c < C ? clamp8(p.r - j) : 0);
          }
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) acc[k] = row[s].with(fv[k], acc[k]);
      }
      // the tile's first adapter fills all rows, the others replace their own
      if (!again) {
#pragma unroll
        for (int k = 0; k < 4; ++k) sum[k] = acc[k];
      } else {
        const bool mine = ids.mine == l;
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
          for (int e = 0; e < 4; ++e) sum[k][e] = mine ? acc[k][e] : sum[k][e];
      }
      again = true;
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      // a row without adapter keeps its base bit for bit, also a NaN's
      bool nan = false;
      if (ids.mine >= 0) {
        nan = any_nan(sum[2 * h]) | any_nan(sum[2 * h + 1]);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          float add = sum[2 * h + (e >> 2)][e & 3];
          if constexpr (dtype_code<T>::value == CAIFX_F16) add *= back;
          old[h][e] = from_f32<T>(to_f32<T>(old[h][e]) + add);
        }
      }
      odd = 2 * odd + nan;
      if (!ids.owned || nan) continue;
      if (kFull || have[h] == 8) {
        __builtin_memcpy(to + 32 * h, &old[h], sizeof old[h]);
      } else {
#pragma unroll
        for (int e = 0; e < 7; ++e)
          if (e < have[h]) to[32 * h + e] = old[h][e];
      }
    }
  };
  if (whole_tile) {
#pragma unroll
    for (int g = 0; g < G; ++g) group(first + g * kExpandCols, early[g], std::true_type{});
  } else {
#pragma unroll 1
    for (int g = 0; g < G; ++g)
      if (first + g * kExpandCols < C) group(first + g * kExpandCols, early[g], std::false_type{});
      else odd *= 4;
  }
  if (__builtin_expect(odd == 0 || !ids.owned, 1)) return;
  const float scale = scaled ? p.scaling[ids.mine] : 1.0f;
  const T *factor = f + static_cast<int64_t>(ids.mine) * p.r * C;
#pragma unroll 1
  for (int n = 0; n < 16 * G; ++n) {
    const int64_t c = first + 8 * q + 32 * (n >> 3) + (n & 7);
    if (!(odd >> (2 * G - 1 - (n >> 3)) & 1) || c >= C) continue;
    float add = 0.0f;
#pragma unroll 1
    for (int j = 0; j < p.r && add == add; ++j) add = __builtin_fmaf(rank1(p, u, m, j) * scale, to_f32<T>(factor[kDown ? j * C + c : c * p.r + j]), add);
    out[m * C + c] = from_f32<T>((base ? to_f32<T>(base[m * C + c]) : 0.0f) + add);
  }
}

// as for the gradients: three waves of a SIMD for fp32 above rank 64 (300 rows, 1024 to 14336, rank 128: with two 60.6 us the pass, with three 57.0)
template <typename T, int RS> constexpr int expand_waves() { return sizeof(T) == 4 && RS == 4 ? 3 : 1; }
template <typename T, int RS, int G> __global__ __launch_bounds__(64 * kExpandWaves, (expand_waves<T, RS>())) void expand_kernel(Problem p, Expand o)
{
  expand_block<T, RS, false, G>(p, o, blockIdx.x, nullptr);
}

// ------------------------------------------------------------------ one row, both products
constexpr int kRowWaves = 8;
constexpr int kRowCols = 64 * kRowWaves;              // of a workgroup at a time
constexpr int kRowRounds = 4;                         // of such columns, all asked for before the first product where registers allow

// A workgroup takes one row and up to 2048 columns of its result and forms the row's h itself: the row's other workgroups do the same from
// the caches, which costs less than a second launch.  Both products use one row (column) of sixteen; the matrix cores are not what
// bounds them, round trips to memory are: a wave asks for eight steps of the first product at a time, and for its part of the second
// factor before the first product is done.
template <typename T, int RS>
__global__ __launch_bounds__(64 * kRowWaves) void row_kernel(Problem p, int rows_padded, const T *__restrict__ x, const T *__restrict__ a, const T *__restrict__ b,
                                                             int64_t per_block, const T *base, T *out, float *__restrict__ hidden)
{
  constexpr bool kHalf = RS == 0, kPieces = kHalf && sizeof(T) == 2;
  constexpr int S = kHalf ? 1 : RS, JT = kHalf ? 1 : 2 * RS, R = 16 * JT;
  constexpr int kAhead = JT * static_cast<int>(sizeof(T)) <= 4 ? 8 : JT * static_cast<int>(sizeof(T)) <= 8 ? 4 : 2;      // steps of the first product
  constexpr int kEarly = S * static_cast<int>(sizeof(T)) <= 2 ? kRowRounds : 1;                                          // rounds of the second
  __shared__ float shares[kRowWaves][R];
  __shared__ __align__(32) float total[S * 32];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i = lane & 15, q = lane >> 4, qj = kPieces ? q & 1 : q;
  // neighbouring workgroups are of neighbouring rows: with a multiple of eight of them a row's workgroups share an L2
  const int64_t part = blockIdx.x / rows_padded, m = blockIdx.x - part * rows_padded;
  if (m >= p.M) return;
  const int64_t lo = part * per_block, hi = lo + per_block < p.N ? lo + per_block : p.N;
  const int l = p.ids[m];
  if (l < 0 || l >= p.L) {
    for (int64_t c = lo + threadIdx.x; c < hi; c += kRowCols) out[m * p.N + c] = base ? base[m * p.N + c] : T(0.0f);
    if (hidden && part == 0 && threadIdx.x < static_cast<unsigned>(p.r)) hidden[m * p.r + threadIdx.x] = 0.0f;
    return;
  }
  const T *fa = a + static_cast<int64_t>(l) * p.r * p.K, *fb = b + static_cast<int64_t>(l) * p.N * p.r, *row = x + m * p.K;
  floatx4_t acc[JT];
#pragma unroll
  for (int j = 0; j < JT; ++j) acc[j] = floatx4_t{0, 0, 0, 0};
  const T *fr[JT];
#pragma unroll
  for (int j = 0; j < JT; ++j) fr[j] = fa + (16 * j + i < p.r ? 16 * j + i : p.r - 1) * p.K;
  vec8<T> fv[kEarly][S][4];
  auto second = [&](int64_t c0, vec8<T> (&to)[S][4]) {
#pragma unroll
    for (int s = 0; s < S; ++s)
#pragma unroll
      for (int t = 0; t < 4; ++t) to[s][t] = load8<T>(fb + (c0 + 16 * t + i) * p.r + 32 * s + 8 * qj, c0 + 16 * t + i < hi ? clamp8(p.r - 32 * s - 8 * qj) : 0);
  };
  int64_t c = wave * 32;
  for (; c + (kAhead - 1) * 32 * kRowWaves + 32 <= p.K; c += kAhead * 32 * kRowWaves) {
    vec8<T> xv[kAhead], av[kAhead][JT];
#pragma unroll
    for (int s = 0; s < kAhead; ++s) {
      const int64_t at = c + s * 32 * kRowWaves + 8 * q;
      xv[s] = load8<T>(row + at);
#pragma unroll
      for (int j = 0; j < JT; ++j) av[s][j] = load8<T>(fr[j] + at);
    }
#pragma unroll
    for (int s = 0; s < kAhead; ++s)
#pragma unroll
      for (int j = 0; j < JT; ++j) acc[j] = mma(av[s][j], xv[s], acc[j]);
  }
  for (; c < p.K; c += 32 * kRowWaves) {
    const int64_t at = c + 8 * q;
    const int have = clamp8(p.K - at);
    const vec8<T> xv = load8<T>(row + at, have);
#pragma unroll
    for (int j = 0; j < JT; ++j) acc[j] = mma(load8<T>(fr[j] + at, have), xv, acc[j]);
  }
#pragma unroll
  for (int e = 0; e < kEarly; ++e)
    if (lo + e * kRowCols + wave * 64 < hi) second(lo + e * kRowCols + wave * 64, fv[e]);
  if (i == 0) {
#pragma unroll
    for (int j = 0; j < JT; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) shares[wave][16 * j + 4 * q + e] = acc[j][e];
  }
  __syncthreads();
  if (threadIdx.x < S * 32) {
    float v = 0.0f;
    if (threadIdx.x < static_cast<unsigned>(p.r)) {
#pragma unroll
      for (int w = 0; w < kRowWaves; ++w) v += shares[w][threadIdx.x];
      if (hidden && part == 0) hidden[m * p.r + threadIdx.x] = v;
      v *= p.scaling[l];
    }
    total[threadIdx.x] = v;
  }
  __syncthreads();
  f32x8_t v[S];
#pragma unroll
  for (int s = 0; s < S; ++s) v[s] = *reinterpret_cast<const f32x8_t *>(total + 32 * s + 8 * qj);
  const float up = row_scale<T>(v);
  const float back = __builtin_bit_cast(float, (254u << 23) - __builtin_bit_cast(uint32_t, up));
  RowOperand<T, kHalf> u[S];
#pragma unroll
  for (int s = 0; s < S; ++s) {
    if constexpr (dtype_code<T>::value == CAIFX_F16) {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[s][e] *= up;
    }
    u[s].set(v[s], q);
  }
#pragma unroll
  for (int e = 0; e < kRowRounds; ++e) {
    const int64_t c0 = lo + e * kRowCols + wave * 64;
    if (c0 >= hi) break;
    if (e >= kEarly) second(c0, fv[0]);
    floatx4_t y[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      y[t] = floatx4_t{0, 0, 0, 0};
#pragma unroll
      for (int s = 0; s < S; ++s) y[t] = u[s].as_rows(fv[e < kEarly ? e : 0][s][t], y[t]);
    }
    // every row of a product is the same: the lanes of q keep column tile q
    float add = q == 0 ? y[0][0] : q == 1 ? y[1][0] : q == 2 ? y[2][0] : y[3][0];
    if constexpr (dtype_code<T>::value == CAIFX_F16) add *= back;
    const int64_t at = c0 + lane;
    if (__builtin_expect(__builtin_isunordered(add, add) && at < hi, 0)) {
      add = 0.0f;
#pragma unroll 1
      for (int j = 0; j < p.r && add == add; ++j) add = __builtin_fmaf(total[j], to_f32<T>(fb[at * p.r + j]), add);
    }
    if (at < hi) out[m * p.N + at] = from_f32<T>((base ? to_f32<T>(base[m * p.N + at]) : 0.0f) + add);
  }
}

// ------------------------------------------------------------------ outer
constexpr int kOuterThreads = 256;
constexpr int kOuterCols = 128;                       // of a workgroup, 32 of a wave; a checkpoint's group
constexpr int kOuterRows = 64;                        // of a step

// what a tensor's values are in LDS: int8 codes are exact in bf16
template <typename Z, typename T> struct Staged { typedef Z type; };
template <typename T> struct Staged<int8_t, T> { typedef bf16_t type; };
template <> struct Staged<int8_t, float> { typedef float type; };
template <typename Z> struct Raw { typedef vec8<Z> type; };
template <> struct Raw<int8_t> { typedef u32x2_t type; };
template <typename S, typename Z> __device__ __forceinline__ vec8<S> staged(const typename Raw<Z>::type &v)
{
  if constexpr (sizeof(Z) > 1) {
    return v;
  } else {
    vec8<S> w;
    float lo[4], hi[4];
    int8x4_to_f32(v[0], lo);
    int8x4_to_f32(v[1], hi);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      w[e] = from_f32<S>(lo[e]);
      w[4 + e] = from_f32<S>(hi[e]);
    }
    return w;
  }
}
template <typename Z> __device__ __forceinline__ typename Raw<Z>::type load_raw(const Z *p, int have)
{
  if constexpr (sizeof(Z) > 1) {
    return load8<Z>(p, have);
  } else {
    typename Raw<Z>::type v;
    __builtin_memset(&v, 0, sizeof v);
    if (have >= 8) {
      __builtin_memcpy(&v, p, 8);
    } else {
      for (int e = 0; e < have; ++e) v[e >> 2] |= static_cast<uint32_t>(static_cast<uint8_t>(p[e])) << (8 * (e & 3));
    }
    return v;
  }
}

struct Outer {
  const void *z;                                      // [M, C], int8 codes with z_scales [M, groups]
  const float *z_scales;
  Rows u;
  int64_t C;
  bool scaled;
  int64_t js, cs;                                     // of the result: [l][j * js + c * cs]
  void *grad;                                         // T
  float *part;                                        // fp32, as many of an adapter's gradients as there are parts
  const int32_t *rows;                                // sorted by adapter, in order for each
  Cut cut;
};

// grad[l][c][j] = scale sum over the rows m of l of z[m][c] u[m][j]: both operands run down their rows, so both are staged in LDS as
// they lie in memory and read with the transposing instruction.  The rows come from the sorted list: whatever their order in the batch,
// they are read once.  The pitches leave the four rows of a transposing read in different banks.
// kRanksDown: of a product's results a lane holds four ranks of one column (grad_a, whose columns are neighbours), else four columns of
// one rank (grad_b, whose ranks are).
constexpr int kOuterList = 1024;                      // rows of a slot at most
constexpr int kZPitch = kOuterCols + 16;
constexpr int u_pitch(int R) { return R + (R == 64 ? 8 : R == 128 ? 16 : 0); }
template <typename T, int JT> constexpr int outer_lds()
{
  return kOuterRows * kZPitch * static_cast<int>(sizeof(T)) + 4 * kOuterRows * u_pitch(16 * JT) + 4 * kOuterList;
}
template <typename Z, typename T, int JT, bool kRanksDown>
__device__ __forceinline__ void outer_block(const Problem &p, const Outer &o, unsigned block, unsigned char *lds)
{
  typedef typename Staged<Z, T>::type S;
  constexpr bool k16 = sizeof(T) == 2;
  typedef typename std::conditional<k16, bf16_t, float>::type UT;
  constexpr int R = 16 * JT, kOf = R / 4;              // values of u of a thread
  constexpr int kUPitch = u_pitch(R);
  static_assert(sizeof(S) == sizeof(T));
  S *zs = reinterpret_cast<S *>(lds);
  UT *us = reinterpret_cast<UT *>(lds + kOuterRows * kZPitch * sizeof(S));             // two of them in 16 bits, one behind the other
  int32_t *list = reinterpret_cast<int32_t *>(lds + kOuterRows * kZPitch * sizeof(S) + 4 * kOuterRows * kUPitch);
  const int64_t tiles = (o.C + kOuterCols - 1) / kOuterCols;
  const int64_t at = block / static_cast<unsigned>(tiles);
  if (at >= o.cut.header[0]) return;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, i = lane & 15, q = lane >> 4;
  const Slot slot = o.cut.slots[at];
  const int64_t c0 = (block - at * tiles) * kOuterCols;
  for (int k = tid; k < slot.count; k += kOuterThreads) list[k] = o.rows[slot.first + k];
  const int64_t groups = (o.C + CAIFX_CHECKPOINT_GROUP - 1) / CAIFX_CHECKPOINT_GROUP, group = c0 / CAIFX_CHECKPOINT_GROUP;
  const float scale = o.scaled && slot.count > 0 ? p.scaling[slot.adapter] : 1.0f;
  floatx4_t acc[2][JT];
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int j = 0; j < JT; ++j) acc[t][j] = floatx4_t{0, 0, 0, 0};
  __syncthreads();

  // a step's values of a thread: four octets of z, a quarter of a row of u
  typename Raw<Z>::type zv[4];
  float uv[kOf];
  const int zrow = tid >> 4, zcol = (tid & 15) * 8, urow = tid >> 2, ucol = (tid & 3) * kOf;
  const Z *z = static_cast<const Z *>(o.z) + c0 + zcol;
  const int zhave = clamp8(o.C - c0 - zcol), uhave = p.r - ucol;
  auto fetch = [&](int s) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int e = s * kOuterRows + zrow + 16 * k;
      if (e < slot.count) zv[k] = load_raw<Z>(z + list[e] * o.C, zhave);
      else __builtin_memset(&zv[k], 0, sizeof zv[k]);
    }
    const int e = s * kOuterRows + urow;
#pragma unroll
    for (int k = 0; k < kOf; ++k) uv[k] = 0.0f;
    if (e < slot.count) {
      const int64_t m = list[e];
      const float by = o.z_scales ? o.z_scales[m * groups + group] : 1.0f;
      const float *from = o.u.at + m * p.r + ucol;
      for (int w = 0; w < o.u.slices; ++w, from += p.M * p.r) {
        if (uhave >= kOf) {
          float add[kOf];
          __builtin_memcpy(add, from, sizeof add);
#pragma unroll
          for (int k = 0; k < kOf; ++k) uv[k] += add[k];
        } else {
#pragma unroll
          for (int k = 0; k < kOf; ++k)
            if (k < uhave) uv[k] += from[k];
        }
      }
      if (o.z_scales) {
#pragma unroll
        for (int k = 0; k < kOf; ++k) uv[k] *= by;
      }
    }
  };
  const int steps = (slot.count + kOuterRows - 1) / kOuterRows;
  if (steps > 0) fetch(0);
  for (int s = 0; s < steps; ++s) {
    if (s > 0) __syncthreads();                       // the step before has been read
#pragma unroll
    for (int k = 0; k < 4; ++k) *reinterpret_cast<vec8<S> *>(zs + (zrow + 16 * k) * kZPitch + zcol) = staged<S, Z>(zv[k]);
    if constexpr (k16) {
      bf16_t hi[kOf], lo[kOf];
#pragma unroll
      for (int k = 0; k < kOf; ++k) {
        hi[k] = from_f32<bf16_t>(uv[k]);
        lo[k] = from_f32<bf16_t>(uv[k] - to_f32<bf16_t>(hi[k]));
      }
      __builtin_memcpy(__builtin_assume_aligned(us + urow * kUPitch + ucol, 8), hi, sizeof hi);
      __builtin_memcpy(__builtin_assume_aligned(us + (kOuterRows + urow) * kUPitch + ucol, 8), lo, sizeof lo);
    } else {
      __builtin_memcpy(__builtin_assume_aligned(us + urow * kUPitch + ucol, 16), uv, sizeof uv);
    }
    __syncthreads();
    if (s + 1 < steps) fetch(s + 1);
#pragma unroll
    for (int h = 0; h < kOuterRows / 32; ++h) {
      typename Fine<T>::type uf[JT];
#pragma unroll
      for (int j = 0; j < JT; ++j) {
        const UT *from = us + 32 * h * kUPitch + 16 * j;
        if constexpr (k16) {
          uf[j].hi = down<UT>(from, kUPitch, 4, lane, q);
          uf[j].lo = down<UT>(from + kOuterRows * kUPitch, kUPitch, 4, lane, q);
        } else {
          uf[j] = down<UT>(from, kUPitch, 4, lane, q);
        }
      }
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const auto w = whole(down<S>(zs + 32 * h * kZPitch + 32 * wave + 16 * t, kZPitch, 4, lane, q));
#pragma unroll
        for (int j = 0; j < JT; ++j) acc[t][j] = kRanksDown ? mma(uf[j], w, acc[t][j], 0) : mma(w, uf[j], acc[t][j], 0);
      }
    }
  }
  const int64_t size = p.r * o.C;
  // a lane's columns and ranks
  const auto column = [&](int t, int e) { return c0 + 32 * wave + 16 * t + (kRanksDown ? i : 4 * q + e); };
  const auto rank = [&](int j, int e) { return 16 * j + (kRanksDown ? 4 * q + e : i); };
  const auto put = [&](int64_t to, float v) {
    if (slot.part >= 0) o.part[slot.part * size + to] = v;
    else static_cast<T *>(o.grad)[slot.adapter * size + to] = from_f32<T>(v);
  };
  bool odd = false;
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int j = 0; j < JT; ++j) {
      odd |= any_nan(acc[t][j]);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (column(t, e) < o.C && rank(j, e) < p.r) put(rank(j, e) * o.js + column(t, e) * o.cs, acc[t][j][e] * scale);
    }
  if (__builtin_expect(odd && scale == scale, 0)) {
#pragma unroll 1
    for (int k = 0; k < 8 * JT; ++k) {
      const int64_t c = column(k / (4 * JT), k % 4);
      const int jj = rank(k / 4 % JT, k % 4);
      if (c >= o.C || jj >= p.r) continue;
      const int64_t to = jj * o.js + c * o.cs;
      const float was = slot.part >= 0 ? o.part[slot.part * size + to] : to_f32<T>(static_cast<const T *>(o.grad)[slot.adapter * size + to]);
      if (was == was) continue;
      float v = 0.0f;
#pragma unroll 1
      for (int n = 0; n < slot.count && v == v; ++n) {
        const int64_t m = list[n];
        float x;
        if constexpr (sizeof(Z) > 1) x = to_f32<Z>(static_cast<const Z *>(o.z)[m * o.C + c]);
        else x = static_cast<float>(static_cast<const Z *>(o.z)[m * o.C + c]) * o.z_scales[m * groups + group];
        v = __builtin_fmaf(rank1(p, o.u, m, jj), x, v);
      }
      put(to, v * scale);
    }
  }
}

// What of the backward needs g or the sorted rows, in one launch: blocks of grad_b, of grad_a, of dx.  Each of the three alone leaves the
// chip half empty at its beginning and its end, and a launch of its own costs the small calls 3 us.
// gradients_waves: waves of a SIMD that registers have to allow, as many as local memory holds where that is a matter of a few registers: three in fp32 up
// to rank 32 (4096 x 11008, rank 16, with two 151 us the pass, with three 141), four with 64 columns in 16 bits
// between ranks 33 and 64 (1200 rows, 1024 to 4096, rank 64: with three 34.0, with four 33.1).
template <typename T, int JT, int G> constexpr int gradients_waves() { return sizeof(T) == 4 && JT <= 2 ? 3 : sizeof(T) == 2 && JT == 4 && G == 1 ? 4 : 1; }
template <typename T, typename Z, int JT, int G>
__global__ __launch_bounds__(kOuterThreads, (gradients_waves<T, JT, G>())) void gradients_kernel(Problem p, Outer b, unsigned blocks_b, Outer a, unsigned blocks_a, Expand dx)
{
  static_assert(kOuterThreads == 64 * kExpandWaves);
  constexpr int RS = JT / 2;
  constexpr int kLds = outer_lds<T, JT>() > expand_lds<T, RS>() ? outer_lds<T, JT>() : expand_lds<T, RS>();
  __shared__ __align__(32) unsigned char lds[kLds];
  if (blockIdx.x < blocks_b) outer_block<T, T, JT, false>(p, b, blockIdx.x, lds);
  else if (blockIdx.x < blocks_b + blocks_a) outer_block<Z, T, JT, true>(p, a, blockIdx.x - blocks_b, lds);
  else expand_block<T, RS, true, G>(p, dx, blockIdx.x - blocks_b - blocks_a, reinterpret_cast<T *>(lds));
}

// the slots of an adapter that has several, added in order
struct Join {
  const float *part;
  void *grad;
  int64_t size;                                       // of an adapter's gradient
  Cut cut;
};
constexpr int kJoinPer = 4;
template <typename T> __device__ __forceinline__ void join(const Join &j, int64_t block, int which)
{
  if (which >= j.cut.header[1]) return;
  const Multi m = j.cut.multi[which];
  const int64_t i = (block * 256 + threadIdx.x) * kJoinPer;
  if (i >= j.size) return;
  const float *from = j.part + m.part * j.size + i;
  T *to = static_cast<T *>(j.grad) + m.adapter * j.size + i;
  if (i + kJoinPer <= j.size) {
    float v[kJoinPer];
    __builtin_memcpy(v, from, sizeof v);
#pragma unroll 4
    for (int s = 1; s < m.parts; ++s) {
      float w[kJoinPer];
      __builtin_memcpy(w, from + s * j.size, sizeof w);
#pragma unroll
      for (int k = 0; k < kJoinPer; ++k) v[k] += w[k];
    }
    T out[kJoinPer];
#pragma unroll
    for (int k = 0; k < kJoinPer; ++k) out[k] = from_f32<T>(v[k]);
    __builtin_memcpy(to, out, sizeof out);
  } else {
    for (int64_t k = 0; i + k < j.size; ++k) {
      float v = from[k];
      for (int s = 1; s < m.parts; ++s) v += from[s * j.size + k];
      to[k] = from_f32<T>(v);
    }
  }
}
template <typename T> __global__ __launch_bounds__(256) void join_kernel(Join a, Join b, unsigned blocks_a)
{
  if (blockIdx.x < blocks_a) join<T>(a, blockIdx.x, blockIdx.y);
  else join<T>(b, blockIdx.x - blocks_a, blockIdx.y);
}

__global__ __launch_bounds__(256) void zero_kernel(unsigned char *at, int64_t bytes)
{
  zero_bytes(at, 0, bytes, static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x, static_cast<int64_t>(gridDim.x) * 256);
}

// ------------------------------------------------------------------ host
int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
int up_to(int rank) { return rank <= 16 ? 16 : rank <= 32 ? 32 : rank <= 64 ? 64 : 128; }      // the ranks that a kernel computes
size_t up16(size_t n) { return (n + 15) & ~static_cast<size_t>(15); }

// rows of a workgroup of the backward's shrinking product
int shrink_rows(int rank, size_t es)
{
  const int bytes = up_to(rank) / 16 * static_cast<int>(es);
  return bytes >= 32 ? 16 : 32;
}

// columns of a unit
int shrink_unit(int rank, size_t es, bool down)
{
  const int bytes = up_to(rank) / 16 * static_cast<int>(es);
  return 32 * shrink_steps(bytes, down);
}

// Workgroups of the shrinking product per `rows` rows: enough that some 512 run, a slice no shorter than one unit for each wave.  Above rank 32
// some 256: every slice is read again by all consumers of the rows (four adapters of rank 64, 4096 rows: 62 + 50 us for the consumers and
// the product, 71 + 51 with twice as many slices; forward of 999 rows to 4096 29.5 and 36.0).
struct Slices {
  int count;
  int64_t columns;
};
Slices plan_slices(int64_t M, int64_t C, int rank, int rows, int unit)
{
  const int64_t tiles = ceil_div(M, rows), whole = ceil_div(C, kShrinkWaves * unit);
  int64_t n = (rank > 32 ? 256 : 512) / (tiles > 0 ? tiles : 1);
  n = n < 1 ? 1 : (n > 16 ? 16 : n);
  if (n > whole) n = whole;
  const int64_t columns = ceil_div(whole, n) * kShrinkWaves * unit;
  return {static_cast<int>(ceil_div(C, columns)), columns};
}

// Rows of a slot of the gradients' products: so many that some 512 workgroups run, in whole steps.
int32_t plan_chunk(int64_t M, int64_t C)
{
  const int64_t rows = ceil_div(ceil_div(M * ceil_div(C, kOuterCols), 512), kOuterRows) * kOuterRows;
  return static_cast<int32_t>(rows < 128 ? 128 : (rows > 1024 ? 1024 : rows));
}

// Whether the forward takes its rows one by one: every workgroup reads its row's first factor again, so that factor must be short (256 KB
// is four memory round trips of a workgroup's waves), the workgroups few enough to run at once, and all reads together less than what the
// caches give in some ten us.  Measured, us,
// row by row / in tiles, rows of one adapter each (neighbours of one adapter), K = 4096, bf16: rank 16, one row 7.4 / 10.1; 32 rows to
// N = 14336 10.1 / 18.6 (8.9 / 10.1); 128 rows to 4096 10.2 / 22.5 (8.8 / 9.8), to 14336 (112 MB) 27.6 / 35.6 (23.9 / 11.8); rank 64
// (512 KB), one row 18.5 / 14.2, 32 rows to 4096 19.9 / 17.3 (19.0 / 13.8).
bool row_at_a_time(int64_t M, int64_t N, int64_t K, int rank, size_t es)
{
  const int64_t factor = static_cast<int64_t>(rank) * K * static_cast<int64_t>(es);
  const int64_t workgroups = M * ceil_div(N, kRowCols * kRowRounds);
  return factor <= 256 << 10 && workgroups <= 512 && workgroups <= (int64_t{64} << 20) / factor;
}

// Workgroups that share the adapters of a tile of 16 rows, `waves` waves working on it otherwise: as many as leave some 4096 in
// all (999 rows in runs, 4096 to 4096, turns of four: 23.5 us, without turns 18.8).
unsigned turns(const Problem &p, int64_t waves)
{
  const int64_t most = p.L < 16 ? p.L : 16, n = 4096 / (ceil_div(p.M, 16) * waves);
  return static_cast<unsigned>(n < 1 ? 1 : (n > most ? most : n));
}

struct Side {                                         // one gradient
  int32_t chunk;
  int64_t slots, parts, multi;                        // at most
  size_t header, slot_bytes, multi_bytes, part_bytes;
};
Side plan_side(int64_t M, int64_t C, int rank, int L)
{
  Side w{};
  w.chunk = plan_chunk(M, C);
  w.slots = M / w.chunk + L;
  w.parts = M > w.chunk ? 2 * (M / w.chunk) : 0;      // an adapter of n > chunk rows has ceil(n / chunk) <= 2 n / chunk
  w.multi = M / (w.chunk + 1) < L ? M / (w.chunk + 1) : L;
  w.header = 16;
  w.slot_bytes = up16(w.slots * sizeof(Slot));
  w.multi_bytes = up16(w.multi * sizeof(Multi));
  w.part_bytes = up16(static_cast<size_t>(w.parts) * rank * C * 4);
  return w;
}
struct Plan {
  Slices slices;
  Side a, b;
  size_t rows, list, spare, total;                    // bytes
};
Plan plan(int64_t M, int64_t N, int64_t K, int rank, int L, size_t es, bool backward)
{
  Plan w{};
  w.slices = plan_slices(M, backward ? N : K, rank, backward ? shrink_rows(rank, es) : 16, shrink_unit(rank, es, backward));
  w.rows = up16(static_cast<size_t>(w.slices.count) * M * rank * 4);
  if (!backward && row_at_a_time(M, N, K, rank, es)) w.rows = 0;
  if (backward) {
    w.a = plan_side(M, K, rank, L);
    w.b = plan_side(M, N, rank, L);
    w.list = up16(static_cast<size_t>(M) * 4);
    w.spare = L > 2048 ? up16(static_cast<size_t>(L) * 4) : 0;      // the sorting workgroup has at least 8 KB of LDS
  }
  w.total = w.rows + w.list + w.spare;
  for (const Side *x : {&w.a, &w.b}) w.total += x->header + x->slot_bytes + x->multi_bytes + x->part_bytes;
  return w;
}

// `product` false: the sorting workgroup alone, which reads neither z nor f
template <typename T, bool kDown>
void shrink(const Problem &p, const Slices &sl, const void *z, int64_t C, const void *f, bool scaled, float *out, const Sort &sort, hipStream_t s,
            bool product = true)
{
  const int rows = kDown ? shrink_rows(p.r, sizeof(T)) : 16;
  const dim3 block(64 * kShrinkWaves),
      grid = product ? dim3(static_cast<unsigned>(ceil_div(p.M, rows) + (sort.rows ? 1 : 0)), sl.count, turns(p, sl.count * kShrinkWaves)) : dim3(1);
  const T *zz = static_cast<const T *>(z), *ff = static_cast<const T *>(f);
  if (p.r <= 16) hipLaunchKernelGGL((shrink_kernel<T, 1, kDown>), grid, block, 0, s, p, zz, C, ff, sl.columns, scaled, out, sort);
  else if (p.r <= 32) hipLaunchKernelGGL((shrink_kernel<T, 2, kDown>), grid, block, 0, s, p, zz, C, ff, sl.columns, scaled, out, sort);
  else if (p.r <= 64) hipLaunchKernelGGL((shrink_kernel<T, 4, kDown>), grid, block, 0, s, p, zz, C, ff, sl.columns, scaled, out, sort);
  else hipLaunchKernelGGL((shrink_kernel<T, 8, kDown>), grid, block, 0, s, p, zz, C, ff, sl.columns, scaled, out, sort);
}

// Whether a wave of the expanding product takes 64 columns, or 256 (in calls of `es` bytes a value).  64 while there are few waves and the rows that
// they read again for each 64 columns (all slices, fp32) are few bytes; fp32 above rank 64 always, where 256 leave registers for one wave of a SIMD.
// Measured, us with 64 / 256 columns, K -> N, runs of 100 rows, bf16 where nothing else is said: rank 16, 1024 -> 14336, 300 rows (4256 waves) 13.6 / 17.2,
// 999 (14112) 22.9 / 23.3; 4096 -> 11008, 600 rows (6536) 19.3 / 20.3, 999 (10836) 25.8 / 24.3.  Rank 64, 1024 -> 14336, 300 rows (33 MB read again)
// 22.3 / 24.3; 4096 -> 14336, 300 rows (133 MB) 36.4 / 30.4; 4096 -> 11008, 999 rows 52.9 / 40.5; its backward to 11008, 600 rows (204 MB) 63.7 / 54.6.
// fp32, rank 64, 4096 -> 11008, 600 rows (102 MB) 54.5 / 57.9, its backward to 11008 (204 MB) 100.7 / 90.7; rank 128, 4096 rows 4096 -> 11008 516 / 530,
// backward 11008 -> 4096 548 / 689.
bool narrow_waves(const Problem &p, const Rows &u, int64_t C, size_t es)
{
  if (es == 4 && p.r > 64) return true;
  const int64_t waves = ceil_div(p.M, 16) * ceil_div(C, kExpandCols), again = waves * u.slices * 16 * 4 * p.r;
  return waves < 8192 && again < (int64_t{es == 4 ? 120 : 72} << 20);
}
template <typename T, int RS> constexpr bool kWideWaves = sizeof(T) == 2 || RS <= 2;      // whether a call may take the wide ones
Expand plan_expand(const Problem &p, const Rows &u, int64_t C, const void *f, bool scaled, const void *base, void *out, float *hidden, bool narrow,
                   unsigned &blocks)
{
  const int64_t tiles = ceil_div(C, kExpandCols * (narrow ? 1 : 4));
  const Expand o{u, C, tiles, f, scaled, base, out, hidden, narrow ? turns(p, tiles) : 1, static_cast<unsigned>(ceil_div(p.M, 16 * kExpandWaves) * tiles)};
  blocks = o.places * o.turns;
  return o;
}

template <typename T> int forward(const Problem &p, const void *x, const void *base, void *y, float *hidden, void *workspace, hipStream_t s)
{
  if (row_at_a_time(p.M, p.N, p.K, p.r, sizeof(T))) {
    // as many parts of the columns as make some 256 workgroups, or as many as are needed
    const int64_t units = ceil_div(p.N, kRowCols), least = ceil_div(units, kRowRounds), most = 256 / p.M < units ? 256 / p.M : units;
    const int64_t per = ceil_div(units, most > least ? most : least) * kRowCols;
    const int padded = static_cast<int>(p.M < 8 ? p.M : ceil_div(p.M, 8) * 8);
    const dim3 grid(static_cast<unsigned>(ceil_div(p.N, per) * padded)), block(64 * kRowWaves);
    const T *xx = static_cast<const T *>(x), *a = static_cast<const T *>(p.a), *b = static_cast<const T *>(p.b), *bb = static_cast<const T *>(base);
    T *yy = static_cast<T *>(y);
    if (p.r <= 16) hipLaunchKernelGGL((row_kernel<T, 0>), grid, block, 0, s, p, padded, xx, a, b, per, bb, yy, hidden);
    else if (p.r <= 32) hipLaunchKernelGGL((row_kernel<T, 1>), grid, block, 0, s, p, padded, xx, a, b, per, bb, yy, hidden);
    else if (p.r <= 64) hipLaunchKernelGGL((row_kernel<T, 2>), grid, block, 0, s, p, padded, xx, a, b, per, bb, yy, hidden);
    else hipLaunchKernelGGL((row_kernel<T, 4>), grid, block, 0, s, p, padded, xx, a, b, per, bb, yy, hidden);
    return launch_status();
  }
  const Plan w = plan(p.M, p.N, p.K, p.r, p.L, sizeof(T), false);
  float *h = static_cast<float *>(workspace);
  if (hidden && w.slices.count == 1) h = hidden, hidden = nullptr;
  shrink<T, false>(p, w.slices, x, p.K, p.a, false, h, Sort{}, s);
  unsigned blocks;
  const Rows rows{h, w.slices.count};
  const bool narrow = narrow_waves(p, rows, p.N, sizeof(T));
  const Expand o = plan_expand(p, rows, p.N, p.b, true, base, y, hidden, narrow, blocks);
  const dim3 grid(blocks), block(64 * kExpandWaves);
#define CAIFX_GO(RS)                                                                                           \
  if (narrow) hipLaunchKernelGGL((expand_kernel<T, RS, 1>), grid, block, 0, s, p, o);                          \
  else if constexpr (kWideWaves<T, RS>) hipLaunchKernelGGL((expand_kernel<T, RS, 4>), grid, block, 0, s, p, o)
  if (p.r <= 16) {
    CAIFX_GO(0);
  } else if (p.r <= 32) {
    CAIFX_GO(1);
  } else if (p.r <= 64) {
    CAIFX_GO(2);
  } else {
    CAIFX_GO(4);
  }
#undef CAIFX_GO
  return launch_status();
}

template <typename T, typename Z>
void gradients(const Problem &p, const Outer &b, unsigned blocks_b, const Outer &a, unsigned blocks_a, const Expand &dx, unsigned blocks_x, bool narrow,
               hipStream_t s)
{
  const dim3 grid(blocks_b + blocks_a + blocks_x), block(kOuterThreads);
  if (grid.x == 0) return;
#define CAIFX_GO(JT)                                                                                                                             \
  if (narrow) hipLaunchKernelGGL((gradients_kernel<T, Z, JT, 1>), grid, block, 0, s, p, b, blocks_b, a, blocks_a, dx);                           \
  else if constexpr (kWideWaves<T, JT / 2>)                                                                                                      \
    hipLaunchKernelGGL((gradients_kernel<T, Z, JT, 4>), grid, block, 0, s, p, b, blocks_b, a, blocks_a, dx)
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
  const int64_t size_a = static_cast<int64_t>(p.r) * p.K, size_b = static_cast<int64_t>(p.r) * p.N;
  if (p.M == 0) {                                     // sums of nothing
    if (ga) hipLaunchKernelGGL(zero_kernel, dim3(1024), dim3(256), 0, s, static_cast<unsigned char *>(ga), static_cast<int64_t>(sizeof(T)) * p.L * size_a);
    if (gb) hipLaunchKernelGGL(zero_kernel, dim3(1024), dim3(256), 0, s, static_cast<unsigned char *>(gb), static_cast<int64_t>(sizeof(T)) * p.L * size_b);
    return launch_status();
  }
  const Plan w = plan(p.M, p.N, p.K, p.r, p.L, sizeof(T), true);
  unsigned char *at = static_cast<unsigned char *>(workspace);
  auto take = [&](size_t n) {
    unsigned char *here = at;
    at += n;
    return here;
  };
  float *g = reinterpret_cast<float *>(take(w.rows));
  Sort sort{};
  sort.rows = reinterpret_cast<int32_t *>(take(w.list));
  sort.spare = reinterpret_cast<int32_t *>(take(w.spare));
  float *part[2];
  for (int k = 0; k < 2; ++k) {
    const Side &side = k ? w.b : w.a;
    Cut &cut = k ? sort.b : sort.a;
    cut.header = reinterpret_cast<int32_t *>(take(side.header));
    cut.slots = reinterpret_cast<Slot *>(take(side.slot_bytes));
    cut.multi = reinterpret_cast<Multi *>(take(side.multi_bytes));
    cut.chunk = side.chunk;
    part[k] = reinterpret_cast<float *>(take(side.part_bytes));
  }
  const Rows rows{g, w.slices.count};
  shrink<T, true>(p, w.slices, dy, p.N, p.b, true, g, ga || gb ? sort : Sort{}, s, dx || ga);      // b may be null for grad_b alone, which needs no g
  unsigned blocks_b = 0, blocks_a = 0, blocks_x = 0;
  const Outer ob{dy, nullptr, Rows{hidden, 1}, p.N, true, 1, p.r, gb, part[1], sort.rows, sort.b};
  const Outer oa{x, x_scales, rows, p.K, false, p.K, 1, ga, part[0], sort.rows, sort.a};
  if (gb) blocks_b = static_cast<unsigned>(ceil_div(p.N, kOuterCols) * w.b.slots);
  if (ga) blocks_a = static_cast<unsigned>(ceil_div(p.K, kOuterCols) * w.a.slots);
  Expand ox{};
  const bool narrow = !dx || narrow_waves(p, rows, p.K, sizeof(T));
  if (dx) ox = plan_expand(p, rows, p.K, p.a, false, base, dx, nullptr, narrow, blocks_x);
  if (x_scales) gradients<T, int8_t>(p, ob, blocks_b, oa, blocks_a, ox, blocks_x, narrow, s);
  else gradients<T, T>(p, ob, blocks_b, oa, blocks_a, ox, blocks_x, narrow, s);
  const int64_t multi_a = ga ? w.a.multi : 0, multi_b = gb ? w.b.multi : 0, multi = multi_a > multi_b ? multi_a : multi_b;
  if (multi > 0) {
    const unsigned blocks_a = multi_a > 0 ? static_cast<unsigned>(ceil_div(size_a, 256 * kJoinPer)) : 0;
    const unsigned blocks_b = multi_b > 0 ? static_cast<unsigned>(ceil_div(size_b, 256 * kJoinPer)) : 0;
    hipLaunchKernelGGL(join_kernel<T>, dim3(blocks_a + blocks_b, static_cast<unsigned>(multi)), dim3(256), 0, s, Join{part[0], ga, size_a, sort.a},
                       Join{part[1], gb, size_b, sort.b}, blocks_a);
  }
  return launch_status();
}

int check(int64_t M, int64_t N, int64_t K, int rank, int num_adapters, int dtype, bool backward)
{
  if (!valid_dtype(dtype) || M < 0 || N <= 0 || K <= 0 || rank <= 0 || num_adapters <= 0) return CAIFX_ERR_INVALID_ARGUMENT;
  if (rank > CAIFX_ADAPTER_RANK_MAX || M > (int64_t{1} << 23) || N > (int64_t{1} << 26) || K > (int64_t{1} << 26)) return CAIFX_ERR_UNSUPPORTED;
  // a grid has fewer than 2^32 threads; the backward's launch holds three kinds of blocks, two of them slots of rows
  constexpr int64_t kBlocks = int64_t{1} << 22;
  for (const int64_t C : {N, K}) {
    if (ceil_div(M, 16 * kExpandWaves) > kBlocks / ceil_div(C, kExpandCols)) return CAIFX_ERR_UNSUPPORTED;
    if (backward && M / plan_chunk(M, C) + num_adapters > kBlocks / ceil_div(C, kOuterCols)) return CAIFX_ERR_UNSUPPORTED;
  }
  return CAIFX_OK;
}

}  // namespace
}  // namespace caifx

using namespace caifx;

extern "C" {

size_t caifx_adapters_workspace_bytes(int64_t M, int64_t N, int64_t K, int rank, int num_adapters, int dtype, int backward)
{
  if (check(M, N, K, rank, num_adapters, dtype, backward != 0) != CAIFX_OK || M == 0) return 0;
  return plan(M, N, K, rank, num_adapters, dtype_size(dtype), backward != 0).total;
}

int caifx_adapters_forward(int64_t M, int64_t N, int64_t K, int rank, int num_adapters, const void *x, const int32_t *ids, const void *a, const void *b,
                           const float *scaling, const void *base, void *y, float *hidden, int dtype, void *workspace, size_t workspace_bytes,
                           caifx_stream_t stream)
{
  const int st = check(M, N, K, rank, num_adapters, dtype, false);
  if (st != CAIFX_OK || M == 0) return st;
  if (!x || !ids || !a || !b || !scaling || !y) return CAIFX_ERR_INVALID_ARGUMENT;
  const size_t es = dtype_size(dtype), need = plan(M, N, K, rank, num_adapters, es, false).total;
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
  const int st = check(M, N, K, rank, num_adapters, dtype, true);
  if (st != CAIFX_OK || ((M == 0 || !dx) && !grad_a && !grad_b)) return st;
  if (M > 0 && (!dy || !ids || !scaling || (dx && !a) || ((dx || grad_a) && !b) || (grad_a && !x) || (grad_b && !hidden))) return CAIFX_ERR_INVALID_ARGUMENT;
  const size_t es = dtype_size(dtype), need = plan(M, N, K, rank, num_adapters, es, true).total;
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
