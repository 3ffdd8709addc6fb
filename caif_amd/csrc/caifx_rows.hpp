// Products with up to some hundred rows of activations and a weight in microscaled 4 bits, or dense in the 16-bit compute type:
//   y[m, n] = sum_k x[m, k] w[n, k]       and, over two weights (gate and up) at once, hidden = silu(x w0^T) * (x w1^T).
//
// Bound by memory with few rows (the weight's bytes), by the L1 from some dozens on: a compute unit has some 100 lines on their way at a
// time, whatever it asks for, and the activations are read anew for every 16 NT weight rows.  So they are asked for in whole lines, only the
// rows that there are, and take the operands' order in a wave's own part of LDS or, in larger calls, beforehand (see pack_rows_kernel).
// Measured, bf16, weights in turn so that none stays in the caches: one row, N = 14336, K = 4096 10.2 us (3.1 TB/s), 16 rows 11.8, one row of a gated
// block over two such weights 19.2 (3.3 TB/s).  A weight used again and again, 31 MB that come half from the memory-side cache: one row 8.0; 24 rows in
// fp16, N = 4096, K = 14336 13.9; eight rows of the gated block 15.2.
// A workgroup of eight waves owns 16 MT rows and 16 NT weight rows of the result; the waves take units of 512 reduction elements in turn and their sums meet in LDS at the end.
// So every wave streams its part of the weight rows straight into matrix-core operands, no wave waits for another in between, and a
// launch of a usual weight has all of it on its way at once.  Lane (j, q) of v_mfma_f32_16x16x32 loads block
// q of four, 16 bytes, of weight row j, and the four lanes of a row exchange their dwords (two swaps of half waves, two of rows of lanes)
// so that instruction i takes block i, lane q its values 8 q .. 8 q + 7.  The codes become operands by
// v_cvt_scalef32_pk_{bf16,f16}_fp4 with the block's scale: exact in bf16, in fp16 rounded like any weight that is cast to it.  Where the
// activations have 4 bits too, the same blocks go into v_mfma_scale_f32_16x16x128_f8f6f4 as they are.
#pragma once

#include "caifx_rows_plan.hpp"
#include "caifx_wide.hpp"

#include <type_traits>

namespace caifx {

constexpr int kRowsChunk = 256;              // reduction elements of a chunk: 128 bytes of codes of a weight row
constexpr int kRowsWaves = 8;

struct RowsArgs {
  const void *x;          // direct: [M, x_pitch] of the compute type, or fp32 for three pieces, x_pitch at least 8, at any address; packed: see pack_rows_kernel
  int64_t x_pitch;
  const void *w[2];       // MX codes or dense rows of the compute type
  const uint8_t *s[2];    // MX scales
  const uint8_t *xs;      // both in 4 bits: scales of x, whose codes are rows of w_pitch bytes
  int64_t M, N, R;        // R: elements of the reduction, a multiple of 8 for dense weights
  int64_t blocks;         // MX blocks of a weight row
  int64_t w_pitch;        // bytes of a weight row
  int chunks, tiles;      // chunks of the reduction, row tiles of 16 in the packed activations
  int span;               // columns of a workgroup, at most 16 for each of its column tiles
  int splits;             // workgroups that share a reduction: the z-th writes its sums to y + z M N (fp32)
  void *y;                // [M, N] result, or hidden
  void *gate, *up;        // two weights: kept projections, or null
  const void *addend;     // one weight: y = T(float(T(acc)) + float(addend))
  int y_dtype;
};

// dword d of lane group q becomes dword q of lane group d
__device__ __forceinline__ u32x4_t exchange(u32x4_t v)
{
  typedef uint32_t two_t __attribute__((ext_vector_type(2)));
  const two_t a = __builtin_bit_cast(two_t, __builtin_amdgcn_permlane32_swap(v[0], v[2], false, false));
  const two_t b = __builtin_bit_cast(two_t, __builtin_amdgcn_permlane32_swap(v[1], v[3], false, false));
  const two_t c = __builtin_bit_cast(two_t, __builtin_amdgcn_permlane16_swap(a[0], b[0], false, false));
  const two_t d = __builtin_bit_cast(two_t, __builtin_amdgcn_permlane16_swap(a[1], b[1], false, false));
  return u32x4_t{c[0], c[1], d[0], d[1]};
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

// A number as three of eight bits of its mantissa each, cut off and so exact, which add up to it; a bf16 in the upper half of every dword.
// (bf16 has no numbers below 2^-133: what a number of less than 2^-109 has beneath that is lost.)
__device__ __forceinline__ void pieces_of_f32(float value, uint32_t (&piece)[3])
{
  const uint32_t bits = __builtin_bit_cast(uint32_t, value), high = bits & 0xFFFF0000u;
  const bool finite = (bits & 0x7F800000u) != 0x7F800000u;
  const float rest = value - __builtin_bit_cast(float, high);
  const uint32_t middle = __builtin_bit_cast(uint32_t, rest) & 0xFFFF0000u;
  const float last = rest - __builtin_bit_cast(float, middle);
  // a NaN whose upper bits alone would be an infinity stays a NaN
  const uint32_t nan = !finite && (bits & 0x007FFFFFu) != 0 ? 0x00400000u : 0u;
  piece[0] = high | nan;
  piece[1] = finite ? middle : 0u;
  piece[2] = finite ? __builtin_bit_cast(uint32_t, last) : 0u;
}

// Eight elements of two bytes (XW = 1) or four, read `gone` elements early: those move out in front, zeros follow behind.
template <int XW> __device__ __forceinline__ void drop_first(u32x4_t (&v)[XW], int gone)
{
  uint32_t a[4 * XW];
#pragma unroll
  for (int i = 0; i < 4 * XW; ++i) a[i] = v[i >> 2][i & 3];
  const auto move = [&](int dwords, bool now) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < 4 * XW; ++i) a[i] = !now ? a[i] : i + dwords < 4 * XW ? a[i + dwords < 4 * XW ? i + dwords : 0] : 0u;
  };
  if constexpr (XW == 1) {
#pragma unroll
    for (int i = 0; i < 4; ++i) a[i] = (gone & 1) ? __builtin_amdgcn_alignbyte(i < 3 ? a[i < 3 ? i + 1 : 0] : 0u, a[i], 2u) : a[i];
  } else {
    move(1, gone & 1);
  }
  move(XW, gone & 2);
  move(2 * XW, gone & 4);
#pragma unroll
  for (int i = 0; i < 4 * XW; ++i) v[i >> 2][i & 3] = gone >= 8 ? 0u : a[i];
}

// P: pieces of an activation (3: fp32).  NW: weights (2: gate and up; the first half of the NT column tiles is gate's).  kWhole: rows of
// at least 16 blocks: a unit's scales of a weight row are one access, at any address (one byte at a time they are more requests than the
// codes; K = 11008, N = 4096, one row 22.0 us instead of 8.6).
// XG: groups of four rows of activations that are read where they are, fp32 ones (up to four) taken
// apart on their way through LDS; 0: packed ones.  kOdd: direct rows that do not end with eight elements, and rows in 4 bits that do not end with
// a block (one kernel for both takes 9.7 us instead of 9.2 for one row, N = 14336, K = 4096, weights in turn, and 75 instead of 71 for 300 packed
// ones; packed first, K = 4095 takes 3 us more).
template <typename CT, int P, int kWeight, int NW, int MT, int NT, int XG, bool kWhole, bool kOdd>
__global__ __launch_bounds__(kRowsWaves * 64) void rows_kernel(RowsArgs g)
{
  constexpr int NC = NT / NW;                // column tiles of one weight
  constexpr bool kMicro = kWeight != ROWS_DENSE, kBoth = kWeight == ROWS_BOTH;
  constexpr bool kDirect = XG > 0 && !kBoth;
  constexpr int WV = kMicro ? 1 : 4, XV = kBoth ? 1 : 4;      // 16-byte pieces of a column tile and of a row tile per half chunk
  constexpr int XW = P == 3 ? 2 : 1;                          // direct: loads of eight elements
  constexpr uint32_t kRoom = kOdd ? 32 : 0;
  constexpr int XL = kDirect ? XG * XW : MT * P * XV;         // loads of activations per half chunk
  // half chunks on their way before the one in hand is used: a second one where a SIMD still holds four waves with it (one row, N = 4096, K =
  // 14336: 10.2 us instead of 13.3; with 32 registers a half chunk, 16 rows, N = 14336, K = 4096: 11.9 instead of 11.4)
  constexpr int kRegs = 4 * (NT * WV + XL);
  constexpr int D = kRegs <= 24 ? 2 : 1;
  static_assert(NT % NW == 0 && (P == 1 || XG <= 1) && (kMicro || !kWhole) && (XG == 0 || XG == 4 * MT || (MT == 1 && XG == 1)) && (kDirect || kWeight == ROWS_MX || !kOdd), "");
  // the activations of a half chunk for each wave, [P][4 XG][16 pieces of 16 bytes]; at the end the waves' sums
  constexpr int kSums = kRowsWaves / 2 * MT * NT * 1024, kOrder = kDirect ? kRowsWaves * P * XG * 1024 : 0;
  __shared__ __attribute__((aligned(16))) unsigned char smem[kSums > kOrder ? kSums : kOrder];
  auto sums = reinterpret_cast<floatx4_t(*)[MT * NT][64]>(smem);
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int j = lane & 15, q = lane >> 4;
  const int64_t n0 = static_cast<int64_t>(blockIdx.x) * g.span, m0 = static_cast<int64_t>(blockIdx.y) * (16 * MT);

  // what each lane reads from, as an offset of 32 bits from the first row of the tile (at most 64 rows of 2^24 bytes): rows past the end
  // are the last one again, and are not stored
  const uint8_t *w_base[NW], *s_base[NW];
#pragma unroll
  for (int v = 0; v < NW; ++v) {
    w_base[v] = static_cast<const uint8_t *>(g.w[v]) + n0 * g.w_pitch;
    s_base[v] = kMicro ? g.s[v] + n0 * g.blocks : nullptr;
  }
  const int columns = g.N - n0 < g.span ? static_cast<int>(g.N - n0) : g.span;
  uint32_t w_off[NC], s_off[NC];
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int n = c * 16 + j;
    const uint32_t row = static_cast<uint32_t>(n < columns ? n : columns - 1);
    w_off[c] = row * static_cast<uint32_t>(g.w_pitch) + q * 16;
    s_off[c] = row * static_cast<uint32_t>(g.blocks);
  }
  const uint8_t *x_base = static_cast<const uint8_t *>(g.x), *xs_base = nullptr;
  uint32_t x_off[kDirect ? XG : MT], xs_off[kBoth ? MT : 1];
  if constexpr (kBoth || kDirect) {
    const int64_t pitch = kBoth ? g.w_pitch : 2 * XW * g.x_pitch;
    x_base += m0 * pitch;
    if constexpr (kBoth) xs_base = g.xs + m0 * g.blocks;
#pragma unroll
    for (int t = 0; t < (kDirect ? XG : MT); ++t) {
      // (direct: lane (j, q) reads piece j of the half chunk of row 4 t + q)
      const int64_t m = m0 + (kDirect ? 4 * t + q : 16 * t + j);
      const uint32_t row = static_cast<uint32_t>((m < g.M ? m : g.M - 1) - m0);
      x_off[t] = row * static_cast<uint32_t>(pitch) + (kDirect ? j * XW : q) * 16 + kRoom;
      if constexpr (kBoth) xs_off[t] = row * static_cast<uint32_t>(g.blocks);
    }
  }
  // 16 bytes at a base that all lanes share, which the asm keeps in scalar registers: otherwise every load of the loop gets a 64-bit pointer
  // of its own in vector registers, a hundred of them
  typedef u32x4_t anywhere_t __attribute__((aligned(1)));
  auto at128 = [](const uint8_t *base, uint32_t off, auto aligned_) __attribute__((always_inline)) {
    uint64_t b = reinterpret_cast<uint64_t>(base);
    asm("" : "+s"(b), "+v"(off));
    if constexpr (decltype(aligned_)::value) return *reinterpret_cast<const __attribute__((address_space(1))) u32x4_t *>(b + off);
    else return static_cast<u32x4_t>(*reinterpret_cast<const __attribute__((address_space(1))) anywhere_t *>(b + off));
  };
  const std::true_type aligned{};

  // A unit is two chunks, four halves of 128 elements; wave w takes units w, w + 8, ..
  struct Half {
    u32x4_t w[NT][WV];
    u32x4_t x[XL];
    uint32_t scale[kMicro && !kWhole ? NT : 1];      // like a dword of Scales; both in 4 bits: the byte of this lane's block
    uint32_t x_scale[kBoth && !kWhole ? MT : 1];
  };
  struct Scales {
    u32x4_t w[kWhole ? NT : 1];              // dword h: the scales of half h, a byte for each of its blocks
    u32x4_t x[kWhole && kBoth ? MT : 1];
  };
  const int length = static_cast<int>(kOdd ? g.x_pitch : g.R);      // (dense rows are filled up to a multiple of eight)
  const int halves = kMicro ? static_cast<int>((g.blocks + 3) >> 2) : static_cast<int>((g.R + 127) >> 7);
  const int units = (halves + 3) >> 2;
  const int z = static_cast<int>(blockIdx.z);
  const int first = units * z / g.splits + wave, end = units * (z + 1) / g.splits;
  const int mine = end > first ? (end - 1 - first) / kRowsWaves + 1 : 0;
  auto load_scales = [&](Scales &to, int unit) __attribute__((always_inline)) {
    if constexpr (kWhole) {
      // (a unit that begins less than 16 blocks before the end of a row: the row's last 16, see `behind`)
      const int64_t at = static_cast<int64_t>(unit) * 16, from = at + 16 <= g.blocks ? at : g.blocks - 16;
#pragma unroll
      for (int c = 0; c < NT; ++c) to.w[c] = at128(s_base[c / NC] + from, s_off[c % NC], std::false_type{});
      if constexpr (kBoth) {
#pragma unroll
        for (int t = 0; t < MT; ++t) to.x[t] = at128(xs_base + from, xs_off[t], std::false_type{});
      }
    }
  };
  // half `at` of all; past the end the last one again (it is not used)
  auto load = [&](Half &b, int at) __attribute__((always_inline)) {
    const int64_t half = at < halves ? at : halves - 1;
    if constexpr (kMicro) {
      // blocks past the end of a row: its last one again, as zeros or (kWhole) under a scale of 2^-127 against activations that are zeros
      const int block = static_cast<int>(half) * 4 + q;
      const bool in = block < g.blocks;
      const uint32_t back = in ? 0u : static_cast<uint32_t>(block - (g.blocks - 1));
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        b.w[t][0] = at128(w_base[t / NC] + half * 64, w_off[t % NC] - back * 16, aligned);
        if constexpr (!kWhole) {
          const uint8_t *from = s_base[t / NC] + half * 4;
          if constexpr (kBoth) {
            b.scale[t] = in ? from[s_off[t % NC] + q - back] : 0u;
          } else {
            // the half's four bytes, those past the end of the row as zeros
            uint32_t dword = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (half * 4 + i < g.blocks) dword |= static_cast<uint32_t>(from[s_off[t % NC] + i]) << (8 * i);
            b.scale[t] = dword;
          }
          if (!in) b.w[t][0] = u32x4_t{0, 0, 0, 0};
        }
      }
      if constexpr (kBoth) {
#pragma unroll
        for (int t = 0; t < MT; ++t) {
          b.x[t] = at128(x_base + half * 64, x_off[t] - back * 16, aligned);
          if constexpr (!kWhole) b.x_scale[t] = in ? (xs_base + half * 4)[xs_off[t] + q - back] : 0u;
        }
        return;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        // pieces of eight elements past the end of a row: its last one again, as zeros once it is used
        const int k = static_cast<int>(half) * 128 + 32 * i + 8 * q;
        const uint32_t back = k < g.R ? 0u : static_cast<uint32_t>(k - (g.R - 8)) * 2;
#pragma unroll
        for (int t = 0; t < NT; ++t) b.w[t][i] = at128(w_base[t / NC] + half * 256, w_off[t % NC] + 64 * i - back, aligned);
      }
    }
    if constexpr (kDirect) {
      // Eight elements that begin past the row, or (kOdd) end there: its last eight.  Those can begin up to 28 bytes before the half chunk, which
      // the offset, without a sign, makes room for.
      const int k = static_cast<int>(half) * 128 + 8 * j;
      uint32_t back;
      if constexpr (kOdd) back = k + 8 > length ? static_cast<uint32_t>(k + 8 - length) * (2 * XW) : 0u;
      else back = k < g.R ? 0u : static_cast<uint32_t>(k - (g.R - 8)) * (2 * XW);
#pragma unroll
      for (int t = 0; t < XG; ++t)
#pragma unroll
        for (int i = 0; i < XW; ++i) b.x[t * XW + i] = at128(x_base + half * (256 * XW) - kRoom, x_off[t] - back + 16 * i, std::false_type{});
    } else {
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        int64_t tile = (m0 >> 4) + t;
        tile = tile < g.tiles ? tile : g.tiles - 1;
        const uint8_t *from = x_base + (tile * g.chunks + (half >> 1)) * (P * 8 * 1024);
#pragma unroll
        for (int p = 0; p < P; ++p)
#pragma unroll
          for (int i = 0; i < 4; ++i) b.x[(t * P + p) * 4 + i] = at128(from + (p * 8 + 4 * (half & 1) + i) * 1024, static_cast<uint32_t>(lane) * 16, aligned);
      }
    }
  };

  floatx4_t acc[MT][NT];
#pragma unroll
  for (int t = 0; t < MT; ++t)
#pragma unroll
    for (int c = 0; c < NT; ++c) acc[t][c] = floatx4_t{0.0f, 0.0f, 0.0f, 0.0f};
  // direct: a wave's rows of a half chunk through its own part of LDS into the operands' order; piece p of row r lies in place p ^ r, so that
  // the reads of sixteen rows use every bank.  Lanes of rows that were not read hold others': their results are not stored.
  unsigned char *const order = smem + (kDirect ? wave * (P * XG * 1024) : 0);
  // kPart: the half may reach past the end of the rows
  auto compute = [&](Half &b, const Scales &s, int h, int half, auto part_) __attribute__((always_inline)) {
    constexpr bool kPart = decltype(part_)::value;
    if constexpr (kPart && kDirect) {
      if constexpr (kOdd) {
        const int past = half * 128 + 8 * j + 8 - length;
        if (past > 0)
#pragma unroll
          for (int t = 0; t < XG; ++t) {
            u32x4_t eight[XW];
#pragma unroll
            for (int i = 0; i < XW; ++i) eight[i] = b.x[t * XW + i];
            drop_first<XW>(eight, past);
#pragma unroll
            for (int i = 0; i < XW; ++i) b.x[t * XW + i] = eight[i];
          }
      } else {
        if (half * 128 + 8 * j >= g.R)
#pragma unroll
          for (int t = 0; t < XL; ++t) b.x[t] = u32x4_t{0, 0, 0, 0};
      }
    }
    if constexpr (kPart && kMicro && kOdd) {
      // codes behind the last column, whose values may be beyond the compute type: an infinity against the activations' zeros would be a NaN
      const int left = static_cast<int>(g.R) - 32 * (4 * half + q);
      if ((g.R & 31) != 0 && left < 32) {
#pragma unroll
        for (int d = 0; d < 4; ++d) {
          const int in = left - 8 * d;
          const uint32_t mask = in >= 8 ? ~0u : in > 0 ? (1u << (4 * in)) - 1u : 0u;
#pragma unroll
          for (int t = 0; t < NT; ++t) b.w[t][0][d] &= mask;
        }
      }
    }
    if constexpr (kPart && !kMicro) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (half * 128 + 32 * i + 8 * q >= g.R)
#pragma unroll
          for (int t = 0; t < NT; ++t) b.w[t][i] = u32x4_t{0, 0, 0, 0};
    }
    u32x4_t ordered[kDirect ? MT * P * 4 : 1];
    if constexpr (kDirect) {
#pragma unroll
      for (int t = 0; t < XG; ++t) {
        unsigned char *to = order + (4 * t + q) * 256 + ((j ^ ((4 * t + q) & 15)) << 4);
        if constexpr (P == 1) {
          *reinterpret_cast<u32x4_t *>(to) = b.x[t];
        } else {
          u32x4_t v[3];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const floatx4_t four = __builtin_bit_cast(floatx4_t, b.x[t * XW + (i >> 1)]);
            uint32_t even[3], odd[3];
            pieces_of_f32(four[2 * (i & 1)], even);
            pieces_of_f32(four[2 * (i & 1) + 1], odd);
#pragma unroll
            for (int p = 0; p < 3; ++p) v[p][i] = __builtin_amdgcn_perm(odd[p], even[p], 0x07060302u);
          }
#pragma unroll
          for (int p = 0; p < 3; ++p) *reinterpret_cast<u32x4_t *>(to + p * (XG * 1024)) = v[p];
        }
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int row = XG < 4 ? j & (4 * XG - 1) : 16 * t + j;
#pragma unroll
          for (int p = 0; p < P; ++p)
            ordered[(t * P + p) * 4 + i] = *reinterpret_cast<const u32x4_t *>(order + p * (XG * 1024) + row * 256 + (((4 * i + q) ^ (row & 15)) << 4));
        }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
    }
#pragma unroll
    for (int c = 0; c < NT; ++c) {
      if constexpr (kBoth) {
        const uint32_t byte = kWhole ? s.w[kWhole ? c : 0][h] >> (8 * q) : b.scale[kWhole ? 0 : c];
#pragma unroll
        for (int t = 0; t < MT; ++t) {
          const uint32_t xb = kWhole ? s.x[kWhole ? t : 0][h] >> (8 * q) : b.x_scale[kWhole ? 0 : t];
          acc[t][c] = mfma_micro(b.x[t], b.w[c][0], acc[t][c], xb, byte);
        }
      } else {
        u32x4_t codes;
        uint32_t bytes = 0;
        if constexpr (kMicro) {
          codes = exchange(b.w[c][0]);
          bytes = kWhole ? s.w[kWhole ? c : 0][h] : b.scale[kWhole ? 0 : c];
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          u32x4_t w;
          if constexpr (kMicro) w = mxfp4_eight<CT>(codes[i], mxfp4_scale((bytes >> (8 * i)) & 255u));
          else w = b.w[c][i];
#pragma unroll
          for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int p = 0; p < P; ++p) acc[t][c] = Mfma16<CT>::run(kDirect ? ordered[kDirect ? (t * P + p) * 4 + i : 0] : b.x[kDirect ? 0 : (t * P + p) * 4 + i], w, acc[t][c]);
        }
      }
    }
  };
  // the halves of unit `unit`; what they leave free is asked for again: the unit's own later halves, then those of unit + 8
  Half ring[D];
  Scales scales;
  auto run = [&](int unit, auto last_, auto part_) __attribute__((always_inline)) {
    constexpr bool kLast = decltype(last_)::value, kPart = decltype(part_)::value;      // kPart: maybe less than four halves
    Scales next;
    if constexpr (!kLast) load_scales(next, unit + kRowsWaves);
    if constexpr (kWhole && kPart) {
      // the row's last 16 blocks begin `behind` before this unit's: the dwords move up, then the bytes, zeros behind them
      const int behind = 16 * unit + 16 - static_cast<int>(g.blocks);
      const auto forth = [&](u32x4_t &v) __attribute__((always_inline)) {
        const int d = behind >> 2;
        const uint32_t t0 = d == 0 ? v[0] : d == 1 ? v[1] : d == 2 ? v[2] : v[3], t1 = d == 0 ? v[1] : d == 1 ? v[2] : d == 2 ? v[3] : 0u,
                       t2 = d == 0 ? v[2] : d == 1 ? v[3] : 0u, t3 = d == 0 ? v[3] : 0u;
        const uint32_t r = static_cast<uint32_t>(behind & 3);
        v = u32x4_t{__builtin_amdgcn_alignbyte(t1, t0, r), __builtin_amdgcn_alignbyte(t2, t1, r), __builtin_amdgcn_alignbyte(t3, t2, r),
                    __builtin_amdgcn_alignbyte(0u, t3, r)};
      };
      if (behind > 0) {
#pragma unroll
        for (int c = 0; c < NT; ++c) forth(scales.w[kWhole ? c : 0]);
        if constexpr (kBoth) {
#pragma unroll
          for (int t = 0; t < MT; ++t) forth(scales.x[kWhole && kBoth ? t : 0]);
        }
      }
    }
#pragma unroll
    for (int h = 0; h < 4; ++h) {
      // (a branch here makes the compiler wait for all that is on its way; without one it asks for more than there are registers for where
      // the tile is large)
      if ((D > 1 && !kPart) || 4 * unit + h < halves) compute(ring[h % D], scales, h, 4 * unit + h, part_);
      __builtin_amdgcn_sched_barrier(0);
      if (h + D < 4) load(ring[h % D], 4 * unit + h + D);
      else if constexpr (!kLast) load(ring[h % D], 4 * (unit + kRowsWaves) + h + D - 4);
      __builtin_amdgcn_sched_barrier(0);
    }
    if constexpr (!kLast) scales = next;
  };
  if (mine > 0) {
    load_scales(scales, first);
#pragma unroll
    for (int h = 0; h < D; ++h) load(ring[h], 4 * first + h);
    int unit = first;
    for (int t = 1; t < mine; ++t, unit += kRowsWaves) run(unit, std::false_type{}, std::false_type{});
    if (D == 1 || 512 * (unit + 1) > (kOdd ? g.x_pitch : g.R)) run(unit, std::true_type{}, std::true_type{});
    else run(unit, std::true_type{}, std::false_type{});
  }

  // the eight waves' sums, in a fixed order: wave w + 4's into wave w's, then those four into the result
  constexpr int kHalf = kRowsWaves / 2;
  if constexpr (kDirect) __syncthreads();      // (their places are others' activations until then)
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
      if (m >= g.M || col >= columns) continue;
      const int tile = (row >> 4) * NT + (col >> 4);
      const float v = total(tile, row & 15, col & 15);
      const int64_t to = (z * g.M + m) * g.N + n;
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

template <typename CT, int P, int kWeight, int NW, int MT, int NT, int XG>
int rows_launch(const RowsArgs &g, hipStream_t s)
{
  const int64_t rows = (g.M + 16 * MT - 1) / (16 * MT), cols = (g.N + g.span - 1) / g.span;
  // a grid's second extent has 65535 blocks: more rows than that go in several launches
  for (int64_t r = 0; r < rows; r += 65535) {
    RowsArgs part = g;
    const int64_t m0 = r * 16 * MT, es = static_cast<int64_t>(dtype_size(g.y_dtype));
    const auto forth = [&](const void *p, int64_t bytes) { return p ? const_cast<char *>(static_cast<const char *>(p)) + bytes : nullptr; };
    part.M = g.M - m0;
    part.tiles = g.tiles - static_cast<int>(m0 / 16);
    part.x = forth(g.x, kWeight == ROWS_BOTH ? m0 * g.w_pitch : XG > 0 ? m0 * g.x_pitch * (P == 3 ? 4 : 2) : m0 / 16 * g.chunks * (P * 8 * 1024));
    part.xs = g.xs ? g.xs + m0 * g.blocks : nullptr;
    part.y = forth(g.y, m0 * g.N * es);
    part.gate = forth(g.gate, m0 * g.N * es);
    part.up = forth(g.up, m0 * g.N * es);
    part.addend = forth(g.addend, m0 * g.N * es);
    const dim3 grid(static_cast<unsigned>(cols), static_cast<unsigned>(rows - r < 65535 ? rows - r : 65535), static_cast<unsigned>(g.splits));
    const auto go = [&](auto whole_, auto odd_) {
      hipLaunchKernelGGL((rows_kernel<CT, P, kWeight, NW, MT, NT, XG, decltype(whole_)::value, decltype(odd_)::value>), grid, dim3(kRowsWaves * 64), 0, s, part);
    };
    const auto pick_odd = [&](auto whole_) {
      if constexpr (kWeight == ROWS_MX || (XG > 0 && kWeight != ROWS_BOTH)) {
        if (g.x_pitch % (kWeight == ROWS_MX ? CAIFX_MXFP4_BLOCK : 8) != 0) return go(whole_, std::true_type{});
      }
      go(whole_, std::false_type{});
    };
    if constexpr (kWeight != ROWS_DENSE) {
      if (g.blocks >= 16) pick_odd(std::true_type{});
      else pick_odd(std::false_type{});
    } else {
      pick_odd(std::false_type{});
    }
  }
  return launch_status();
}

template <typename CT, int P, int kWeight, int NW, int MT, int XG>
int rows_pick_columns(const RowsArgs &g, hipStream_t s)
{
  const int tiles = rows_column_tiles(g.span, NW);
  if constexpr (P == 1 || MT == 1) {
    if (tiles == 4) return rows_launch<CT, P, kWeight, NW, MT, 4, XG>(g, s);
  }
  if constexpr (NW == 1) {
    if (tiles == 1) return rows_launch<CT, P, kWeight, NW, MT, 1, XG>(g, s);
  }
  return rows_launch<CT, P, kWeight, NW, MT, 2, XG>(g, s);
}
// XG for activations that are read where they are, unless no call does so: a dense copy of one weight is a gradient's, with packed activations
template <typename CT, int P, int kWeight, int NW, int MT, int XG> int rows_pick_direct(const RowsArgs &g, bool direct, hipStream_t s)
{
  if constexpr (kWeight == ROWS_MX || NW == 2) {
    if (direct) return rows_pick_columns<CT, P, kWeight, NW, MT, XG>(g, s);
  }
  return rows_pick_columns<CT, P, kWeight, NW, MT, 0>(g, s);
}
template <typename CT, int kWeight, int NW> int rows_pick(const RowsArgs &g, int pieces, bool direct, hipStream_t s)
{
  const bool four = direct && g.M <= 4;
  // (two stored weights are of the 16-bit compute type)
  if constexpr (dtype_code<CT>::value == CAIFX_BF16 && (kWeight == ROWS_MX || NW == 1)) {
    if (pieces == 3) {
      if (rows_tile(g.M, 3) == 32) return rows_pick_columns<CT, 3, kWeight, NW, 2, 0>(g, s);
      return rows_pick_direct<CT, 3, kWeight, NW, 1, 1>(g, direct, s);
    }
  }
  switch (rows_tile(g.M, 1)) {
    case 16: return four ? rows_pick_direct<CT, 1, kWeight, NW, 1, 1>(g, direct, s) : rows_pick_direct<CT, 1, kWeight, NW, 1, 4>(g, direct, s);
    case 32: return rows_pick_direct<CT, 1, kWeight, NW, 2, 8>(g, direct, s);
    default: return rows_pick_direct<CT, 1, kWeight, NW, 4, 16>(g, direct, s);
  }
}

int rows_both(const RowsArgs &g, hipStream_t s);
int rows_bf16(const RowsArgs &g, int weight, int weights, int pieces, bool direct, hipStream_t s);
int rows_f16(const RowsArgs &g, int weight, int weights, bool direct, hipStream_t s);

}  // namespace caifx
