// Product of two tensors in microscaled 4 bits on the 4-bit matrix cores: y[m, n] = sum over the blocks of 2^(sa + sb) sum a b.
//
// v_mfma_scale_f32_16x16x128_f8f6f4 takes codes and scales as they are stored: lane (r, q) holds block q of row r, 16 bytes, and the
// block's byte.  Four times the rate of bf16 from a quarter of the bytes, so the operands' way is the same as in caifx_gemm_wide.hip: a
// step is 128 bytes of every row (256 values, two instructions deep), tiles of 64 WI x 64 WJ, four waves of a quarter each, half tiles
// asked for three ahead straight into LDS.  Beside them the scales of two steps, 16 bytes of every row, in a ring of two, from a copy that
// holds the 1 KB of 64 rows together (from the rows themselves each request touches 64 lines, eight times over: 157 us instead of 141 at
// M = 4096, N = 14336, K = 4096).
// The columns' operand is the instruction's first one, so that a lane's four sums are neighbours of a row and go to LDS, on their way into
// whole rows, 8 bytes (fp32: 16) at a time.
// M = 4096, N = 14336, K = 4096: 137 us, 3.5 PFLOP/s, behind 5.5 for the scales' order.  A step takes 1.59 us where the matrix pipes alone
// take 1.32, and a tile 9 us more for its first requests and its results, which all compute units write at once.
// Blocks past the end of a row count for nothing: both scales are 2^-127 there, and codes have no infinities or NaN.
#include "caifx_mxfp4.hpp"

#include <atomic>
#include <type_traits>

namespace caifx {
namespace {

constexpr int kBandRows = 1024;            // rows of a band of the tile order

struct MxGemmArgs {
  const uint8_t *a, *b;         // codes [M, pitch], [C, pitch] bytes
  const uint8_t *sa, *sb;       // scales in the order of order_scales_kernel, `groups` pieces of 16 bytes a row
  void *d;                      // [M, C]
  int64_t M, C, pitch;
  int groups, d_dtype;
  int parts;                    // workgroups that share a tile's steps: the z-th writes its sums to d + z M C (fp32)
  int halved;                   // tiles at the end of each XCD's list that two workgroups of half the rows take
};

__device__ __forceinline__ void mfma_mx(floatx4_t &acc, const u32x4_t &a, const u32x4_t &b, uint32_t sa, uint32_t sb)
{
  asm volatile("v_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel_hi:[0,0,0] cbsz:4 blgp:4" : "+a"(acc) : "v"(a), "v"(b), "v"(sa), "v"(sb));
}

// A step runs through the quadrants (h, g) = (0,0) (0,1) (1,1) (1,0) of its tile, h the half of the rows and g that of the columns; the
// operands of a quadrant are read during the one before it.  Half 1 of step s has been read by everybody in the middle of quadrant (1,1)
// and half 0 in the middle of the next step's (0,0): there the waves meet, and behind the barrier the freed slot is requested for step
// s + 2.  Requests complete in issue order, so each wait is an exact count: WI + WJ requests of a wave per half, and two more, the
// scales of steps s + 2 and s + 3, with half 0 where s + 2 is even.
template <int WI, int WJ, bool kTail> __device__ __forceinline__ void mx_tile(MxGemmArgs &g, unsigned char *smem, int64_t row0, int64_t col0)
{
  constexpr int BM = 64 * WI, BN = 64 * WJ;
  constexpr int kASlot = BM / 2 * 128, kBSlot = BN / 2 * 128;      // LDS bytes of half an operand tile
  constexpr int kBBase = 4 * kASlot;
  constexpr int kScales = kBBase + 4 * kBSlot;                     // scales: [slot][BM + BN rows][16 bytes]
  constexpr int kScaleSlot = (BM + BN) * 16;
  constexpr int kReq = WI + WJ;            // requests of a wave per half step
  constexpr int kMore = 2;                 // requests of a wave for the scales of two steps
  constexpr int Q = 2 * WI * WJ;           // products per quadrant
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave >> 1, wn = wave & 1;
  const int r16 = lane & 15, kq = lane >> 4;

  // this workgroup's steps, from an even one on (two share their scales)
  const int total = static_cast<int>((g.pitch + 127) / 128), z = static_cast<int>(blockIdx.y);
  const int begin = static_cast<int>(static_cast<int64_t>(total) * z / g.parts) & ~1;
  const int steps = (z + 1 == g.parts ? total : static_cast<int>(static_cast<int64_t>(total) * (z + 1) / g.parts) & ~1) - begin, last = steps - 1;
  const bool ends = z + 1 == g.parts;      // it has the rows' last step
  if (z > 0) g.d = static_cast<float *>(g.d) + z * g.M * g.C;
  // request i of a wave for half h of an operand: 8 rows x 128 bytes; LDS position p of row r holds 16-byte chunk p ^ (r ^ r >> 3) & 7 of
  // the row, so that eight neighbouring lanes' operand reads use eight times four banks (the counters call half of the cycles in which LDS
  // is busy conflicts all the same, as they do in caifx_gemm_wide.hip, which has no scales).  Rows past the end are the last one again and
  // never stored; of a row's last step chunks past its end are its last one again (their scales are 2^-127).
  const uint32_t lds0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(smem));
  uint32_t a_voff[2][WI], b_voff[2][WJ], past[2];
  const int in_last = static_cast<int>((g.pitch - static_cast<int64_t>(total - 1) * 128) >> 4);      // chunks of the last step
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int lrow = 8 * (wave + 4 * i) + (lane >> 3);
    const int chunk = (lane & 7) ^ ((lrow ^ (lrow >> 3)) & 7);
    past[i] = ends && chunk >= in_last ? static_cast<uint32_t>(chunk - in_last + 1) * 16 : 0;
  }
#pragma unroll
  for (int h = 0; h < 2; ++h) {
#pragma unroll
    for (int i = 0; i < WI; ++i) {
      const int lrow = 8 * (wave + 4 * i) + (lane >> 3);
      int64_t m = row0 + h * (BM / 2) + lrow;
      m = m < g.M ? m : g.M - 1;
      a_voff[h][i] = static_cast<uint32_t>((m - row0) * g.pitch + (((lane & 7) ^ ((lrow ^ (lrow >> 3)) & 7)) << 4));
    }
#pragma unroll
    for (int i = 0; i < WJ; ++i) {
      const int lrow = 8 * (wave + 4 * i) + (lane >> 3);
      int64_t c = col0 + h * (BN / 2) + lrow;
      c = c < g.C ? c : g.C - 1;
      b_voff[h][i] = static_cast<uint32_t>((c - col0) * g.pitch + (((lane & 7) ^ ((lrow ^ (lrow >> 3)) & 7)) << 4));
    }
  }
  const uint64_t a_base = uniform64(reinterpret_cast<uint64_t>(g.a) + static_cast<uint64_t>(row0 * g.pitch + begin * 128));
  const uint64_t b_base = uniform64(reinterpret_cast<uint64_t>(g.b) + static_cast<uint64_t>(col0 * g.pitch + begin * 128));
  auto request = [&](int s, int h, int slot, int x) __attribute__((always_inline)) {
    const uint32_t k0 = static_cast<uint32_t>(s < last ? s : last) * 128;          // past the end: the last step again
    const bool is_a = x < WI;
    const int i = is_a ? x : x - WI;
    const uint64_t src = (is_a ? a_base : b_base) + k0;
    const uint32_t dst = lds0 + (is_a ? slot * kASlot : kBBase + slot * kBSlot) + (wave + 4 * i) * 1024;
    uint32_t voff = is_a ? a_voff[h][is_a ? i : 0] : b_voff[h][is_a ? 0 : i];
    if constexpr (kTail) voff -= s >= last ? past[i & 1] : 0u;
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(dst), "v"(voff), "s"(src) : "memory");
  };
  // the scales of steps 2 group and 2 group + 1: a wave takes 64 rows of either operand (with 128 rows two waves the same ones)
  const int groups = g.groups, group0 = begin >> 1;
  const uint32_t s_voff = static_cast<uint32_t>(lane) * 16;
  const auto scales_of = [&](const uint8_t *scales, int64_t row) __attribute__((always_inline)) {
    return uniform64(reinterpret_cast<uint64_t>(scales) + static_cast<uint64_t>((row >> 6) * groups) * 1024);
  };
  const uint64_t sa_base = scales_of(g.sa, row0 + (64 * wave) % BM < g.M ? row0 + (64 * wave) % BM : row0);      // (past the last row: others' scales)
  const uint64_t sb_base = scales_of(g.sb, col0 + (64 * wave) % BN < g.C ? col0 + (64 * wave) % BN : col0);
  auto request_scales = [&](int group, int x) __attribute__((always_inline)) {
    const uint32_t k0 = static_cast<uint32_t>(group0 + group < groups ? group0 + group : groups - 1) * 1024;
    const uint64_t src = (x == 0 ? sa_base : sb_base) + k0;
    const uint32_t dst = lds0 + kScales + (group & 1) * kScaleSlot + (x == 0 ? (64 * wave) % BM : BM + (64 * wave) % BN) * 16;
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(dst), "v"(s_voff), "s"(src) : "memory");
  };

  // operand (row tile i of 16 rows, reduction half kk): tiles i and i + 2 lie 32 rows apart, which flips the
  // swizzle's third bit, the one that kk selects
  uint32_t a_addr[2][2], b_addr[2][2];
#pragma unroll
  for (int kk = 0; kk < 2; ++kk)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int ra = wm * 16 * WI + i * 16 + r16;
      a_addr[i][kk] = ra * 128 + (((4 * kk + kq) ^ ((ra ^ (ra >> 3)) & 7)) << 4);
      const int rb = wn * 16 * WJ + i * 16 + r16;
      b_addr[i][kk] = kBBase + rb * 128 + (((4 * kk + kq) ^ ((rb ^ (rb >> 3)) & 7)) << 4);
    }
  const uint32_t sa_addr = kScales + (wm * 16 * WI + r16) * 16 + kq, sb_addr = kScales + (BM + wn * 16 * WJ + r16) * 16 + kq;
  struct Operand {
    u32x4_t v;
    uint32_t s;
  };
  // par: the step's parity, which half of its 16 bytes of scales it is; pair: the parity of its two steps
  auto read_a = [&](int half, int par, int pair, int i, int kk) __attribute__((always_inline)) {
    Operand o;
    o.v = *reinterpret_cast<const u32x4_t *>(smem + (2 * par + half) * kASlot + (i >> 1) * 4096 + a_addr[i & 1][kk ^ (i >> 1)]);
    o.s = smem[sa_addr + pair * kScaleSlot + (half * (BM / 2) + i * 16) * 16 + par * 8 + 4 * kk];
    return o;
  };
  auto read_b = [&](int half, int par, int pair, int i, int kk) __attribute__((always_inline)) {
    Operand o;
    o.v = *reinterpret_cast<const u32x4_t *>(smem + (2 * par + half) * kBSlot + (i >> 1) * 4096 + b_addr[i & 1][kk ^ (i >> 1)]);
    o.s = smem[sb_addr + pair * kScaleSlot + (half * (BN / 2) + i * 16) * 16 + par * 8 + 4 * kk];
    return o;
  };

  floatx4_t acc[2][2][WI][WJ];     // [h][g][row tile][column tile]
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int q = 0; q < 2; ++q)
#pragma unroll
      for (int i = 0; i < WI; ++i)
#pragma unroll
        for (int c = 0; c < WJ; ++c) acc[h][q][i][c] = floatx4_t{0.0f, 0.0f, 0.0f, 0.0f};

#pragma unroll
  for (int u = 0; u < 4; ++u) {
#pragma unroll
    for (int x = 0; x < kReq; ++x) request(u >> 1, u & 1, u, x);
    if (u == 0)
      for (int x = 0; x < kMore; ++x) request_scales(0, x);
  }
  asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"(3 * kReq) : "memory");
  Operand a0[WI][2], a1[WI][2], b0[WJ][2], b1[WJ][2];
#pragma unroll
  for (int kk = 0; kk < 2; ++kk) {
#pragma unroll
    for (int i = 0; i < WJ; ++i) b0[i][kk] = read_b(0, 0, 0, i, kk);
#pragma unroll
    for (int i = 0; i < WI; ++i) a0[i][kk] = read_a(0, 0, 0, i, kk);
  }

  auto quadrant = [&](floatx4_t(&d)[WI][WJ], const Operand(&a)[WI][2], const Operand(&b)[WJ][2], auto first, auto each) __attribute__((always_inline)) {
#pragma unroll
    for (int t = 0; t < Q; ++t) {
      if (t == Q / 2) first();
      const int u = t % (WI * WJ), kk = t / (WI * WJ);
      const int c = u / WI, i = (c & 1) ? WI - 1 - u % WI : u % WI;
      mfma_mx(d[i][c], b[c][kk].v, a[i][kk].v, b[c][kk].s, a[i][kk].s);
      each(t);
      if (t & 1) __builtin_amdgcn_sched_barrier(0);
    }
  };
  // the n reads or requests of half a quadrant, spread over its Q / 2 products (t = 0 .. Q / 2 - 1)
  auto spread = [&](int t, int n, auto op) __attribute__((always_inline)) {
#pragma unroll
    for (int x = 0; x < n; ++x)
      if (x * (Q / 2) / n == t) op(x);
  };
  auto nothing = []() __attribute__((always_inline)) {};
  auto step = [&](auto par_, int s) __attribute__((always_inline)) {
    constexpr int p = decltype(par_)::value, np = p ^ 1;
    const int pair = (s >> 1) & 1, next = p == 1 ? pair ^ 1 : pair;       // (pair of this step's scales, of the next step's)
    // what may still be on its way when half 1 of this step, then half 0 of the next, has to be there
    auto meet_first = [&]() __attribute__((always_inline)) {
      asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(2 * kReq + (p == 1 ? kMore : 0)) : "memory");
      __builtin_amdgcn_sched_barrier(0);
    };
    auto meet_second = [&]() __attribute__((always_inline)) {
      asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(2 * kReq + (p == 0 ? kMore : 0)) : "memory");
      __builtin_amdgcn_sched_barrier(0);
    };
    quadrant(acc[0][0], a0, b0, meet_first, [&](int t) __attribute__((always_inline)) {
      spread(t - Q / 2, 2 * WJ, [&](int x) __attribute__((always_inline)) { b1[x % WJ][x / WJ] = read_b(1, p, pair, x % WJ, x / WJ); });
      spread(t - Q / 2, kReq + (p == 0 ? kMore : 0), [&](int x) __attribute__((always_inline)) {
        if (x < kReq) request(s + 2, 0, 2 * p, x);
        else request_scales((s >> 1) + 1, x - kReq);
      });
    });
    quadrant(acc[0][1], a0, b1, nothing, [&](int t) __attribute__((always_inline)) {
      spread(t, 2 * WI, [&](int x) __attribute__((always_inline)) { a1[x % WI][x / WI] = read_a(1, p, pair, x % WI, x / WI); });
    });
    quadrant(acc[1][1], a1, b1, meet_second, [&](int t) __attribute__((always_inline)) {
      spread(t - Q / 2, 2 * WI, [&](int x) __attribute__((always_inline)) { a0[x % WI][x / WI] = read_a(0, np, next, x % WI, x / WI); });
      spread(t - Q / 2, kReq, [&](int x) __attribute__((always_inline)) { request(s + 2, 1, 2 * p + 1, x); });
    });
    quadrant(acc[1][0], a1, b0, nothing, [&](int t) __attribute__((always_inline)) {
      if (t % WI == WI - 1) b0[(t / WI) % WJ][t / (WI * WJ)] = read_b(0, np, next, (t / WI) % WJ, t / (WI * WJ));
    });
  };
  int s = 0;
  for (; s + 2 <= steps; s += 2) {
    step(std::integral_constant<int, 0>{}, s);
    step(std::integral_constant<int, 1>{}, s + 1);
  }
  if (s < steps) step(std::integral_constant<int, 0>{}, s);
  // the last products have to leave the pipe before their registers are read (the compiler does not see the asm's
  // latency), requests past the last step may still be writing LDS, and other waves may still be reading
  asm volatile("s_nop 15\n\ts_nop 15\n\ts_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");

  // store through LDS, whole tile rows at a time (fp32: half of them), row pitch = row + 32 bytes so that the rows spread over the banks;
  // 16 bytes per lane where the result's rows start at multiples of that, one value otherwise
  auto store = [&](auto type_) __attribute__((always_inline)) {
    typedef decltype(type_) T;
    constexpr int kPitch = BN * sizeof(T) + 32;
    constexpr int kPer16 = 16 / sizeof(T);
    constexpr int kLanesPerRow = BN / kPer16;
    constexpr int kPassHalves = sizeof(T) == 2 ? 2 : 1;
    constexpr int kRows = kPassHalves * (BM / 2);
    constexpr int kRowsPerInstr = 64 / kLanesPerRow;
    T *dp = static_cast<T *>(g.d);
    const bool whole = g.C % kPer16 == 0 && (reinterpret_cast<uintptr_t>(g.d) & 15) == 0;
#pragma unroll
    for (int pass = 0; pass < 2 / kPassHalves; ++pass) {
      if (pass > 0) __syncthreads();
#pragma unroll
      for (int hh = 0; hh < kPassHalves; ++hh)
#pragma unroll
        for (int q = 0; q < 2; ++q)
#pragma unroll
          for (int i = 0; i < WI; ++i)
#pragma unroll
            for (int c = 0; c < WJ; ++c) {
              const floatx4_t v = acc[pass * kPassHalves + hh][q][i][c];
              unsigned char *to = smem + (hh * (BM / 2) + wm * 16 * WI + i * 16 + r16) * kPitch + (q * (BN / 2) + wn * 16 * WJ + c * 16 + 4 * kq) * sizeof(T);
              if constexpr (sizeof(T) == 2) *reinterpret_cast<u32x2_t *>(to) = u32x2_t{pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3])};
              else *reinterpret_cast<floatx4_t *>(to) = v;
            }
      __syncthreads();
      if (whole) {
#pragma unroll
        for (int b = 0; b < kRows / (4 * kRowsPerInstr); ++b) {
          const int lrow = (b * 4 + wave) * kRowsPerInstr + lane / kLanesPerRow, chunk = lane % kLanesPerRow;
          const int64_t grow = row0 + pass * (BM / 2) + lrow, gcol = col0 + chunk * kPer16;
          const u32x4_t v = *reinterpret_cast<const u32x4_t *>(smem + lrow * kPitch + chunk * 16);
          if (grow < g.M && gcol < g.C) *reinterpret_cast<u32x4_t *>(dp + grow * g.C + gcol) = v;
        }
      } else {
        for (int at = threadIdx.x; at < kRows * BN; at += 256) {
          const int lrow = at / BN, col = at % BN;
          const int64_t grow = row0 + pass * (BM / 2) + lrow, gcol = col0 + col;
          if (grow < g.M && gcol < g.C) dp[grow * g.C + gcol] = *reinterpret_cast<const T *>(smem + lrow * kPitch + col * sizeof(T));
        }
      }
    }
  };
  if (g.d_dtype == CAIFX_BF16) store(bf16_t{});
  else if (g.d_dtype == CAIFX_F16) store(f16_t{});
  else store(float{});
}

// XCD x (workgroup id mod 8) walks the x-th contiguous eighth of a list that runs through bands of 1024 rows column by column.  A last round
// that fills less than half of the compute units is run as twice as many tiles of half the rows.
template <int WI, int WJ, bool kTail, bool kHalves> __global__ __launch_bounds__(256, WI + WJ <= 4 ? 2 : 1) void mx_gemm_kernel(MxGemmArgs g)
{
  constexpr int BM = 64 * WI, BN = 64 * WJ, kBand = kBandRows / BM;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  const int64_t col_tiles = (g.C + BN - 1) / BN, row_tiles = (g.M + BM - 1) / BM;
  const int64_t per_xcd = (row_tiles * col_tiles + 7) >> 3, whole = per_xcd - g.halved;
  int64_t at = blockIdx.x >> 3;
  const bool half = kHalves && at >= whole, lower = half && ((at - whole) & 1);
  if (half) at = whole + ((at - whole) >> 1);
  const int64_t pos = static_cast<int64_t>(blockIdx.x & 7) * per_xcd + at;
  if (pos >= row_tiles * col_tiles) return;
  const int64_t band = pos / (kBand * col_tiles);
  const int64_t within = pos - band * kBand * col_tiles;
  const int64_t left = row_tiles - band * kBand;
  const int64_t band_rows = left < kBand ? left : kBand;
  const int64_t col0 = (within / band_rows) * BN, row0 = (band * kBand + within % band_rows) * BM + (lower ? BM / 2 : 0);
  if constexpr (kHalves) {
    if (half) {
      if (row0 < g.M) mx_tile<WI / 2, WJ, kTail>(g, smem, row0, col0);
      return;
    }
  }
  mx_tile<WI, WJ, kTail>(g, smem, row0, col0);
}

// Scales [rows, blocks] of both operands as [rows / 64][groups][64][16]: the 16 bytes of a row that two steps need, 64 rows together, zeros
// (2^-127) for blocks and rows that there are not.
__global__ __launch_bounds__(256) void order_scales_kernel(const uint8_t *__restrict__ a, int64_t a_rows, const uint8_t *__restrict__ b, int64_t b_rows,
                                                           u32x4_t *__restrict__ out, int blocks, int groups)
{
  const int64_t a_pieces = (a_rows + 63) / 64 * groups * 64, pieces = a_pieces + (b_rows + 63) / 64 * groups * 64;
  const bool dwords = blocks % 4 == 0 && (reinterpret_cast<uintptr_t>(a) & 3) == 0 && (reinterpret_cast<uintptr_t>(b) & 3) == 0;
  for (int64_t at = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; at < pieces; at += static_cast<int64_t>(gridDim.x) * 256) {
    const bool second = at >= a_pieces;
    const int64_t in = second ? at - a_pieces : at, tile = in / (64 * groups);
    const int within = static_cast<int>(in - tile * 64 * groups), group = within >> 6;
    const int64_t row = tile * 64 + (within & 63);
    u32x4_t v = {0, 0, 0, 0};
    if (row < (second ? b_rows : a_rows)) {
      const uint8_t *from = (second ? b : a) + row * blocks + group * 16;
      const int left = blocks - group * 16;
#pragma unroll
      for (int d = 0; d < 4; ++d) {
        if (dwords) {
          if (4 * d < left) v[d] = *reinterpret_cast<const uint32_t *>(from + 4 * d);
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (4 * d + i < left) v[d] |= static_cast<uint32_t>(from[4 * d + i]) << (8 * i);
        }
      }
    }
    out[at] = v;
  }
}

template <int WI, int WJ, bool kTail, bool kHalves = false>
int launch_mx(const MxGemmArgs &g, hipStream_t s)
{
  constexpr int BM = 64 * WI, BN = 64 * WJ;
  constexpr int kRing = (BM + BN) * 256 + 2 * (BM + BN) * 16, kStore16 = BM * (BN * 2 + 32), kStore32 = BM / 2 * (BN * 4 + 32);
  constexpr int kStore = kStore16 > kStore32 ? kStore16 : kStore32;
  constexpr int kLds = kRing > kStore ? kRing : kStore;
  auto kern = mx_gemm_kernel<WI, WJ, kTail, kHalves>;
  static std::atomic<bool> raised{false};
  if (!raised.load(std::memory_order_relaxed)) {
    // the attribute is per kernel and sticky; two threads racing here both set it, which is harmless
    if (hipFuncSetAttribute(reinterpret_cast<const void *>(kern), hipFuncAttributeMaxDynamicSharedMemorySize, kLds) != hipSuccess)
      return CAIFX_ERR_LAUNCH_FAILED;
    raised.store(true, std::memory_order_relaxed);
  }
  const int64_t tiles = ((g.M + BM - 1) / BM) * ((g.C + BN - 1) / BN);
  hipLaunchKernelGGL(kern, dim3(static_cast<unsigned>(((tiles + 7) / 8 + g.halved) * 8), static_cast<unsigned>(g.parts)), dim3(256), kLds, s, g);
  return launch_status();
}

int64_t groups_of(int64_t blocks) { return (blocks + 15) / 16; }
int64_t scale_bytes(int64_t rows, int64_t blocks) { return (rows + 63) / 64 * groups_of(blocks) * 1024; }

}  // namespace

bool mx_gemm_takes(int64_t M, int64_t C, int64_t blocks)
{
  // (row offsets inside a tile have 32 bits; a grid has fewer than 2^31 workgroups)
  return blocks < (int64_t{1} << 17) && ((M + 127) / 128) * ((C + 127) / 128) <= (int64_t{1} << 30);
}

namespace {

// One workgroup of 256 x 256 per compute unit or two of 128 x 128: the large tile reads each operand half as often.  Few tiles and many steps: up
// to eight workgroups share a tile's steps, and a second launch adds their sums.  Measured with the scales' order, us, small / large / large with
// the last round halved: M = 4096, N = 14336, K = 4096 178 / 157 / 147; M = 1536 72 / 74 / 66; M = 512, N = K = 4096 17 / 34 / 23; small in one / four
// parts: M = 256, N = 4096, K = 14336 42 / 26, N = 14336, K = 4096 20 / 44.
struct MxPlan {
  bool large;
  int halved, parts;
  double us;
};
MxPlan mx_plan(int64_t M, int64_t C, int64_t blocks)
{
  const int64_t large = ((M + 255) / 256) * ((C + 255) / 256), small = ((M + 127) / 128) * ((C + 127) / 128);
  const int64_t steps = (blocks + 7) / 8;
  MxPlan best{};
  // us of a step: full rounds, and a last one that costs less the fewer tiles it has
  const auto rounds = [](int64_t tiles, int64_t slots, double full, double base, double per) {
    const int64_t rest = tiles % slots;
    return full * static_cast<double>(tiles / slots) + (rest == 0 ? 0.0 : base + per * static_cast<double>(rest));
  };
  const auto consider = [&](bool is_large, int halved, int parts, double step) {
    const double us = 9.0 + step * static_cast<double>((steps + parts - 1) / parts) + (parts > 1 ? 4.0 + 1.4e-6 * parts * static_cast<double>(M) * static_cast<double>(C) : 0.0);
    if (best.parts == 0 || us < best.us) best = MxPlan{is_large, halved, parts, us};
  };
  for (int parts = 1; parts <= 8 && (parts == 1 || steps >= 8 * parts); ++parts) {
    const int64_t t = small * parts;
    consider(false, 0, parts, t % 512 <= 256 ? rounds(t, 512, 1.35, 0.58, 0.0004) : rounds(t, 512, 1.35, 0.65, 0.0012));
    consider(true, 0, parts, rounds(large * parts, 256, 2.2, 1.3, 0.003));
  }
  const int64_t rest = (large + 7) / 8 % 32;
  if (rest > 0 && rest <= 16) consider(true, static_cast<int>(rest), 1, rounds((large + 7) / 8 * 8, 256, 2.2, 0.9, 0.0025));
  return best;
}

}  // namespace

double mx_gemm_us(int64_t M, int64_t C, int64_t blocks) { return mx_plan(M, C, blocks).us; }

size_t mx_gemm_workspace_bytes(int64_t M, int64_t C, int64_t blocks)
{
  const MxPlan p = mx_plan(M, C, blocks);
  return static_cast<size_t>(scale_bytes(M, blocks) + scale_bytes(C, blocks)) + (p.parts > 1 ? static_cast<size_t>(p.parts) * static_cast<size_t>(M) * static_cast<size_t>(C) * 4 : 0);
}

int mx_gemm(int64_t M, int64_t C, int64_t blocks, const void *a, const void *sa, const void *b, const void *sb, void *d, int d_dtype, void *workspace, hipStream_t s)
{
  const MxPlan p = mx_plan(M, C, blocks);
  MxGemmArgs g{};
  g.a = static_cast<const uint8_t *>(a);
  g.b = static_cast<const uint8_t *>(b);
  g.M = M;
  g.C = C;
  g.pitch = 16 * blocks;
  g.groups = static_cast<int>(groups_of(blocks));
  g.parts = p.parts;
  g.halved = p.halved;
  g.sa = static_cast<const uint8_t *>(workspace);
  g.sb = g.sa + scale_bytes(M, blocks);
  void *partial = static_cast<char *>(workspace) + scale_bytes(M, blocks) + scale_bytes(C, blocks);
  g.d = p.parts > 1 ? partial : d;
  g.d_dtype = p.parts > 1 ? static_cast<int>(CAIFX_F32) : d_dtype;
  const int64_t grid = (scale_bytes(M, blocks) + scale_bytes(C, blocks)) / 16 / 256;
  hipLaunchKernelGGL(order_scales_kernel, dim3(static_cast<unsigned>(grid < 1 ? 1 : grid < (1 << 20) ? grid : (1 << 20))), dim3(256), 0, s, static_cast<const uint8_t *>(sa), M,
                     static_cast<const uint8_t *>(sb), C, static_cast<u32x4_t *>(workspace), static_cast<int>(blocks), g.groups);
  const bool tail = blocks % 8 != 0;
  int st;
  if (p.halved) st = tail ? launch_mx<4, 4, true, true>(g, s) : launch_mx<4, 4, false, true>(g, s);
  else if (p.large) st = tail ? launch_mx<4, 4, true>(g, s) : launch_mx<4, 4, false>(g, s);
  else st = tail ? launch_mx<2, 2, true>(g, s) : launch_mx<2, 2, false>(g, s);
  return st != CAIFX_OK || p.parts == 1 ? st : join_sums(static_cast<const float *>(partial), p.parts, M * C, d, d_dtype, nullptr, s);
}

}  // namespace caifx
