// Tiles and shares of the dense product (caifx_gemm_wide.hip), and what it takes (host only).
#pragma once

#include <cstdint>

namespace caifx {

constexpr int kWideStep = 64;              // reduction extent of a step

// What a 64-deep step of the whole launch costs with one of the three tiles, in us: the number of rounds the tiles take
// times the time of one, measured on N(0,1) x N(0,0.02) bf16 values at R = 4096.  256 x 256 (one workgroup per compute
// unit) 1.39 per round of 256, 128 x 256 (one) 0.87, 128 x 128 (two) 0.91 per round of 512 and 0.49 for a last round of
// at most 256.  M = 4096, C = 11008: 265 / 300 / 300 us; M = 2048, C = 11008: 166 / 149 / 162; M = 1024, C = 4096: 72 /
// 44 / 32.
enum { TILE_256 = 0, TILE_128x256 = 1, TILE_128 = 2 };
// row tiles of bm rows; over expert segments of unknown lengths the last tile of each is taken as half full
inline int64_t row_tiles_of(int64_t M, int experts, int64_t bm)
{
  if (experts == 0) return (M + bm - 1) / bm;
  const int64_t t = (M + bm - 1) / bm + experts / 2, least = M < experts ? M : experts;
  return t > least ? t : least;
}
// parts: workgroups that share a tile's steps
inline double step_cost(int tile, int64_t M, int64_t C, int experts, int parts)
{
  const auto tiles = [&](int64_t bm, int64_t bn) { return row_tiles_of(M, experts, bm) * ((C + bn - 1) / bn) * parts; };
  if (tile == TILE_256) return 1.39 * static_cast<double>((tiles(256, 256) + 255) / 256);
  if (tile == TILE_128x256) return 0.87 * static_cast<double>((tiles(128, 256) + 255) / 256);
  const int64_t t = tiles(128, 128), rest = t % 512;
  return 0.91 * static_cast<double>(t / 512) + (rest == 0 ? 0.0 : rest <= 256 ? 0.49 : 0.91);
}
inline int best_tile(int64_t M, int64_t C, int experts, int parts = 1)
{
  int best = TILE_256;
  for (int t = TILE_128x256; t <= TILE_128; ++t)
    if (step_cost(t, M, C, experts, parts) < step_cost(best, M, C, experts, parts)) best = t;
  return best;
}

// A partly filled round costs less than a full one: `base` + `per` for each of its tiles.
inline double rounds_cost(int64_t tiles, int64_t slots, double full, double base, double per)
{
  const int64_t rest = tiles % slots;
  return full * static_cast<double>(tiles / slots) + (rest == 0 ? 0.0 : base + per * static_cast<double>(rest));
}
inline double wide_us_of(int64_t M, int64_t C, int64_t R, int parts = 1)      // the product alone
{
  const auto tiles = [&](int64_t bm, int64_t bn) { return (M + bm - 1) / bm * ((C + bn - 1) / bn) * parts; };
  double step;
  switch (best_tile(M, C, 0, parts)) {
    case TILE_256: step = rounds_cost(tiles(256, 256), 256, 1.42, 0.75, 0.0026); break;
    case TILE_128x256: step = rounds_cost(tiles(128, 256), 256, 0.81, 0.25, 0.0022); break;
    default: {
      const int64_t t = tiles(128, 128);
      step = t % 512 <= 256 ? rounds_cost(t, 512, 0.82, 0.24, 0.0008) : rounds_cost(t, 512, 0.82, 0.30, 0.0010);
    }
  }
  return step * static_cast<double>((R / kWideStep + parts - 1) / parts);
}

// into how many parts a product that is not gated is best cut, and what it takes with their joining, in us, estimated
struct WideParts {
  int parts;
  double us;
};
// Few tiles and many steps: up to eight workgroups share a tile's steps, each at least eight of them, and a second launch adds their sums.
// us in one part / in the best, with the copies before it: M = 512, C = 4096, R = 14336 126 / 105, in fp32 (three times the steps) 291 / 200; M = 2048,
// C = 4096, R = 22016 (a gated block's gradient) 418 / 387; M = 1024, C = R = 4096 48 / 59, not taken.
inline WideParts wide_parts(int64_t M, int64_t C, int64_t R)
{
  WideParts best{1, wide_us_of(M, C, R)};
  for (int parts = 2; parts <= 8 && R / kWideStep >= 8 * parts; ++parts) {
    const double us = wide_us_of(M, C, R, parts) + 4.0 + 1.4e-6 * parts * static_cast<double>(M) * static_cast<double>(C);
    if (us < best.us) best = WideParts{parts, us};
  }
  return best;
}

}  // namespace caifx
