// How xv_mxfp4_gemm cuts a product, as rules over sizes (host code without HIP:
// a test asks them which kernels its shapes reach).
#pragma once
#include <algorithm>
#include <cmath>

constexpr int kFp4Waves = 8;  // waves of a workgroup
constexpr int kShort = 64;    // rows of x up to which the per-wave rings take a product, the shared tiles above
constexpr int kMaxM = 7;      // shared tiles: column tiles per wave at most (224 rows of x)

// How a product of up to kShort rows is cut: tiles per workgroup, parts of K.
// The cheapest by cycles, a workgroup per CU at a time.  Up to 16 rows a
// workgroup costs its tiles and its start and end, about one and a half tiles.
// Of more, it costs what goes through its LDS-DMA, about 40 bytes a cycle, most
// of it x: more tiles on parts of K read less of that, where it pays for the second
// kernel (64 rows through 4096 x 12288 17.6 us against 23.2 with K whole, 32 rows
// 13.6 against 14.8; through 4096 x 4096 K stays whole, 11.5).
struct ShortPlan { int tiles, parts; };
inline ShortPlan short_plan(int m, int rows, int k, bool silu) {
  const int tiles = (rows / (silu ? 2 : 1) + 15) / 16 * (silu ? 2 : 1);
  const int xr = (m + 15) / 16 * 16;  // rows of x that are fetched
  ShortPlan best = {silu ? 2 : 1, 1};
  double cost = 1e300;
  for (int t : {1, 2, 4, 6}) {
    if (silu && t % 2) continue;
    const int groups = (tiles + t - 1) / t;
    if (m <= 16) {
      const double c = ((groups + 255) / 256) * (t + 1.5);
      if (c <= cost) { cost = c; best = {t, 1}; }
      continue;
    }
    for (int parts : {1, 2, 4, 8}) {
      if (parts > 1 && k / parts < 128 * kFp4Waves) break;
      const double bytes = (double)k / parts * (2 * xr + t * 8.5);
      double c = std::ceil((double)groups * parts / 256) * (bytes / 40 + 6000);
      if (parts > 1) c += 8000 + (double)parts * m * rows * 8 / 2000;
      if (c <= cost) { cost = c; best = {t, parts}; }
    }
  }
  return best;
}

// How a product of more than kShort rows is cut: column tiles per wave, row
// tiles of the weight per wave, parts of K.  The cheapest by cycles: a step costs its
// matrix instructions (16 cycles each, two waves a SIMD) or its x through
// LDS-DMA (about 40 bytes a cycle), a workgroup about 8000 more at its ends, parts
// their second kernel and the traffic between.
struct TilePlan { int mtw, nt, parts; };
inline TilePlan tile_plan(int m, int rows, int k, bool silu) {
  const int gy = (m + 32 * kMaxM - 1) / (32 * kMaxM);
  const int mtw = std::max(3, ((m + gy - 1) / gy + 31) / 32);
  const int steps = (k + 127) / 128;
  TilePlan best = {mtw, 4, 1};
  double cost = 1e300;
  for (int nt : {4, 2, 1}) {
    if (silu && nt == 1) continue;
    for (int parts : {1, 2, 3, 4, 6, 8, 12, 16}) {
      if (parts > 1 && steps / parts < 4) break;
      const double groups = (double)((rows + 64 * nt - 1) / (64 * nt)) * ((m + 32 * mtw - 1) / (32 * mtw)) * parts;
      const double step = std::max(128.0 * nt * mtw, 200.0 * mtw) + 700.0;
      double c = std::ceil(groups / 256) * ((steps + parts - 1) / parts * step + 8000.0);
      if (parts > 1) c += 7000.0 + (double)parts * m * rows * 8.0 / 2000.0;
      if (c < cost) { cost = c; best = {mtw, nt, parts}; }
    }
  }
  return best;
}
