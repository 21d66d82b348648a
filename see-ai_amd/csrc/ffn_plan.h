// ffn_plan.h -- which tile a product of the feed-forward block (k_ffn.hip) runs
// on, and over how many workgroups its K is shared out.  Plain C++ without HIP,
// so the rule runs where there is no GPU.
#pragma once

#include <algorithm>
#include <cmath>
#include <cstddef>
#include <initializer_list>

namespace seeai::ffn {

// How a launch runs: its tile, and over how many workgroups the K of the tiles
// past `whole` is shared out.
struct Plan {
  int tile = 0;  // of kTiles
  int tiles = 0, whole = 0, splits = 1, per_split = 0;
};
struct TileShape {
  int rows, cols, rows_dual, cols_dual, per_cu;  // output's; workgroups a CU holds
  int bm(bool dual) const { return dual ? rows_dual : rows; }
  int bn(bool dual) const { return dual ? cols_dual : cols; }
  // us of a stage of one product and of two side by side: on an idle chip, and
  // more for every workgroup a CU holds.
  double alone, shared, alone_dual, shared_dual;
};
// bf16, fitted to some 600 timings (K shared out over 1 to 32, 39 products from
// 1 x 5632 x 2048 to 8192 x 2048 x 5632), mean error 12 %; the tile and sharing
// it picks were within 6 % of the best on average (16 % the worst that was no
// outlier).  Few tokens take the 64-row tile with K shared out -- 24 x 2048 x
// 5632: 10 us over 8, 25 us over 1, 95 us on 256 x 256 -- many the 256 x 256:
// 8192 x 2048 x 11264 333 us against 443 on 128 x 128.
constexpr TileShape kTiles[3] = {{256, 256, 256, 128, 1, 1.07, 0.37, 1.11, 0.43},
                                 {128, 128, 128, 64, 2, 0.47, 0.21, 0.58, 0.24},
                                 {64, 64, 64, 64, 2, 0.18, 0.10, 0.27, 0.29}};
// f32, stages of 32 with all three planes of each operand in LDS, fitted to 490
// timings (K shared out over 1 to 16, ten blocks from 150 x 128 x 512 to 200 x
// 2048 x 5632), mean error 15 %.  dW of 1001 x 776 x 2048: 73 us (103 with a
// stage a plane product on 128 x 128 x 64, which loads each plane twice).
constexpr TileShape kTiles32[2] = {{256, 128, 128, 128, 1, 1.5, 1.5, 1.44, 1.5},
                                   {64, 128, 64, 64, 2, 0.56, 0.52, 0.68, 0.55}};
constexpr int Deep(bool f32) { return f32 ? 32 : 64; }
inline const TileShape& ShapeOf(bool f32, int tile) { return f32 ? kTiles32[tile] : kTiles[tile]; }
constexpr size_t kMostPart = size_t{64} << 20;  // bytes of shared-out sums
struct Shape {
  size_t M, N;
};
// Either every tile's K is shared out, or, with more tiles than the chip holds
// at once, that of the tiles left over after whole rounds: 528 tiles of the
// weights' gradients run as two rounds and a sixteenth instead of three.
inline Plan Choose(bool f32, bool dual, std::initializer_list<Shape> products, size_t K, int nseg) {
  const double stages = static_cast<double>((K + Deep(f32) - 1) / Deep(f32)) * nseg;
  Plan best;
  double least = 1e30;
  for (int t = 0; t < (f32 ? 2 : 3); ++t) {
    const TileShape& s = ShapeOf(f32, t);
    const int bm = s.bm(dual), bn = s.bn(dual);
    const double alone = dual ? s.alone_dual : s.alone, shared = dual ? s.shared_dual : s.shared;
    const double tile_bytes = bm * bn * (dual ? 2 : 1) * 4.0, chip = 256.0 * s.per_cu;
    double tiles = 0;
    for (const Shape& q : products)
      tiles += std::ceil(static_cast<double>(q.M) / bm) * std::ceil(static_cast<double>(q.N) / bn);
    // us of `wgs` workgroups of `per` stages.
    auto run = [&](double wgs, double per) {
      return std::ceil(wgs / chip) * per * (alone + std::min<double>(s.per_cu, wgs / 256.0) * shared);
    };
    const double full = std::floor(tiles / chip) * chip;
    for (double whole : {0.0, full}) {
      const double rest = tiles - whole;
      if (whole > 0 && rest == 0) continue;
      for (int k : {1, 2, 3, 4, 6, 8, 12, 16, 24, 32}) {
        if (whole > 0 && k == 1) continue;  // the same as sharing nothing out
        if (k > 1 && (k * 2 > stages || k * rest * tile_bytes > kMostPart)) break;
        const double per = std::ceil(stages / k), n = std::ceil(stages / per);
        double us = (whole > 0 ? run(whole, stages) : 0) + run(rest * n, per) + 7;
        if (k > 1) us += 1 + 0.1 * k + k * rest * tile_bytes * 2 / 5.5e6;
        if (us < least) {
          least = us;
          best = {t, static_cast<int>(tiles), static_cast<int>(k == 1 ? tiles : whole),
                  static_cast<int>(n), static_cast<int>(per)};
        }
      }
      if (full == 0) break;
    }
  }
  return best;
}

}  // namespace seeai::ffn
