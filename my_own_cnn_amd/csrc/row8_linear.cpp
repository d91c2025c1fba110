// Products of 8-bit rows with 8-bit weights (miq_row8_linear, miq_row8_experts):
//
//   y[m, j] = float(sum over i of x[m, i] * w[j, i]) * x_scale[m] * w_scale[j] + bias[j] + add[m, j]
//
// on v_mfma_i32_16x16x64_i8, by one of two kernels and in one of their tiles, whichever a model of their
// times gives as the fastest.
#include <algorithm>

#include "row8_internal.h"

namespace miq {
namespace {

struct Shape {
  bool few;
  int rows, channels;
};

// Tiles through LDS: us for a step of 64 codes of one workgroup that has its CU for itself, and of a CU that
// has many; us for a tile's output.
struct Tile {
  int rows, channels;
  double alone, each, output;
};
constexpr Tile kTiles[] = {{64, 64, 0.18, 0.13, 0.4},
                           {64, 128, 0.205, 0.21, 0.7},
                           {128, 128, 0.24, 0.31, 1.3},
                           {128, 256, 0.36, 0.57, 2.5},
                           {256, 256, 0.55, 0.84, 7}};
// Rows that do not start on 16 bytes go through registers.
constexpr double kThroughRegisters = 1.5;
// Few rows: bound by what a CU takes in, 38 KB a us (21 where rows do not start on 4 bytes); us for a tile's
// sums beyond the first two of a CU.
struct Few {
  int rows, channels;
  double sums;
};
constexpr Few kFew[] = {{16, 16, 0.7}, {16, 32, 1.4}, {32, 16, 0.85}, {32, 32, 1.1}, {64, 32, 2.6}};
constexpr double kIntake = 38e3, kOddIntake = 21e3, kLaunch = 3.5;

Shape shape_of(int64_t rows, int64_t c, int64_t k, int64_t experts) {
  const auto over = [](int64_t n, int64_t by) { return (n + by - 1) / by; };
  // experts: as if all that can have rows had as many
  const int64_t groups = std::min(rows, experts), part = over(rows, groups);
  // what no kernel is faster than: the weights read and y written
  const double bytes = (static_cast<double>(groups) * k * c + 2.6 * rows * k) / 4.6e6;
  Shape best{};
  double least = 0.0;
  const auto take = [&](const Shape& s, double us) {
    us = std::max(us, bytes);
    if (best.rows == 0 || us < least) {
      best = s;
      least = us;
    }
  };
  for (const Few& t : kFew) {
    const int64_t tiles = groups * over(part, t.rows) * over(k, t.channels), rounds = over(tiles, 256);
    const double in = static_cast<double>(std::min<int64_t>(part, t.rows) + t.channels) * c;
    take({true, t.rows, t.channels},
         kLaunch + rounds * in / (c % 4 == 0 ? kIntake : kOddIntake) + std::max<int64_t>(rounds - 2, 0) * t.sums);
  }
  const double steps = static_cast<double>(over(c, 64)) * (c % 16 == 0 ? 1.0 : kThroughRegisters);
  for (const Tile& t : kTiles) {
    if (c < 16 || (t.rows == 256 && c % 16 != 0)) continue;
    // of experts the last row tile is half full
    const double high = groups == 1 ? over(part, t.rows) : std::max(1.0, static_cast<double>(part) / t.rows + 0.5);
    const int64_t tiles = static_cast<int64_t>(groups * high) * over(k, t.channels), rounds = over(tiles, 256);
    take({false, t.rows, t.channels}, kLaunch + steps * std::max(t.alone, t.each * rounds) + t.output * rounds);
  }
  return best;
}

}  // namespace

void plan_row8_linear(int32_t rows, int32_t c, int32_t k, int32_t experts, int32_t plan[3]) {
  const Shape s = shape_of(rows, c, k, experts);
  plan[0] = s.few;
  plan[1] = s.rows;
  plan[2] = s.channels;
}

hipError_t launch_row8_linear(const Row8LinearArgs& a, hipStream_t stream) {
  Row8LinearArgs b = a;
  if (b.x_rows == 0) b.c = 0;  // every row stands for zeros
  const Shape s = shape_of(b.rows, b.c, b.k, b.experts);
  return s.few ? launch_row8_few(b, s.rows, s.channels, stream) : launch_row8_tile(b, s.rows, s.channels, stream);
}

}  // namespace miq
