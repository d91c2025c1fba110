// Products of 8-bit rows with 8-bit weights (miq_row8_linear, miq_row8_experts):
//
//   y[m, j] = float(sum over i of x[m, i] * w[j, i]) * x_scale[m] * w_scale[j] + bias[j] + add[m, j]
//
// on v_mfma_i32_16x16x64_i8, by one of two kernels and in one of their tiles, whichever a model of their
// times gives as the fastest: on 600 problems spread over rows, c, k and experts its choice took 3% longer
// than the fastest of all on average, 46% at most.
#include <algorithm>

#include "row8_internal.h"

namespace miq {
namespace {

struct Shape {
  bool few, pad;
  int rows, channels;
};

// Tiles through LDS: us for a step of 128 codes of one workgroup that has its CU for itself, and of a CU that
// has many; us for a tile's output.
struct Tile {
  int rows, channels;
  double alone, each, output;
};
constexpr Tile kTiles[] = {{64, 64, 0.17, 0.19, 0.4},
                           {64, 128, 0.275, 0.31, 0.7},
                           {128, 128, 0.44, 0.5, 1.3},
                           {128, 256, 0.61, 0.94, 2.5},
                           {256, 256, 1.1, 1.5, 7}};
// Rows that do not start on 16 bytes go through registers, or are first copied to rows of whole lines in the
// workspace, which takes a launch and moves them twice: 1003 x 2051 x 1537 19.7 us and 16.6, 4096 x 1023 x 4096
// 43 and 32, 8192 x 8193 x 8192 805 and 446.
constexpr double kThroughRegisters = 2.5, kCopy = 3, kCopyRate = 3.2e6;
// Few rows: bound by what a CU takes in, 38 KB a us (21 where rows do not start on 4 bytes); us for a tile's
// sums beyond the first two of a CU.
struct Few {
  int rows, channels;
  double sums;
};
constexpr Few kFew[] = {{16, 16, 1.85}, {16, 32, 1.4}, {32, 16, 2.4}, {32, 32, 1.9}, {64, 32, 2.6}};
constexpr double kIntake = 38e3, kOddIntake = 21e3, kLaunch = 3.5;

Shape shape_of(int64_t x_rows, int64_t rows, int64_t c, int64_t k, int64_t experts) {
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
    take({true, false, t.rows, t.channels},
         kLaunch + rounds * in / (c % 4 == 0 ? kIntake : kOddIntake) + std::max<int64_t>(rounds - 2, 0) * t.sums);
  }
  if (c < 16) return best;
  const double steps = static_cast<double>(over(c, 128));
  const double copied = 2.0 * (x_rows + static_cast<double>(experts) * k) * c;
  for (const Tile& t : kTiles) {
    // of experts the last row tile is half full
    const double high = groups == 1 ? over(part, t.rows) : std::max(1.0, static_cast<double>(part) / t.rows + 0.5);
    const int64_t rounds = over(static_cast<int64_t>(groups * high) * over(k, t.channels), 256);
    const double each = steps * std::max(t.alone, t.each * rounds), rest = kLaunch + t.output * rounds;
    if (c % 16 == 0) {
      take({false, false, t.rows, t.channels}, each + rest);
    } else {
      if (t.rows != 256) take({false, false, t.rows, t.channels}, kThroughRegisters * each + rest);
      take({false, true, t.rows, t.channels}, each + rest + kCopy + copied / kCopyRate);
    }
  }
  return best;
}

// Codes of a copied row.
int64_t padded(int64_t c) { return (c + 127) / 128 * 128; }

}  // namespace

void plan_row8_linear(int32_t rows, int32_t c, int32_t k, int32_t experts, int32_t plan[4]) {
  const Shape s = shape_of(rows, rows, c, k, experts);
  plan[0] = s.few;
  plan[1] = s.rows;
  plan[2] = s.channels;
  plan[3] = s.pad;
}

size_t row8_workspace_bytes(int32_t x_rows, int32_t rows, int32_t c, int32_t k, int32_t experts) {
  if (x_rows == 0 || !shape_of(x_rows, rows, c, k, experts).pad) return 0;
  return static_cast<size_t>((x_rows + static_cast<int64_t>(experts) * k) * padded(c));
}

hipError_t launch_row8_linear(const Row8LinearArgs& a, hipStream_t stream) {
  Row8LinearArgs b = a;
  if (b.x_rows == 0) b.c = 0;  // every row stands for zeros
  const Shape s = shape_of(b.x_rows, b.rows, b.c, b.k, b.experts);
  if (s.pad) {
    const int64_t weights = static_cast<int64_t>(b.experts) * b.k;
    int8_t* const to = static_cast<int8_t*>(a.ws);
    const int32_t width = static_cast<int32_t>(padded(a.c));
    const hipError_t e = launch_row8_pad(a.x, a.x_rows, a.w, weights, a.c, width, to, stream);
    if (e != hipSuccess) return e;
    b.x = to;
    b.w = to + static_cast<int64_t>(a.x_rows) * width;
    b.c = width;
  }
  return s.few ? launch_row8_few(b, s.rows, s.channels, stream) : launch_row8_tile(b, s.rows, s.channels, stream);
}

}  // namespace miq
