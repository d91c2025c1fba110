// What the int8 product kernels of 8-bit rows share: problems and their tiles, the output stage.
#pragma once

#include "row8_device.h"

namespace miq {
namespace {

typedef v4i v4i_any __attribute__((aligned(1)));

// Rows [row0, end) of y, at most a tile of them, by the weights of `expert`; expert < 0: no such tile.
struct RowTile {
  int expert, row0, end;
};

// Tile number `tile` of the experts' row tiles of `high` rows, in their order: every wave looks for it by
// itself, 64 experts at a time.  Offsets are held to 0 .. rows and to rising order.
__device__ __forceinline__ RowTile find_tile(const int32_t* offsets, int experts, int rows, int high, int tile) {
  const int lane = static_cast<int>(threadIdx.x) & 63;
  for (int base = 0; base < experts; base += 64) {
    const int e = min(base + lane, experts - 1);
    const int lo = min(max(offsets[e], 0), rows);
    const int hi = min(max(offsets[e + 1], lo), rows);
    const int count = base + lane < experts ? (hi - lo + high - 1) / high : 0;
    int upto = count;  // this expert's tiles and those before it
    for (int step = 1; step < 64; step *= 2) {
      const int other = __shfl_up(upto, step);
      if (lane >= step) upto += other;
    }
    const uint64_t past = __ballot(upto > tile);
    if (past != 0) {
      const int at = __builtin_ctzll(past);
      const int row0 = __shfl(lo, at) + (tile - (__shfl(upto, at) - __shfl(count, at))) * high;
      const int end = min(__shfl(hi, at), row0 + high);
      return {__builtin_amdgcn_readfirstlane(base + at), __builtin_amdgcn_readfirstlane(row0),
              __builtin_amdgcn_readfirstlane(end)};
    }
    tile -= __shfl(upto, 63);
  }
  return {-1, 0, 0};
}

// The most row tiles that rows in `experts` groups can have.
inline int64_t most_tiles(int64_t rows, int64_t experts, int64_t high) {
  const int64_t parts = rows / high + experts;
  return parts < rows ? parts : rows;
}

// A value of y: the sum of the codes' products, exact in 32 bits, is rounded once to fp32, then times
// the row's and the channel's scale.
__device__ __forceinline__ float scaled(int sum, float x_scale, float w_scale) {
  return static_cast<float>(sum) * x_scale * w_scale;
}

}  // namespace
}  // namespace miq
