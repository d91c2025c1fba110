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

// An expert's rows, held to 0 .. rows and to rising order, and its row tiles of `high` rows.
struct ExpertRows {
  int lo, hi, tiles;
};
__device__ __forceinline__ ExpertRows expert_rows(const int32_t* offsets, int experts, int rows, int high, int expert) {
  const int e = min(expert, experts - 1);
  const int lo = min(max(offsets[e], 0), rows);
  const int hi = min(max(offsets[e + 1], lo), rows);
  return {lo, hi, expert < experts && hi > lo ? (hi - lo - 1) / high + 1 : 0};
}

// All experts' row tiles; every wave counts them by itself, 64 experts at a time.
__device__ __forceinline__ int count_tiles(const int32_t* offsets, int experts, int rows, int high) {
  int count = 0;
  for (int base = 0; base < experts; base += 64)
    count += expert_rows(offsets, experts, rows, high, base + (static_cast<int>(threadIdx.x) & 63)).tiles;
  for (int step = 1; step < 64; step *= 2) count += __shfl_xor(count, step);
  return __builtin_amdgcn_readfirstlane(count);
}

// Tile number `tile` of the experts' row tiles, in their order.
__device__ __forceinline__ RowTile find_tile(const int32_t* offsets, int experts, int rows, int high, int tile) {
  const int lane = static_cast<int>(threadIdx.x) & 63;
  for (int base = 0; base < experts; base += 64) {
    const ExpertRows e = expert_rows(offsets, experts, rows, high, base + lane);
    int upto = e.tiles;  // this expert's tiles and those before it
    for (int step = 1; step < 64; step *= 2) {
      const int other = __shfl_up(upto, step);
      if (lane >= step) upto += other;
    }
    const uint64_t past = __ballot(upto > tile);
    if (past != 0) {
      const int at = __builtin_ctzll(past);
      // Uniform before the branch: a tile whose rows might differ by lane puts every load of the product in a loop.
      const int first = __builtin_amdgcn_readfirstlane(__shfl(e.lo, at));
      const int last = __builtin_amdgcn_readfirstlane(__shfl(e.hi, at));
      const int before = __builtin_amdgcn_readfirstlane(__shfl(upto, at) - __shfl(e.tiles, at));
      const int row0 = first + (__builtin_amdgcn_readfirstlane(tile) - before) * high;
      if (row0 < first || row0 >= last) return {-1, 0, 0};  // only where offsets fall
      return {base + at, row0, last - row0 < high ? last : row0 + high};
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

// 16 codes at p, which starts on 4 bytes or (ODD) anywhere: 16-byte loads run at their rate from multiples
// of 4 and at a third of it from other addresses, so there the dwords that hold the codes are loaded and
// shifted.  These dwords each hold a code, so none lies in another page than the codes.
template <bool ODD>
__device__ __forceinline__ v4i load16(const int8_t* p) {
  if constexpr (!ODD) {
    return *reinterpret_cast<const v4i_any*>(p);
  } else {
    typedef v4i v4i_dwords __attribute__((aligned(4)));
    const unsigned by = static_cast<unsigned>(reinterpret_cast<uintptr_t>(p)) & 3;
    const v4i v = *reinterpret_cast<const v4i_dwords*>(p - by);
    const int8_t* const end = p + 15;
    const int e = *reinterpret_cast<const int*>(end - (reinterpret_cast<uintptr_t>(end) & 3));
    return v4i{static_cast<int>(__builtin_amdgcn_alignbyte(v[1], v[0], by)),
               static_cast<int>(__builtin_amdgcn_alignbyte(v[2], v[1], by)),
               static_cast<int>(__builtin_amdgcn_alignbyte(v[3], v[2], by)),
               static_cast<int>(__builtin_amdgcn_alignbyte(e, v[3], by))};
  }
}

// 16 codes of a row of c at channel `at`, zeros past the row's end: there, the row's last 16 codes shifted
// down, or, of a row shorter than that, code by code.
__device__ __forceinline__ v4i load_codes16(const int8_t* row, int at, int c) {
  const int left = c - at;
  if (left >= 16) return *reinterpret_cast<const v4i_any*>(row + at);
  if (left <= 0) return v4i{};
  if (c >= 16) {
    const v4i last = *reinterpret_cast<const v4i_any*>(row + c - 16);
    return __builtin_bit_cast(v4i, __builtin_bit_cast(unsigned __int128, last) >> (8 * (16 - left)));
  }
  v4i v = {};
#pragma unroll
  for (int i = 0; i < 16; ++i)
    if (i < left) v[i / 4] |= (row[at + i] & 0xff) << (8 * (i & 3));
  return v;
}

// Whether rows of codes start on multiples of `to` bytes.
inline bool codes_on(const Row8LinearArgs& a, int to) {
  return a.c % to == 0 && reinterpret_cast<uintptr_t>(a.x) % to == 0 && reinterpret_cast<uintptr_t>(a.w) % to == 0;
}

// A value of y: the sum of the codes' products, exact in 32 bits, is rounded once to fp32, then times
// the row's and the channel's scale.
__device__ __forceinline__ float scaled(int sum, float x_scale, float w_scale) {
  return static_cast<float>(sum) * x_scale * w_scale;
}

// The first `left` (at most W) of W floats, zeros after them.
template <int W>
__device__ __forceinline__ typename Vec<W>::type load_floats(const float* p, int left) {
  if constexpr (W == 8) {
    return load8_of(p, left);
  } else {
    if (left >= 4) return load4(p);
    v4f v = {};
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < left) v[i] = p[i];
    return v;
  }
}

// Four values of a row of y at any address.
__device__ __forceinline__ void store_four(float* p, const v4f& v) { store_run<false>(p, v); }
__device__ __forceinline__ void store_four(__bf16* p, const v4f& v) {
  *reinterpret_cast<v4bf_any*>(p) = __builtin_convertvector(v, v4bf);  // to nearest even
}

}  // namespace
}  // namespace miq
