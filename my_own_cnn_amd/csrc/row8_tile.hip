// Products of 8-bit rows with 8-bit weights in tiles held by LDS (row8_linear.cpp has the formula).
//
// A workgroup computes BM rows by BN channels of y, 128 codes of the reduction a step: whole lines of the
// caches.  Both operands lie in LDS as rows of 128 bytes, STAGES steps of them; a step's bytes travel
// straight from global memory to LDS (DMA), or, where rows do not start on 16 bytes, through registers.  A
// wave reads the fragments of the next half step while its matrix instructions run on this half, and meets
// the others once a step.
//
// 16384 x 4096 x 8192 on 256-square tiles 464 us, 2370 TOP/s, 8192 cubed 420 us, 2620 (a library product of
// the same codes to int32: 488 and 510 us): bound by the power that the matrix instructions draw (1.5 to 1.9 GHz,
// the matrix units busy 54 to 67% of the cycles).  What it took, for 16384 x 4096 x 8192 in us: 64-square tiles
// through registers 1342; 256-square tiles in steps of 64 codes straight to LDS 503 to 525; whole lines, half as many
// requests to the L2 478; rows of y written whole 464.  32 x 32 x 32 matrix instructions 639 (they draw more for
// the same product), four waves of 128 x 128 596, a workgroup that goes from tile to tile with the next one's
// loads ahead of its output 537.  Few tiles are bound by the loads' latency: 64 rows by 8192 x 4096 on two buffers
// 16.5 us, on four 9.0.
#include <algorithm>

#include "row8_product.h"

namespace miq {
namespace {

constexpr int kStep = 128;  // codes, and bytes of a row of LDS

struct Tiling {
  int from, high, wide;  // the launch's first row tile and their number (the most, of experts), channel tiles
};

// The 16-byte units of a row of LDS are permuted by its number: an LDS read serves in one cycle the lanes
// 0-3, 12-15, 20-23, 24-27 of a half-wave or the other 16, that is of a fragment the rows 0-3 and 12-15 at one
// unit and 4-11 at the next one, or the other way round, and these lie in different banks.
__device__ __forceinline__ int unit(int row, int at) { return at ^ ((row >> 1) & 7); }

// The channel in row p of LDS.  Matrix instruction f of a group of 64 rows of LDS leaves its rows 4q .. 4q + 3
// in lane group q: for 16-byte stores whose four lanes lie side by side a lane's channels are 8q .. 8q + 7 of
// 32 (bf16, of two instructions), or 4q .. 4q + 3 of 16.
template <typename T>
__device__ __forceinline__ int channel_of(int p) {
  if constexpr (sizeof(T) == 4) return p;
  return (p & ~31) + ((p >> 2) & 3) * 8 + ((p >> 4) & 1) * 4 + (p & 3);
}

// Tile `id` of a launch: tiles go in bands of eight rows of tiles, so that neighbours share their rows and
// channels in an L2.  Experts' tiles are dealt to the XCDs by their real number (`high` row tiles), not by
// the most that the launch allows for.
struct Place {
  RowTile r;
  int n0;
};
template <int BM, int BN>
__device__ __forceinline__ Place place_of(const Row8LinearArgs& a, const Tiling& tiling, int high, int id) {
  constexpr int kBand = 8;
  const int at = xcd_tile(id, high * tiling.wide);
  const int band = at / (kBand * tiling.wide);
  const int band_high = min(kBand, high - band * kBand);
  const int in = at - band * kBand * tiling.wide;
  const int row_tile = tiling.from + band * kBand + in % band_high, n0 = in / band_high * BN;
  if (a.offsets != nullptr) return {find_tile(a.offsets, a.experts, a.rows, BM, row_tile), n0};
  return {{0, row_tile * BM, a.rows - row_tile * BM < BM ? a.rows : (row_tile + 1) * BM}, n0};
}
template <int BM>
__device__ __forceinline__ int row_tiles(const Row8LinearArgs& a, const Tiling& tiling) {
  if (a.offsets == nullptr) return tiling.high;
  return min(tiling.high, count_tiles(a.offsets, a.experts, a.rows, BM) - tiling.from);
}

template <typename T, bool DMA, int BM, int BN, int WM, int WN, int STAGES, bool STREAM>
__global__ __launch_bounds__(WM* WN * 64, 2) void row8_tile_kernel(Row8LinearArgs a, Tiling tiling) {
  constexpr int kWaves = WM * WN;
  constexpr int NX = BM / 8 / kWaves, NW = BN / 8 / kWaves;  // runs of 8 rows that a wave stages
  constexpr int kStage = (BM + BN) * kStep;
  constexpr int FM = BM / WM / 16, FN = BN / WN / 16;  // a wave's fragments
  static_assert(NX >= 1 && NW >= 1 && FN % 2 == 0 && (DMA || STAGES == 2), "whole runs and groups of 32 channels");
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);

  const int high = row_tiles<BM>(a, tiling);
  if (static_cast<int>(blockIdx.x) >= high * tiling.wide) return;
  const Place place = place_of<BM, BN>(a, tiling, high, blockIdx.x);
  const RowTile r = place.r;
  if (r.expert < 0) return;
  const int n0 = place.n0, rows = r.end - r.row0, channels = min(BN, a.k - n0);

  // The output stage takes U runs of a lane's channels of each row, W values each.  Its scales are loaded first,
  // where registers are left for them.
  constexpr int W = kWide<T>, U = FN * 4 / W;
  constexpr bool kEarly = FM * FN < 32;
  const int wm = wave / WN, wn = wave % WN;
  const int f_row = lane & 15, f_at = lane >> 4;
  const int64_t w_of0 = static_cast<int64_t>(r.expert) * a.k;
  const int k0 = n0 + wn * FN * 16 + f_at * W;  // of run u: k0 + u * 4 * W
  float x_scale[FM];
  typename Vec<W>::type w_scale[U];
  auto load_scales = [&]() {
#pragma unroll
    for (int j = 0; j < FM; ++j) {
      const int row = (wm * FM + j) * 16 + f_row;
      int from = row < rows ? r.row0 + row : -1;
      if (a.index != nullptr && from >= 0) from = a.index[from];
      x_scale[j] = from >= 0 && from < a.x_rows ? a.x_scales[from] : 0.0f;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) w_scale[u] = load_floats<W>(a.w_scales + w_of0 + k0 + u * 4 * W, a.k - (k0 + u * 4 * W));
  };
  if constexpr (kEarly) load_scales();

  // A wave's runs: lane l stages one unit of row l >> 3 of each.  Rows and channels beyond the tile's read
  // another's: they reach no sum that is stored.
  int x_row[NX], w_row[NW];
#pragma unroll
  for (int i = 0; i < NX; ++i) {
    const int row = (wave * NX + i) * 8 + (lane >> 3);
    x_row[i] = row < rows ? row : 0;
    if (a.index != nullptr) {
      const int from = a.index[r.row0 + x_row[i]];
      x_row[i] = from >= 0 && from < a.x_rows ? from : 0;
    }
  }
#pragma unroll
  for (int i = 0; i < NW; ++i) w_row[i] = min(channel_of<T>((wave * NW + i) * 8 + (lane >> 3)), channels - 1);
  const int8_t* const x_base = a.index != nullptr ? a.x : a.x + static_cast<int64_t>(r.row0) * a.c;
  const int8_t* const w_base = a.w + (w_of0 + n0) * a.c;
  const int steps = (a.c + kStep - 1) / kStep;
  // the lane's channel in run i: its rows are 8i .. 8i + 7
  auto run_at = [&](int i) { return unit(i * 8 + (lane >> 3), lane & 7) * 16; };

  // DMA: offsets of a wave's runs; past the tensor's end they read zeros.
  unsigned x_of[NX], w_of[NW];
  __amdgpu_buffer_rsrc_t x_rsrc, w_rsrc;
  // registers: where a wave's runs start, and a step of them on its way
  const int8_t* x_from[NX];
  const int8_t* w_from[NW];
  v4i x_set[NX], w_set[NW];
  if constexpr (DMA) {
#pragma unroll
    for (int i = 0; i < NX; ++i)
      x_of[i] = static_cast<unsigned>(x_row[i]) * static_cast<unsigned>(a.c) + run_at(wave * NX + i);
#pragma unroll
    for (int i = 0; i < NW; ++i)
      w_of[i] = static_cast<unsigned>(w_row[i]) * static_cast<unsigned>(a.c) + run_at(wave * NW + i);
    x_rsrc = make_rsrc(x_base, static_cast<int>(static_cast<unsigned>(a.index != nullptr ? a.x_rows : rows) *
                                                static_cast<unsigned>(a.c)));
    w_rsrc = make_rsrc(w_base, channels * a.c);
  } else {
#pragma unroll
    for (int i = 0; i < NX; ++i) x_from[i] = x_base + static_cast<int64_t>(x_row[i]) * a.c;
#pragma unroll
    for (int i = 0; i < NW; ++i) w_from[i] = w_base + static_cast<int64_t>(w_row[i]) * a.c;
  }
  auto stage = [&](int step, int buffer) {
    const unsigned k = static_cast<unsigned>(min(step, steps - 1)) * kStep;
    char* const to = lds + buffer * kStage;
#pragma unroll
    for (int i = 0; i < NX; ++i)
      load_lds16(x_rsrc, reinterpret_cast<v4i*>(to + (wave * NX + i) * 1024), x_of[i], k);
#pragma unroll
    for (int i = 0; i < NW; ++i)
      load_lds16(w_rsrc, reinterpret_cast<v4i*>(to + BM * kStep + (wave * NW + i) * 1024), w_of[i], k);
  };
  auto load = [&](int step) {
    const int k = min(step, steps - 1) * kStep;
    if (step < steps - 1) {
#pragma unroll
      for (int i = 0; i < NX; ++i) x_set[i] = load16<false>(x_from[i] + k + run_at(wave * NX + i));
#pragma unroll
      for (int i = 0; i < NW; ++i) w_set[i] = load16<false>(w_from[i] + k + run_at(wave * NW + i));
    } else {
#pragma unroll
      for (int i = 0; i < NX; ++i) x_set[i] = load_codes16(x_from[i], k + run_at(wave * NX + i), a.c);
#pragma unroll
      for (int i = 0; i < NW; ++i) w_set[i] = load_codes16(w_from[i], k + run_at(wave * NW + i), a.c);
    }
  };
  auto write = [&](int buffer) {
    char* const to = lds + buffer * kStage + lane * 16;
#pragma unroll
    for (int i = 0; i < NX; ++i) *reinterpret_cast<v4i*>(to + (wave * NX + i) * 1024) = x_set[i];
#pragma unroll
    for (int i = 0; i < NW; ++i) *reinterpret_cast<v4i*>(to + BM * kStep + (wave * NW + i) * 1024) = w_set[i];
  };

  typedef __attribute__((address_space(3))) const char lds_char;
  typedef __attribute__((address_space(3))) const v4i lds_v4i;
  lds_char* f_from[2];  // of a half step
#pragma unroll
  for (int h = 0; h < 2; ++h) f_from[h] = (lds_char*)lds + f_row * kStep + unit(f_row, 4 * h + f_at) * 16;  // an address-space cast
  v4i fx[2][FM], fw[2][FN];
  auto read = [&](int buffer, int half) {
    lds_char* const x = f_from[half] + wm * FM * 16 * kStep + buffer * kStage;
    lds_char* const w = f_from[half] + BM * kStep + wn * FN * 16 * kStep + buffer * kStage;
#pragma unroll
    for (int i = 0; i < FN; ++i) fw[half][i] = *reinterpret_cast<lds_v4i*>(w + i * 16 * kStep);
#pragma unroll
    for (int i = 0; i < FM; ++i) fx[half][i] = *reinterpret_cast<lds_v4i*>(x + i * 16 * kStep);
  };
  v4i acc[FN][FM] = {};
  auto multiply = [&](int half) {
#pragma unroll
    for (int i = 0; i < FN; ++i)
#pragma unroll
      for (int j = 0; j < FM; ++j)
        acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fw[half][i], fx[half][j], acc[i][j], 0, 0, 0);
  };
  // a read or a load after each matrix instruction
  auto mix = [&]() {
    if constexpr (DMA) {
#pragma unroll
      for (int i = 0; i < FN * FM; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);  // matrix
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);  // LDS reads
        __builtin_amdgcn_sched_group_barrier(0x020, 1, 0);  // loads
      }
    }
    __builtin_amdgcn_sched_barrier(0);
  };

  // The middle of step t is where the waves meet: each has read all of its buffer, so the loads of step t +
  // STAGES (registers: the values of t + 2, loaded a step ago) go into it, and each has its part of t + 1 in
  // LDS, so the fragments of that can be read.  STAGES - 2 steps stay in flight.  Past the last step the
  // loads repeat it.
  constexpr int kLoads = NX + NW;
  static_assert((STAGES - 1) * kLoads <= 63, "the counter has 6 bits");
  if constexpr (DMA) {
#pragma unroll
    for (int i = 0; i < STAGES; ++i) stage(i, i);
    wait_vmcnt63((STAGES - 1) * kLoads);
  } else {
    load(0);
    write(0);
    load(1);
    write(1);
    load(2);
    __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
  }
  barrier_only();
  read(0, 0);
  int now = 0;  // buffer of step t
  for (int t = 0; t + 1 < steps; ++t) {
    const int next = now + 1 == STAGES ? 0 : now + 1;
    read(now, 1);
    multiply(0);
    mix();
    if constexpr (DMA) wait_vmcnt63((STAGES - 2) * kLoads);
    __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
    barrier_only();
    if constexpr (DMA) {
      stage(t + STAGES, now);
    } else {
      write(now);
      load(t + 3);
    }
    read(next, 0);
    multiply(1);
    mix();
    now = next;
  }
  // the last step: codes past the rows' end do not count
  read(now, 1);
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const bool there = (steps - 1) * kStep + (4 * h + f_at) * 16 < a.c;
#pragma unroll
    for (int j = 0; j < FM; ++j) fx[h][j] = there ? fx[h][j] : v4i{};
    multiply(h);
  }
  wait_vmcnt(0);  // no load into LDS outlives the workgroup

  if constexpr (!kEarly) load_scales();
  typename Vec<W>::type bias[U] = {};
  if (a.bias != nullptr) {
#pragma unroll
    for (int u = 0; u < U; ++u) bias[u] = load_floats<W>(a.bias + w_of0 + k0 + u * 4 * W, a.k - (k0 + u * 4 * W));
  }
  // row by row, so that the halves of a line are written one after the other
#pragma unroll
  for (int j = 0; j < FM; ++j) {
    const int row = (wm * FM + j) * 16 + f_row;
    if (row >= rows) continue;
    T* const y = static_cast<T*>(a.y) + (r.row0 + row) * a.ld_y + k0;
    const T* const add = static_cast<const T*>(a.add) + (r.row0 + row) * a.ld_add + k0;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int left = a.k - (k0 + u * 4 * W);
      if (left <= 0) continue;
      typename Vec<W>::type v;
#pragma unroll
      for (int i = 0; i < W; ++i) v[i] = scaled(acc[(u * W + i) / 4][j][i % 4], x_scale[j], w_scale[u][i]);
      if (a.bias != nullptr) v += bias[u];
      if (a.add != nullptr) v += load_some<false>(add + u * 4 * W, left);
      store_some<STREAM>(y + u * 4 * W, v, left);
    }
  }
}

template <typename T, bool DMA, int BM, int BN, int WM, int WN, int STAGES, bool STREAM = false>
hipError_t launch(const Row8LinearArgs& a, int wide, int64_t high, hipStream_t stream) {
  constexpr int kSize = STAGES * (BM + BN) * kStep;
  auto* const kernel = row8_tile_kernel<T, DMA, BM, BN, WM, WN, STAGES, STREAM>;
  if (kSize > 64 * 1024) {
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                             hipFuncAttributeMaxDynamicSharedMemorySize, kSize);
    if (e != hipSuccess) return e;
  }
  // at most 2^22 tiles a launch, whole row tiles each
  const int64_t most = std::max<int64_t>((int64_t{1} << 22) / wide, 1);
  for (int64_t from = 0; from < high; from += most) {
    const Tiling t{static_cast<int>(from), static_cast<int>(std::min(most, high - from)), wide};
    kernel<<<static_cast<unsigned>(static_cast<int64_t>(t.high) * wide), WM * WN * 64, kSize, stream>>>(a, t);
    if (const hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  }
  return hipSuccess;
}

template <typename T, bool DMA>
hipError_t by_tile(const Row8LinearArgs& a, int rows, int channels, hipStream_t stream) {
  const int wide = (a.k + channels - 1) / channels;
  const int64_t high = a.offsets != nullptr ? most_tiles(a.rows, a.experts, rows)
                                            : (static_cast<int64_t>(a.rows) + rows - 1) / rows;
  if constexpr (DMA) {
    // Few tiles: as many steps in flight as LDS holds for the one or two workgroups of a CU.
    const bool few = high * wide <= 512, one = high * wide <= 256;
    // a large y past the caches: 16384 x 2048 x 8192 281 -> 255 us, 16384 x 4096 x 8192 the same
    const bool past = channels == 256 && stream_stores(a.y, a.rows, a.k, a.ld_y, sizeof(T));
    if (rows == 256 && past) return launch<T, DMA, 256, 256, 2, 4, 2, true>(a, wide, high, stream);
    if (rows == 256) return launch<T, DMA, 256, 256, 2, 4, 2>(a, wide, high, stream);
    if (channels == 256 && past) return launch<T, DMA, 128, 256, 2, 4, 3, true>(a, wide, high, stream);
    if (channels == 256) return launch<T, DMA, 128, 256, 2, 4, 3>(a, wide, high, stream);
    if (rows == 128 && one) return launch<T, DMA, 128, 128, 2, 2, 4>(a, wide, high, stream);
    if (rows == 128) return launch<T, DMA, 128, 128, 2, 2, 2>(a, wide, high, stream);
    if (channels == 128 && few) return launch<T, DMA, 64, 128, 2, 2, 3>(a, wide, high, stream);
    if (channels == 128) return launch<T, DMA, 64, 128, 2, 2, 2>(a, wide, high, stream);
    if (few) return launch<T, DMA, 64, 64, 2, 2, 4>(a, wide, high, stream);
    return launch<T, DMA, 64, 64, 2, 2, 2>(a, wide, high, stream);
  } else {
    if (rows == 64 && channels == 64) return launch<T, DMA, 64, 64, 2, 2, 2>(a, wide, high, stream);
    if (rows == 64) return launch<T, DMA, 64, 128, 2, 2, 2>(a, wide, high, stream);
    if (channels == 128) return launch<T, DMA, 128, 128, 2, 2, 2>(a, wide, high, stream);
    // (256 rows would spill)
    return launch<T, DMA, 128, 256, 2, 4, 2>(a, (a.k + 255) / 256,
                                                a.offsets != nullptr ? most_tiles(a.rows, a.experts, 128)
                                                                     : (static_cast<int64_t>(a.rows) + 127) / 128, stream);
  }
}

template <typename T>
hipError_t by_way(const Row8LinearArgs& a, int rows, int channels, hipStream_t stream) {
  // straight to LDS: rows that start on 16 bytes, and rows of an index within 32-bit offsets
  if (codes_on(a, 16) && (a.index == nullptr || static_cast<int64_t>(a.x_rows) * a.c < (int64_t{1} << 32) - (1 << 20))) {
    return by_tile<T, true>(a, rows, channels, stream);
  }
  // Through registers a load from an odd address costs less than the second load and the shifts that few rows
  // take.
  return by_tile<T, false>(a, rows, channels, stream);
}

}  // namespace

hipError_t launch_row8_tile(const Row8LinearArgs& a, int rows, int channels, hipStream_t stream) {
  return a.bf16 ? by_way<__bf16>(a, rows, channels, stream) : by_way<float>(a, rows, channels, stream);
}

}  // namespace miq
