// Products of few 8-bit rows with 8-bit weights (row8_linear.cpp has the formula): the weights are read
// once, at the memory's rate, and never pass through LDS.
//
// A workgroup computes 16 * MT rows by 16 * NT channels.  Its eight waves share the reduction: wave w takes
// steps w, w + 8, ... of 64 codes, straight from global memory into the operands of its matrix
// instructions, U steps in flight; their sums meet in LDS at the end.  U leaves registers for two workgroups a
// CU (four steps of 16 x 32, 108 registers), so one's search for its rows and its sums hide behind the other's
// loads: with eight (156) the 16 rows below took 22 us.
//
// Bound by the weights: one row by 4096 x 4096 (16.8 MB) 6.2 us, 2 of them the launch; 14 of 64 experts' 2048 x
// 2048 for 16 rows (59 MB) 17 us.  With more rows by what a CU takes in, 38 KB a us in segments of 64 bytes:
// 64 rows by 8192 x 4096 15 us, where tiles take 9.
#include "row8_product.h"

namespace miq {
namespace {

constexpr int kStep = 64, kWaves = 8;

template <typename T, bool ODD, int NT, int MT, int U>
__global__ __launch_bounds__(kWaves * 64) void row8_few_kernel(Row8LinearArgs a, int64_t total, int wide) {
  __shared__ v4i sums[kWaves][NT * MT][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int f_row = lane & 15, f_at = (lane >> 4) * 16;
  for (int64_t tile = blockIdx.x; tile < total; tile += gridDim.x) {
    const int row_tile = static_cast<int>(tile / wide);
    const int n0 = static_cast<int>(tile - static_cast<int64_t>(row_tile) * wide) * (16 * NT);
    const int first = row_tile * 16 * MT;
    RowTile r = {0, first, a.rows - first < 16 * MT ? a.rows : first + 16 * MT};
    if (a.offsets != nullptr) {  // `first` may lie past the rows
      r = find_tile(a.offsets, a.experts, a.rows, 16 * MT, row_tile);
      if (r.expert < 0) return;  // nor has any tile after it
    }
    // Rows and channels beyond the tile's read another's: they reach no sum that is stored.
    const int8_t* x[MT];
    const int8_t* w[NT];
#pragma unroll
    for (int j = 0; j < MT; ++j) {
      int from = r.row0 + j * 16 + f_row;
      from = from < r.end ? from : r.row0;
      if (a.index != nullptr) from = a.index[from];
      x[j] = a.x + static_cast<int64_t>(from >= 0 && from < a.x_rows ? from : 0) * a.c;
    }
#pragma unroll
    for (int i = 0; i < NT; ++i)
      w[i] = a.w + (static_cast<int64_t>(r.expert) * a.k + min(n0 + i * 16 + f_row, a.k - 1)) * a.c;
    v4i acc[NT][MT] = {};
    const int whole = a.c / kStep;
    for (int s = wave; s < whole; s += kWaves * U) {
      v4i fx[U][MT], fw[U][NT];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int at = (s + kWaves * u) * kStep + f_at;
        if (s + kWaves * u < whole) {
#pragma unroll
          for (int i = 0; i < NT; ++i) fw[u][i] = load16<ODD>(w[i] + at);
#pragma unroll
          for (int j = 0; j < MT; ++j) fx[u][j] = load16<ODD>(x[j] + at);
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (s + kWaves * u < whole) {
#pragma unroll
          for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int j = 0; j < MT; ++j)
              acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fw[u][i], fx[u][j], acc[i][j], 0, 0, 0);
        }
    }
    if (whole * kStep < a.c && wave == whole % kWaves) {  // the rest of a step
      v4i fx[MT], fw[NT];
#pragma unroll
      for (int i = 0; i < NT; ++i) fw[i] = load_codes16(w[i], whole * kStep + f_at, a.c);
#pragma unroll
      for (int j = 0; j < MT; ++j) fx[j] = load_codes16(x[j], whole * kStep + f_at, a.c);
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int j = 0; j < MT; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fw[i], fx[j], acc[i][j], 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int j = 0; j < MT; ++j) sums[wave][i * MT + j][lane] = acc[i][j];
    __syncthreads();
    // four channels of a row a thread
    for (int at = threadIdx.x; at < NT * MT * 64; at += kWaves * 64) {
      const int f = at >> 6, l = at & 63;
      v4i sum = sums[0][f][l];
#pragma unroll
      for (int i = 1; i < kWaves; ++i) sum += sums[i][f][l];
      const int row = r.row0 + (f % MT) * 16 + (l & 15), k = n0 + (f / MT) * 16 + (l >> 4) * 4, left = a.k - k;
      if (row >= r.end || left <= 0) continue;
      const int from = a.index != nullptr ? a.index[row] : row;
      const float x_scale = from >= 0 && from < a.x_rows ? a.x_scales[from] : 0.0f;
      const int64_t of = static_cast<int64_t>(r.expert) * a.k + k;
      const v4f w_scale = load_floats<4>(a.w_scales + of, left);
      v4f v;
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = scaled(sum[i], x_scale, w_scale[i]);
      if (a.bias != nullptr) v += load_floats<4>(a.bias + of, left);
      T* const y = static_cast<T*>(a.y) + row * a.ld_y + k;
      const T* const add = static_cast<const T*>(a.add) + row * a.ld_add + k;
      if (left >= 4) {
        if (a.add != nullptr) v += load4(add);
        store_four(y, v);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (i < left) y[i] = static_cast<T>(v[i] + (a.add != nullptr ? static_cast<float>(add[i]) : 0.0f));
      }
    }
    __syncthreads();
  }
}

template <typename T, bool ODD, int NT, int MT, int U>
hipError_t launch(const Row8LinearArgs& a, hipStream_t stream) {
  const int wide = (a.k + 16 * NT - 1) / (16 * NT);
  const int64_t high = a.offsets != nullptr ? most_tiles(a.rows, a.experts, 16 * MT)
                                            : (static_cast<int64_t>(a.rows) + 16 * MT - 1) / (16 * MT);
  const int64_t total = high * wide;
  const unsigned grid = static_cast<unsigned>(total < (1 << 21) ? total : (1 << 21));
  row8_few_kernel<T, ODD, NT, MT, U><<<grid, kWaves * 64, 0, stream>>>(a, total, wide);
  return hipGetLastError();
}

template <typename T, bool ODD>
hipError_t by_tile(const Row8LinearArgs& a, int rows, int channels, hipStream_t stream) {
  if (rows == 16) return channels == 16 ? launch<T, ODD, 1, 1, 8>(a, stream) : launch<T, ODD, 2, 1, 4>(a, stream);
  if (rows == 32) return channels == 16 ? launch<T, ODD, 1, 2, 4>(a, stream) : launch<T, ODD, 2, 2, 4>(a, stream);
  return launch<T, ODD, 2, 4, 4>(a, stream);
}

template <typename T>
hipError_t by_address(const Row8LinearArgs& a, int rows, int channels, hipStream_t stream) {
  return codes_on(a, 4) ? by_tile<T, false>(a, rows, channels, stream) : by_tile<T, true>(a, rows, channels, stream);
}

}  // namespace

hipError_t launch_row8_few(const Row8LinearArgs& a, int rows, int channels, hipStream_t stream) {
  return a.bf16 ? by_address<__bf16>(a, rows, channels, stream) : by_address<float>(a, rows, channels, stream);
}

}  // namespace miq
