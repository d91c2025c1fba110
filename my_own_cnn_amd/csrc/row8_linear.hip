// Products of 8-bit rows with 8-bit weights (miq_row8_linear, miq_row8_experts):
//
//   y[m, j] = float(sum over i of x[m, i] * w[j, i]) * x_scale[m] * w_scale[j] + bias[j] + add[m, j]
//
// on v_mfma_i32_16x16x64_i8.  The channels are the rows of a matrix instruction and y's rows its
// columns, so that a lane holds four consecutive channels of one row of y.
#include "row8_product.h"

namespace miq {
namespace {

constexpr int kTile = 64, kStep = 64, kPitch = kStep + 16;

// 16 codes of a row of c at channel `at`, zeros past the row's end.
__device__ __forceinline__ v4i load_codes16(const int8_t* row, int at, int c) {
  if (at + 16 <= c) return *reinterpret_cast<const v4i_any*>(row + at);
  v4i v = {};
#pragma unroll
  for (int i = 0; i < 16; ++i)
    if (at + i < c) v[i / 4] |= (row[at + i] & 0xff) << (8 * (i & 3));
  return v;
}

template <typename T>
__global__ __launch_bounds__(256) void row8_linear_any_kernel(Row8LinearArgs a, int64_t total, int wide_tiles) {
  __shared__ __attribute__((aligned(16))) int8_t xs[kTile * kPitch], ws[kTile * kPitch];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  for (int64_t tile = blockIdx.x; tile < total; tile += gridDim.x) {
    const int high_at = static_cast<int>(tile / wide_tiles);
    const int k0 = static_cast<int>(tile - static_cast<int64_t>(high_at) * wide_tiles) * kTile;
    RowTile r = {0, high_at * kTile, min(a.rows, (high_at + 1) * kTile)};
    if (a.offsets != nullptr) r = find_tile(a.offsets, a.experts, a.rows, kTile, high_at);
    if (r.expert < 0) return;  // nor has any tile after it
    const int8_t* const w = a.w + static_cast<int64_t>(r.expert) * a.k * a.c;
    // a thread stages 16 codes of one row of each operand
    const int s_row = tid >> 2, s_at = (tid & 3) * 16;
    int from = r.row0 + s_row < r.end ? r.row0 + s_row : -1;
    if (a.index != nullptr && from >= 0) from = a.index[from];
    const bool has_x = from >= 0 && from < a.x_rows, has_w = k0 + s_row < a.k;
    const int8_t* const x_row = a.x + static_cast<int64_t>(has_x ? from : 0) * a.c;
    const int8_t* const w_row = w + static_cast<int64_t>(has_w ? k0 + s_row : 0) * a.c;
    v4i acc[2][2] = {};
    const int wk = (wave & 1) * 32, wm = (wave >> 1) * 32;
    for (int at = 0; at < a.c; at += kStep) {
      const v4i x16 = has_x ? load_codes16(x_row, at + s_at, a.c) : v4i{};
      const v4i w16 = has_w ? load_codes16(w_row, at + s_at, a.c) : v4i{};
      __syncthreads();
      *reinterpret_cast<v4i*>(xs + s_row * kPitch + s_at) = x16;
      *reinterpret_cast<v4i*>(ws + s_row * kPitch + s_at) = w16;
      __syncthreads();
      v4i fx[2], fw[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        fx[i] = *reinterpret_cast<const v4i*>(xs + (wm + 16 * i + (lane & 15)) * kPitch + (lane >> 4) * 16);
        fw[i] = *reinterpret_cast<const v4i*>(ws + (wk + 16 * i + (lane & 15)) * kPitch + (lane >> 4) * 16);
      }
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fw[i], fx[j], acc[i][j], 0, 0, 0);
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int row = r.row0 + wm + 16 * j + (lane & 15);
      if (row >= r.end) continue;
      int source = row;
      if (a.index != nullptr) source = a.index[row];
      const float x_scale = source >= 0 && source < a.x_rows ? a.x_scales[source] : 0.0f;
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int k = k0 + wk + 16 * i + (lane >> 4) * 4 + q;
          if (k >= a.k) continue;
          const int64_t of = static_cast<int64_t>(r.expert) * a.k + k;
          float v = scaled(acc[i][j][q], x_scale, a.w_scales[of]);
          if (a.bias != nullptr) v += a.bias[of];
          if (a.add != nullptr) v += static_cast<float>(static_cast<const T*>(a.add)[row * a.ld_add + k]);
          static_cast<T*>(a.y)[row * a.ld_y + k] = static_cast<T>(v);
        }
    }
  }
}

}  // namespace

size_t row8_linear_workspace_bytes(int32_t, int32_t, int32_t) { return 0; }

hipError_t launch_row8_linear(const Row8LinearArgs& a, hipStream_t stream) {
  const int wide_tiles = (a.k + kTile - 1) / kTile;
  const int64_t high = a.offsets != nullptr ? most_tiles(a.rows, a.experts, kTile)
                                            : (static_cast<int64_t>(a.rows) + kTile - 1) / kTile;
  const int64_t total = high * wide_tiles;
  const unsigned grid = static_cast<unsigned>(total < (1 << 22) ? total : (1 << 22));
  if (a.bf16) row8_linear_any_kernel<__bf16><<<grid, 256, 0, stream>>>(a, total, wide_tiles);
  else row8_linear_any_kernel<float><<<grid, 256, 0, stream>>>(a, total, wide_tiles);
  return hipGetLastError();
}

}  // namespace miq
