// dw[j, i] = sum over m of dy[m, j] * x'[m, i] with x' kept in 8 bits (miq_act8_grad).
//
// A kept value, code * 2^e with |code| <= 127, is exact in bf16: bf16 dy multiplies it directly
// on the bf16 matrix instructions with fp32 sums; fp32 dy is split into three bf16 numbers that
// add up to it (8 + 8 + 8 significant bits), three products a term.  The terms m are split over
// workgroups where the output has few tiles, and the partial sums added in order.
#include "train_device.h"

namespace miq {
namespace {

constexpr int kThreads = 256;
constexpr int kTile = 128;    // output rows and columns per workgroup
constexpr int kStep = 32;     // terms per step
constexpr int kPitch = 40;    // bf16 per LDS row: 80 bytes

struct Grad {
  const void* dy;
  const int8_t* codes;
  const uint8_t* scales;
  void* out;
  int64_t ld_dy, ld_out;
  int rows, c, k, groups, tiles_k, tiles_c, per_split;
  bool accumulate, to_parts;
};

template <int P>
__device__ __forceinline__ void split(float v, __bf16 (&p)[P]) {
  if constexpr (P == 1) {
    p[0] = static_cast<__bf16>(v);
  } else {
    // Truncation leaves at most 16, then 8 significant bits; an infinity or a NaN stays in the
    // first part alone.
    const unsigned bits = __float_as_uint(v);
    const bool finite = (bits & 0x7f800000u) != 0x7f800000u;
    const unsigned quiet = (bits & 0x7fffffffu) > 0x7f800000u ? 0x400000u : 0u;
    const float a = __uint_as_float((bits | quiet) & 0xffff0000u);
    const float r = finite ? v - a : 0.0f;
    const float b = __uint_as_float(__float_as_uint(r) & 0xffff0000u);
    p[0] = static_cast<__bf16>(a);
    p[1] = static_cast<__bf16>(b);
    p[2] = static_cast<__bf16>(r - b);
  }
}

template <typename T, typename TO, int P>
__global__ __launch_bounds__(kThreads) void act8_grad_kernel(Grad g) {
  __shared__ __bf16 lds_a[P][kTile][kPitch];
  __shared__ __bf16 lds_b[kTile][kPitch];
  const int tile = blockIdx.x % (g.tiles_k * g.tiles_c);
  const int part = blockIdx.x / (g.tiles_k * g.tiles_c);
  const int k0 = (tile / g.tiles_c) * kTile;
  const int c0 = (tile % g.tiles_c) * kTile;
  const int64_t m0 = static_cast<int64_t>(part) * g.per_split;
  const int64_t m1 = min(m0 + g.per_split, static_cast<int64_t>(g.rows));
  const T* dy = static_cast<const T*>(g.dy);
  const int lane = threadIdx.x & 63;
  const int wave = threadIdx.x >> 6;
  const int wk = (wave >> 1) * 64, wc = (wave & 1) * 64;
  const int col = threadIdx.x & (kTile - 1);
  v4f acc[4][4] = {};
  for (int64_t m = m0; m < m1; m += kStep) {
    for (int i = threadIdx.x / kTile; i < kStep; i += kThreads / kTile) {
      const bool there = m + i < m1;
      const float a = there && k0 + col < g.k ? static_cast<float>(dy[(m + i) * g.ld_dy + k0 + col]) : 0.0f;
      float b = 0.0f;
      if (there && c0 + col < g.c) {
        b = static_cast<float>(g.codes[(m + i) * g.c + c0 + col]) *
            __uint_as_float(static_cast<unsigned>(g.scales[(m + i) * g.groups + (c0 + col) / kAct8Group]) << 23);
      }
      __bf16 p[P];
      split(a, p);
#pragma unroll
      for (int q = 0; q < P; ++q) lds_a[q][col][i] = p[q];
      lds_b[col][i] = static_cast<__bf16>(b);
    }
    __syncthreads();
    v8bf fb[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) fb[j] = *reinterpret_cast<const v8bf*>(&lds_b[wc + j * 16 + (lane & 15)][(lane >> 4) * 8]);
#pragma unroll
    for (int q = P - 1; q >= 0; --q)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const v8bf fa = *reinterpret_cast<const v8bf*>(&lds_a[q][wk + i * 16 + (lane & 15)][(lane >> 4) * 8]);
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fa, fb[j], acc[i][j], 0, 0, 0);
      }
    __syncthreads();
  }
  TO* out = static_cast<TO*>(g.out) + (g.to_parts ? static_cast<int64_t>(part) * g.k * g.c : 0);
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int row = k0 + wk + i * 16 + (lane >> 4) * 4 + r;
        const int at = c0 + wc + j * 16 + (lane & 15);
        if (row < g.k && at < g.c) {
          TO* to = out + row * g.ld_out + at;
          float v = acc[i][j][r];
          if (g.accumulate) v += static_cast<float>(*to);
          *to = static_cast<TO>(v);
        }
      }
}

template <typename TO>
__global__ __launch_bounds__(kThreads) void act8_grad_join_kernel(Grad g, const float* __restrict__ parts, int splits) {
  const int64_t n = static_cast<int64_t>(g.k) * g.c;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; i < n;
       i += static_cast<int64_t>(gridDim.x) * kThreads) {
    float v = 0.0f;
    for (int s = 0; s < splits; ++s) v += parts[s * n + i];
    TO* to = static_cast<TO*>(g.out) + (i / g.c) * g.ld_out + i % g.c;
    if (g.accumulate) v += static_cast<float>(*to);
    *to = static_cast<TO>(v);
  }
}

// Splits of the terms: enough workgroups for two on each of the 256 CUs, 256 terms each or more.
int splits_of(int32_t rows, int32_t c, int32_t k, int* per) {
  const int64_t tiles = ((static_cast<int64_t>(c) + kTile - 1) / kTile) * ((static_cast<int64_t>(k) + kTile - 1) / kTile);
  int64_t n = 512 / tiles;
  const int64_t most = (static_cast<int64_t>(rows) + 255) / 256;
  if (n > most) n = most;
  if (n < 1) n = 1;
  int64_t each = (rows + n - 1) / n;
  each = (each + kStep - 1) / kStep * kStep;
  if (each < kStep) each = kStep;
  *per = static_cast<int>(each);
  n = (rows + each - 1) / each;
  return static_cast<int>(n < 1 ? 1 : n);
}

template <typename T, typename TO, int P>
void launch(const Act8GradArgs& a, hipStream_t stream) {
  Grad g{};
  g.dy = a.dy;
  g.codes = a.codes;
  g.scales = a.scales;
  g.ld_dy = a.ld_dy;
  g.rows = a.rows;
  g.c = a.c;
  g.k = a.k;
  g.groups = (a.c + kAct8Group - 1) / kAct8Group;
  g.tiles_k = (a.k + kTile - 1) / kTile;
  g.tiles_c = (a.c + kTile - 1) / kTile;
  const int splits = splits_of(a.rows, a.c, a.k, &g.per_split);
  const unsigned blocks = static_cast<unsigned>(static_cast<int64_t>(g.tiles_k) * g.tiles_c * splits);
  g.out = a.dw;
  g.ld_out = a.ld_dw;
  g.accumulate = a.accumulate;
  if (splits == 1) {
    act8_grad_kernel<T, TO, P><<<blocks, kThreads, 0, stream>>>(g);
    return;
  }
  Grad h = g;
  h.out = a.ws;
  h.ld_out = a.c;
  h.accumulate = false;
  h.to_parts = true;
  act8_grad_kernel<T, float, P><<<blocks, kThreads, 0, stream>>>(h);
  const int64_t n = static_cast<int64_t>(a.k) * a.c;
  const int64_t join = (n + kThreads - 1) / kThreads;
  act8_grad_join_kernel<TO><<<static_cast<unsigned>(join < 4096 ? join : 4096), kThreads, 0, stream>>>(
      g, static_cast<const float*>(a.ws), splits);
}

}  // namespace

size_t act8_grad_workspace_bytes(int32_t rows, int32_t c, int32_t k, bool) {
  int per;
  const int splits = splits_of(rows, c, k, &per);
  return splits > 1 ? static_cast<size_t>(splits) * c * k * 4 : 0;
}

hipError_t launch_act8_grad(const Act8GradArgs& a, hipStream_t stream) {
  if (!a.dy_bf16) {
    launch<float, float, 3>(a, stream);
  } else if (a.dw_bf16) {
    launch<__bf16, __bf16, 1>(a, stream);
  } else {
    launch<__bf16, float, 1>(a, stream);
  }
  return hipGetLastError();
}

}  // namespace miq
