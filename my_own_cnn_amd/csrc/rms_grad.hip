// The backward pass of the root-mean-square norm (miq_rms_bprop).
//
//   n = s * r, r = 1 / sqrt(mean s^2 + eps), dn = dy * gain
//   ds = r * (dn - n * mean(dn * n)) + dsum,   dgain = sum over the rows of dy * n
//
// One read of s, dy and dsum and one write of ds: a row stays in the registers of a wave or a
// workgroup, both sums of a row (s^2 and dn * s) meet once, and dgain's terms are added in registers over
// the rows that a workgroup takes.  The workgroups' sums go to the workspace and are added by a second
// launch, both in an order fixed by the sizes.
//
// Bound by memory: 16384 x 2048 bf16 with dsum (268 MB) 49 us, 5.5 TB/s, and 4.7 us for the sum of 768 rows of the
// workspace: 53 us a call, without dsum 49.  With x and dy loaded when their row comes and not a row ahead 58 and 52,
// 8192 x 4096 65 (56 ahead), 16384 x 1000 38 (31).
#include <algorithm>

#include "row8_device.h"

namespace miq {
namespace {

constexpr int64_t kWorkspace = 1 << 25;  // values of the workspace, while that leaves a workgroup

// Whether the sum of dn * s over a row lost nothing that matters: it did not overflow, and what its terms lost below
// the normal numbers is far below it.  Otherwise (zeros of dy among them) mean(dn * n) is summed over n / c.
__device__ __forceinline__ bool in_range(float dot) { return fabsf(dot) > 1e-27f && fabsf(dot) < 1e38f; }

// 16 bytes of a row as they lie in memory, zeros past its end.
template <typename T>
struct RawOf;
template <>
struct RawOf<__bf16> {
  typedef v8bf type;
  typedef v8bf_any any;
};
template <>
struct RawOf<float> {
  typedef v4f type;
  typedef v4f_any any;
};
template <typename T>
__device__ __forceinline__ typename RawOf<T>::type load_raw(const T* p, int left) {
  if (left >= kWide<T>) return *reinterpret_cast<const typename RawOf<T>::any*>(p);
  typename RawOf<T>::type v = {};
#pragma unroll
  for (int i = 0; i < kWide<T>; ++i)
    if (i < left) v[i] = p[i];
  return v;
}

template <int W, typename G>
__device__ __forceinline__ typename Vec<W>::type load_gain(const G* p, int left) {
  typename Vec<W>::type v = {};
#pragma unroll
  for (int i = 0; i < W; ++i)
    if (i < left) v[i] = static_cast<float>(p[i]);
  return v;
}

template <typename T, typename G, int THREADS, int V>
__global__ __launch_bounds__(kRowBlock<THREADS>, THREADS == 1024 ? 4 : 2) void rms_grad_kernel(RmsGradArgs a) {
  constexpr int W = kWide<T>;
  constexpr int kThreads = kRowBlock<THREADS>, kRows = kThreads / THREADS;
  typedef typename Vec<W>::type Run;
  __shared__ RowSums<THREADS> lds;
  __shared__ float sums[kRows > 1 ? kRows * THREADS * V * W : 1];
  const int t = static_cast<int>(threadIdx.x) % THREADS;
  const int own = static_cast<int>(threadIdx.x) / THREADS;
  Run g[V], total[V];
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int col = (j * THREADS + t) * W;
    g[j] = load_gain<W>(static_cast<const G*>(a.gain) + col, a.c - col);
    total[j] = Run{};
  }
  // The next row's values travel while this one is summed, where registers hold both: more than 16 values a thread (8
  // of 1024 threads, which have 128 VGPRs each) would spill and are loaded when their row comes.
  constexpr bool kAhead = V * W * (THREADS == 1024 ? 2 : 1) <= 16;
  typename RawOf<T>::type next_s[V], next_d[V], next_e[V];
  auto load = [&](int64_t row) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int col = (j * THREADS + t) * W;
      next_s[j] = load_raw(static_cast<const T*>(a.x) + row * a.ld_x + col, a.c - col);
      next_d[j] = load_raw(static_cast<const T*>(a.dy) + row * a.ld_dy + col, a.c - col);
      if (a.dsum != nullptr) next_e[j] = load_raw(static_cast<const T*>(a.dsum) + row * a.ld_dsum + col, a.c - col);
    }
  };
  const int64_t step = static_cast<int64_t>(gridDim.x) * kRows;
  int64_t row = static_cast<int64_t>(blockIdx.x) * kRows + own;
  if (kAhead && row < a.rows) load(row);
  int turn = 0;
  for (; row < a.rows; row += step) {
    Run s[V], d[V];
    typename RawOf<T>::type e[V];
    if (!kAhead) load(row);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      s[j] = __builtin_convertvector(next_s[j], Run);
      d[j] = __builtin_convertvector(next_d[j], Run);
      e[j] = next_e[j];
    }
    if (kAhead && row + step < a.rows) load(row + step);
    float squares = 0.0f, dot = 0.0f;
#pragma unroll
    for (int j = 0; j < V; ++j)
#pragma unroll
      for (int i = 0; i < W; ++i) {
        squares += s[j][i] * s[j][i];
        dot += d[j][i] * g[j][i] * s[j][i];
      }
    reduce_row<THREADS>(lds, turn, &squares, &dot, nullptr);
    turn ^= 1;
    float eps = a.eps, down = 1.0f;
    if (overflowed(squares)) {  // the same for all of the row's threads
      squares = dot = 0.0f;
      down = kDown;
      eps = eps * kDown * kDown;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        s[j] *= kDown;
#pragma unroll
        for (int i = 0; i < W; ++i) {
          squares += s[j][i] * s[j][i];
          dot += d[j][i] * g[j][i] * s[j][i];
        }
      }
      reduce_row<THREADS>(lds, turn, &squares, &dot, nullptr);
      turn ^= 1;
    }
    const float r = inverse_rms(squares, a.c, eps);
    float along = dot * r / static_cast<float>(a.c);
    if (!in_range(dot)) {  // the same for all of the row's threads
      const float each = r / static_cast<float>(a.c);
      along = 0.0f;
#pragma unroll
      for (int j = 0; j < V; ++j)
#pragma unroll
        for (int i = 0; i < W; ++i) along += d[j][i] * g[j][i] * (s[j][i] * each);
      reduce_row<THREADS>(lds, turn, &along, nullptr, nullptr);
      turn ^= 1;
    }
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int col = (j * THREADS + t) * W;
      const Run n = s[j] * r;
      total[j] += d[j] * n;
      Run dx = (d[j] * g[j] - n * along) * (r * down);
      if (a.dsum != nullptr) dx += __builtin_convertvector(e[j], Run);
      store_some<false>(static_cast<T*>(a.dx) + row * a.ld_dx + col, dx, a.c - col);
    }
  }
  // The workgroup's row of the workspace.
  float* const out = a.ws + static_cast<int64_t>(blockIdx.x) * a.c;
  if constexpr (kRows > 1) {
#pragma unroll
    for (int j = 0; j < V; ++j)
#pragma unroll
      for (int i = 0; i < W; ++i) sums[own * (THREADS * V * W) + (j * THREADS + t) * W + i] = total[j][i];
    __syncthreads();
    for (int col = threadIdx.x; col < a.c; col += kThreads) {
      float s = 0.0f;
#pragma unroll
      for (int k = 0; k < kRows; ++k) s += sums[k * (THREADS * V * W) + col];
      out[col] = s;
    }
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int col = (j * THREADS + t) * W;
#pragma unroll
      for (int i = 0; i < W; ++i)
        if (i < a.c - col) out[col + i] = total[j][i];
    }
  }
}

// Rows longer than the registers of a workgroup: read again for ds and dgain; dgain's terms are added
// in the workgroup's row of the workspace, each by the thread that reads it next.
template <typename T, typename G>
__global__ __launch_bounds__(1024) void rms_grad_long_kernel(RmsGradArgs a) {
  constexpr int W = kWide<T>, kThreads = 1024;
  typedef typename Vec<W>::type Run;
  __shared__ RowSums<kThreads> lds;
  float* const out = a.ws + static_cast<int64_t>(blockIdx.x) * a.c;
  int turn = 0;
  bool first = true;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* const x = static_cast<const T*>(a.x) + row * a.ld_x;
    const T* const dy = static_cast<const T*>(a.dy) + row * a.ld_dy;
    const G* const gain = static_cast<const G*>(a.gain);
    float squares = 0.0f, dot = 0.0f, down = 1.0f, eps = a.eps;
    for (int again = 0; again < 2; ++again) {
      squares = dot = 0.0f;
      for (int64_t at = static_cast<int64_t>(threadIdx.x) * W; at < a.c; at += kThreads * W) {
        const int left = static_cast<int>(a.c - at);
        const Run s = load_some<false>(x + at, left) * down, d = load_some<false>(dy + at, left);
        const Run g = load_gain<W>(gain + at, left);
#pragma unroll
        for (int i = 0; i < W; ++i) {
          squares += s[i] * s[i];
          dot += d[i] * g[i] * s[i];
        }
      }
      reduce_row<kThreads>(lds, turn, &squares, &dot, nullptr);
      turn ^= 1;
      if (!overflowed(squares) || again) break;
      down = kDown;
      eps = a.eps * kDown * kDown;
    }
    const float r = inverse_rms(squares, a.c, eps);
    float along = dot * r / static_cast<float>(a.c);
    if (!in_range(dot)) {  // the same for all of the row's threads
      const float each = r / static_cast<float>(a.c);
      along = 0.0f;
      for (int64_t at = static_cast<int64_t>(threadIdx.x) * W; at < a.c; at += kThreads * W) {
        const int left = static_cast<int>(a.c - at);
        const Run s = load_some<false>(x + at, left) * down, d = load_some<false>(dy + at, left);
        const Run g = load_gain<W>(gain + at, left);
#pragma unroll
        for (int i = 0; i < W; ++i) along += d[i] * g[i] * (s[i] * each);
      }
      reduce_row<kThreads>(lds, turn, &along, nullptr, nullptr);
      turn ^= 1;
    }
    for (int64_t at = static_cast<int64_t>(threadIdx.x) * W; at < a.c; at += kThreads * W) {
      const int left = static_cast<int>(a.c - at);
      const Run n = load_some<false>(x + at, left) * down * r, d = load_some<false>(dy + at, left);
      const Run g = load_gain<W>(gain + at, left);
      Run dx = (d * g - n * along) * (r * down);
      if (a.dsum != nullptr) dx += load_some<false>(static_cast<const T*>(a.dsum) + row * a.ld_dsum + at, left);
#pragma unroll
      for (int i = 0; i < W; ++i)
        if (i < left) out[at + i] = (first ? 0.0f : out[at + i]) + d[i] * n[i];
      store_some<false>(static_cast<T*>(a.dx) + row * a.ld_dx + at, dx, left);
    }
    first = false;
  }
}

// dgain[col] = the sum of the workspace's rows, 32 columns a workgroup, 32 threads a column.
template <typename D>
__global__ __launch_bounds__(1024) void rms_grad_join_kernel(const float* __restrict__ ws, D* __restrict__ dgain, int c,
                                                             int parts, bool accumulate) {
  __shared__ float lds[32][33];
  const int x = threadIdx.x & 31, y = threadIdx.x >> 5;
  for (int base = blockIdx.x * 32; base < c; base += gridDim.x * 32) {
    float s = 0.0f;
    if (base + x < c) {
      const float* from = ws + base + x;
#pragma unroll 8
      for (int p = y; p < parts; p += 32) s += from[static_cast<int64_t>(p) * c];
    }
    lds[y][x] = s;
    __syncthreads();
    if (y == 0 && base + x < c) {
      float total = accumulate ? static_cast<float>(dgain[base + x]) : 0.0f;
      for (int i = 0; i < 32; ++i) total += lds[i][x];
      dgain[base + x] = static_cast<D>(total);
    }
    __syncthreads();
  }
}

// Four waves on rows of 1025 to 2048 bf16: a thread's 8 values leave room for the next row's, a wave's 32 a thread
// do not.  16384 x 2048 with dsum 53 us, a wave a row 57; without dsum 49 and 44.  fp32 rows of as many bytes have 16
// values a thread and stay with a wave (5003 x 1001 17 us, 18 with four).
RowShape shape_of(int64_t c, int wide, int64_t rows) {
  const RowShape s = row_shape(c, wide, rows);
  return wide == 8 && s.threads == 64 && s.runs == 4 ? RowShape{256, 1} : s;
}

// Workgroups, each with a row of the workspace, while there are rows for them.  With the loads ahead few a CU keep
// the memory busy, and more of them only add to the sum of the workspace: over 64 to 4096 channels of both types
// with dsum 3 a CU took 1 to 11% less than 5 where a thread has one run, and 2 a CU 3 to 8% less than 3 where it
// has more.
int64_t parts_of(int64_t rows, int64_t c, int wide) {
  const RowShape s = shape_of(c, wide, rows);
  const int64_t per_cu = s.threads == 1024 ? 1 : (s.runs == 1 ? 3 : 2);
  const int64_t at_once = s.threads < 256 ? 256 / s.threads : 1;  // rows of a workgroup
  return std::min({(rows + at_once - 1) / at_once, 256 * per_cu, std::max<int64_t>(kWorkspace / c, 1)});
}

template <typename T, typename G>
void launch(const RmsGradArgs& a, int64_t parts, hipStream_t stream) {
  by_shape(shape_of(a.c, kWide<T>, a.rows), [&](auto threads, auto runs) {
    constexpr int THREADS = threads.value, V = runs.value;
    if constexpr (V == 0) {
      rms_grad_long_kernel<T, G><<<static_cast<unsigned>(parts), 1024, 0, stream>>>(a);
    } else {
      rms_grad_kernel<T, G, THREADS, V><<<static_cast<unsigned>(parts), kRowBlock<THREADS>, 0, stream>>>(a);
    }
  });
}

}  // namespace

size_t rms_grad_workspace_bytes(int64_t rows, int32_t c) { return static_cast<size_t>(std::max(parts_of(rows, c, 8), parts_of(rows, c, 4))) * c * sizeof(float); }

hipError_t launch_rms_grad(const RmsGradArgs& a, hipStream_t stream) {
  const int64_t parts = parts_of(a.rows, a.c, a.bf16 ? 8 : 4);
  if (parts > 0) {
    if (a.bf16) a.gain_bf16 ? launch<__bf16, __bf16>(a, parts, stream) : launch<__bf16, float>(a, parts, stream);
    else a.gain_bf16 ? launch<float, __bf16>(a, parts, stream) : launch<float, float>(a, parts, stream);
    if (const hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  }
  const unsigned grid = static_cast<unsigned>(std::min<int64_t>((static_cast<int64_t>(a.c) + 31) / 32, 1 << 20));
  const int n = static_cast<int>(parts);
  if (a.dgain_bf16) rms_grad_join_kernel<<<grid, 1024, 0, stream>>>(a.ws, static_cast<__bf16*>(a.dgain), a.c, n, a.accumulate);
  else rms_grad_join_kernel<<<grid, 1024, 0, stream>>>(a.ws, static_cast<float*>(a.dgain), a.c, n, a.accumulate);
  return hipGetLastError();
}

}  // namespace miq
