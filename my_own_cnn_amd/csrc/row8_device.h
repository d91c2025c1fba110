// Device helpers of kernels that hold a row of a tensor in the registers of a wave or a workgroup.
#pragma once

#include "row8_internal.h"
#include "train_device.h"

namespace miq {
namespace {

// A row's values stand for code * scale with scale = m / 127, m its largest magnitude, held to 2^-110
// from below so that 127 / m stays finite.
constexpr float kLeastTop = 7.703719777548943e-34f;  // 2^-110

// Bits of a magnitude order as the magnitudes do, NaN above infinity.
__device__ __forceinline__ unsigned magnitude(float v) { return __float_as_uint(v) & 0x7fffffffu; }

template <typename V, int N>
__device__ __forceinline__ void zero(V (&v)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = V{};
}

// The sums of `a` and `b` and the largest `top` over the THREADS that hold a row: a quarter, a half or all of a
// wave, or a whole workgroup, which meets once.  `turn` alternates between rows, so that a wave that is a row ahead
// writes where nobody reads any more.
template <int THREADS>
struct RowSums {
  static constexpr int kWaves = THREADS > 64 ? THREADS / 64 : 1;
  float a[2][kWaves], b[2][kWaves];
  unsigned top[2][kWaves];
};
template <int THREADS>
__device__ __forceinline__ void reduce_row(RowSums<THREADS>& lds, int turn, float* a, float* b, unsigned* top) {
  for (int step = 1; step < (THREADS < 64 ? THREADS : 64); step *= 2) {
    if (a != nullptr) *a += __shfl_xor(*a, step);
    if (b != nullptr) *b += __shfl_xor(*b, step);
    if (top != nullptr) *top = max(*top, static_cast<unsigned>(__shfl_xor(static_cast<int>(*top), step)));
  }
  if constexpr (THREADS > 64) {
    constexpr int N = THREADS / 64;
    const int wave = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) {
      if (a != nullptr) lds.a[turn][wave] = *a;
      if (b != nullptr) lds.b[turn][wave] = *b;
      if (top != nullptr) lds.top[turn][wave] = *top;
    }
    __syncthreads();
    if (a != nullptr) {
      float s = 0.0f;
#pragma unroll
      for (int i = 0; i < N; ++i) s += lds.a[turn][i];
      *a = s;
    }
    if (b != nullptr) {
      float s = 0.0f;
#pragma unroll
      for (int i = 0; i < N; ++i) s += lds.b[turn][i];
      *b = s;
    }
    if (top != nullptr) {
      unsigned t = 0;
#pragma unroll
      for (int i = 0; i < N; ++i) t = max(t, lds.top[turn][i]);
      *top = t;
    }
  }
}

// A row of W-value runs held by THREADS threads: run j of a thread starts at channel (j * THREADS + t) * W.
// V runs a thread in registers.
struct RowShape {
  int threads, runs;
};
// The fewest threads that leave a thread few runs; runs == 0: more than registers hold.
inline RowShape row_shape(int64_t c, int wide, int64_t rows) {
  const int64_t n = (c + wide - 1) / wide;
  if (n <= 16) return {16, 1};
  if (n <= 32) return {32, 1};
  if (n <= 64) return {64, 1};
  if (n <= 128) return {64, 2};
  if (n <= 256) return rows >= 1024 ? RowShape{64, 4} : RowShape{256, 1};
  if (n <= 512) return {256, 2};
  if (n <= 1024) return {256, 4};
  if (n <= 2048) return {1024, 2};
  return {1024, 0};
}
// Calls go(threads, runs) with both as compile-time values.
template <typename F>
void by_shape(const RowShape& s, F&& go) {
  using std::integral_constant;
  if (s.threads == 16) {
    go(integral_constant<int, 16>{}, integral_constant<int, 1>{});
  } else if (s.threads == 32) {
    go(integral_constant<int, 32>{}, integral_constant<int, 1>{});
  } else if (s.threads == 64) {
    if (s.runs == 1) go(integral_constant<int, 64>{}, integral_constant<int, 1>{});
    else if (s.runs == 2) go(integral_constant<int, 64>{}, integral_constant<int, 2>{});
    else go(integral_constant<int, 64>{}, integral_constant<int, 4>{});
  } else if (s.threads == 256) {
    if (s.runs == 1) go(integral_constant<int, 256>{}, integral_constant<int, 1>{});
    else if (s.runs == 2) go(integral_constant<int, 256>{}, integral_constant<int, 2>{});
    else go(integral_constant<int, 256>{}, integral_constant<int, 4>{});
  } else if (s.runs == 2) {
    go(integral_constant<int, 1024>{}, integral_constant<int, 2>{});
  } else {
    go(integral_constant<int, 1024>{}, integral_constant<int, 0>{});
  }
}

// Workgroups (of at least 256 threads) of a kernel that loops over rows.
inline unsigned row_blocks(const RowShape& s, int64_t rows, int64_t most) {
  const int64_t per = s.threads < 256 ? 256 / s.threads : 1;
  const int64_t blocks = (rows + per - 1) / per;
  return static_cast<unsigned>(blocks < most ? blocks : most);
}
template <int THREADS>
constexpr int kRowBlock = THREADS < 256 ? 256 : THREADS;

// W values times `inverse` as codes of the row's channels col ..; |value * inverse| <= 127, or `bad` (codes 0).
// Adding 1.5 * 2^23 rounds to nearest even into the low byte.
template <int W>
__device__ __forceinline__ void store_codes(int8_t* p, const typename Vec<W>::type& v, float inverse, bool bad, int left) {
  int q[W / 4];
#pragma unroll
  for (int i = 0; i < W; i += 4) {
    const int four = static_cast<int>(pack4_magic(v[i] * inverse + 12582912.0f, v[i + 1] * inverse + 12582912.0f,
                                                  v[i + 2] * inverse + 12582912.0f, v[i + 3] * inverse + 12582912.0f));
    q[i / 4] = bad ? 0 : four;
  }
  if (left >= W) {
    if constexpr (W == 8) *reinterpret_cast<v2i_any*>(p) = v2i{q[0], q[1]};
    else *reinterpret_cast<int_any*>(p) = q[0];
  } else {
#pragma unroll
    for (int i = 0; i < W; ++i)
      if (i < left) p[i] = static_cast<int8_t>(q[i / 4] >> (8 * (i & 3)));
  }
}

// The mean square's reciprocal root, from the sum of squares.  A sum that overflows is summed again
// over values times 2^-80, by the caller.
constexpr float kDown = 8.271806125530277e-25f;  // 2^-80
__device__ __forceinline__ bool overflowed(float squares) { return !(squares < 1e38f); }
__device__ __forceinline__ float inverse_rms(float squares, int c, float eps) {
  return 1.0f / sqrtf(squares / static_cast<float>(c) + eps);
}

}  // namespace
}  // namespace miq
