// The root-mean-square norm of rows, with the residual's addition, as real rows or as 8-bit rows
// (miq_rms_fprop, miq_rms_row8).
//
//   s = x + add (rounded to the type), r = 1 / sqrt(mean s^2 + eps), y = s * r * gain
//
// A row stays in the registers of a wave or a workgroup between its one read and its one write.  For
// 8-bit rows the codes need no r: the largest |s * gain| is found in the same pass as the sum of
// squares, and a code is s * gain times 127 over it; only the row's scale is multiplied by r.  Where
// s * gain or the norm leaves 2^-110 .. infinity, the codes are those of s * r * gain, looked at once more.
//
// Bound by memory: 16384 x 4096 bf16 with an addend as 8-bit rows (470 MB) 95 us, 4.9 TB/s; 16384 x 2048 bf16
// with an addend as real rows (268 MB) 53 us, 5.0 TB/s: a large copy's rate.  Rows of 64 channels share a
// wave four at a time (65536 x 64 bf16 29 -> 12 us a call).  Four rows of 4096 take 3.8 us, 2 of them the launch.
#include "row8_device.h"

namespace miq {
namespace {

template <int W, typename G>
__device__ __forceinline__ typename Vec<W>::type load_gain(const G* p, int left) {
  if constexpr (W == 8) {
    return load8_of(p, left);
  } else {
    if (left >= 4) return load4(p);
    v4f v = {};
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < left) v[i] = static_cast<float>(p[i]);
    return v;
  }
}

// Whether codes of a row can be taken from s * gain, whose largest magnitude has the bits `top`: it and the norm's own
// lie above the least one of a row and are finite.  False for rows with an infinity (r is 0) or a NaN.
__device__ __forceinline__ bool in_range(unsigned top, float r) {
  const float m = __uint_as_float(top), of_norm = m * r;
  return m >= kLeastTop && top < 0x7f800000u && of_norm >= kLeastTop && __float_as_uint(of_norm) < 0x7f800000u;
}

// Values as the type holds them.
template <typename T, typename V>
__device__ __forceinline__ V as_held(V v) {
  if constexpr (sizeof(T) == 2) {
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(V) / 4); ++i) v[i] = static_cast<float>(static_cast<T>(v[i]));
  }
  return v;
}

template <typename T, typename G, int THREADS, int V, bool ADD, bool CODES>
__global__ __launch_bounds__(kRowBlock<THREADS>) void rms_kernel(RmsArgs a) {
  constexpr int W = kWide<T>;
  constexpr int kRows = kRowBlock<THREADS> / THREADS;
  typedef typename Vec<W>::type Run;
  __shared__ RowSums<THREADS> lds;
  const int t = static_cast<int>(threadIdx.x) % THREADS;
  int turn = 0;
  for (int64_t row = static_cast<int64_t>(blockIdx.x) * kRows + static_cast<int>(threadIdx.x) / THREADS; row < a.rows;
       row += static_cast<int64_t>(gridDim.x) * kRows) {
    Run s[V], g[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int col = (j * THREADS + t) * W;
      s[j] = load_some<false>(static_cast<const T*>(a.x) + row * a.ld_x + col, a.c - col);
      if constexpr (ADD) s[j] += load_some<false>(static_cast<const T*>(a.add) + row * a.ld_add + col, a.c - col);
      g[j] = load_gain<W>(static_cast<const G*>(a.gain) + col, a.c - col);
    }
    float squares = 0.0f;
    unsigned top = 0;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      if constexpr (ADD) {
        const int col = (j * THREADS + t) * W;
        s[j] = as_held<T>(s[j]);
        store_some<false>(static_cast<T*>(a.sum) + row * a.ld_sum + col, s[j], a.c - col);
      }
#pragma unroll
      for (int i = 0; i < W; ++i) {
        squares += s[j][i] * s[j][i];
        if constexpr (CODES) top = max(top, magnitude(s[j][i] * g[j][i]));
      }
    }
    reduce_row<THREADS>(lds, turn, &squares, nullptr, CODES ? &top : nullptr);
    turn ^= 1;
    float eps = a.eps;
    if (overflowed(squares)) {  // the same for all of the row's threads
      squares = 0.0f;
      top = 0;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        s[j] *= kDown;
#pragma unroll
        for (int i = 0; i < W; ++i) {
          squares += s[j][i] * s[j][i];
          if constexpr (CODES) top = max(top, magnitude(s[j][i] * g[j][i]));
        }
      }
      reduce_row<THREADS>(lds, turn, &squares, nullptr, CODES ? &top : nullptr);
      turn ^= 1;
      eps = eps * kDown * kDown;
    }
    float r = inverse_rms(squares, a.c, eps);
    if constexpr (CODES) {
      if (!in_range(top, r)) {  // the same for all of the row's threads
        top = 0;
#pragma unroll
        for (int j = 0; j < V; ++j) {
          s[j] *= r;
#pragma unroll
          for (int i = 0; i < W; ++i) top = max(top, magnitude(s[j][i] * g[j][i]));
        }
        reduce_row<THREADS>(lds, turn, nullptr, nullptr, &top);
        turn ^= 1;
        r = 1.0f;
      }
      const float m = fmaxf(__uint_as_float(top), kLeastTop);
      const bool bad = top >= 0x7f800000u;
      const float inverse = 127.0f / m;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const int col = (j * THREADS + t) * W;
        store_codes<W>(a.codes + row * a.c + col, s[j] * g[j], inverse, bad, a.c - col);
      }
      if (t == 0) a.scales[row] = bad ? __uint_as_float(0x7fc00000u) : m * r / 127.0f;
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const int col = (j * THREADS + t) * W;
        store_some<false>(static_cast<T*>(a.y) + row * a.ld_y + col, s[j] * r * g[j], a.c - col);
      }
    }
  }
}

// Rows longer than the registers of a workgroup: read again for the output, and with a sum from there.
template <typename T, typename G, bool ADD, bool CODES>
__global__ __launch_bounds__(1024) void rms_long_kernel(RmsArgs a) {
  constexpr int W = kWide<T>, kThreads = 1024;
  typedef typename Vec<W>::type Run;
  __shared__ RowSums<kThreads> lds;
  int turn = 0;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* const x = static_cast<const T*>(a.x) + row * a.ld_x;
    const T* const add = static_cast<const T*>(a.add) + row * a.ld_add;
    T* const sum = static_cast<T*>(a.sum) + row * a.ld_sum;
    const T* const from = ADD ? sum : x;
    const G* const gain = static_cast<const G*>(a.gain);
    float squares = 0.0f, down = 1.0f, by = 1.0f, eps = a.eps;  // codes are of s * down * by * gain
    unsigned top = 0;
    for (int again = 0; again < 2; ++again) {
      squares = 0.0f;
      top = 0;
      for (int64_t at = static_cast<int64_t>(threadIdx.x) * W; at < a.c; at += kThreads * W) {
        const int left = static_cast<int>(a.c - at);
        Run s;
        if (again) {
          s = load_some<false>(from + at, left) * kDown;
        } else {
          s = load_some<false>(x + at, left);
          if constexpr (ADD) {
            s = as_held<T>(s + load_some<false>(add + at, left));
            store_some<false>(sum + at, s, left);
          }
        }
        Run g;
        if constexpr (CODES) g = load_gain<W>(gain + at, left);
#pragma unroll
        for (int i = 0; i < W; ++i) {
          squares += s[i] * s[i];
          if constexpr (CODES) top = max(top, magnitude(s[i] * g[i]));
        }
      }
      reduce_row<kThreads>(lds, turn, &squares, nullptr, CODES ? &top : nullptr);
      turn ^= 1;
      if (!overflowed(squares) || again) break;
      down = kDown;
      eps = a.eps * kDown * kDown;
    }
    float r = inverse_rms(squares, a.c, eps);
    if (CODES && !in_range(top, r)) {  // the same for all of the row's threads
      top = 0;
      for (int64_t at = static_cast<int64_t>(threadIdx.x) * W; at < a.c; at += kThreads * W) {
        const int left = static_cast<int>(a.c - at);
        const Run s = load_some<false>(from + at, left) * down * r;
        const Run g = load_gain<W>(gain + at, left);
#pragma unroll
        for (int i = 0; i < W; ++i) top = max(top, magnitude(s[i] * g[i]));
      }
      reduce_row<kThreads>(lds, turn, nullptr, nullptr, &top);
      turn ^= 1;
      by = r;
      r = 1.0f;
    }
    const float m = fmaxf(__uint_as_float(top), kLeastTop), inverse = 127.0f / m;
    const bool bad = top >= 0x7f800000u;
    for (int64_t at = static_cast<int64_t>(threadIdx.x) * W; at < a.c; at += kThreads * W) {
      const int left = static_cast<int>(a.c - at);
      const Run s = load_some<false>(from + at, left) * down;
      const Run g = load_gain<W>(gain + at, left);
      if constexpr (CODES) store_codes<W>(a.codes + row * a.c + at, s * by * g, inverse, bad, left);
      else store_some<false>(static_cast<T*>(a.y) + row * a.ld_y + at, s * r * g, left);
    }
    if (CODES && threadIdx.x == 0) a.scales[row] = bad ? __uint_as_float(0x7fc00000u) : m * r / 127.0f;
  }
}

template <typename T, typename G, bool ADD, bool CODES>
hipError_t launch(const RmsArgs& a, hipStream_t stream) {
  const RowShape shape = row_shape(a.c, kWide<T>, a.rows);
  by_shape(shape, [&](auto threads, auto runs) {
    constexpr int THREADS = threads.value, V = runs.value;
    if constexpr (V == 0) {
      rms_long_kernel<T, G, ADD, CODES><<<row_blocks(shape, a.rows, 1 << 16), 1024, 0, stream>>>(a);
    } else {
      rms_kernel<T, G, THREADS, V, ADD, CODES>
          <<<row_blocks(shape, a.rows, 1 << 20), kRowBlock<THREADS>, 0, stream>>>(a);
    }
  });
  return hipGetLastError();
}

template <typename T, typename G>
hipError_t by_form(const RmsArgs& a, hipStream_t stream) {
  if (a.add != nullptr) return a.codes ? launch<T, G, true, true>(a, stream) : launch<T, G, true, false>(a, stream);
  return a.codes ? launch<T, G, false, true>(a, stream) : launch<T, G, false, false>(a, stream);
}

}  // namespace

hipError_t launch_rms(const RmsArgs& a, hipStream_t stream) {
  if (a.bf16) return a.gain_bf16 ? by_form<__bf16, __bf16>(a, stream) : by_form<__bf16, float>(a, stream);
  return a.gain_bf16 ? by_form<float, __bf16>(a, stream) : by_form<float, float>(a, stream);
}

}  // namespace miq
