// 8-bit rows: int8 codes and one scale a row (miq_act_row8, miq_row8_expand).
//
// v = act(x), or act(gate) * up; m = max(max |v|, 2^-110); code = rint(v * (127 / m)), scale = m / 127.
// A row stays in the registers of a wave or a workgroup: one read, one write.
//
// Bound by memory: gated silu of 16384 x 8192 bf16 (671 MB) 138 us, 4.9 TB/s (150 with the library's expf and a
// division); the values of its codes (403 MB) 64 us, 6.3 TB/s.  gelu of 4099 x 1003 fp32 8.3 us (12.7 with erfcf).
#include "row8_product.h"

namespace miq {
namespace {

// A row that holds an infinity or a NaN has codes 0 and a NaN scale.
struct RowCode {
  float inverse, scale;
  bool bad;
};
__device__ __forceinline__ RowCode code_of(unsigned top) {
  const float m = fmaxf(__uint_as_float(top), kLeastTop);
  const bool bad = top >= 0x7f800000u;
  return {127.0f / m, bad ? __uint_as_float(0x7fc00000u) : m / 127.0f, bad};
}

// act(v) for codes, which keep 8 bits of it: on the exponential and reciprocal instructions (1 unit each; the
// rounded argument moves the exponential by |v| / 2 units), and erfc by the Chebyshev fit "erfcc" of Press et
// al., Numerical Recipes, within 1.2e-7 of its value everywhere.
__device__ __forceinline__ float exp_of(float v) { return __builtin_amdgcn_exp2f(v * 1.44269504088896341f); }
template <int ACT>
__device__ __forceinline__ float code_act(float v) {
  if constexpr (ACT == kSilu) return v * __builtin_amdgcn_rcpf(1.0f + exp_of(-v));
  if constexpr (ACT == kGelu) {
    const float z = v * -0.70710678118654752f, x = fabsf(z);
    const float t = __builtin_amdgcn_rcpf(fmaf(0.5f, x, 1.0f));
    float p = 0.17087277f;
    p = fmaf(p, t, -0.82215223f);
    p = fmaf(p, t, 1.48851587f);
    p = fmaf(p, t, -1.13520398f);
    p = fmaf(p, t, 0.27886807f);
    p = fmaf(p, t, -0.18628806f);
    p = fmaf(p, t, 0.09678418f);
    p = fmaf(p, t, 0.37409196f);
    p = fmaf(p, t, 1.00002368f);
    p = fmaf(p, t, -1.26551223f);
    const float tail = t * exp_of(fmaf(-x, x, p));
    const float erfc = z >= 0.0f ? tail : 2.0f - tail;
    // v = -infinity: 0 * infinity is NaN, as its row stands for anyway
    return 0.5f * v * (z == z ? erfc : z);
  }
  return act_of<ACT>(v);
}

template <typename T, int ACT, bool GATED>
__device__ __forceinline__ typename Vec<kWide<T>>::type activated(const T* row, int64_t at, int c, int left) {
  auto v = load_some<false>(row + at, left);
  if constexpr (GATED) {
    const auto up = load_some<false>(row + c + at, left);
#pragma unroll
    for (int i = 0; i < kWide<T>; ++i) v[i] = code_act<ACT>(v[i]) * up[i];
  } else {
#pragma unroll
    for (int i = 0; i < kWide<T>; ++i) v[i] = code_act<ACT>(v[i]);
  }
  return v;
}

template <typename T, int ACT, bool GATED, int THREADS, int V>
__global__ __launch_bounds__(kRowBlock<THREADS>) void act_row8_kernel(ActRow8Args a) {
  constexpr int W = kWide<T>;
  constexpr int kRows = kRowBlock<THREADS> / THREADS;
  typedef typename Vec<W>::type Run;
  __shared__ RowSums<THREADS> lds;
  const int t = static_cast<int>(threadIdx.x) % THREADS;
  int turn = 0;
  for (int64_t row = static_cast<int64_t>(blockIdx.x) * kRows + static_cast<int>(threadIdx.x) / THREADS; row < a.rows;
       row += static_cast<int64_t>(gridDim.x) * kRows) {
    Run v[V];
    unsigned top = 0;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int col = (j * THREADS + t) * W;
      v[j] = activated<T, ACT, GATED>(static_cast<const T*>(a.x) + row * a.ld_x, col, a.c, a.c - col);
#pragma unroll
      for (int i = 0; i < W; ++i) top = max(top, magnitude(v[j][i]));
    }
    reduce_row<THREADS>(lds, turn, nullptr, nullptr, &top);
    turn ^= 1;
    const RowCode code = code_of(top);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int col = (j * THREADS + t) * W;
      store_codes<W>(a.codes + row * a.c + col, v[j], code.inverse, code.bad, a.c - col);
    }
    if (t == 0) a.scales[row] = code.scale;
  }
}

// Rows longer than the registers of a workgroup: read twice.
template <typename T, int ACT, bool GATED>
__global__ __launch_bounds__(1024) void act_row8_long_kernel(ActRow8Args a) {
  constexpr int W = kWide<T>, kThreads = 1024;
  __shared__ RowSums<kThreads> lds;
  int turn = 0;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* const x = static_cast<const T*>(a.x) + row * a.ld_x;
    unsigned top = 0;
    for (int64_t at = static_cast<int64_t>(threadIdx.x) * W; at < a.c; at += kThreads * W) {
      const auto v = activated<T, ACT, GATED>(x, at, a.c, static_cast<int>(a.c - at));
#pragma unroll
      for (int i = 0; i < W; ++i) top = max(top, magnitude(v[i]));
    }
    reduce_row<kThreads>(lds, turn, nullptr, nullptr, &top);
    turn ^= 1;
    const RowCode code = code_of(top);
    for (int64_t at = static_cast<int64_t>(threadIdx.x) * W; at < a.c; at += kThreads * W) {
      const int left = static_cast<int>(a.c - at);
      const auto v = activated<T, ACT, GATED>(x, at, a.c, left);
      store_codes<W>(a.codes + row * a.c + at, v, code.inverse, code.bad, left);
    }
    if (threadIdx.x == 0) a.scales[row] = code.scale;
  }
}

// What the codes stand for: 16 bytes of output a lane.
struct Expand {
  int64_t total, ld_y;  // lanes
  int c, per_row;
  FastDivM div;  // by per_row
};
template <typename T>
__global__ __launch_bounds__(256) void row8_expand_kernel(Expand e, const int8_t* __restrict__ codes,
                                                          const float* __restrict__ scales, T* __restrict__ y) {
  constexpr int W = kWide<T>;
  typedef typename Vec<W>::type Run;
  for (int64_t base = static_cast<int64_t>(blockIdx.x) * 256; base < e.total; base += static_cast<int64_t>(gridDim.x) * 256) {
    if (base + threadIdx.x >= e.total) continue;
    const int64_t row0 = base / e.per_row;  // the workgroup's, one division
    const int at = static_cast<int>(base - row0 * e.per_row) + static_cast<int>(threadIdx.x);
    const int over = fdiv(at, e.div);
    const int64_t row = row0 + over;
    const int col = (at - over * e.per_row) * W, left = e.c - col;
    const int8_t* const from = codes + row * e.c + col;
    int q[W / 4] = {};
    if (left >= W) {
      if constexpr (W == 8) {
        const v2i w = *reinterpret_cast<const v2i_any*>(from);
        q[0] = w[0];
        q[1] = w[1];
      } else {
        q[0] = *reinterpret_cast<const int_any*>(from);
      }
    } else {
#pragma unroll
      for (int i = 0; i < W; ++i)
        if (i < left) q[i / 4] |= (from[i] & 0xff) << (8 * (i & 3));
    }
    const float scale = scales[row];
    Run v;
#pragma unroll
    for (int i = 0; i < W; i += 4) {
      const v4f four = codes4(q[i / 4]) * scale;
#pragma unroll
      for (int j = 0; j < 4; ++j) v[i + j] = four[j];
    }
    store_some<false>(y + row * e.ld_y + col, v, left);
  }
}

// Rows of codes to rows of whole lines, 16 bytes a lane.
struct Pad {
  int64_t total, x_rows;  // lanes
  int c, per_row;
  FastDivM div;  // by per_row
};
__global__ __launch_bounds__(256) void row8_pad_kernel(Pad p, const int8_t* __restrict__ x, const int8_t* __restrict__ w,
                                                       int8_t* __restrict__ to) {
  for (int64_t base = static_cast<int64_t>(blockIdx.x) * 256; base < p.total; base += static_cast<int64_t>(gridDim.x) * 256) {
    const int64_t lane = base + threadIdx.x;
    if (lane >= p.total) continue;
    const int64_t row0 = base / p.per_row;  // the workgroup's, one division
    const int at = static_cast<int>(base - row0 * p.per_row) + static_cast<int>(threadIdx.x);
    const int over = fdiv(at, p.div);
    const int64_t row = row0 + over;
    const int col = (at - over * p.per_row) * 16;
    const int8_t* const from = row < p.x_rows ? x + row * p.c : w + (row - p.x_rows) * p.c;
    const v4i v = col + 16 <= p.c ? load16<true>(from + col) : load_codes16(from, col, p.c);
    reinterpret_cast<v4i*>(to)[lane] = v;
    store_gap(v);
  }
}

template <typename T, int ACT, bool GATED>
void launch_act(const ActRow8Args& a, hipStream_t stream) {
  const RowShape shape = row_shape(a.c, kWide<T>, a.rows);
  by_shape(shape, [&](auto threads, auto runs) {
    constexpr int THREADS = threads.value, V = runs.value;
    if constexpr (V == 0) {
      act_row8_long_kernel<T, ACT, GATED><<<row_blocks(shape, a.rows, 1 << 16), 1024, 0, stream>>>(a);
    } else {
      act_row8_kernel<T, ACT, GATED, THREADS, V>
          <<<row_blocks(shape, a.rows, 1 << 20), kRowBlock<THREADS>, 0, stream>>>(a);
    }
  });
}

template <typename T, int ACT>
void by_gate(const ActRow8Args& a, hipStream_t stream) {
  a.gated ? launch_act<T, ACT, true>(a, stream) : launch_act<T, ACT, false>(a, stream);
}

template <typename T>
void by_act(const ActRow8Args& a, hipStream_t stream) {
  switch (a.act) {
    case kRelu: by_gate<T, kRelu>(a, stream); break;
    case kSilu: by_gate<T, kSilu>(a, stream); break;
    case kGelu: by_gate<T, kGelu>(a, stream); break;
    default: by_gate<T, kNone>(a, stream); break;
  }
}

}  // namespace

hipError_t launch_act_row8(const ActRow8Args& a, hipStream_t stream) {
  a.bf16 ? by_act<__bf16>(a, stream) : by_act<float>(a, stream);
  return hipGetLastError();
}

hipError_t launch_row8_pad(const int8_t* x, int64_t x_rows, const int8_t* w, int64_t w_rows, int32_t c, int32_t width,
                           int8_t* to, hipStream_t stream) {
  Pad p{};
  p.c = c;
  p.x_rows = x_rows;
  p.per_row = width / 16;
  p.total = (x_rows + w_rows) * p.per_row;
  p.div = fastdiv_m(static_cast<uint32_t>(p.per_row));
  const int64_t blocks = (p.total + 255) / 256;
  const unsigned grid = static_cast<unsigned>(blocks < (1 << 23) ? blocks : (1 << 23));
  row8_pad_kernel<<<grid, 256, 0, stream>>>(p, x, w, to);
  return hipGetLastError();
}

hipError_t launch_row8_expand(const Row8ExpandArgs& a, hipStream_t stream) {
  const int wide = a.bf16 ? 8 : 4;
  Expand e{};
  e.per_row = static_cast<int>((static_cast<int64_t>(a.c) + wide - 1) / wide);
  e.total = a.rows * e.per_row;
  e.ld_y = a.ld_y;
  e.c = a.c;
  e.div = fastdiv_m(static_cast<uint32_t>(e.per_row));
  const int64_t blocks = (e.total + 255) / 256;
  const unsigned grid = static_cast<unsigned>(blocks < (1 << 23) ? blocks : (1 << 23));
  if (a.bf16) row8_expand_kernel<<<grid, 256, 0, stream>>>(e, a.codes, a.scales, static_cast<__bf16*>(a.y));
  else row8_expand_kernel<<<grid, 256, 0, stream>>>(e, a.codes, a.scales, static_cast<float*>(a.y));
  return hipGetLastError();
}

}  // namespace miq
