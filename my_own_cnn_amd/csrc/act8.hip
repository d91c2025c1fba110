// Activations whose input is kept in 8 bits (miq_act8_fprop, _bprop, _expand).
//
// Every kernel is one pass over its tensors.  A lane holds 16 bytes of consecutive channels (8 of
// bf16, 4 of fp32), so 4 or 8 neighbouring lanes share one exponent byte; a row's chunks are padded
// to whole groups, which keeps those lanes in one row whatever the row's length.  The largest
// magnitude of a group goes round its lanes by two or three exchanges; scaling by a power of two is
// exact, so the codes depend on no rounding but their own.
//
// Bound by memory in fp32 and with relu: 4.8 TB/s, what a large copy reaches, and more.  bf16 moves
// half the bytes a value, so there the exponential, the division and erfc of silu and gelu take the
// longer: ungated on 16384 x 8192, forward and backward, relu 5.9 and 5.9 TB/s, silu 4.4 and 4.1, gelu
// 3.4 and 2.8 (243 us); gated 6.1 and 6.4, 5.3 and 4.5, 4.5 and 3.7.  Vector instructions per value,
// forward and backward: relu 20 and 16, silu 43 and 41, gelu 69 and 79; ungated silu and gelu issue one
// each 3.4 to 4.8 cycles and SIMD at 2.4 GHz, and are bound by that.  fp32 on 8192 x 8192, gelu: 4.7 and
// 4.2 TB/s ungated, 5.7 and 5.4 gated.
//
// Gated silu on 16384 x 8192 bf16, one after the other: 453 us, 436 with stores past the caches, 427 to
// 435 with loads past them too.  50176 x 128 fp32 kept and expanded: 8.7 and 7.8 us for 32 MB each,
// some 2 of them the launch.  Stores of 32 bytes per lane of fp32 took 8.7 us to expand; lanes of 8 fp32
// values kept faster (7.6 us) and expanded slower.
#include "train_device.h"

namespace miq {
namespace {

constexpr int kThreads = 256;

enum Act : int { kNone = 0, kRelu = 1, kSilu = 2, kGelu = 3 };

// act(v).  NaN stays NaN.
template <int ACT>
__device__ __forceinline__ float act_of(float v) {
  if constexpr (ACT == kRelu) return v < 0.0f ? 0.0f : v;
  if constexpr (ACT == kSilu) return v / (1.0f + expf(-v));
  if constexpr (ACT == kGelu) return 0.5f * v * erfcf(v * -0.70710678118654752f);
  return v;
}

// act'(v); 0 at relu's corner.
template <int ACT>
__device__ __forceinline__ float slope_of(float v) {
  if constexpr (ACT == kRelu) return v > 0.0f ? 1.0f : (v <= 0.0f ? 0.0f : v);
  if constexpr (ACT == kSilu) {
    const float s = 1.0f / (1.0f + expf(-v));
    return s * (1.0f + v * (1.0f - s));
  }
  if constexpr (ACT == kGelu)
    return 0.5f * erfcf(v * -0.70710678118654752f) + v * expf(-0.5f * v * v) * 0.39894228040143268f;
  return 1.0f;
}

struct Rows {
  int64_t total;     // chunks of a lane's channels, rows padded to whole groups
  int64_t ld_x, ld_dy, ld_y;
  int c, groups, per_row;  // chunks per row: groups * (32 / a lane's channels)
  FastDivM div;            // by per_row
};

// A lane's channels: 16 bytes of the tensor's type.
template <typename T>
constexpr int kWide = 16 / static_cast<int>(sizeof(T));

template <int W>
struct Vec;
template <>
struct Vec<8> {
  typedef v8f type;
};
template <>
struct Vec<4> {
  typedef v4f type;
};

// Past the caches too where the output is (STREAM): what is read once leaves no room for what is not.
template <bool STREAM>
__device__ __forceinline__ v8f load_run(const __bf16* p) {
  const v8bf_any* const q = reinterpret_cast<const v8bf_any*>(p);
  if constexpr (STREAM) return __builtin_convertvector(__builtin_nontemporal_load(q), v8f);
  else return __builtin_convertvector(*q, v8f);
}
template <bool STREAM>
__device__ __forceinline__ v4f load_run(const float* p) {
  const v4f_any* const q = reinterpret_cast<const v4f_any*>(p);
  if constexpr (STREAM) return __builtin_nontemporal_load(q);
  else return *q;
}
template <bool STREAM>
__device__ __forceinline__ void load_codes(const int8_t* p, int (&q)[2]) {
  const v2i_any* const from = reinterpret_cast<const v2i_any*>(p);
  v2i w;
  if constexpr (STREAM) w = __builtin_nontemporal_load(from);
  else w = *from;
  q[0] = w[0];
  q[1] = w[1];
}
template <bool STREAM>
__device__ __forceinline__ void load_codes(const int8_t* p, int (&q)[1]) {
  const int_any* const from = reinterpret_cast<const int_any*>(p);
  if constexpr (STREAM) q[0] = __builtin_nontemporal_load(from);
  else q[0] = *from;
}

// The first `left` of a lane's channels; the rest read zero and are not stored.
template <bool STREAM, typename T>
__device__ __forceinline__ typename Vec<kWide<T>>::type load_some(const T* p, int left) {
  if (left >= kWide<T>) return load_run<STREAM>(p);
  typename Vec<kWide<T>>::type v = {};
#pragma unroll
  for (int i = 0; i < kWide<T>; ++i)
    if (i < left) v[i] = static_cast<float>(p[i]);
  return v;
}
template <bool STREAM, typename T>
__device__ __forceinline__ void store_some(T* p, const typename Vec<kWide<T>>::type& v, int left) {
  if (left >= kWide<T>) {
    store_run<STREAM>(p, v);
    return;
  }
#pragma unroll
  for (int i = 0; i < kWide<T>; ++i)
    if (i < left) p[i] = static_cast<T>(v[i]);
}

// (row, channel, channels left) of this thread's chunk of W; false past the end
template <int W>
__device__ __forceinline__ bool place(const Rows& r, int64_t block, int64_t* row, int* col, int* left) {
  const int64_t base = block * kThreads;
  const int64_t row0 = base / r.per_row;  // the workgroup's, one division
  const int at = static_cast<int>(base - row0 * r.per_row) + threadIdx.x;
  const int over = fdiv(at, r.div);
  *row = row0 + over;
  *col = (at - over * r.per_row) * W;
  *left = r.c - *col;
  return base + threadIdx.x < r.total;
}

// The exponent byte of a group, from its largest magnitude (as fp32 bits) in all of its lanes (4 of
// bf16, 8 of fp32).
__device__ __forceinline__ int exponent_byte(unsigned top) {
  const int e = static_cast<int>(top >> 23) - 6 + ((top & 0x7fffffu) >= 0x7f0000u ? 1 : 0);
  return top >= 0x7f800000u ? 255 : min(max(e, 1), 248);
}

// Keeps a lane's W values: codes at `codes`, the group's byte at `scale` (by its first lane).
template <int W>
__device__ __forceinline__ void keep(const typename Vec<W>::type& v, int left, int8_t* codes, uint8_t* scale) {
  unsigned top = 0;  // magnitudes order as their bits do, NaN above infinity
#pragma unroll
  for (int i = 0; i < W; ++i) top = max(top, __float_as_uint(v[i]) & 0x7fffffffu);
#pragma unroll
  for (int step = 1; step < kAct8Group / W; step *= 2)
    top = max(top, static_cast<unsigned>(__shfl_xor(static_cast<int>(top), step)));
  const int byte = exponent_byte(top);
  // 2^(127 - byte), a normal number for every byte below 254; the products are exact or below half
  // a code, and adding 1.5 * 2^23 rounds them to nearest even into the low byte
  const float inverse = __uint_as_float(static_cast<unsigned>(254 - min(byte, 253)) << 23);
  float r[W];
#pragma unroll
  for (int i = 0; i < W; ++i) r[i] = __builtin_amdgcn_fmed3f(v[i] * inverse, -127.0f, 127.0f) + 12582912.0f;
  int q[W / 4];
#pragma unroll
  for (int i = 0; i < W; i += 4)
    q[i / 4] = byte == 255 ? 0 : static_cast<int>(pack4_magic(r[i], r[i + 1], r[i + 2], r[i + 3]));  // 255: not finite
  if (left >= W) {
    if constexpr (W == 8) *reinterpret_cast<v2i_any*>(codes) = v2i{q[0], q[1]};
    else *reinterpret_cast<int_any*>(codes) = q[0];
  } else {
#pragma unroll
    for (int i = 0; i < W; ++i)
      if (i < left) codes[i] = static_cast<int8_t>(q[i / 4] >> (8 * (i & 3)));
  }
  if ((threadIdx.x & (kAct8Group / W - 1)) == 0) *scale = static_cast<uint8_t>(byte);
}

template <bool STREAM, int W>
__device__ __forceinline__ typename Vec<W>::type kept(const int8_t* codes, const uint8_t* scale, int left) {
  int q[W / 4] = {};
  if (left >= W) {
    load_codes<STREAM>(codes, q);
  } else {
#pragma unroll
    for (int i = 0; i < W; ++i)
      if (i < left) q[i / 4] |= (codes[i] & 0xff) << (8 * (i & 3));
  }
  // byte 255 is the bits of infinity, which a zero code makes NaN
  const float s = __uint_as_float(static_cast<unsigned>(*scale) << 23);
  typename Vec<W>::type v;
#pragma unroll
  for (int i = 0; i < W; i += 4) {
    const v4f four = codes4(q[i / 4]) * s;
#pragma unroll
    for (int j = 0; j < 4; ++j) v[i + j] = four[j];
  }
  return v;
}

template <typename T, int ACT, bool GATED, bool STREAM>
__global__ __launch_bounds__(kThreads) void act8_fprop_kernel(Rows r, const T* __restrict__ x, T* __restrict__ y,
                                                              int8_t* __restrict__ codes, uint8_t* __restrict__ scales) {
  constexpr int H = GATED ? 2 : 1, W = kWide<T>;
  typedef typename Vec<W>::type V;
  for (int64_t b = blockIdx.x; b * kThreads < r.total; b += gridDim.x) {
    int64_t row;
    int at, left;
    if (!place<W>(r, b, &row, &at, &left)) continue;  // whole groups of lanes leave together
    V v[H];
#pragma unroll
    for (int h = 0; h < H; ++h) {
      const int col = h * r.c + at;
      v[h] = load_some<STREAM>(x + row * r.ld_x + col, left);
      keep<W>(v[h], left, codes + row * (H * static_cast<int64_t>(r.c)) + col,
              scales + (row * H + h) * r.groups + at / kAct8Group);
    }
    if (y != nullptr) {
      V out;
#pragma unroll
      for (int i = 0; i < W; ++i) out[i] = act_of<ACT>(v[0][i]) * (GATED ? v[H - 1][i] : 1.0f);
      store_some<STREAM>(y + row * r.ld_y + at, out, left);
    }
  }
}

template <typename T, int ACT, bool GATED, bool STREAM>
__global__ __launch_bounds__(kThreads) void act8_bprop_kernel(Rows r, const T* __restrict__ dy,
                                                              const int8_t* __restrict__ codes,
                                                              const uint8_t* __restrict__ scales, T* __restrict__ dx) {
  constexpr int H = GATED ? 2 : 1, W = kWide<T>;
  typedef typename Vec<W>::type V;
  for (int64_t b = blockIdx.x; b * kThreads < r.total; b += gridDim.x) {
    int64_t row;
    int at, left;
    if (!place<W>(r, b, &row, &at, &left) || left <= 0) continue;
    const V d = load_some<STREAM>(dy + row * r.ld_dy + at, left);
    V v[H];
#pragma unroll
    for (int h = 0; h < H; ++h)
      v[h] = kept<STREAM, W>(codes + row * (H * static_cast<int64_t>(r.c)) + h * r.c + at,
                     scales + (row * H + h) * r.groups + at / kAct8Group, left);
    V g;
#pragma unroll
    for (int i = 0; i < W; ++i) g[i] = d[i] * (GATED ? v[H - 1][i] : 1.0f) * slope_of<ACT>(v[0][i]);
    store_some<STREAM>(dx + row * r.ld_y + at, g, left);
    if constexpr (GATED) {
#pragma unroll
      for (int i = 0; i < W; ++i) g[i] = d[i] * act_of<ACT>(v[0][i]);
      store_some<STREAM>(dx + row * r.ld_y + r.c + at, g, left);
    }
  }
}

template <typename T, int ACT, bool GATED, bool STREAM>
__global__ __launch_bounds__(kThreads) void act8_expand_kernel(Rows r, const int8_t* __restrict__ codes,
                                                               const uint8_t* __restrict__ scales, T* __restrict__ y) {
  constexpr int H = GATED ? 2 : 1, W = kWide<T>;
  typedef typename Vec<W>::type V;
  for (int64_t b = blockIdx.x; b * kThreads < r.total; b += gridDim.x) {
    int64_t row;
    int at, left;
    if (!place<W>(r, b, &row, &at, &left) || left <= 0) continue;
    V v[H];
#pragma unroll
    for (int h = 0; h < H; ++h)
      v[h] = kept<STREAM, W>(codes + row * (H * static_cast<int64_t>(r.c)) + h * r.c + at,
                     scales + (row * H + h) * r.groups + at / kAct8Group, left);
    V out;
#pragma unroll
    for (int i = 0; i < W; ++i) out[i] = act_of<ACT>(v[0][i]) * (GATED ? v[H - 1][i] : 1.0f);
    store_some<STREAM>(y + row * r.ld_y + at, out, left);
  }
}

Rows rows_of(const Act8Args& a) {
  Rows r{};
  const int64_t groups = (static_cast<int64_t>(a.c) + kAct8Group - 1) / kAct8Group;
  r.groups = static_cast<int>(groups);
  r.per_row = static_cast<int>(groups * (a.bf16 ? 4 : 8));
  r.total = a.rows * r.per_row;
  r.ld_x = a.ld_x;
  r.ld_dy = a.ld_dy;
  r.ld_y = a.ld_y;
  r.c = a.c;
  r.div = fastdiv_m(static_cast<uint32_t>(r.per_row));
  return r;
}

// Calls go(type, act, gated, stream) with the four as compile-time values; `wide`: the length of an
// output row in units of c.
template <typename F>
void dispatch(const Act8Args& a, int wide, F&& go) {
  const bool stream = stream_stores(a.y, a.rows, static_cast<int64_t>(a.c) * wide, a.ld_y, a.bf16 ? 2 : 4);
  auto by_stream = [&](auto type, auto act, auto gated) {
    stream ? go(type, act, gated, std::true_type{}) : go(type, act, gated, std::false_type{});
  };
  auto by_gate = [&](auto type, auto act) {
    a.gated ? by_stream(type, act, std::true_type{}) : by_stream(type, act, std::false_type{});
  };
  auto by_act = [&](auto type) {
    switch (a.act) {
      case kRelu: by_gate(type, std::integral_constant<int, kRelu>{}); break;
      case kSilu: by_gate(type, std::integral_constant<int, kSilu>{}); break;
      case kGelu: by_gate(type, std::integral_constant<int, kGelu>{}); break;
      default: by_gate(type, std::integral_constant<int, kNone>{}); break;
    }
  };
  a.bf16 ? by_act(__bf16{}) : by_act(float{});
}

unsigned blocks_of(const Rows& r) {
  const int64_t blocks = (r.total + kThreads - 1) / kThreads;
  return static_cast<unsigned>(blocks < (1 << 23) ? blocks : (1 << 23));
}

}  // namespace

hipError_t launch_act8_fprop(const Act8Args& a, hipStream_t stream) {
  const Rows r = rows_of(a);
  dispatch(a, 1, [&](auto type, auto act, auto gated, auto past) {
    using T = decltype(type);
    act8_fprop_kernel<T, act.value, gated.value, past.value><<<blocks_of(r), kThreads, 0, stream>>>(
        r, static_cast<const T*>(a.x), static_cast<T*>(a.y), a.codes, a.scales);
  });
  return hipGetLastError();
}

hipError_t launch_act8_bprop(const Act8Args& a, hipStream_t stream) {
  const Rows r = rows_of(a);
  dispatch(a, a.gated ? 2 : 1, [&](auto type, auto act, auto gated, auto past) {
    using T = decltype(type);
    act8_bprop_kernel<T, act.value, gated.value, past.value><<<blocks_of(r), kThreads, 0, stream>>>(
        r, static_cast<const T*>(a.dy), a.codes, a.scales, static_cast<T*>(a.y));
  });
  return hipGetLastError();
}

hipError_t launch_act8_expand(const Act8Args& a, hipStream_t stream) {
  const Rows r = rows_of(a);
  dispatch(a, 1, [&](auto type, auto act, auto gated, auto past) {
    using T = decltype(type);
    act8_expand_kernel<T, act.value, gated.value, past.value><<<blocks_of(r), kThreads, 0, stream>>>(
        r, a.codes, a.scales, static_cast<T*>(a.y));
  });
  return hipGetLastError();
}

}  // namespace miq
