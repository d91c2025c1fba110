// Device helpers shared by the token-network kernels: runs of a row's values as fp32, codes as fp32,
// activations, token ids.
#pragma once

#include "qconv_device.h"
#include "train_internal.h"

namespace miq {
namespace {

typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef float v8f __attribute__((ext_vector_type(8)));
typedef int v2i __attribute__((ext_vector_type(2)));
// Rows start at any multiple of the element's size: global memory takes 16-byte accesses at any
// address, so odd row lengths run the same loads and stores as aligned ones.
typedef v8bf v8bf_any __attribute__((aligned(2)));
typedef v4f v4f_any __attribute__((aligned(4)));
typedef v2i v2i_any __attribute__((aligned(1)));
typedef int int_any __attribute__((aligned(1)));

__device__ __forceinline__ v8f load8(const float* p) {
  const v4f a = *reinterpret_cast<const v4f_any*>(p), b = *reinterpret_cast<const v4f_any*>(p + 4);
  return v8f{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
}
__device__ __forceinline__ v8f load8(const __bf16* p) {
  return __builtin_convertvector(*reinterpret_cast<const v8bf_any*>(p), v8f);
}
// The first n (0 .. 8) of eight values; the rest read zero.
template <typename T>
__device__ __forceinline__ v8f load8_of(const T* p, int n) {
  if (n >= 8) return load8(p);
  v8f v = {};
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i < n) v[i] = static_cast<float>(p[i]);
  return v;
}

// 16 bytes of a row; past the caches (STREAM) for outputs that no cache holds until they are read, as
// stream_stores() says.
template <bool STREAM>
__device__ __forceinline__ void store_run(__bf16* p, const v8f& v) {
  const v8bf b = __builtin_convertvector(v, v8bf);  // to nearest even
  if constexpr (STREAM) __builtin_nontemporal_store(b, reinterpret_cast<v8bf_any*>(p));
  else *reinterpret_cast<v8bf_any*>(p) = b;
  store_gap(__builtin_bit_cast(v4i, b));
}
template <bool STREAM>
__device__ __forceinline__ void store_run(float* p, const v4f& v) {
  if constexpr (STREAM) __builtin_nontemporal_store(v, reinterpret_cast<v4f_any*>(p));
  else *reinterpret_cast<v4f_any*>(p) = v;
  store_gap(v);
}

// Eight values as two runs of four, `apart` elements from each other: neighbouring lanes' runs are
// neighbours in memory, so that every store of a wave covers whole lines.
typedef __bf16 v4bf __attribute__((ext_vector_type(4)));
typedef v4bf v4bf_any __attribute__((aligned(2)));

__device__ __forceinline__ v4f load4(const float* p) { return *reinterpret_cast<const v4f_any*>(p); }
__device__ __forceinline__ v4f load4(const __bf16* p) {
  return __builtin_convertvector(*reinterpret_cast<const v4bf_any*>(p), v4f);
}
template <typename T>
__device__ __forceinline__ v8f load44(const T* p, int apart) {
  return __builtin_shufflevector(load4(p), load4(p + apart), 0, 1, 2, 3, 4, 5, 6, 7);
}
__device__ __forceinline__ void store44(float* p, int apart, const v8f& v) {
  store_run<false>(p, __builtin_shufflevector(v, v, 0, 1, 2, 3));
  store_run<false>(p + apart, __builtin_shufflevector(v, v, 4, 5, 6, 7));
}
// Of a row that ends n elements after p.
template <typename T>
__device__ __forceinline__ v8f load44_of(const T* p, int apart, int n) {
  v8f v = {};
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (h * apart + i < n) v[4 * h + i] = static_cast<float>(p[h * apart + i]);
  return v;
}
template <typename T>
__device__ __forceinline__ void store44_of(T* p, int apart, const v8f& v, int n) {
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (h * apart + i < n) p[h * apart + i] = static_cast<T>(v[4 * h + i]);
}

// Four int8 codes of a word as fp32, one conversion with a byte select each.  (A vector conversion
// of eight chars takes the last one through 64-bit integers.)
__device__ __forceinline__ v4f codes4(int w) {
  return v4f{static_cast<float>(static_cast<signed char>(w)), static_cast<float>(static_cast<signed char>(w >> 8)),
             static_cast<float>(static_cast<signed char>(w >> 16)), static_cast<float>(w >> 24)};
}

__device__ __forceinline__ int64_t load_id(const void* ids, bool wide, int64_t t) {
  return wide ? static_cast<const int64_t*>(ids)[t] : static_cast<const int32_t*>(ids)[t];
}

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

// Whether an output of `rows` rows of `width` values, `ld` apart, is written past the caches: rows of
// whole 64-byte lines, and more than half of the 256 MB last-level cache, so that little of it
// would be there for a reader.  Lookup of 65536 rows of 2048, 268 MB: 95 -> 86 us; gated act8 of
// 16384 x 8192 forward and backward 453 -> 442 us.  Rows that share lines lose: 73 -> 87 us on a
// table gradient of 50021 x 1001.
inline bool stream_stores(const void* p, int64_t rows, int64_t width, int64_t ld, int64_t size) {
  return reinterpret_cast<uintptr_t>(p) % 64 == 0 && ld * size % 64 == 0 && rows * width * size > (int64_t{128} << 20);
}

}  // namespace
}  // namespace miq
