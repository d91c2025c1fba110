// dw[j, i] = sum over m of dy[m, j] * x'[m, i] with x' kept in 8 bits (miq_act8_grad).
//
// A kept value, code * 2^e with |code| <= 127, is exact in bf16: bf16 dy multiplies it directly
// on the bf16 matrix instructions with fp32 sums; fp32 dy is split into three bf16 numbers that
// add up to it (8 + 8 + 8 significant bits, exactly from 2^-110 up), three products a term where
// two fp32 operands would need six.
//
// A workgroup computes a square tile of dw over a range of the rows m, 32 rows a step.  A step's
// values travel global memory -> registers -> LDS, where both operands lie as bf16 rows [m][j] and
// [m][i]; the codes are turned into bf16 on that way, once per value (a byte-select conversion, a
// product, half a pack).  The matrix instructions want eight consecutive m of one column per lane:
// the transposing LDS read gives a lane four m of its column at once.  The rows of LDS are permuted
// in units of 16 columns (32 bytes) by their m, so that a read meets no bank twice.
//
// Bound by the matrix instructions and the power they draw: 4096 x 4096 over 16384 bf16 rows takes 460
// to 471 us from card to card, 1168 to 1195 TFLOP/s, at some 2.0 GHz, the matrix units busy 56% of the
// cycles (a library product of the same operands in bf16: 552 us).  What it took, in us: 128-square
// tiles and transposed 2-byte LDS stores 7386; this layout 629; loads without branches, two steps of
// them in flight and the conversions spread between the matrix instructions 485; eight waves of
// 64 x 128 instead of four of 128 x 128 472; no bank conflicts, and five stages with a barrier every
// second step 460.  fp32, 4096 cubed: 349 to 360 us, 381 to 394 TFLOP/s (three times that of bf16),
// on two stages.  512 x 128 over 50176 fp32 rows, the reading of 110 MB: 39 us, 32 in the product
// (3.4 TB/s) and 6 in the join of 63 partial sums.  The smaller tiles do less: 2048 cubed in bf16 33 to
// 37 us, 470 to 520 TFLOP/s.
#include "train_device.h"

namespace miq {
namespace {

constexpr int kThreads = 256;
constexpr int kStep = 32;  // rows m per step

typedef short v4s __attribute__((ext_vector_type(4)));
typedef float v16f __attribute__((ext_vector_type(16)));
typedef v4i v4i_any __attribute__((aligned(1)));

struct Grad {
  const void* dy;
  const int8_t* codes;
  const uint8_t* scales;
  void* out;
  int64_t ld_dy, ld_out;
  int rows, c, k, groups, tiles_k, tiles_c, per_split;
  bool accumulate, to_parts;
};

// Eight values of dy on their way to LDS.
template <typename T>
struct Raw;
template <>
struct Raw<__bf16> {
  v8bf v;
};
template <>
struct Raw<float> {
  v8f v;
};

__device__ __forceinline__ void load_raw(Raw<__bf16>& r, const __bf16* p, int n) {
  if (n >= 8) {
    r.v = *reinterpret_cast<const v8bf_any*>(p);
  } else {
    r.v = v8bf{};
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) r.v[i] = p[i];
  }
}
__device__ __forceinline__ void load_raw(Raw<float>& r, const float* p, int n) { r.v = load8_of(p, n); }

// The P bf16 numbers that add up to each of eight values.
__device__ __forceinline__ void split8(const Raw<__bf16>& r, v8bf (&p)[1]) { p[0] = r.v; }
__device__ __forceinline__ void split8(const Raw<float>& r, v8bf (&p)[3]) {
  v8f a, b, c;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    // Truncation leaves at most 16, then 8 significant bits; an infinity or a NaN stays in the
    // first number alone.
    const unsigned bits = __float_as_uint(r.v[i]);
    const bool finite = (bits & 0x7f800000u) != 0x7f800000u;
    const unsigned quiet = (bits & 0x7fffffffu) > 0x7f800000u ? 0x400000u : 0u;
    a[i] = __uint_as_float((bits | quiet) & 0xffff0000u);
    const float rest = finite ? r.v[i] - a[i] : 0.0f;
    b[i] = __uint_as_float(__float_as_uint(rest) & 0xffff0000u);
    c[i] = rest - b[i];
  }
  p[0] = __builtin_convertvector(a, v8bf);
  p[1] = __builtin_convertvector(b, v8bf);
  p[2] = __builtin_convertvector(c, v8bf);
}

// The permutation of a row's 32-byte units: the 32 lanes that a transposing read serves at once take
// two neighbouring units of four rows, and these eight lie in different banks, 256 bytes in all.
template <int W>
__device__ __forceinline__ int turn(int m) {
  return W >= 128 ? ((m & 3) << 1) | ((m >> 2) & 1) : (m & 2) | ((m >> 2) & 1);
}

template <typename T, typename TO, int P, int TK, int TC, int VK, int VC, int STAGES, int SETS>
__global__ __launch_bounds__(VK* VC * 64, TK* TC >= 256 * 256 ? 1 : 2) void act8_grad_kernel(Grad g) {
  constexpr int kThreads = VK * VC * 64;
  constexpr int kPitchA = TK * 2, kPitchB = TC * 2;      // bytes
  constexpr int kPlane = kStep * kPitchA;
  constexpr int kStage = P * kPlane + kStep * kPitchB;
  constexpr int NA = kStep * TK / 8 / kThreads;          // chunks of eight values of dy per thread
  constexpr int CB = kStep * TC / kThreads < 16 ? 8 : 16;  // codes per chunk
  constexpr int NB = kStep * TC / CB / kThreads;
  constexpr int WK = TK / VK, WC = TC / VC;              // a wave's part
  constexpr int IA = WK / 32, IB = WC / 32;
  extern __shared__ __attribute__((aligned(16))) char lds[];

  const int tiles = g.tiles_k * g.tiles_c;
  const int at = xcd_tile(blockIdx.x, gridDim.x);
  const int part = at / tiles;
  // tiles in bands of four along k: neighbours share their rows of both operands in L2
  const int tile = at - part * tiles;
  const int band = tile / (4 * g.tiles_c);
  const int high = min(4, g.tiles_k - 4 * band);
  const int in = tile - band * 4 * g.tiles_c;
  const int k0 = (band * 4 + in % high) * TK;
  const int c0 = (in / high) * TC;
  const int m0 = part * g.per_split;  // below rows
  const int m1 = static_cast<int>(min(static_cast<int64_t>(m0) + g.per_split, static_cast<int64_t>(g.rows)));
  const int steps = m1 > m0 ? (m1 - m0 + kStep - 1) / kStep : 0;

  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = tid >> 6;
  const int wk = (wave / VC) * WK, wc = (wave % VC) * WC;

  // a thread's chunks: rows a_row + i * kRowsA and b_row + i * kRowsB, always the same columns
  const int a_row = tid / (TK / 8), a_col = (tid % (TK / 8)) * 8;
  const int b_row = tid / (TC / CB), b_col = (tid % (TC / CB)) * CB;
  constexpr int kRowsA = kThreads * 8 / TK, kRowsB = kThreads * CB / TC;
  const int a_left = g.k - k0 - a_col;
  const int b_left = g.c - c0 - b_col;
  const T* a_from = static_cast<const T*>(g.dy) + (m0 + a_row) * g.ld_dy + k0 + a_col;
  const int8_t* b_from = g.codes + (static_cast<int64_t>(m0) + b_row) * g.c + c0 + b_col;
  const uint8_t* s_from = g.scales + (static_cast<int64_t>(m0) + b_row) * g.groups + (c0 + b_col) / kAct8Group;

  struct Staged {
    Raw<T> a[NA];
    v4i b[NB];
    unsigned scale[NB];
  };
  // Steps whose 32 rows can be read whole, columns beyond the tensors' widths (other rows' values,
  // which reach only sums that are not stored) among them: inside the range, and not so near the
  // tensors' ends that such a column lies beyond them.
  auto whole = [&](int64_t ld, int64_t width, int64_t first, int64_t span) {
    const int64_t last = (g.rows - 1) * ld + width - first - span;  // where a row's reads may start at most
    return last < 0 ? int64_t{0} : last / ld + 1;
  };
  // Spreads a half step's other instructions between its matrix instructions: left alone, the
  // compiler issues the matrix instructions in one run and the conversions after them.
  auto mix = [&]() {
    constexpr int kMul = P * IA * IB;
    constexpr int kReads = 2 * (P * IA + IB), kWrites = P * NA + NB * CB / 8;
#pragma unroll
    for (int i = 0; i < kMul; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);                                 // matrix
      __builtin_amdgcn_sched_group_barrier(0x100, 2 * ((kReads + kMul - 1) / kMul), 0);  // LDS reads
      __builtin_amdgcn_sched_group_barrier(0x002, 8, 0);                                 // vector ALU
      __builtin_amdgcn_sched_group_barrier(0x200, (kWrites + kMul - 1) / kMul, 0);       // LDS writes
      __builtin_amdgcn_sched_group_barrier(0x020, 1, 0);                                 // loads
    }
  };
  const int64_t safe = min(min(whole(g.ld_dy, g.k, k0, TK), whole(g.c, g.c, c0, TC)),
                           whole(g.groups, g.groups, c0 / kAct8Group, (TC + kAct8Group - 1) / kAct8Group));
  const int fast = static_cast<int>(max(min(safe, static_cast<int64_t>(m1)) - m0, int64_t{0})) / kStep;
  auto load = [&](Staged& r, int step) {
    const int64_t down = static_cast<int64_t>(step) * kStep;
    const T* a = a_from + down * g.ld_dy;
    const int8_t* b = b_from + down * g.c;
    const uint8_t* s = s_from + down * g.groups;
#pragma unroll
    for (int i = 0; i < NA; ++i) load_raw(r.a[i], a + i * (kRowsA * g.ld_dy), 8);
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      const int8_t* p = b + i * (kRowsB * static_cast<int64_t>(g.c));
      if constexpr (CB == 16) {
        r.b[i] = *reinterpret_cast<const v4i_any*>(p);
      } else {
        const v2i w = *reinterpret_cast<const v2i_any*>(p);
        r.b[i][0] = w[0];
        r.b[i][1] = w[1];
      }
      r.scale[i] = s[i * (kRowsB * static_cast<int64_t>(g.groups))];
    }
  };
  auto load_edge = [&](Staged& r, int step) {  // value by value at the edges, zeros beyond them
    const int64_t down = static_cast<int64_t>(step) * kStep;
    const int m = m0 + step * kStep;
#pragma unroll
    for (int i = 0; i < NA; ++i)
      load_raw(r.a[i], a_from + (down + i * kRowsA) * g.ld_dy, m + a_row + i * kRowsA < m1 ? a_left : 0);
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      const bool there = m + b_row + i * kRowsB < m1 && b_left > 0;
      const int8_t* p = b_from + (down + i * kRowsB) * g.c;
      r.b[i] = v4i{};
#pragma unroll
      for (int j = 0; j < CB; ++j)
        if (there && j < b_left) r.b[i][j / 4] |= (p[j] & 0xff) << (8 * (j & 3));
      r.scale[i] = there ? s_from[(down + i * kRowsB) * g.groups] : 0;
    }
  };
  auto write = [&](const Staged& r, int stage) {
    char* const base = lds + stage * kStage;
#pragma unroll
    for (int i = 0; i < NA; ++i) {
      const int row = a_row + i * kRowsA;
      v8bf p[P];
      split8(r.a[i], p);
      char* const to = base + row * kPitchA + (((a_col >> 4) ^ turn<TK>(row)) * 32) + (a_col & 8) * 2;
#pragma unroll
      for (int q = 0; q < P; ++q) *reinterpret_cast<v8bf*>(to + q * kPlane) = p[q];
    }
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      const int row = b_row + i * kRowsB;
      const float scale = __uint_as_float(r.scale[i] << 23);  // byte 255: infinity, NaN times a zero code
      char* const to = base + P * kPlane + row * kPitchB + (((b_col >> 4) ^ turn<TC>(row)) * 32) + (b_col & 8) * 2;
#pragma unroll
      for (int j = 0; j < CB / 8; ++j) {
        const v4f lo = codes4(r.b[i][2 * j]) * scale, hi = codes4(r.b[i][2 * j + 1]) * scale;
        *reinterpret_cast<v8bf*>(to + j * 16) =
            __builtin_convertvector(__builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7), v8bf);
      }
    }
  };

  // Fragments: lane l's column is l & 31, its rows of a 16-row half are (l >> 5) * 4 .. + 3 and
  // those plus 8; one transposing read takes four rows of a 16-column unit per 16 lanes.
  const int f_row = (lane >> 5) * 4 + ((lane & 15) >> 2);
  const int f_unit = (lane >> 4) & 1;
  int a_at[IA], b_at[IB];
#pragma unroll
  for (int i = 0; i < IA; ++i)
    a_at[i] = f_row * kPitchA + (((wk / 16 + 2 * i + f_unit) ^ turn<TK>(f_row)) * 32) + (lane & 3) * 8;
#pragma unroll
  for (int i = 0; i < IB; ++i)
    b_at[i] = P * kPlane + f_row * kPitchB + (((wc / 16 + 2 * i + f_unit) ^ turn<TC>(f_row)) * 32) + (lane & 3) * 8;
  typedef __attribute__((address_space(3))) char lds_char;
  typedef __attribute__((address_space(3))) v4s lds_v4s;
  lds_char* const lds3 = (lds_char*)lds;  // an address-space cast
  auto fragment = [&](lds_char* from, int pitch) {
    // rows + 8 have the same permutation
    const v4s lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<lds_v4s*>(from));
    const v4s hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<lds_v4s*>(from + 8 * pitch));
    return __builtin_bit_cast(v8bf, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
  };

  v16f acc[IA][IB] = {};
  v8bf fa[2][P][IA], fb[2][IB];
  auto read = [&](int stage, int half, int to) {
    lds_char* const base = lds3 + stage * kStage;
#pragma unroll
    for (int i = 0; i < IB; ++i) fb[to][i] = fragment(base + b_at[i] + half * 16 * kPitchB, kPitchB);
#pragma unroll
    for (int i = 0; i < IA; ++i) {
      lds_char* const column = base + a_at[i] + half * 16 * kPitchA;
#pragma unroll
      for (int q = 0; q < P; ++q) fa[to][q][i] = fragment(column + q * kPlane, kPitchA);
    }
  };
  auto multiply = [&](int from) {
#pragma unroll
    for (int q = P - 1; q >= 0; --q)  // the smallest pieces first
#pragma unroll
      for (int i = 0; i < IA; ++i)
#pragma unroll
        for (int j = 0; j < IB; ++j)
          acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fa[from][q][i], fb[from][j], acc[i][j], 0, 0, 0);
  };

  // Three stages: a step multiplies its own, reads the next one's first half and writes the third.
  // Two, where three do not fit: a step reads and multiplies its own and writes the other.  Five:
  // a step writes the one three ahead, so that a barrier after every second step is enough: between
  // two barriers steps t and t + 1 read the stages t to t + 2, all written before, and write t + 3
  // and t + 4, in place of t - 2 and t - 1.  Either way the values written were loaded SETS steps
  // before.  Past the last step the loads, writes and reads repeat that step: their values go unused.
  constexpr int kAhead = STAGES == 5 ? 3 : STAGES - 1;  // a step writes the values of step t + kAhead
  static_assert(STAGES != 5 || SETS == 2, "the barrier goes by the place in the loop");
  if (fast > 0) {
    Staged first[kAhead], r[SETS];  // step s >= kAhead in r[s % SETS]
    // the sets' loads in order: the waits for one of them do not include the next
#pragma unroll
    for (int i = 0; i < kAhead; ++i) load(first[i], min(i, fast - 1));
#pragma unroll
    for (int i = kAhead; i < kAhead + SETS; ++i) {
      __builtin_amdgcn_sched_barrier(0);
      load(r[i % SETS], min(i, fast - 1));
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < kAhead; ++i) write(first[i], i);
    __syncthreads();
    if constexpr (STAGES >= 3) read(0, 0, 0);
    int now = 0;
    auto step = [&](Staged& set, int t, bool barrier) {
      const int next = now == STAGES - 1 ? 0 : now + 1;
      if constexpr (STAGES == 2) read(now, 0, 0);
      read(now, 1, 1);
      write(set, now + kAhead >= STAGES ? now + kAhead - STAGES : now + kAhead);
      multiply(0);
      mix();
      __builtin_amdgcn_sched_barrier(0);
      load(set, min(t + kAhead + SETS, fast - 1));
      if constexpr (STAGES >= 3) read(next, 0, 0);
      multiply(1);
      mix();
      if (barrier) __syncthreads();
      now = next;
    };
    int t = 0;
    for (; t + SETS <= fast; t += SETS) {  // no other way round the loop: its waits count on the loads' order
#pragma unroll
      for (int u = 0; u < SETS; ++u) step(r[(u + kAhead) % SETS], t + u, STAGES != 5 || u == 1);
    }
#pragma unroll
    for (int u = 0; u + 1 < SETS; ++u)
      if (t + u < fast) step(r[(u + kAhead) % SETS], t + u, STAGES != 5);
  }
  for (int t = fast; t < steps; ++t) {
    Staged r;
    load_edge(r, t);
    __syncthreads();
    write(r, 0);
    __syncthreads();
    read(0, 0, 0);
    read(0, 1, 1);
    multiply(0);
    multiply(1);
  }

  TO* out = static_cast<TO*>(g.out) + (g.to_parts ? static_cast<int64_t>(part) * g.k * g.c : 0);
#pragma unroll
  for (int i = 0; i < IA; ++i)
#pragma unroll
    for (int j = 0; j < IB; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int row = k0 + wk + i * 32 + (r >> 2) * 8 + (lane >> 5) * 4 + (r & 3);
        const int col = c0 + wc + j * 32 + (lane & 31);
        if (row < g.k && col < g.c) {
          TO* to = out + row * g.ld_out + col;
          float v = acc[i][j][r];
          if (g.accumulate) v += static_cast<float>(*to);
          *to = static_cast<TO>(v);
        }
      }
}

// Adds the splits' partial sums in order, four values per lane: `parts_of` lanes of a workgroup
// share the splits of the same values, and their sums are added in order.
template <typename TO>
__global__ __launch_bounds__(kThreads) void act8_grad_join_kernel(Grad g, const float* __restrict__ parts, int splits,
                                                                  int parts_of) {
  __shared__ v4f sums[kThreads];
  const int64_t n = static_cast<int64_t>(g.k) * g.c;
  const int wide = kThreads / parts_of;  // lanes along the values
  const int at = threadIdx.x % wide;
  const int share = threadIdx.x / wide;
  const int each = (splits + parts_of - 1) / parts_of;
  const int end = min((share + 1) * each, splits);
  for (int64_t i0 = static_cast<int64_t>(blockIdx.x) * wide * 4; i0 < n; i0 += static_cast<int64_t>(gridDim.x) * wide * 4) {
    const int64_t i = i0 + at * 4;
    const int left = static_cast<int>(min(n - i, int64_t{4}));
    v4f v = {};
    if (left == 4) {
#pragma unroll 8
      for (int s = share * each; s < end; ++s) v += *reinterpret_cast<const v4f_any*>(parts + s * n + i);
    } else {
      for (int s = share * each; s < end; ++s)
        for (int j = 0; j < left; ++j) v[j] += parts[s * n + i + j];
    }
    if (parts_of > 1) {
      sums[threadIdx.x] = v;
      __syncthreads();
      if (share == 0)
        for (int s = 1; s < parts_of; ++s) v += sums[s * wide + at];
      __syncthreads();
    }
    if (share == 0 && left > 0) {
      int64_t row = i / g.c;
      int col = static_cast<int>(i - row * g.c);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (j < left) {
          TO* to = static_cast<TO*>(g.out) + row * g.ld_out + col;
          float sum = v[j];
          if (g.accumulate) sum += static_cast<float>(*to);
          *to = static_cast<TO>(sum);
          if (++col == g.c) {
            col = 0;
            ++row;
          }
        }
      }
    }
  }
}

struct Shape {
  int tile, splits, per;
};

// The tile (64, 128 or 256 square) and the splits of the rows: the pair with the least estimated
// time.  A step of 32 rows takes `alone` us with one workgroup on a CU and `each` apiece with several;
// 5 us to launch, fill and drain; dw and partial sums are written and read at 5.9 TB/s; the launch
// that joins them costs 5 us more.  Fitted to every pair's time on 46 problems from 128 x 1024 x 1024
// to 65536 x 1024 x 1024 (rows, c, k) in both types: the pair chosen is the fastest or within 5% of
// it on 44 of them, within 18% on all.
Shape shape_of(int32_t rows, int32_t c, int32_t k, bool dy_bf16) {
  struct Rate {
    int tile;
    double alone, each;
  };
  static constexpr Rate kBf16[3] = {{64, 0.18, 0.16}, {128, 0.47, 0.43}, {256, 1.0, 1.0}};
  static constexpr Rate kF32[3] = {{64, 0.51, 0.43}, {128, 1.01, 0.96}, {256, 2.62, 2.62}};
  const Rate* rates = dy_bf16 ? kBf16 : kF32;
  const double values = static_cast<double>(k) * c * 4e-6 / 5.9;  // us to move one fp32 dw
  const double inputs = rows * (k * (dy_bf16 ? 2.0 : 4.0) + c) * 1e-6 / 4.5;
  Shape best{};
  double least = 0.0;
  for (int i = 0; i < 3; ++i) {
    const int tile = rates[i].tile;
    const int64_t tiles = ((static_cast<int64_t>(c) + tile - 1) / tile) * ((static_cast<int64_t>(k) + tile - 1) / tile);
    for (int s = 1; s <= 256 && (s == 1 || tiles * s <= 2048); s *= 2) {
      int64_t per = (static_cast<int64_t>(rows) + s - 1) / s;
      per = (per + kStep - 1) / kStep * kStep;
      if (per < kStep) per = kStep;
      if (s > 1 && per < 2 * kStep) break;
      const int64_t splits = rows > 0 ? (rows + per - 1) / per : 1;
      const double steps = static_cast<double>(per / kStep);
      const double rounds = static_cast<double>((tiles * splits + 255) / 256);
      double us = steps * rates[i].each * rounds;
      if (us < steps * rates[i].alone) us = steps * rates[i].alone;
      if (us < inputs) us = inputs;
      us += 5 + values * splits;
      if (splits > 1) us += 5 + values * (splits + 1);
      if (best.tile == 0 || us < least) {
        best = Shape{tile, static_cast<int>(splits), static_cast<int>(per)};
        least = us;
      }
    }
  }
  return best;
}

template <typename T, typename TO, int P, int TK, int TC, int VK, int VC, int STAGES, int SETS>
hipError_t launch_tile(const Grad& g, unsigned blocks, hipStream_t stream) {
  constexpr int kBytes = STAGES * (P * kStep * TK * 2 + kStep * TC * 2);
  auto* kernel = &act8_grad_kernel<T, TO, P, TK, TC, VK, VC, STAGES, SETS>;
  if (kBytes > 64 * 1024) {
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                             hipFuncAttributeMaxDynamicSharedMemorySize, kBytes);
    if (e != hipSuccess) return e;
  }
  kernel<<<blocks, VK * VC * 64, kBytes, stream>>>(g);
  return hipGetLastError();
}

template <typename T, typename TO, int P>
hipError_t launch_product(const Grad& g, const Shape& s, hipStream_t stream) {
  const unsigned blocks = static_cast<unsigned>(static_cast<int64_t>(g.tiles_k) * g.tiles_c * s.splits);
  if constexpr (P == 1) {
    if (s.tile == 256) return launch_tile<T, TO, P, 256, 256, 4, 2, 5, 2>(g, blocks, stream);
  } else {
    if (s.tile == 256) return launch_tile<T, TO, P, 256, 256, 4, 2, 2, 1>(g, blocks, stream);
  }
  if (s.tile == 128) return launch_tile<T, TO, P, 128, 128, 4, 2, 3, 2>(g, blocks, stream);
  return launch_tile<T, TO, P, 64, 64, 2, 2, 3, 2>(g, blocks, stream);
}

template <typename T, typename TO, int P>
hipError_t launch(const Act8GradArgs& a, hipStream_t stream) {
  const Shape s = shape_of(a.rows, a.c, a.k, a.dy_bf16);
  Grad g{};
  g.dy = a.dy;
  g.codes = a.codes;
  g.scales = a.scales;
  g.ld_dy = a.ld_dy;
  g.rows = a.rows;
  g.c = a.c;
  g.k = a.k;
  g.groups = (a.c + kAct8Group - 1) / kAct8Group;
  g.tiles_k = (a.k + s.tile - 1) / s.tile;
  g.tiles_c = (a.c + s.tile - 1) / s.tile;
  g.per_split = s.per;
  g.out = a.dw;
  g.ld_out = a.ld_dw;
  g.accumulate = a.accumulate;
  if (s.splits == 1) return launch_product<T, TO, P>(g, s, stream);
  Grad h = g;
  h.out = a.ws;
  h.ld_out = a.c;
  h.accumulate = false;
  h.to_parts = true;
  const hipError_t e = launch_product<T, float, P>(h, s, stream);
  if (e != hipSuccess) return e;
  // lanes that share a value's splits: eight splits each or so, while workgroups are few
  const int64_t n = static_cast<int64_t>(a.k) * a.c;
  int parts_of = 1;
  while (parts_of < 64 && parts_of * 8 < s.splits && n * parts_of < 4 * 256 * 2048) parts_of *= 2;
  const int64_t join = (n + 4 * (kThreads / parts_of) - 1) / (4 * (kThreads / parts_of));
  act8_grad_join_kernel<TO><<<static_cast<unsigned>(join < 65536 ? join : 65536), kThreads, 0, stream>>>(
      g, static_cast<const float*>(a.ws), s.splits, parts_of);
  return hipGetLastError();
}

}  // namespace

void plan_act8_grad(int32_t rows, int32_t c, int32_t k, bool dy_bf16, int32_t* tile, int32_t* splits) {
  const Shape s = shape_of(rows, c, k, dy_bf16);
  *tile = s.tile;
  *splits = s.splits;
}

size_t act8_grad_workspace_bytes(int32_t rows, int32_t c, int32_t k, bool dy_bf16) {
  const Shape s = shape_of(rows, c, k, dy_bf16);
  return s.splits > 1 ? static_cast<size_t>(s.splits) * c * k * 4 : 0;
}

hipError_t launch_act8_grad(const Act8GradArgs& a, hipStream_t stream) {
  if (!a.dy_bf16) return launch<float, float, 3>(a, stream);
  return a.dw_bf16 ? launch<__bf16, __bf16, 1>(a, stream) : launch<__bf16, float, 1>(a, stream);
}

}  // namespace miq
