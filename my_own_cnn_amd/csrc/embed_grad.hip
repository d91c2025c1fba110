// The embedding table's gradient by sorted tokens (miq_embed_grad).
//
// The (row, position) pairs of the tokens are sorted, stably, so that a row's tokens stand together
// in order of position; a position without a token has the key `vocab` and sorts to the end.  Up to
// kRankTokens tokens each token counts the ones before it directly, in one launch (a call of 4096
// tokens 24 us, 30 with the counting passes; of 8192 31 and 38); above that the keys go through
// stable counting passes of up to 10 bits, two launches each.  The sorted list is then cut into
// chunks of a fixed length: a group of lanes walks one chunk and 512 channels, adds the rows of dy
// of each run of equal keys in fp32 and writes the runs that lie within its chunk.  A run that
// reaches over a chunk's end leaves one partial sum per chunk in the workspace, and a last launch
// adds those in order.  The cuts depend on the sizes alone: every call gives the same bits.
//
// Up to kDirectTokens tokens (kDirectShort on the largest tables) nothing is sorted: one launch in
// which each token's workgroup looks at all tokens and adds its row if it is the row's first (1 to
// 256 tokens of 512 channels 8 us instead of 12 to 16).
//
// Rows without a token, most of the table in a common batch, are zeroed by workgroups of the
// launch that adds.  A row has a token exactly if where[row] is a place of the sorted list that
// holds its key: the sort writes where[] for the rows that it sees, and what the others hold is
// tested, not trusted, so nothing has to be cleared.
//
// Bound by memory: dy once, the table once.  65536 tokens on 65536 x 2048, bf16 to fp32: 806 MB in
// 201 us, of them the launch that adds and zeros 162 (5 TB/s; a large copy reaches 4.8), the sort
// 28, the join 9.  A lane stores runs of 16 bytes next to its neighbours' (two runs of an fp32 row):
// with 32 bytes per lane the call took 217 us, and 20011 tokens on 50021 x 1001 99 instead of 73
// (into memory that the last-level cache still holds; 87 into other).
// Six workgroups per CU with four rows in flight per lane (five for fp32 rows): 198 us, with eight
// rows and four workgroups 206.  A chunk's length goes by the tokens and channels, so that a call
// has some 262144 lanes; zeros after the sums, not among them (61 -> 87 us on the odd table).
#include "train_device.h"

namespace miq {
namespace {

constexpr int kThreads = 256;
constexpr int kDirectTokens = 1024; // most tokens that take no sort
constexpr int kDirectShort = 256;   // most of them in workgroups of 256 threads
constexpr int kDirectUnits = 2048;  // and most workgroups that add them
constexpr int kRankTokens = 8192;   // most tokens that are ranked by counting
constexpr int kDigitBits = 10;      // most bits of a counting pass
constexpr int kDigits = 1 << kDigitBits;
constexpr int kSortThreads = 512;
constexpr int kSortWaves = kSortThreads / 64;
constexpr int kCached = 4;          // keys per lane that a counting pass reads once
constexpr int kSortBlocks = 64;     // most workgroups of a counting pass
constexpr int kCols = 512;          // channels per wave: 64 lanes of 8
constexpr int kZeroRows = 32;       // table rows per workgroup that zeros rows without a token
constexpr int kAhead = 4;           // rows of dy in flight per lane

struct Plan {
  int bits, passes, digit_bits, blocks, per_block;  // counting passes
  int lanes, col_tiles, len, chunks;                // lanes per chunk, chunk length
  bool direct;                                      // no sort
  size_t keys0, keys1, order0, order1, hist, where, part, total;
};

size_t up(size_t v) { return (v + 255) & ~static_cast<size_t>(255); }

Plan make_plan(int32_t vocab, int32_t c, int32_t tokens) {
  Plan p{};
  p.bits = 1;
  while ((static_cast<int64_t>(vocab) >> p.bits) != 0) ++p.bits;  // keys 0 .. vocab
  p.passes = (p.bits + kDigitBits - 1) / kDigitBits;
  p.digit_bits = (p.bits + p.passes - 1) / p.passes;
  // workgroups of the counting passes: 1024 tokens or more each
  const int64_t t = tokens;
  int64_t per = (t + kSortBlocks - 1) / kSortBlocks;
  per = ((per < 1024 ? 1024 : per) + kSortThreads - 1) / kSortThreads * kSortThreads;
  p.per_block = static_cast<int>(per);
  p.blocks = static_cast<int>((t + per - 1) / per);
  if (t <= kRankTokens) p.passes = 0;
  p.lanes = 8;
  while (p.lanes < 64 && p.lanes * 8 < c) p.lanes *= 2;
  p.col_tiles = (c + kCols - 1) / kCols;
  // The last bound keeps the grid of workgroups of 512 threads below 2^32 threads, with the 2^23 of
  // them that zero 2^28 rows; of 256 threads it is below for every table, so that a call without
  // tokens, which has no workspace, never comes to the sort.
  p.direct = t <= kDirectTokens && t * p.col_tiles <= kDirectUnits && (t <= kDirectShort || vocab <= 1 << 27);
  if (p.direct) return p;  // without a workspace
  // chunks enough for about 1024 lanes on each of the 256 CUs
  const int64_t want = 262144 / (static_cast<int64_t>(p.col_tiles) * p.lanes);
  int64_t len = (t + (want < 1 ? 1 : want) - 1) / (want < 1 ? 1 : want);
  len = (len + 3) / 4 * 4;
  p.len = static_cast<int>(len < 4 ? 4 : len);
  p.chunks = static_cast<int>((t + p.len - 1) / p.len);
  size_t at = 0;
  const size_t list = up(static_cast<size_t>(tokens) * 4);
  p.keys0 = at; at += list;
  p.order0 = at; at += list;
  if (p.passes > 0) {
    p.keys1 = at; at += list;
    p.order1 = at; at += list;
    p.hist = at; at += up((static_cast<size_t>(p.blocks) << p.digit_bits) * 4);
  }
  p.where = at; at += up(static_cast<size_t>(vocab) * 4);
  p.part = at; at += static_cast<size_t>(p.chunks) * 2 * p.col_tiles * (p.lanes * 8) * 4;
  p.total = at;
  return p;
}

__device__ __forceinline__ unsigned key_of(const void* ids, bool wide, int64_t t, unsigned vocab) {
  const uint64_t id = static_cast<uint64_t>(load_id(ids, wide, t));
  return id < vocab ? static_cast<unsigned>(id) : vocab;
}

// ---- up to kRankTokens tokens: a token's place is the number of tokens that sort before it -----

// 64 / SHARES tokens per workgroup, each held by SHARES lanes of every wave; these and the 16 waves
// share the tokens to compare with.
template <int SHARES>
__global__ __launch_bounds__(1024) void embed_rank_kernel(const void* __restrict__ ids, bool ids64, int tokens,
                                                          unsigned vocab, unsigned* __restrict__ keys,
                                                          int* __restrict__ order, unsigned* __restrict__ where) {
  constexpr int kRanked = 64 / SHARES;
  typedef unsigned v4u __attribute__((ext_vector_type(4)));
  __shared__ __attribute__((aligned(16))) unsigned all[kRankTokens];
  __shared__ int counts[16][64];
  const int padded = (tokens + 63) & ~63;  // past the tokens: keys that sort before nothing
  for (int i = threadIdx.x; i < padded; i += 1024) all[i] = i < tokens ? key_of(ids, ids64, i, vocab) : ~0u;
  __syncthreads();
  const int lane = threadIdx.x & 63;
  const int wave = threadIdx.x >> 6;
  const int share = lane / kRanked;
  const int t = blockIdx.x * kRanked + lane % kRanked;
  const unsigned mine = all[t];
  const int t0 = t & ~63;  // the group of 64 that holds the workgroup's tokens
  int n = 0;
  // equal keys count where they come before; a group's keys in turns that keep the shares in
  // different banks
  for (int g = (wave * SHARES + share) * 64; g < padded; g += 1024 * SHARES) {
    if (g != t0) {
      const unsigned least = g < t0 ? mine : mine - 1;  // all[i] <= least; a key 0 has none below it
      if (g < t0 || mine != 0) {
#pragma unroll
        for (int i = 0; i < 64; i += 4) {
          const v4u k = *reinterpret_cast<const v4u*>(&all[g + ((i + 4 * share) & 63)]);
          n += (k[0] <= least) + (k[1] <= least) + (k[2] <= least) + (k[3] <= least);
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < 64; i += 4) {
        const v4u k = *reinterpret_cast<const v4u*>(&all[g + i]);
#pragma unroll
        for (int j = 0; j < 4; ++j) n += k[j] < mine || (k[j] == mine && g + i + j < t);
      }
    }
  }
  counts[wave][lane] = n;
  __syncthreads();
  if (threadIdx.x < kRanked && t < tokens) {
    int place = 0;
#pragma unroll
    for (int w = 0; w < 16; ++w)
#pragma unroll
      for (int s = 0; s < SHARES; ++s) place += counts[w][s * kRanked + lane];
    keys[place] = mine;
    order[place] = t;
    if (mine < vocab) where[mine] = static_cast<unsigned>(place);
  }
}

// ---- more tokens: stable counting passes -------------------------------------------------------

struct Pass {
  const unsigned* keys_in;  // NULL in the first pass: keys come from the ids, order is 0, 1, ...
  const int* order_in;
  const void* ids;
  bool ids64;
  unsigned vocab;
  int tokens, per_block, blocks, shift, digits;
};

__device__ __forceinline__ unsigned pass_key(const Pass& p, int t) {
  return p.keys_in != nullptr ? p.keys_in[t] : key_of(p.ids, p.ids64, t, p.vocab);
}

// hist[workgroup][digit]: the tokens of each workgroup's range by digit
__global__ __launch_bounds__(kSortThreads) void embed_hist_kernel(Pass p, unsigned* __restrict__ hist) {
  __shared__ unsigned n[kDigits];
  for (int d = threadIdx.x; d < p.digits; d += kSortThreads) n[d] = 0;
  __syncthreads();
  const int64_t begin = static_cast<int64_t>(blockIdx.x) * p.per_block;
  const int64_t end = min(begin + p.per_block, static_cast<int64_t>(p.tokens));
  for (int64_t t = begin + threadIdx.x; t < end; t += kSortThreads)
    atomicAdd(&n[(pass_key(p, static_cast<int>(t)) >> p.shift) & (p.digits - 1)], 1u);
  __syncthreads();
  for (int d = threadIdx.x; d < p.digits; d += kSortThreads) hist[blockIdx.x * p.digits + d] = n[d];
}

// Each wave takes a contiguous part of its workgroup's range, 64 tokens at a time in order: a
// token's place is its wave's running place of its digit plus the lanes before it with that digit.
// `where` (or NULL): a place of each key.
__global__ __launch_bounds__(kSortThreads) void embed_scatter_kernel(Pass p, const unsigned* __restrict__ hist,
                                                                     unsigned* __restrict__ keys,
                                                                     int* __restrict__ order,
                                                                     unsigned* __restrict__ where) {
  __shared__ unsigned at[kSortWaves][kDigits];
  __shared__ unsigned sums[kSortWaves];
  const int wave = threadIdx.x >> 6;
  const int lane = threadIdx.x & 63;
  const int part = p.per_block / kSortWaves;  // a multiple of 64
  const int64_t begin = static_cast<int64_t>(blockIdx.x) * p.per_block + wave * static_cast<int64_t>(part);
  const int64_t end = min(begin + part, static_cast<int64_t>(p.tokens));
  // the wave's first keys stay in registers between counting and placing
  auto pass_pos = [&](int64_t t) { return p.order_in != nullptr ? p.order_in[t] : static_cast<int>(t); };
  unsigned cache[kCached];
  int cached_pos[kCached];
#pragma unroll
  for (int i = 0; i < kCached; ++i) {
    const int64_t t = begin + i * 64 + lane;
    cache[i] = t < end ? pass_key(p, static_cast<int>(t)) : 0;
    cached_pos[i] = t < end ? pass_pos(t) : 0;
  }
  // two digits per thread: the tokens of a digit in all workgroups, and in those before this one
  static_assert(kDigits == 2 * kSortThreads, "");
  const int d0 = threadIdx.x * 2;
  unsigned total[2] = {}, before[2] = {};
  if (d0 < p.digits) {
#pragma unroll 16
    for (int b = 0; b < p.blocks; ++b) {
      const v2i h = *reinterpret_cast<const v2i*>(hist + b * p.digits + d0);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        total[i] += static_cast<unsigned>(h[i]);
        before[i] += b < static_cast<int>(blockIdx.x) ? static_cast<unsigned>(h[i]) : 0;
      }
    }
  }
  for (int w = 0; w < kSortWaves; ++w)
    for (int d = threadIdx.x; d < p.digits; d += kSortThreads) at[w][d] = 0;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kCached; ++i)
    if (begin + i * 64 + lane < end) atomicAdd(&at[wave][(cache[i] >> p.shift) & (p.digits - 1)], 1u);
  for (int64_t t = begin + kCached * 64 + lane; t < end; t += 64)
    atomicAdd(&at[wave][(pass_key(p, static_cast<int>(t)) >> p.shift) & (p.digits - 1)], 1u);
  // the place of this thread's first digit: the tokens of all digits before it
  unsigned first = total[0] + total[1];
#pragma unroll
  for (int step = 1; step < 64; step *= 2) {
    const unsigned left = __shfl_up(first, step);
    first += lane >= step ? left : 0;
  }
  if (lane == 63) sums[wave] = first;
  first -= total[0] + total[1];
  __syncthreads();
  for (int w = 0; w < wave; ++w) first += sums[w];
  if (d0 < p.digits) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      unsigned place = first + before[i];
#pragma unroll
      for (int w = 0; w < kSortWaves; ++w) {
        const unsigned n = at[w][d0 + i];
        at[w][d0 + i] = place;
        place += n;
      }
      first += total[i];
    }
  }
  __syncthreads();
  auto put = [&](bool there, unsigned key, int pos) {
    const unsigned digit = (key >> p.shift) & (p.digits - 1);
    uint64_t same = __ballot(there);
    for (int bit = 1; bit < p.digits; bit *= 2) {
      const uint64_t set = __ballot((digit & bit) != 0);
      same &= (digit & bit) != 0 ? set : ~set;
    }
    const int earlier = __popcll(same & ((uint64_t{1} << lane) - 1));
    unsigned place = 0;
    if (there) place = at[wave][digit] + earlier;
    __builtin_amdgcn_wave_barrier();
    if (there && earlier == 0) at[wave][digit] += __popcll(same);
    __builtin_amdgcn_wave_barrier();
    if (there) {
      keys[place] = key;
      order[place] = pos;
      if (where != nullptr && key < p.vocab) where[key] = place;
    }
  };
#pragma unroll
  for (int i = 0; i < kCached; ++i)
    if (begin + i * 64 < end) put(begin + i * 64 + lane < end, cache[i], cached_pos[i]);
  for (int64_t t0 = begin + kCached * 64; t0 < end; t0 += 64) {
    const int64_t t = t0 + lane;
    put(t < end, t < end ? pass_key(p, static_cast<int>(t)) : 0, t < end ? pass_pos(t) : 0);
  }
}

// ---- the sums ------------------------------------------------------------------------------------

template <typename TI, typename TO>
struct Sum {
  const TI* dy;
  TO* table;
  const unsigned* keys;
  const int* order;
  const unsigned* where;  // a place of each row's key, for rows that have a token
  float* part;
  int64_t ld_dy, ld_table;
  int tokens, c, lanes, col_tiles, len, chunks, sum_blocks;
  unsigned vocab;
  float scale;
  bool accumulate;

  // partial sums: [chunk][0: the run that reaches in, 1: the run that starts here and reaches on]
  __device__ float* slot(int chunk, int which, int tile, int lane) const {
    return part + ((static_cast<int64_t>(chunk) * 2 + which) * col_tiles + tile) * (lanes * 8) + lane * 4;
  }
  // A lane's channels, so that neighbouring lanes store neighbouring runs of 16 bytes: of an fp32
  // table four from `col` and four `apart` from there, of a bf16 table eight from `col` (apart = 4).
  // Where the row ends within a run, the lane takes the row's last run instead, as its neighbour
  // does in part: both write the same values.  Adding to the table is no place for that; there such
  // a lane is not `whole` and goes value by value.  False for a lane beyond the row.
  static constexpr bool kPairs = sizeof(TO) == 4;
  __device__ bool place(int tile, int lane, int* col, int* apart, bool* whole) const {
    const int first = tile * kCols + lane * (kPairs ? 4 : 8);
    *col = first;
    if constexpr (kPairs) {
      const int second = first + lanes * 4;
      *whole = second + 4 <= c || (c >= 4 && !accumulate);
      *apart = lanes * 4;
      if (second + 4 > c && *whole) {
        *col = min(first, c - 4);
        *apart = second < c ? c - 4 - *col : 0;
      }
    } else {
      *whole = first + 8 <= c || (c >= 8 && !accumulate);
      *apart = 4;
      if (*whole) *col = min(first, c - 8);
    }
    return first < c;
  }
  __device__ void finish(unsigned row, int col, int apart, bool whole, v8f acc) const {
    TO* to = table + row * ld_table + col;
    acc *= scale;
    if (whole) {
      if constexpr (kPairs) {
        if (accumulate) acc += load44(to, apart);
        store44(to, apart, acc);
      } else {
        if (accumulate) acc += load8(to);
        store_run<false>(to, acc);
      }
    } else {
      if (accumulate) acc += load44_of(to, apart, c - col);
      store44_of(to, apart, acc, c - col);
    }
  }
};

// Zeros in the rows from `first` on that are marked empty, a row per wave and turn.
template <int THREADS, typename TI, typename TO>
__device__ __forceinline__ void zero_marked(const Sum<TI, TO>& s, int64_t first, const int* empty) {
  const int rows = static_cast<int>(min(static_cast<int64_t>(kZeroRows), s.vocab - first));
  const int lane = threadIdx.x & 63;
  for (int r = threadIdx.x >> 6; r < rows; r += THREADS / 64) {
    if (!empty[r]) continue;
    TO* const row = s.table + (first + r) * s.ld_table;
    constexpr int W = 16 / static_cast<int>(sizeof(TO));
    if (s.c < W) {
      if (lane < s.c) row[lane] = static_cast<TO>(0.0f);
    } else {
#pragma unroll 4
      for (int col = lane * W; col < s.c; col += 64 * W) {
        if constexpr (W == 4) store_run<false>(row + min(col, s.c - 4), v4f{});
        else store_run<false>(row + min(col, s.c - 8), v8f{});
      }
    }
  }
}

// The rows [first, first + kZeroRows) that no token names.
template <typename TI, typename TO>
__device__ __forceinline__ void zero_rows(const Sum<TI, TO>& s, int64_t first) {
  __shared__ int empty[kZeroRows];
  if (threadIdx.x < kZeroRows && first + threadIdx.x < s.vocab) {
    const unsigned row = static_cast<unsigned>(first) + threadIdx.x;
    const unsigned at = s.where[row];
    empty[threadIdx.x] = at >= static_cast<unsigned>(s.tokens) || s.keys[at] != row;
  }
  __syncthreads();
  zero_marked<kThreads>(s, first, empty);
}

// A lane's eight values of a row of dy, as loaded.
template <typename T>
struct Raw8;
template <>
struct Raw8<float> {
  v4f lo, hi;
};
template <>
struct Raw8<__bf16> {
  v4bf lo, hi;
};
template <bool PAIRS>
__device__ __forceinline__ void load_raw(Raw8<float>& r, const float* p, int apart) {
  r.lo = *reinterpret_cast<const v4f_any*>(p);
  r.hi = *reinterpret_cast<const v4f_any*>(p + (PAIRS ? apart : 4));
}
template <bool PAIRS>
__device__ __forceinline__ void load_raw(Raw8<__bf16>& r, const __bf16* p, int apart) {
  if constexpr (PAIRS) {
    r.lo = *reinterpret_cast<const v4bf_any*>(p);
    r.hi = *reinterpret_cast<const v4bf_any*>(p + apart);
  } else {
    const v8bf v = *reinterpret_cast<const v8bf_any*>(p);
    r.lo = __builtin_shufflevector(v, v, 0, 1, 2, 3);
    r.hi = __builtin_shufflevector(v, v, 4, 5, 6, 7);
  }
}
template <typename T>
__device__ __forceinline__ v8f value(const Raw8<T>& r) {
  return __builtin_convertvector(__builtin_shufflevector(r.lo, r.hi, 0, 1, 2, 3, 4, 5, 6, 7), v8f);
}

// WHOLE: the lane's loads of kAhead rows leave together.
template <bool WHOLE, typename TI, typename TO>
__device__ __forceinline__ void sum_chunk(const Sum<TI, TO>& s, int chunk, int tile, int lane, int col, int apart) {
  const int begin = chunk * s.len;
  const int end = min(static_cast<int64_t>(begin) + s.len, static_cast<int64_t>(s.tokens));
  unsigned cur = s.keys[begin];
  if (cur >= s.vocab) return;
  bool reaches_in = begin > 0 && s.keys[begin - 1] == cur;
  const int left = s.c - col;
  v8f acc = {};
  auto flush = [&]() {
    if (reaches_in) {
      store44(s.slot(chunk, 0, tile, lane), s.lanes * 4, acc);
    } else {
      s.finish(cur, col, apart, WHOLE, acc);
    }
    reaches_in = false;
    acc = v8f{};
  };
  // The lists are read kAhead entries at a time, past the chunk's end too: they are padded to that.
  v4i key[kAhead / 4], pos[kAhead / 4];
  auto list = [&](int i) {
#pragma unroll
    for (int j = 0; j < kAhead / 4; ++j) {
      key[j] = *reinterpret_cast<const v4i*>(s.keys + i + 4 * j);
      pos[j] = *reinterpret_cast<const v4i*>(s.order + i + 4 * j);
    }
  };
  list(begin);
  for (int i = begin; i < end; i += kAhead) {
    unsigned k[kAhead];
    Raw8<TI> row[kAhead];
    v8f part[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      // a token without a row is read like any other, an entry past the end as the chunk's first
      k[j] = static_cast<unsigned>(key[j / 4][j & 3]);
      const int64_t t = i + j < end ? pos[j / 4][j & 3] : s.order[begin];
      const TI* from = s.dy + t * s.ld_dy + col;
      if constexpr (WHOLE) {
        load_raw<Sum<TI, TO>::kPairs>(row[j], from, apart);
      } else {
        part[j] = load44_of(from, apart, left);
      }
    }
    if (i + kAhead < end) list(i + kAhead);
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      if (i + j < end) {
        if (k[j] != cur) {
          flush();
          cur = k[j];
        }
        if (cur >= s.vocab) return;  // the rest are tokens without a row
        acc += WHOLE ? value(row[j]) : part[j];
      }
    }
  }
  if (end < s.tokens && s.keys[end] == cur) {
    store44(s.slot(chunk, reaches_in ? 0 : 1, tile, lane), s.lanes * 4, acc);
  } else {
    flush();
  }
}

// ---- up to kDirectTokens tokens: no sort -----------------------------------------------------------

// A workgroup per token and 512 channels: every thread looks at KEYS of the tokens, so that the ones
// of this token's row are found in order at once, and where the token is the row's first the
// workgroup adds them, its waves a contiguous part each and the parts in order.  The workgroups after
// these zero the rows that no token names, kZeroRows each.
//
// Bound by launch and latency.  257 to 1024 tokens take workgroups of 512 threads: 1024 tokens on
// 16384 x 512, fp32, in 9.9 us with all tokens apart, 12.4 with skewed ids and 27.4 with one id (with
// the sort 15.6, 18.5 and 29.4; of 256 threads 8.3, 17.2 and 54; of 1024 17.1, 16.8 and 27.3).  2048
// tokens apart would take 21 to 31 us, 17 with the sort: kDirectTokens ends before.  At most
// kDirectUnits workgroups: 1024 tokens of 1024 channels 11 us instead of 15, of 2048 channels 21 to 27
// instead of 16.
template <int THREADS, int KEYS, typename TI, typename TO>
__global__ __launch_bounds__(THREADS, 8) void embed_direct_kernel(Sum<TI, TO> s, const void* __restrict__ ids, bool ids64) {
  constexpr int kWaves = THREADS / 64;
  constexpr int kRows = sizeof(TI) == 2 ? 8 : 6;  // of dy in flight per lane
  __shared__ uint64_t found[KEYS * kWaves];
  __shared__ int pos[KEYS * THREADS];
  __shared__ v8f parts[kWaves][64];
  __shared__ int empty[kZeroRows];
  const int lane = threadIdx.x & 63;
  const int wave = threadIdx.x >> 6;
  const int token = blockIdx.x / s.col_tiles;
  const unsigned mine = token < s.tokens ? key_of(ids, ids64, token, s.vocab) : s.vocab;
  unsigned key[KEYS];
#pragma unroll
  for (int k = 0; k < KEYS; ++k) {
    const int t = k * THREADS + threadIdx.x;
    key[k] = t < s.tokens ? key_of(ids, ids64, t, s.vocab) : s.vocab;
  }
  if (token >= s.tokens) {
    const int64_t first = static_cast<int64_t>(blockIdx.x - s.sum_blocks) * kZeroRows;
    if (threadIdx.x < kZeroRows) empty[threadIdx.x] = 1;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < KEYS; ++k)
      if (key[k] >= first && key[k] < first + kZeroRows && key[k] < s.vocab) empty[key[k] - first] = 0;
    __syncthreads();
    zero_marked<THREADS>(s, first, empty);
    return;
  }
  if (mine >= s.vocab) return;
  uint64_t same[KEYS];
#pragma unroll
  for (int k = 0; k < KEYS; ++k) {
    same[k] = __ballot(key[k] == mine);
    if (lane == 0) found[k * kWaves + wave] = same[k];
  }
  __syncthreads();
  int n = 0;
#pragma unroll
  for (int w = 0; w < KEYS * kWaves; ++w) {
    const int here = __popcll(found[w]);
    if (w % kWaves == wave && key[w / kWaves] == mine)
      pos[n + __popcll(same[w / kWaves] & ((uint64_t{1} << lane) - 1))] = w * 64 + lane;
    n += here;
  }
  __syncthreads();
  if (pos[0] != token) return;  // another token is the row's first
  const int tile = blockIdx.x % s.col_tiles;
  int col, apart;
  bool whole;
  const bool there = s.place(tile, lane, &col, &apart, &whole);
  const int each = (n + kWaves - 1) / kWaves;
  const int from = min(wave * each, n), to = min(from + each, n);
  v8f acc = {};
  if (there && whole) {
    for (int i = from; i < to; i += kRows) {
      Raw8<TI> row[kRows];
#pragma unroll
      for (int j = 0; j < kRows; ++j)
        load_raw<Sum<TI, TO>::kPairs>(row[j], s.dy + pos[min(i + j, to - 1)] * s.ld_dy + col, apart);
#pragma unroll
      for (int j = 0; j < kRows; ++j)
        if (i + j < to) acc += value(row[j]);
    }
  } else if (there) {
    for (int i = from; i < to; ++i) acc += load44_of(s.dy + pos[i] * s.ld_dy + col, apart, s.c - col);
  }
  if (n > 1) {
    parts[wave][lane] = acc;
    __syncthreads();
    acc = parts[0][lane];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) acc += parts[w][lane];
  }
  if (wave == 0 && there) s.finish(mine, col, apart, whole, acc);
}

template <typename TI, typename TO>
__global__ __launch_bounds__(kThreads, sizeof(TI) == 2 ? 6 : 5) void embed_sum_kernel(Sum<TI, TO> s) {
  if (static_cast<int>(blockIdx.x) >= s.sum_blocks) {
    zero_rows(s, static_cast<int64_t>(blockIdx.x - s.sum_blocks) * kZeroRows);
    return;
  }
  const int64_t unit = (static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x) / s.lanes;
  const int chunk = static_cast<int>(unit / s.col_tiles), tile = static_cast<int>(unit % s.col_tiles);
  const int lane = threadIdx.x & (s.lanes - 1);
  int col, apart;
  bool whole;
  if (!s.place(tile, lane, &col, &apart, &whole) || chunk >= s.chunks) return;
  if (whole) sum_chunk<true>(s, chunk, tile, lane, col, apart);
  else sum_chunk<false>(s, chunk, tile, lane, col, apart);
}

// Adds the partial sums of the run that starts in chunk blockIdx.x / col_tiles and reaches over
// its end: each of the four waves a contiguous part of the chunks, the four parts in order.
template <typename TI, typename TO>
__global__ __launch_bounds__(kThreads) void embed_join_kernel(Sum<TI, TO> s) {
  __shared__ v8f parts[4][64];
  const int chunk = blockIdx.x / s.col_tiles;
  const int tile = blockIdx.x % s.col_tiles;
  const int begin = chunk * s.len;
  const int end = begin + s.len;  // the grid leaves out the last chunk: end < tokens
  const unsigned key = s.keys[end - 1];
  if (key >= s.vocab || s.keys[end] != key || (begin > 0 && s.keys[begin - 1] == key)) return;
  const int lane = threadIdx.x & 63;
  const int wave = threadIdx.x >> 6;
  int more = 0;  // chunks after this one that the run reaches into
  for (;;) {
    const int64_t at = static_cast<int64_t>(chunk) + 1 + more + lane;
    const uint64_t same = __ballot(at < s.chunks && s.keys[min(at * s.len, static_cast<int64_t>(s.tokens) - 1)] == key);
    more += __popcll(same);
    if (same != ~uint64_t{0}) break;
  }
  int col, apart;
  bool whole;
  const bool there = s.place(tile, lane, &col, &apart, &whole) && lane < s.lanes;
  const int each = (more + 1 + 3) / 4;
  const int from = wave * each;
  const int to = min(from + each, more + 1);
  v8f acc = {};
  if (there) {
#pragma unroll 8
    for (int i = from; i < to; ++i) acc += load44(s.slot(chunk + i, i == 0 ? 1 : 0, tile, lane), s.lanes * 4);
  }
  parts[wave][lane] = acc;
  __syncthreads();
  if (wave == 0 && there) {
#pragma unroll
    for (int w = 1; w < 4; ++w) acc += parts[w][lane];
    s.finish(key, col, apart, whole, acc);
  }
}

template <typename TI, typename TO>
hipError_t launch(const EmbedGradArgs& a, hipStream_t stream) {
  const Plan p = make_plan(a.vocab, a.c, a.tokens);
  const int64_t zero_blocks = a.accumulate ? 0 : (static_cast<int64_t>(a.vocab) + kZeroRows - 1) / kZeroRows;
  Sum<TI, TO> s{};
  s.dy = static_cast<const TI*>(a.dy);
  s.table = static_cast<TO*>(a.dtable);
  s.ld_dy = a.ld_dy;
  s.ld_table = a.ld_dtable;
  s.tokens = a.tokens;
  s.c = a.c;
  s.lanes = p.lanes;
  s.col_tiles = p.col_tiles;
  s.len = p.len;
  s.chunks = p.chunks;
  s.vocab = static_cast<unsigned>(a.vocab);
  s.scale = a.scale;
  s.accumulate = a.accumulate;
  if (p.direct) {
    s.lanes = 64;
    s.sum_blocks = a.tokens * p.col_tiles;
    const unsigned blocks = static_cast<unsigned>(s.sum_blocks + zero_blocks);
    if (a.tokens <= kDirectShort) embed_direct_kernel<kDirectShort, 1><<<blocks, kDirectShort, 0, stream>>>(s, a.ids, a.ids64);
    else embed_direct_kernel<512, kDirectTokens / 512><<<blocks, 512, 0, stream>>>(s, a.ids, a.ids64);
    return hipGetLastError();
  }
  char* ws = static_cast<char*>(a.ws);
  const unsigned vocab = static_cast<unsigned>(a.vocab);
  unsigned* keys = reinterpret_cast<unsigned*>(ws + p.keys0);
  int* order = reinterpret_cast<int*>(ws + p.order0);
  unsigned* where = reinterpret_cast<unsigned*>(ws + p.where);
  if (p.passes == 0) {
    // two lanes per token where 64 tokens a workgroup leave half of the CUs without one and the work
    // counts: 8192 tokens 34.0 -> 30.8 us a call, 1024 tokens 16.9 -> 17.4 (sorted)
    if (a.tokens <= kRankTokens / 2) {
      embed_rank_kernel<1><<<(a.tokens + 63) / 64, 1024, 0, stream>>>(a.ids, a.ids64, a.tokens, vocab, keys, order, where);
    } else {
      embed_rank_kernel<2><<<(a.tokens + 31) / 32, 1024, 0, stream>>>(a.ids, a.ids64, a.tokens, vocab, keys, order, where);
    }
  } else {
    unsigned* keys_to = reinterpret_cast<unsigned*>(ws + p.keys1);
    int* order_to = reinterpret_cast<int*>(ws + p.order1);
    unsigned* hist = reinterpret_cast<unsigned*>(ws + p.hist);
    for (int i = 0; i < p.passes; ++i) {
      Pass pass{i == 0 ? nullptr : keys, i == 0 ? nullptr : order, a.ids, a.ids64, vocab, a.tokens, p.per_block, p.blocks,
                i * p.digit_bits, 1 << p.digit_bits};
      embed_hist_kernel<<<p.blocks, kSortThreads, 0, stream>>>(pass, hist);
      embed_scatter_kernel<<<p.blocks, kSortThreads, 0, stream>>>(pass, hist, keys_to, order_to,
                                                                  i == p.passes - 1 ? where : nullptr);
      unsigned* k = keys;
      keys = keys_to;
      keys_to = k;
      int* o = order;
      order = order_to;
      order_to = o;
    }
  }
  s.keys = keys;
  s.order = order;
  s.where = where;
  s.part = reinterpret_cast<float*>(ws + p.part);
  const int64_t units = static_cast<int64_t>(p.chunks) * p.col_tiles;
  const int64_t per = kThreads / p.lanes;
  s.sum_blocks = static_cast<int>((units + per - 1) / per);
  embed_sum_kernel<TI, TO><<<static_cast<unsigned>(s.sum_blocks + zero_blocks), kThreads, 0, stream>>>(s);
  if (p.chunks > 1)
    embed_join_kernel<TI, TO><<<static_cast<unsigned>((p.chunks - 1) * p.col_tiles), kThreads, 0, stream>>>(s);
  return hipGetLastError();
}

}  // namespace

size_t embed_grad_workspace_bytes(int32_t vocab, int32_t c, int32_t tokens) {
  return make_plan(vocab, c, tokens).total;
}

void plan_embed_grad(int32_t vocab, int32_t c, int32_t tokens, int32_t* sorts, int32_t* chunks) {
  const Plan p = make_plan(vocab, c, tokens);
  *sorts = p.direct ? 0 : p.passes == 0 ? 1 : 2 * p.passes;
  *chunks = p.chunks;
}

hipError_t launch_embed_grad(const EmbedGradArgs& a, hipStream_t stream) {
  if (a.dy_bf16) return a.dtable_bf16 ? launch<__bf16, __bf16>(a, stream) : launch<__bf16, float>(a, stream);
  return a.dtable_bf16 ? launch<float, __bf16>(a, stream) : launch<float, float>(a, stream);
}

}  // namespace miq
