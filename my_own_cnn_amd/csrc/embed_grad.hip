// The embedding table's gradient by sorted tokens (miq_embed_grad).
//
// The (row, position) pairs of the tokens are sorted, stably, so that a row's tokens stand together
// in order of position; a position without a token has the key `vocab` and sorts to the end.  Up
// to kRankTokens tokens each token counts the ones before it directly, in one launch; above that
// the keys go through stable counting passes of up to 10 bits.  The sorted list is then cut into
// chunks of a fixed length: a group of lanes walks one chunk and 512 channels, adds the rows of dy
// of each run of equal keys in fp32 and writes the runs that lie within its chunk.  A run that
// reaches over a chunk's end leaves one partial sum per chunk in the workspace, and a last launch
// adds those in order.  The cuts depend on the number of tokens and channels alone: every call
// gives the same bits.
#include "train_device.h"

namespace miq {
namespace {

constexpr int kThreads = 256;
constexpr int kRankTokens = 8192;   // most tokens that are ranked by counting
constexpr int kDigitBits = 10;      // most bits of a counting pass
constexpr int kSortThreads = 512;
constexpr int kSortWaves = kSortThreads / 64;
constexpr int kCols = 512;          // channels per wave: 64 lanes of 8
constexpr int kZeroRows = 32;       // table rows per workgroup that zeros rows without a token
constexpr int kAhead = 8;           // rows of dy in flight per lane

struct Plan {
  int bits, passes, digit_bits, blocks, per_block;  // counting passes
  int lanes, col_tiles, len, chunks;                // lanes per chunk, chunk length
  size_t keys0, keys1, order0, order1, hist, part, total;
};

size_t up(size_t v) { return (v + 255) & ~static_cast<size_t>(255); }

Plan make_plan(int32_t vocab, int32_t c, int32_t tokens) {
  Plan p{};
  p.bits = 1;
  while ((static_cast<int64_t>(vocab) >> p.bits) != 0) ++p.bits;  // keys 0 .. vocab
  p.passes = (p.bits + kDigitBits - 1) / kDigitBits;
  p.digit_bits = (p.bits + p.passes - 1) / p.passes;
  // workgroups of the counting passes: 2048 tokens or more each, at most 256
  const int64_t t = tokens;
  int64_t per = (t + 255) / 256;
  per = (per < 2048 ? 2048 : per + kSortThreads - 1) / kSortThreads * kSortThreads;
  p.per_block = static_cast<int>(per);
  p.blocks = static_cast<int>((t + per - 1) / per);
  if (t <= kRankTokens) p.passes = 0;
  p.lanes = 8;
  while (p.lanes < 64 && p.lanes * 8 < c) p.lanes *= 2;
  p.col_tiles = (c + kCols - 1) / kCols;
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
  p.part = at; at += static_cast<size_t>(p.chunks) * 2 * p.col_tiles * (p.lanes * 8) * 4;
  p.total = at;
  return p;
}

__device__ __forceinline__ unsigned key_of(const void* ids, bool wide, int64_t t, unsigned vocab) {
  const uint64_t id = static_cast<uint64_t>(load_id(ids, wide, t));
  return id < vocab ? static_cast<unsigned>(id) : vocab;
}

// ---- up to kRankTokens tokens: a token's place is the number of tokens that sort before it -----

// 64 tokens per workgroup, one per lane; the 16 waves share the tokens to compare with.
__global__ __launch_bounds__(1024) void embed_rank_kernel(const void* __restrict__ ids, bool ids64, int tokens,
                                                          unsigned vocab, unsigned* __restrict__ keys,
                                                          int* __restrict__ order) {
  __shared__ unsigned all[kRankTokens];
  __shared__ int counts[16][64];
  for (int i = threadIdx.x; i < tokens; i += 1024) all[i] = key_of(ids, ids64, i, vocab);
  __syncthreads();
  const int lane = threadIdx.x & 63;
  const int wave = threadIdx.x >> 6;
  const int t0 = blockIdx.x * 64;
  const int t = t0 + lane;
  const unsigned mine = t < tokens ? all[t] : 0;
  int n = 0;
  // waves 0 .. 15 take every 16th group of 64 tokens
  for (int g = wave * 64; g < tokens; g += 1024) {
    const int end = min(g + 64, tokens);
    if (g < t0) {
      for (int i = g; i < end; ++i) n += all[i] <= mine;
    } else if (g > t0) {
      for (int i = g; i < end; ++i) n += all[i] < mine;
    } else {
      for (int i = g; i < end; ++i) n += all[i] < mine || (all[i] == mine && i < t);
    }
  }
  counts[wave][lane] = n;
  __syncthreads();
  if (wave == 0 && t < tokens) {
    int place = 0;
#pragma unroll
    for (int w = 0; w < 16; ++w) place += counts[w][lane];
    keys[place] = mine;
    order[place] = t;
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

// hist[digit][block]: the tokens of each workgroup's range by digit
__global__ __launch_bounds__(kSortThreads) void embed_hist_kernel(Pass p, unsigned* __restrict__ hist) {
  __shared__ unsigned n[1 << kDigitBits];
  for (int d = threadIdx.x; d < p.digits; d += kSortThreads) n[d] = 0;
  __syncthreads();
  const int64_t begin = static_cast<int64_t>(blockIdx.x) * p.per_block;
  const int64_t end = min(begin + p.per_block, static_cast<int64_t>(p.tokens));
  for (int64_t t = begin + threadIdx.x; t < end; t += kSortThreads)
    atomicAdd(&n[(pass_key(p, static_cast<int>(t)) >> p.shift) & (p.digits - 1)], 1u);
  __syncthreads();
  for (int d = threadIdx.x; d < p.digits; d += kSortThreads) hist[static_cast<size_t>(d) * p.blocks + blockIdx.x] = n[d];
}

// hist -> the place of each (digit, workgroup)'s first token; one workgroup, one digit per thread
__global__ __launch_bounds__(1 << kDigitBits) void embed_scan_kernel(unsigned* __restrict__ hist, int digits,
                                                                     int blocks) {
  __shared__ unsigned sums[1 << kDigitBits];
  const int d = threadIdx.x;
  unsigned total = 0;
  if (d < digits)
    for (int b = 0; b < blocks; ++b) total += hist[static_cast<size_t>(d) * blocks + b];
  sums[d] = total;
  __syncthreads();
  for (int step = 1; step < (1 << kDigitBits); step *= 2) {
    const unsigned before = d >= step ? sums[d - step] : 0;
    __syncthreads();
    sums[d] += before;
    __syncthreads();
  }
  if (d < digits) {
    unsigned at = sums[d] - total;
    for (int b = 0; b < blocks; ++b) {
      unsigned& h = hist[static_cast<size_t>(d) * blocks + b];
      const unsigned n = h;
      h = at;
      at += n;
    }
  }
}

// Each wave takes a contiguous part of its workgroup's range, 64 tokens at a time in order: a
// token's place is its wave's running place of its digit plus the lanes before it with that digit.
__global__ __launch_bounds__(kSortThreads) void embed_scatter_kernel(Pass p, const unsigned* __restrict__ hist,
                                                                     unsigned* __restrict__ keys,
                                                                     int* __restrict__ order) {
  __shared__ unsigned at[kSortWaves][1 << kDigitBits];
  const int wave = threadIdx.x >> 6;
  const int lane = threadIdx.x & 63;
  for (int i = threadIdx.x; i < kSortWaves * p.digits; i += kSortThreads) at[i / p.digits][i % p.digits] = 0;
  __syncthreads();
  const int part = p.per_block / kSortWaves;  // a multiple of 64
  const int64_t begin = static_cast<int64_t>(blockIdx.x) * p.per_block + wave * part;
  const int64_t end = min(begin + part, static_cast<int64_t>(p.tokens));
  for (int64_t t = begin + lane; t < end; t += 64)
    atomicAdd(&at[wave][(pass_key(p, static_cast<int>(t)) >> p.shift) & (p.digits - 1)], 1u);
  __syncthreads();
  for (int d = threadIdx.x; d < p.digits; d += kSortThreads) {
    unsigned place = hist[static_cast<size_t>(d) * p.blocks + blockIdx.x];
    for (int w = 0; w < kSortWaves; ++w) {
      const unsigned n = at[w][d];
      at[w][d] = place;
      place += n;
    }
  }
  __syncthreads();
  for (int64_t t0 = begin; t0 < end; t0 += 64) {
    const int64_t t = t0 + lane;
    const bool there = t < end;
    const unsigned key = there ? pass_key(p, static_cast<int>(t)) : 0;
    const int pos = there ? (p.order_in != nullptr ? p.order_in[t] : static_cast<int>(t)) : 0;
    const unsigned digit = (key >> p.shift) & (p.digits - 1);
    uint64_t same = __ballot(there);
    for (int bit = 1; bit < p.digits; bit *= 2) {
      const uint64_t set = __ballot((digit & bit) != 0);
      same &= (digit & bit) != 0 ? set : ~set;
    }
    const int before = __popcll(same & ((uint64_t{1} << lane) - 1));
    unsigned place = 0;
    if (there) place = at[wave][digit] + before;
    __builtin_amdgcn_wave_barrier();
    if (there && before == 0) at[wave][digit] += __popcll(same);
    __builtin_amdgcn_wave_barrier();
    if (there) {
      keys[place] = key;
      order[place] = pos;
    }
  }
}

// ---- the sums ------------------------------------------------------------------------------------

template <typename TI, typename TO>
struct Sum {
  const TI* dy;
  TO* table;
  const unsigned* keys;
  const int* order;
  float* part;
  int64_t ld_dy, ld_table;
  int tokens, c, lanes, col_tiles, len, chunks, sum_blocks;
  unsigned vocab;
  float scale;
  bool accumulate;

  // partial sums: [chunk][0: the run that reaches in, 1: the run that starts here and reaches on]
  __device__ float* slot(int chunk, int which, int tile, int lane) const {
    return part + ((static_cast<int64_t>(chunk) * 2 + which) * col_tiles + tile) * (lanes * 8) + lane * 8;
  }
  __device__ void finish(unsigned row, int col, v8f acc) const {
    TO* to = table + row * ld_table + col;
    acc *= scale;
    if (accumulate) acc += load8_of(to, c - col);
    store8_of(to, acc, c - col);
  }
};

template <typename TI, typename TO>
__device__ __forceinline__ void sum_chunk(const Sum<TI, TO>& s, int chunk, int tile, int lane) {
  const int col = tile * kCols + lane * 8;
  if (chunk >= s.chunks || col >= s.c) return;
  const int begin = chunk * s.len;
  const int end = min(static_cast<int64_t>(begin) + s.len, static_cast<int64_t>(s.tokens));
  unsigned cur = s.keys[begin];
  if (cur >= s.vocab) return;
  bool reaches_in = begin > 0 && s.keys[begin - 1] == cur;
  const int left = s.c - col;
  v8f acc = {};
  auto flush = [&]() {
    if (reaches_in) {
      store8(s.slot(chunk, 0, tile, lane), acc);
    } else {
      s.finish(cur, col, acc);
    }
    reaches_in = false;
    acc = v8f{};
  };
  for (int i = begin; i < end; i += kAhead) {
    unsigned key[kAhead];
    v8f row[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      key[j] = i + j < end ? s.keys[i + j] : s.vocab;
      const int t = i + j < end ? s.order[i + j] : 0;
      row[j] = key[j] < s.vocab ? load8_of(s.dy + t * s.ld_dy + col, left) : v8f{};
    }
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      if (i + j < end && cur < s.vocab) {
        if (key[j] != cur) {
          flush();
          cur = key[j];
        }
        acc += row[j];
      }
    }
  }
  if (cur >= s.vocab) return;
  if (end < s.tokens && s.keys[end] == cur) {
    store8(s.slot(chunk, reaches_in ? 0 : 1, tile, lane), acc);
  } else {
    flush();
  }
}

// Zeros in the rows [first, first + kZeroRows) that no token names.
template <typename TI, typename TO>
__device__ __forceinline__ void zero_rows(const Sum<TI, TO>& s, int64_t first) {
  __shared__ int starts[kZeroRows + 1];
  const int rows = static_cast<int>(min(static_cast<int64_t>(kZeroRows), s.vocab - first));
  if (threadIdx.x <= rows) {  // the first place of row first + threadIdx.x
    const unsigned row = static_cast<unsigned>(first) + threadIdx.x;
    int lo = 0, hi = s.tokens;
    while (lo < hi) {
      const int mid = lo + (hi - lo) / 2;
      if (s.keys[mid] < row) lo = mid + 1;
      else hi = mid;
    }
    starts[threadIdx.x] = lo;
  }
  __syncthreads();
  for (int r = 0; r < rows; ++r) {
    if (starts[r] != starts[r + 1]) continue;
    for (int col = threadIdx.x * 8; col < s.c; col += kThreads * 8)
      store8_of(s.table + (first + r) * s.ld_table + col, v8f{}, s.c - col);
  }
}

template <typename TI, typename TO>
__global__ __launch_bounds__(kThreads) void embed_sum_kernel(Sum<TI, TO> s) {
  if (static_cast<int>(blockIdx.x) < s.sum_blocks) {
    const int64_t unit = (static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x) / s.lanes;
    sum_chunk(s, static_cast<int>(unit / s.col_tiles), static_cast<int>(unit % s.col_tiles), threadIdx.x & (s.lanes - 1));
  } else {
    zero_rows(s, static_cast<int64_t>(blockIdx.x - s.sum_blocks) * kZeroRows);
  }
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
  const int col = tile * kCols + lane * 8;
  const bool there = lane < s.lanes && col < s.c;
  const int each = (more + 1 + 3) / 4;
  const int from = wave * each;
  const int to = min(from + each, more + 1);
  v8f acc = {};
  if (there) {
#pragma unroll 4
    for (int i = from; i < to; ++i) acc += load8(s.slot(chunk + i, i == 0 ? 1 : 0, tile, lane));
  }
  parts[wave][lane] = acc;
  __syncthreads();
  if (wave == 0 && there) {
#pragma unroll
    for (int w = 1; w < 4; ++w) acc += parts[w][lane];
    s.finish(key, col, acc);
  }
}

template <typename TI, typename TO>
hipError_t launch_sums(const EmbedGradArgs& a, const Plan& p, const unsigned* keys, const int* order,
                       hipStream_t stream) {
  Sum<TI, TO> s{};
  s.dy = static_cast<const TI*>(a.dy);
  s.table = static_cast<TO*>(a.dtable);
  s.keys = keys;
  s.order = order;
  s.part = reinterpret_cast<float*>(static_cast<char*>(a.ws) + p.part);
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
  const int64_t units = static_cast<int64_t>(p.chunks) * p.col_tiles;
  const int64_t per = kThreads / p.lanes;
  s.sum_blocks = static_cast<int>((units + per - 1) / per);
  const int64_t zero_blocks = a.accumulate ? 0 : (static_cast<int64_t>(a.vocab) + kZeroRows - 1) / kZeroRows;
  embed_sum_kernel<TI, TO><<<static_cast<unsigned>(s.sum_blocks + zero_blocks), kThreads, 0, stream>>>(s);
  if (p.chunks > 1)
    embed_join_kernel<TI, TO><<<static_cast<unsigned>((p.chunks - 1) * p.col_tiles), kThreads, 0, stream>>>(s);
  return hipGetLastError();
}

}  // namespace

size_t embed_grad_workspace_bytes(int32_t vocab, int32_t c, int32_t tokens) {
  return make_plan(vocab, c, tokens).total;
}

hipError_t launch_embed_grad(const EmbedGradArgs& a, hipStream_t stream) {
  const Plan p = make_plan(a.vocab, a.c, a.tokens);
  char* ws = static_cast<char*>(a.ws);
  unsigned* keys = reinterpret_cast<unsigned*>(ws + p.keys0);
  int* order = reinterpret_cast<int*>(ws + p.order0);
  const unsigned vocab = static_cast<unsigned>(a.vocab);
  if (a.tokens > 0 && p.passes == 0) {
    embed_rank_kernel<<<(a.tokens + 63) / 64, 1024, 0, stream>>>(a.ids, a.ids64, a.tokens, vocab, keys, order);
  } else if (a.tokens > 0) {
    unsigned* keys_to = reinterpret_cast<unsigned*>(ws + p.keys1);
    int* order_to = reinterpret_cast<int*>(ws + p.order1);
    unsigned* hist = reinterpret_cast<unsigned*>(ws + p.hist);
    for (int i = 0; i < p.passes; ++i) {
      Pass s{i == 0 ? nullptr : keys, i == 0 ? nullptr : order, a.ids, a.ids64, vocab, a.tokens, p.per_block, p.blocks,
             i * p.digit_bits, 1 << p.digit_bits};
      embed_hist_kernel<<<p.blocks, kSortThreads, 0, stream>>>(s, hist);
      embed_scan_kernel<<<1, 1 << kDigitBits, 0, stream>>>(hist, s.digits, p.blocks);
      embed_scatter_kernel<<<p.blocks, kSortThreads, 0, stream>>>(s, hist, keys_to, order_to);
      unsigned* k = keys;
      keys = keys_to;
      keys_to = k;
      int* o = order;
      order = order_to;
      order_to = o;
    }
  }
  if (a.dy_bf16) {
    return a.dtable_bf16 ? launch_sums<__bf16, __bf16>(a, p, keys, order, stream)
                         : launch_sums<__bf16, float>(a, p, keys, order, stream);
  }
  return a.dtable_bf16 ? launch_sums<float, __bf16>(a, p, keys, order, stream)
                       : launch_sums<float, float>(a, p, keys, order, stream);
}

}  // namespace miq
