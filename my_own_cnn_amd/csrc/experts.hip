// Rows sorted by expert, and their way back (miq_experts_plan, miq_experts_join).
#include "row8_device.h"

namespace miq {
namespace {

// One workgroup per expert looks at all ids twice: it counts those of the experts before its own, which
// is where its rows start, and its own per wave, and then writes each of its own at its place.  No
// workgroup waits for another, and the places depend on the ids alone.  16384 ids on 32 experts 8 us (14 without
// runs loaded together); 262144 on 64 68 us, bound by what one CU reads twice.
constexpr int kPlanThreads = 1024, kPlanWaves = kPlanThreads / 64;

template <typename ID>
__global__ __launch_bounds__(kPlanThreads) void experts_plan_kernel(ExpertsPlanArgs a, FastDivM by_slots) {
  __shared__ int before[kPlanWaves], own[kPlanWaves];
  const ID* const ids = static_cast<const ID*>(a.ids);
  const int expert = blockIdx.x, wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  // a wave's ids: whole runs of 64, none past n
  const int64_t runs = (static_cast<int64_t>(a.n) + 63) / 64;
  const int64_t each = (runs + kPlanWaves - 1) / kPlanWaves;
  const int64_t from = min(wave * each, runs) * 64;
  const int64_t to = min((wave + 1) * each, runs) * 64;
  // eight runs of 64 at a time, loaded together
  constexpr int kRuns = 8;
  auto load = [&](int64_t base, ID (&id)[kRuns]) {
#pragma unroll
    for (int u = 0; u < kRuns; ++u) {
      const int64_t i = base + u * 64 + lane;
      id[u] = i < to && i < a.n ? ids[i] : -1;
    }
  };
  int less = 0, same = 0;
  for (int64_t base = from; base < to; base += 64 * kRuns) {
    ID id[kRuns];
    load(base, id);
#pragma unroll
    for (int u = 0; u < kRuns; ++u) {
      less += id[u] >= 0 && id[u] < expert;
      same += id[u] == expert;
    }
  }
  for (int step = 1; step < 64; step *= 2) {
    less += __shfl_xor(less, step);
    same += __shfl_xor(same, step);
  }
  if (lane == 0) {
    before[wave] = less;
    own[wave] = same;
  }
  __syncthreads();
  int start = 0, count = 0, at = 0;
  for (int w = 0; w < kPlanWaves; ++w) {
    start += before[w];
    at += w < wave ? own[w] : 0;
    count += own[w];
  }
  at += start;
  for (int64_t base = from; base < to; base += 64 * kRuns) {
    ID id[kRuns];
    load(base, id);
#pragma unroll
    for (int u = 0; u < kRuns; ++u) {
      const int64_t i = base + u * 64 + lane;
      const uint64_t mine = __ballot(id[u] == expert);
      if (mine >> lane & 1) {
        const int place = at + __popcll(mine & ((uint64_t{1} << lane) - 1));
        a.rows[place] = fdiv(static_cast<int>(i), by_slots);
        a.places[i] = place;
      }
      if (expert == 0 && i < to && i < a.n && (id[u] < 0 || id[u] >= a.experts)) a.places[i] = -1;
      at += __popcll(mine);
    }
  }
  if (threadIdx.x == 0) a.offsets[expert] = start;
  if (expert == a.experts - 1) {
    const int total = start + count;
    if (threadIdx.x == 0) a.offsets[a.experts] = total;
    for (int64_t i = total + static_cast<int64_t>(threadIdx.x); i < a.n; i += kPlanThreads) a.rows[i] = -1;
  }
}

// out[t] = add[t] + sum over j of share[t, j] * y[places[t, j]], in the order of j: 16 bytes of a row a lane.
// Bound by memory: 8192 x 2 rows of 2048 bf16 (101 MB) 19 us, 5.2 TB/s.
struct Join {
  int64_t total;  // lanes
  int per_row;
  FastDivM div;  // by per_row
};
template <typename T>
__global__ __launch_bounds__(256) void experts_join_kernel(ExpertsJoinArgs a, Join e) {
  constexpr int W = kWide<T>;
  typedef typename Vec<W>::type Run;
  for (int64_t base = static_cast<int64_t>(blockIdx.x) * 256; base < e.total; base += static_cast<int64_t>(gridDim.x) * 256) {
    if (base + threadIdx.x >= e.total) continue;
    const int64_t t0 = base / e.per_row;  // the workgroup's, one division
    const int at = static_cast<int>(base - t0 * e.per_row) + static_cast<int>(threadIdx.x);
    const int over = fdiv(at, e.div);
    const int64_t t = t0 + over;
    const int col = (at - over * e.per_row) * W, left = a.c - col;
    Run sum = {};
    if (a.add != nullptr) sum = load_some<false>(static_cast<const T*>(a.add) + t * a.ld_add + col, left);
    for (int j = 0; j < a.slots; ++j) {
      const int place = a.places[t * a.slots + j];
      if (place < 0 || place >= a.rows) continue;
      const float share = a.share != nullptr ? a.share[t * a.slots + j] : 1.0f;
      sum += load_some<false>(static_cast<const T*>(a.y) + place * a.ld_y + col, left) * share;
    }
    store_some<false>(static_cast<T*>(a.out) + t * a.ld_out + col, sum, left);
  }
}

}  // namespace

hipError_t launch_experts_plan(const ExpertsPlanArgs& a, hipStream_t stream) {
  const FastDivM div = fastdiv_m(static_cast<uint32_t>(a.slots));
  const unsigned grid = static_cast<unsigned>(a.experts);
  if (a.ids64) experts_plan_kernel<int64_t><<<grid, kPlanThreads, 0, stream>>>(a, div);
  else experts_plan_kernel<int32_t><<<grid, kPlanThreads, 0, stream>>>(a, div);
  return hipGetLastError();
}

hipError_t launch_experts_join(const ExpertsJoinArgs& a, hipStream_t stream) {
  const int wide = a.bf16 ? 8 : 4;
  Join e{};
  e.per_row = static_cast<int>((static_cast<int64_t>(a.c) + wide - 1) / wide);
  e.total = a.tokens * e.per_row;
  e.div = fastdiv_m(static_cast<uint32_t>(e.per_row));
  const int64_t blocks = (e.total + 255) / 256;
  const unsigned grid = static_cast<unsigned>(blocks < (1 << 23) ? blocks : (1 << 23));
  if (a.bf16) experts_join_kernel<__bf16><<<grid, 256, 0, stream>>>(a, e);
  else experts_join_kernel<float><<<grid, 256, 0, stream>>>(a, e);
  return hipGetLastError();
}

}  // namespace miq
