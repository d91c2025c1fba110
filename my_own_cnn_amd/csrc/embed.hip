// y[t, :] = scale * table[ids[t], :] (miq_embed_fprop).
//
// Bound by memory: the rows read and the rows written, each once.  A lane writes runs of 16 bytes,
// neighbouring lanes neighbouring runs, so that every store of a wave covers whole lines: eight
// channels of bf16, or four of fp32 twice (fp32 rows to bf16, 65536 rows of 2048: 95 us, and 111
// with stores of 8 bytes).  Where a row ends within a run, the lane takes the row's last run
// instead: it writes what its neighbour writes in part, the same values.
#include "train_device.h"

namespace miq {
namespace {

constexpr int kThreads = 256;

template <bool STREAM, typename TI>
__device__ __forceinline__ void move(const TI* from, __bf16* to, float scale, bool there) {
  v8f v = {};
  if (there) v = load8(from) * scale;
  store_run<STREAM>(to, v);
}
template <bool STREAM, typename TI>
__device__ __forceinline__ void move(const TI* from, float* to, float scale, bool there) {
  v4f v = {};
  if (there) v = load4(from) * scale;
  store_run<STREAM>(to, v);
}

// One row per 2^row_log threads.
template <bool STREAM, typename TI, typename TO>
__global__ __launch_bounds__(kThreads) void embed_fprop_kernel(const TI* __restrict__ table, const void* __restrict__ ids,
                                                               TO* __restrict__ y, int vocab, int c, int64_t tokens,
                                                               int64_t ld_table, int64_t ld_y, float scale, bool ids64,
                                                               int row_log) {
  constexpr int W = 16 / static_cast<int>(sizeof(TO)), kRuns = 8 / W;
  const int rows = kThreads >> row_log;
  const int lane = threadIdx.x & ((1 << row_log) - 1);
  for (int64_t t = static_cast<int64_t>(blockIdx.x) * rows + (threadIdx.x >> row_log); t < tokens;
       t += static_cast<int64_t>(gridDim.x) * rows) {
    const int64_t id = load_id(ids, ids64, t);
    const bool there = id >= 0 && id < vocab;
    const TI* from = table + (there ? id : 0) * ld_table;
    TO* to = y + t * ld_y;
    if (c < W) {
      if (lane < c) to[lane] = there ? static_cast<TO>(static_cast<float>(from[lane]) * scale) : static_cast<TO>(0.0f);
      continue;
    }
    for (int base = lane * W; base < c; base += (kRuns * W) << row_log) {
#pragma unroll
      for (int r = 0; r < kRuns; ++r) {
        const int col = base + ((r * W) << row_log);
        if (col < c) move<STREAM>(from + min(col, c - W), to + min(col, c - W), scale, there);
      }
    }
  }
}

template <typename TI, typename TO>
void launch(const EmbedArgs& a, int blocks, int row_log, hipStream_t stream) {
  auto* kernel = stream_stores(a.y, a.tokens, a.c, a.ld_y, sizeof(TO)) ? &embed_fprop_kernel<true, TI, TO>
                                                                       : &embed_fprop_kernel<false, TI, TO>;
  kernel<<<blocks, kThreads, 0, stream>>>(static_cast<const TI*>(a.table), a.ids, static_cast<TO*>(a.y), a.vocab, a.c,
                                          a.tokens, a.ld_table, a.ld_y, a.scale, a.ids64, row_log);
}

}  // namespace

hipError_t launch_embed_fprop(const EmbedArgs& a, hipStream_t stream) {
  int row_log = 3;
  while (row_log < 8 && (8 << row_log) < a.c) ++row_log;
  const int64_t per = kThreads >> row_log;
  const int64_t want = (a.tokens + per - 1) / per;
  const int blocks = static_cast<int>(want < (1 << 20) ? want : (1 << 20));
  if (a.table_bf16) {
    a.y_bf16 ? launch<__bf16, __bf16>(a, blocks, row_log, stream) : launch<__bf16, float>(a, blocks, row_log, stream);
  } else {
    a.y_bf16 ? launch<float, __bf16>(a, blocks, row_log, stream) : launch<float, float>(a, blocks, row_log, stream);
  }
  return hipGetLastError();
}

}  // namespace miq
