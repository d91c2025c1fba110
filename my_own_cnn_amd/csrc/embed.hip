// y[t, :] = scale * table[ids[t], :] (miq_embed_fprop).
#include "train_device.h"

namespace miq {
namespace {

constexpr int kThreads = 256;

// One row per 2^row_log threads, eight channels per thread and step.
template <typename TI, typename TO>
__global__ __launch_bounds__(kThreads) void embed_fprop_kernel(const TI* __restrict__ table, const void* __restrict__ ids,
                                                               TO* __restrict__ y, int vocab, int c, int64_t tokens,
                                                               int64_t ld_table, int64_t ld_y, float scale, bool ids64,
                                                               int row_log) {
  const int rows = kThreads >> row_log;
  const int lane = threadIdx.x & ((1 << row_log) - 1);
  for (int64_t t = static_cast<int64_t>(blockIdx.x) * rows + (threadIdx.x >> row_log); t < tokens;
       t += static_cast<int64_t>(gridDim.x) * rows) {
    const int64_t id = load_id(ids, ids64, t);
    const bool there = id >= 0 && id < vocab;
    for (int col = lane * 8; col < c; col += 8 << row_log) {
      v8f v = {};
      if (there) v = load8_of(table + id * ld_table + col, c - col) * scale;
      store8_of(y + t * ld_y + col, v, c - col);
    }
  }
}

template <typename TI, typename TO>
void launch(const EmbedArgs& a, int blocks, int row_log, hipStream_t stream) {
  embed_fprop_kernel<TI, TO><<<blocks, kThreads, 0, stream>>>(static_cast<const TI*>(a.table), a.ids,
                                                              static_cast<TO*>(a.y), a.vocab, a.c, a.tokens, a.ld_table,
                                                              a.ld_y, a.scale, a.ids64, row_log);
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
