// Internal interface between train_capi.cpp and the kernels of the token-network entry points
// (embed.hip, embed_grad.hip, act8.hip, act8_grad.hip).
#pragma once

#include <hip/hip_runtime.h>

#include <cstddef>
#include <cstdint>

namespace miq {

constexpr int kAct8Group = 32;  // channels that share an exponent byte

struct EmbedArgs {
  const void* table;
  const void* ids;
  void* y;
  int64_t ld_table, ld_y, tokens;
  int32_t vocab, c;
  float scale;
  bool table_bf16, ids64, y_bf16;
};
hipError_t launch_embed_fprop(const EmbedArgs& a, hipStream_t stream);

struct EmbedGradArgs {
  const void* dy;
  const void* ids;
  void* dtable;
  void* ws;
  int64_t ld_dy, ld_dtable;
  int32_t tokens, vocab, c;
  float scale;
  bool accumulate, dy_bf16, ids64, dtable_bf16;
};
size_t embed_grad_workspace_bytes(int32_t vocab, int32_t c, int32_t tokens);
void plan_embed_grad(int32_t vocab, int32_t c, int32_t tokens, int32_t* sorts, int32_t* chunks);
hipError_t launch_embed_grad(const EmbedGradArgs& a, hipStream_t stream);

// x, y: act8_fprop; dy, y (= dx): act8_bprop; y: act8_expand.
struct Act8Args {
  const void* x;
  const void* dy;
  void* y;
  int8_t* codes;
  uint8_t* scales;
  int64_t rows, ld_x, ld_dy, ld_y;
  int32_t c, act;
  bool gated, bf16;
};
hipError_t launch_act8_fprop(const Act8Args& a, hipStream_t stream);
hipError_t launch_act8_bprop(const Act8Args& a, hipStream_t stream);
hipError_t launch_act8_expand(const Act8Args& a, hipStream_t stream);

struct Act8GradArgs {
  const void* dy;
  const int8_t* codes;
  const uint8_t* scales;
  void* dw;
  void* ws;
  int64_t ld_dy, ld_dw;
  int32_t rows, c, k;
  bool accumulate, dy_bf16, dw_bf16;
};
size_t act8_grad_workspace_bytes(int32_t rows, int32_t c, int32_t k, bool dy_bf16);
void plan_act8_grad(int32_t rows, int32_t c, int32_t k, bool dy_bf16, int32_t* tile, int32_t* splits);
hipError_t launch_act8_grad(const Act8GradArgs& a, hipStream_t stream);

}  // namespace miq
