// Internal interface between row8_capi.cpp and the kernels of 8-bit rows (rms.hip, rms_grad.hip,
// row8.hip, row8_linear.cpp, row8_few.hip, row8_tile.hip, experts.hip).
#pragma once

#include <hip/hip_runtime.h>

#include <cstddef>
#include <cstdint>

namespace miq {

// sum, add: both or neither.  y: rms_fprop; codes, scales: rms_row8.
struct RmsArgs {
  const void* x;
  const void* add;
  const void* gain;
  void* sum;
  void* y;
  int8_t* codes;
  float* scales;
  int64_t rows, ld_x, ld_add, ld_sum, ld_y;
  int32_t c;
  float eps;
  bool bf16, gain_bf16;
};
hipError_t launch_rms(const RmsArgs& a, hipStream_t stream);

struct RmsGradArgs {
  const void* dy;
  const void* x;
  const void* gain;
  const void* dsum;
  void* dx;
  void* dgain;
  float* ws;
  int64_t rows, ld_dy, ld_x, ld_dsum, ld_dx;
  int32_t c;
  float eps;
  bool accumulate, bf16, gain_bf16, dgain_bf16;
};
size_t rms_grad_workspace_bytes(int64_t rows, int32_t c);
hipError_t launch_rms_grad(const RmsGradArgs& a, hipStream_t stream);

struct ActRow8Args {
  const void* x;
  int8_t* codes;
  float* scales;
  int64_t rows, ld_x;
  int32_t c, act;
  bool gated, bf16;
};
hipError_t launch_act_row8(const ActRow8Args& a, hipStream_t stream);

struct Row8ExpandArgs {
  const int8_t* codes;
  const float* scales;
  void* y;
  int64_t rows, ld_y;
  int32_t c;
  bool bf16;
};
hipError_t launch_row8_expand(const Row8ExpandArgs& a, hipStream_t stream);

// One product, or (offsets not NULL) `experts` of them: rows offsets[e] .. offsets[e + 1] - 1 of y by
// w[e].  index (or NULL): the row of x of each row of y.
struct Row8LinearArgs {
  const int8_t* x;
  const float* x_scales;
  const int8_t* w;
  const float* w_scales;
  const float* bias;
  const void* add;
  const int32_t* offsets;
  const int32_t* index;
  void* y;
  void* ws;  // of row8_workspace_bytes
  int64_t ld_add, ld_y;
  int32_t x_rows, rows, c, k, experts;
  bool bf16;
};
hipError_t launch_row8_few(const Row8LinearArgs& a, int rows, int channels, hipStream_t stream);
hipError_t launch_row8_tile(const Row8LinearArgs& a, int rows, int channels, hipStream_t stream);
// Two tensors' rows of c codes to rows of `width`, the rest zeros: x's, then w's.
hipError_t launch_row8_pad(const int8_t* x, int64_t x_rows, const int8_t* w, int64_t w_rows, int32_t c, int32_t width,
                           int8_t* to, hipStream_t stream);
// plan: whether the weights go straight to the matrix instructions (few rows), a tile's rows and channels, whether
// rows are first copied to the workspace.
void plan_row8_linear(int32_t rows, int32_t c, int32_t k, int32_t experts, int32_t plan[4]);
size_t row8_workspace_bytes(int32_t x_rows, int32_t rows, int32_t c, int32_t k, int32_t experts);
hipError_t launch_row8_linear(const Row8LinearArgs& a, hipStream_t stream);

struct ExpertsPlanArgs {
  const void* ids;
  int32_t* offsets;
  int32_t* rows;
  int32_t* places;
  int32_t n, slots, experts;
  bool ids64;
};
hipError_t launch_experts_plan(const ExpertsPlanArgs& a, hipStream_t stream);

struct ExpertsJoinArgs {
  const void* y;
  const int32_t* places;
  const float* share;  // or NULL: ones
  const void* add;     // or NULL
  void* out;
  int64_t tokens, ld_y, ld_add, ld_out;
  int32_t rows, slots, c;
  bool bf16;
};
hipError_t launch_experts_join(const ExpertsJoinArgs& a, hipStream_t stream);

}  // namespace miq
