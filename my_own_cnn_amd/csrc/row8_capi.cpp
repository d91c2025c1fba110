// extern "C" entry points of the norm and of products on 8-bit rows: host-side validation and dispatch.
// Nothing is enqueued before the arguments are validated, and nothing is allocated.
#include <cstdint>

#include "miq_qconv.h"
#include "qconv_internal.h"
#include "row8_internal.h"

namespace {

constexpr int64_t kMaxPositions = 0x7fffffffLL - 64;  // rows of a product are counted in int32
constexpr int32_t kMaxChannels = 1 << 29;             // two halves of a gated row stay in int32
constexpr int64_t kMaxRows = 1LL << 40;
constexpr int64_t kMaxValues = 1LL << 46;             // byte offsets stay far inside int64
constexpr int32_t kMaxSum = 131071;                   // products of 8-bit codes whose sum stays in int32
constexpr int32_t kMaxSide = 1 << 22;
constexpr int32_t kMaxExperts = 4096;

int bad(const char* msg) { return miq::record_error(MIQ_ERR_INVALID_ARGUMENT, msg); }
int null(const char* msg) { return miq::record_error(MIQ_ERR_NULL_POINTER, msg); }

int done(hipError_t e) { return e == hipSuccess ? MIQ_OK : miq::record_error(MIQ_ERR_HIP, hipGetErrorString(e)); }

bool real_type(int32_t t) { return t == MIQ_F32 || t == MIQ_BF16; }
bool aligned(const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }
uintptr_t size_of(int32_t type) { return type == MIQ_BF16 ? 2 : type == MIQ_I64 ? 8 : 4; }
bool stride_ok(int64_t ld, int64_t width) { return ld >= width && ld <= kMaxValues; }

constexpr const char* kShortRows = "row distance is smaller than the row";
constexpr const char* kUnaligned = "a pointer is not aligned to its element";

int check_rows(int64_t rows, int32_t c) {
  if (rows < 0 || c < 0) return bad("extents of rows must be >= 0");
  if (c > kMaxChannels || rows > kMaxRows || (c > 0 && rows > kMaxValues / c)) {
    return bad("rows exceed 2^29 channels, 2^40 rows or 2^46 values");
  }
  return MIQ_OK;
}

int check_norm(int64_t rows, int32_t c, float eps, int32_t type, int32_t gain_type) {
  const int st = check_rows(rows, c);
  if (st != MIQ_OK) return st;
  if (!(eps >= 1e-30f && eps <= 1e30f)) return bad("eps must lie in 1e-30 .. 1e30");
  if (!real_type(type) || !real_type(gain_type)) return bad("type and gain_type must be MIQ_F32 or MIQ_BF16");
  return MIQ_OK;
}

int norm(const void* x, const void* add, const void* gain, void* sum, void* y, int8_t* codes, float* scales,
         int64_t rows, int32_t c, int64_t ld_x, int64_t ld_add, int64_t ld_sum, int64_t ld_y, float eps, int32_t type,
         int32_t gain_type, bool real, void* stream) {
  const int st = check_norm(rows, c, eps, type, gain_type);
  if (st != MIQ_OK) return st;
  if (!stride_ok(ld_x, c) || (real && !stride_ok(ld_y, c)) ||
      (add != nullptr && (!stride_ok(ld_add, c) || !stride_ok(ld_sum, c)))) {
    return bad(kShortRows);
  }
  if (rows == 0 || c == 0) return MIQ_OK;
  if (x == nullptr) return null("input pointer is NULL");
  if (gain == nullptr) return null("gain pointer is NULL");
  if ((add == nullptr) != (sum == nullptr)) return null("add and sum come together, one of them is NULL");
  if (real ? y == nullptr : codes == nullptr || scales == nullptr) return null("output pointer is NULL");
  const uintptr_t size = size_of(type);
  if (!aligned(x, size) || !aligned(add, size) || !aligned(sum, size) || !aligned(y, size) ||
      !aligned(gain, size_of(gain_type)) || !aligned(scales, 4)) {
    return bad(kUnaligned);
  }
  miq::RmsArgs a{};
  a.x = x;
  a.add = add;
  a.gain = gain;
  a.sum = sum;
  a.y = y;
  a.codes = codes;
  a.scales = scales;
  a.rows = rows;
  a.ld_x = ld_x;
  a.ld_add = ld_add;
  a.ld_sum = ld_sum;
  a.ld_y = ld_y;
  a.c = c;
  a.eps = eps;
  a.bf16 = type == MIQ_BF16;
  a.gain_bf16 = gain_type == MIQ_BF16;
  return done(miq::launch_rms(a, static_cast<hipStream_t>(stream)));
}

int check_product(int64_t rows, int32_t c, int32_t k, int32_t experts) {
  if (rows < 0 || c < 0 || k < 0) return bad("extents of a product must be >= 0");
  if (rows > kMaxPositions) return bad("a product takes at most 2^31 - 65 rows");
  if (c > kMaxSum) return bad("a product takes at most 131071 channels: sums of more leave 32 bits");
  if (k > kMaxSide) return bad("a product has at most 2^22 output channels");
  if (experts < 1 || experts > kMaxExperts) return bad("experts must lie in 1 .. 4096");
  return MIQ_OK;
}

int check_plan(int64_t tokens, int32_t slots, int32_t experts) {
  if (tokens < 0 || slots < 1) return bad("tokens must be >= 0 and slots >= 1");
  if (tokens > kMaxPositions / slots) return bad("a plan takes at most 2^31 - 65 ids");
  if (experts < 1 || experts > kMaxExperts) return bad("experts must lie in 1 .. 4096");
  return MIQ_OK;
}

}  // namespace

extern "C" {

int miq_rms_fprop(const void* x, const void* add, const void* gain, void* sum, void* y, int64_t rows, int32_t c,
                  int64_t ld_x, int64_t ld_add, int64_t ld_sum, int64_t ld_y, float eps, int32_t type,
                  int32_t gain_type, void* stream) {
  return norm(x, add, gain, sum, y, nullptr, nullptr, rows, c, ld_x, ld_add, ld_sum, ld_y, eps, type, gain_type, true,
              stream);
}

int miq_rms_row8(const void* x, const void* add, const void* gain, void* sum, int8_t* codes, float* scales, int64_t rows,
                 int32_t c, int64_t ld_x, int64_t ld_add, int64_t ld_sum, float eps, int32_t type, int32_t gain_type,
                 void* stream) {
  return norm(x, add, gain, sum, nullptr, codes, scales, rows, c, ld_x, ld_add, ld_sum, 0, eps, type, gain_type, false,
              stream);
}

int miq_rms_bprop_workspace_size(int64_t rows, int32_t c, size_t* bytes) {
  if (bytes == nullptr) return null("bytes pointer is NULL");
  const int st = check_rows(rows, c);
  if (st != MIQ_OK) return st;
  *bytes = rows == 0 || c == 0 ? 0 : miq::rms_grad_workspace_bytes(rows, c);
  return MIQ_OK;
}

int miq_rms_bprop(const void* dy, const void* x, const void* gain, const void* dsum, void* dx, void* dgain, int64_t rows,
                  int32_t c, int64_t ld_dy, int64_t ld_x, int64_t ld_dsum, int64_t ld_dx, float eps, int32_t accumulate,
                  int32_t type, int32_t gain_type, int32_t dgain_type, void* workspace, size_t workspace_bytes,
                  void* stream) {
  const int st = check_norm(rows, c, eps, type, gain_type);
  if (st != MIQ_OK) return st;
  if (!real_type(dgain_type)) return bad("dgain_type must be MIQ_F32 or MIQ_BF16");
  if (accumulate != 0 && accumulate != 1) return bad("accumulate must be 0 or 1");
  if (!stride_ok(ld_dy, c) || !stride_ok(ld_x, c) || !stride_ok(ld_dx, c) || (dsum != nullptr && !stride_ok(ld_dsum, c))) {
    return bad(kShortRows);
  }
  if (c == 0 || (rows == 0 && accumulate != 0)) return MIQ_OK;
  if (dgain == nullptr) return null("dgain pointer is NULL");
  const size_t need = rows == 0 ? 0 : miq::rms_grad_workspace_bytes(rows, c);
  if (rows > 0) {
    if (dy == nullptr || x == nullptr || gain == nullptr) return null("dy, x or gain pointer is NULL");
    if (dx == nullptr) return null("output pointer is NULL");
    if (workspace == nullptr) return null("workspace pointer is NULL");
  }
  if (workspace_bytes < need) return bad("workspace is smaller than miq_rms_bprop_workspace_size reports");
  const uintptr_t size = size_of(type);
  if (!aligned(dy, size) || !aligned(x, size) || !aligned(dsum, size) || !aligned(dx, size) ||
      !aligned(gain, size_of(gain_type)) || !aligned(dgain, size_of(dgain_type)) || !aligned(workspace, 16)) {
    return bad("a pointer is not aligned to its element, or the workspace to 16 bytes");
  }
  miq::RmsGradArgs a{};
  a.dy = dy;
  a.x = x;
  a.gain = gain;
  a.dsum = dsum;
  a.dx = dx;
  a.dgain = dgain;
  a.ws = static_cast<float*>(workspace);
  a.rows = rows;
  a.ld_dy = ld_dy;
  a.ld_x = ld_x;
  a.ld_dsum = ld_dsum;
  a.ld_dx = ld_dx;
  a.c = c;
  a.eps = eps;
  a.accumulate = accumulate != 0;
  a.bf16 = type == MIQ_BF16;
  a.gain_bf16 = gain_type == MIQ_BF16;
  a.dgain_bf16 = dgain_type == MIQ_BF16;
  return done(miq::launch_rms_grad(a, static_cast<hipStream_t>(stream)));
}

int miq_act_row8(const void* x, int8_t* codes, float* scales, int64_t rows, int32_t c, int64_t ld_x, int32_t act,
                 int32_t gated, int32_t type, void* stream) {
  const int st = check_rows(rows, c);
  if (st != MIQ_OK) return st;
  if (act < MIQ_ACT_NONE || act > MIQ_ACT_GELU) return bad("act must be NONE, RELU, SILU or GELU");
  if (gated != 0 && gated != 1) return bad("gated must be 0 or 1");
  if (!real_type(type)) return bad("type must be MIQ_F32 or MIQ_BF16");
  if (!stride_ok(ld_x, static_cast<int64_t>(c) * (1 + gated))) return bad(kShortRows);
  if (rows == 0) return MIQ_OK;
  if (x == nullptr && c > 0) return null("input pointer is NULL");
  if ((codes == nullptr && c > 0) || scales == nullptr) return null("codes or scales pointer is NULL");
  if (!aligned(x, size_of(type)) || !aligned(scales, 4)) return bad(kUnaligned);
  miq::ActRow8Args a{};
  a.x = x;
  a.codes = codes;
  a.scales = scales;
  a.rows = rows;
  a.ld_x = ld_x;
  a.c = c;
  a.act = act;
  a.gated = gated != 0;
  a.bf16 = type == MIQ_BF16;
  return done(miq::launch_act_row8(a, static_cast<hipStream_t>(stream)));
}

int miq_row8_expand(const int8_t* codes, const float* scales, void* y, int64_t rows, int32_t c, int64_t ld_y,
                    int32_t type, void* stream) {
  const int st = check_rows(rows, c);
  if (st != MIQ_OK) return st;
  if (!real_type(type)) return bad("type must be MIQ_F32 or MIQ_BF16");
  if (!stride_ok(ld_y, c)) return bad(kShortRows);
  if (rows == 0 || c == 0) return MIQ_OK;
  if (codes == nullptr || scales == nullptr) return null("codes or scales pointer is NULL");
  if (y == nullptr) return null("output pointer is NULL");
  if (!aligned(y, size_of(type)) || !aligned(scales, 4)) return bad(kUnaligned);
  miq::Row8ExpandArgs a{};
  a.codes = codes;
  a.scales = scales;
  a.y = y;
  a.rows = rows;
  a.ld_y = ld_y;
  a.c = c;
  a.bf16 = type == MIQ_BF16;
  return done(miq::launch_row8_expand(a, static_cast<hipStream_t>(stream)));
}

int miq_plan_row8_linear(int64_t rows, int32_t c, int32_t k, int32_t experts, int32_t plan[4]) {
  if (plan == nullptr) return null("plan pointer is NULL");
  const int st = check_product(rows, c, k, experts);
  if (st != MIQ_OK) return st;
  plan[0] = plan[1] = plan[2] = plan[3] = 0;
  if (rows > 0 && k > 0) miq::plan_row8_linear(static_cast<int32_t>(rows), c, k, experts, plan);
  return MIQ_OK;
}

int miq_row8_workspace_size(int64_t x_rows, int64_t rows, int32_t c, int32_t k, int32_t experts, size_t* bytes) {
  if (bytes == nullptr) return null("bytes pointer is NULL");
  const int st = check_product(rows, c, k, experts);
  if (st != MIQ_OK) return st;
  if (x_rows < 0 || x_rows > kMaxPositions) return bad("x_rows must lie in 0 .. 2^31 - 65");
  *bytes = rows == 0 || k == 0 ? 0
                               : miq::row8_workspace_bytes(static_cast<int32_t>(x_rows), static_cast<int32_t>(rows), c, k,
                                                           experts);
  return MIQ_OK;
}

int miq_row8_linear(const int8_t* codes, const float* scales, const int8_t* w_codes, const float* w_scales,
                    const float* bias, const void* add, void* y, int64_t rows, int32_t c, int32_t k, int64_t ld_add,
                    int64_t ld_y, int32_t type, void* workspace, size_t workspace_bytes, void* stream) {
  size_t need = 0;
  const int st = miq_row8_workspace_size(rows, rows, c, k, 1, &need);
  if (st != MIQ_OK) return st;
  if (!real_type(type)) return bad("type must be MIQ_F32 or MIQ_BF16");
  if (!stride_ok(ld_y, k) || (add != nullptr && !stride_ok(ld_add, k))) return bad(kShortRows);
  if (rows == 0 || k == 0) return MIQ_OK;
  if (scales == nullptr || w_scales == nullptr || (c > 0 && (codes == nullptr || w_codes == nullptr))) {
    return null("codes or scales pointer is NULL");
  }
  if (y == nullptr) return null("output pointer is NULL");
  if (need > 0 && workspace == nullptr) return null("workspace pointer is NULL");
  if (workspace_bytes < need) return bad("workspace is smaller than miq_row8_workspace_size reports");
  if (!aligned(scales, 4) || !aligned(w_scales, 4) || !aligned(bias, 4) || !aligned(add, size_of(type)) ||
      !aligned(y, size_of(type)) || !aligned(workspace, 16)) {
    return bad("a pointer is not aligned to its element, or the workspace to 16 bytes");
  }
  miq::Row8LinearArgs a{};
  a.x = codes;
  a.x_scales = scales;
  a.w = w_codes;
  a.w_scales = w_scales;
  a.bias = bias;
  a.add = add;
  a.y = y;
  a.ws = workspace;
  a.ld_add = ld_add;
  a.ld_y = ld_y;
  a.x_rows = a.rows = static_cast<int32_t>(rows);
  a.c = c;
  a.k = k;
  a.experts = 1;
  a.bf16 = type == MIQ_BF16;
  return done(miq::launch_row8_linear(a, static_cast<hipStream_t>(stream)));
}

int miq_row8_experts(const int8_t* codes, const float* scales, const int8_t* w_codes, const float* w_scales,
                     const float* bias, const int32_t* offsets, const int32_t* index, void* y, int64_t x_rows,
                     int64_t rows, int32_t c, int32_t k, int32_t experts, int64_t ld_y, int32_t type,
                     void* workspace, size_t workspace_bytes, void* stream) {
  size_t need = 0;
  const int st = miq_row8_workspace_size(x_rows, rows, c, k, experts, &need);
  if (st != MIQ_OK) return st;
  if (index == nullptr && x_rows < rows) return bad("without an index x has as many rows as y");
  if (!real_type(type)) return bad("type must be MIQ_F32 or MIQ_BF16");
  if (!stride_ok(ld_y, k)) return bad(kShortRows);
  if (rows == 0 || k == 0) return MIQ_OK;
  if (offsets == nullptr) return null("offsets pointer is NULL");
  if ((x_rows > 0 && scales == nullptr) || w_scales == nullptr ||
      (c > 0 && ((x_rows > 0 && codes == nullptr) || w_codes == nullptr))) {
    return null("codes or scales pointer is NULL");
  }
  if (y == nullptr) return null("output pointer is NULL");
  if (need > 0 && workspace == nullptr) return null("workspace pointer is NULL");
  if (workspace_bytes < need) return bad("workspace is smaller than miq_row8_workspace_size reports");
  if (!aligned(scales, 4) || !aligned(w_scales, 4) || !aligned(bias, 4) || !aligned(offsets, 4) || !aligned(index, 4) ||
      !aligned(y, size_of(type)) || !aligned(workspace, 16)) {
    return bad("a pointer is not aligned to its element, or the workspace to 16 bytes");
  }
  miq::Row8LinearArgs a{};
  a.x = codes;
  a.x_scales = scales;
  a.w = w_codes;
  a.w_scales = w_scales;
  a.bias = bias;
  a.offsets = offsets;
  a.index = index;
  a.y = y;
  a.ws = workspace;
  a.ld_y = ld_y;
  a.x_rows = static_cast<int32_t>(x_rows);
  a.rows = static_cast<int32_t>(rows);
  a.c = c;
  a.k = k;
  a.experts = experts;
  a.bf16 = type == MIQ_BF16;
  return done(miq::launch_row8_linear(a, static_cast<hipStream_t>(stream)));
}

int miq_experts_plan(const void* ids, int32_t* offsets, int32_t* rows, int32_t* places, int64_t tokens, int32_t slots,
                     int32_t experts, int32_t id_type, void* stream) {
  const int st = check_plan(tokens, slots, experts);
  if (st != MIQ_OK) return st;
  if (id_type != MIQ_I32 && id_type != MIQ_I64) return bad("id_type must be MIQ_I32 or MIQ_I64");
  if (offsets == nullptr) return null("offsets pointer is NULL");
  if (tokens > 0 && ids == nullptr) return null("ids pointer is NULL");
  if (tokens > 0 && (rows == nullptr || places == nullptr)) return null("output pointer is NULL");
  if (!aligned(ids, size_of(id_type)) || !aligned(offsets, 4) || !aligned(rows, 4) || !aligned(places, 4)) {
    return bad(kUnaligned);
  }
  miq::ExpertsPlanArgs a{};
  a.ids = ids;
  a.offsets = offsets;
  a.rows = rows;
  a.places = places;
  a.n = static_cast<int32_t>(tokens * slots);
  a.slots = slots;
  a.experts = experts;
  a.ids64 = id_type == MIQ_I64;
  return done(miq::launch_experts_plan(a, static_cast<hipStream_t>(stream)));
}

int miq_experts_join(const void* y, const int32_t* places, const float* share, const void* add, void* out, int64_t rows,
                     int64_t tokens, int32_t slots, int32_t c, int64_t ld_y, int64_t ld_add, int64_t ld_out, int32_t type,
                     void* stream) {
  if (rows < 0 || rows > kMaxPositions) return bad("rows must lie in 0 .. 2^31 - 65");
  int st = check_plan(tokens, slots, 1);
  if (st == MIQ_OK) st = check_rows(tokens, c);
  if (st != MIQ_OK) return st;
  if (!real_type(type)) return bad("type must be MIQ_F32 or MIQ_BF16");
  if (!stride_ok(ld_y, c) || !stride_ok(ld_out, c) || (add != nullptr && !stride_ok(ld_add, c))) return bad(kShortRows);
  if (tokens == 0 || c == 0) return MIQ_OK;
  if (rows > 0 && y == nullptr) return null("input pointer is NULL");
  if (places == nullptr) return null("places pointer is NULL");
  if (out == nullptr) return null("output pointer is NULL");
  const uintptr_t size = size_of(type);
  if (!aligned(y, size) || !aligned(add, size) || !aligned(out, size) || !aligned(places, 4) || !aligned(share, 4)) {
    return bad(kUnaligned);
  }
  miq::ExpertsJoinArgs a{};
  a.y = y;
  a.places = places;
  a.share = share;
  a.add = add;
  a.out = out;
  a.tokens = tokens;
  a.ld_y = ld_y;
  a.ld_add = ld_add;
  a.ld_out = ld_out;
  a.rows = static_cast<int32_t>(rows);
  a.slots = slots;
  a.c = c;
  a.bf16 = type == MIQ_BF16;
  return done(miq::launch_experts_join(a, static_cast<hipStream_t>(stream)));
}

}  // extern "C"
