// extern "C" entry points of the token-network operators: host-side validation and dispatch.
// Nothing is enqueued before the arguments are validated, and nothing is allocated.
#include <cstdint>

#include "miq_qconv.h"
#include "qconv_internal.h"
#include "train_internal.h"

namespace {

constexpr int64_t kMaxPositions = 0x7fffffffLL - 64;  // positions are sorted as int32
constexpr int64_t kMaxVocab = 1LL << 28;              // one workgroup per 32 table rows in a launch
constexpr int32_t kMaxChannels = 1 << 29;             // two halves of a gated row stay in int32
constexpr int64_t kMaxRows = 1LL << 40;
constexpr int64_t kMaxValues = 1LL << 46;             // byte offsets stay far inside int64
constexpr int32_t kMaxSide = 1 << 22;                 // of a weight gradient
constexpr int64_t kMaxTiles = 1LL << 23;              // of 128 x 128 in a launch

int bad(const char* msg) { return miq::record_error(MIQ_ERR_INVALID_ARGUMENT, msg); }
int null(const char* msg) { return miq::record_error(MIQ_ERR_NULL_POINTER, msg); }

int done(hipError_t e) { return e == hipSuccess ? MIQ_OK : miq::record_error(MIQ_ERR_HIP, hipGetErrorString(e)); }

bool real_type(int32_t t) { return t == MIQ_F32 || t == MIQ_BF16; }
bool id_type_ok(int32_t t) { return t == MIQ_I32 || t == MIQ_I64; }

bool aligned(const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }
uintptr_t size_of(int32_t type) { return type == MIQ_BF16 ? 2 : type == MIQ_I64 ? 8 : 4; }

int check_embed_sizes(int64_t vocab, int32_t c, int64_t tokens) {
  if (vocab < 0 || c < 0 || tokens < 0) return bad("embedding extents must be >= 0");
  if (vocab > kMaxVocab || c > kMaxChannels) return bad("embedding table exceeds 2^28 rows or 2^29 channels");
  if (tokens > kMaxPositions) return bad("embedding takes at most 2^31 - 65 tokens");
  return MIQ_OK;
}

int check_act8(int64_t rows, int32_t c, int32_t act, int32_t gated, int32_t type) {
  if (rows < 0 || c < 0) return bad("act8 extents must be >= 0");
  if (c > kMaxChannels || rows > kMaxRows || (c > 0 && rows > kMaxValues / c)) {
    return bad("act8 tensor exceeds 2^29 channels, 2^40 rows or 2^46 values");
  }
  if (act < MIQ_ACT_NONE || act > MIQ_ACT_GELU) return bad("act must be NONE, RELU, SILU or GELU");
  if (gated != 0 && gated != 1) return bad("gated must be 0 or 1");
  if (!real_type(type)) return bad("type must be MIQ_F32 or MIQ_BF16");
  return MIQ_OK;
}

int check_side(int64_t rows, int32_t c, int32_t k, int32_t dy_type) {
  if (rows < 0 || c < 0 || k < 0) return bad("act8 weight gradient extents must be >= 0");
  if (rows > kMaxPositions) return bad("act8 weight gradient takes at most 2^31 - 65 rows");
  if (c > kMaxSide || k > kMaxSide) return bad("act8 weight gradient exceeds 2^22 channels");
  if (((c + 127LL) / 128) * ((k + 127LL) / 128) > kMaxTiles) {
    return miq::record_error(MIQ_ERR_UNSUPPORTED, "act8 weight gradient has more than 2^23 128x128 tiles");
  }
  if (!real_type(dy_type)) return bad("dy_type must be MIQ_F32 or MIQ_BF16");
  return MIQ_OK;
}

bool stride_ok(int64_t ld, int64_t width) { return ld >= width && ld <= kMaxValues; }

}  // namespace

extern "C" {

int miq_embed_fprop(const void* table, const void* ids, void* y, int64_t vocab, int32_t c, int64_t tokens,
                    int64_t ld_table, int64_t ld_y, float scale, int32_t table_type, int32_t id_type, int32_t y_type,
                    void* stream) {
  const int st = check_embed_sizes(vocab, c, tokens);
  if (st != MIQ_OK) return st;
  if (!real_type(table_type) || !real_type(y_type)) return bad("table_type and y_type must be MIQ_F32 or MIQ_BF16");
  if (!id_type_ok(id_type)) return bad("id_type must be MIQ_I32 or MIQ_I64");
  if (!stride_ok(ld_table, c) || !stride_ok(ld_y, c)) return bad("row distance is smaller than the row");
  if (tokens == 0 || c == 0) return MIQ_OK;
  if (ids == nullptr) return null("ids pointer is NULL");
  if (y == nullptr) return null("output pointer is NULL");
  if (vocab > 0 && table == nullptr) return null("table pointer is NULL");
  if (!aligned(table, size_of(table_type)) || !aligned(y, size_of(y_type)) || !aligned(ids, size_of(id_type))) {
    return bad("a pointer is not aligned to its element");
  }
  miq::EmbedArgs a{};
  a.table = table;
  a.ids = ids;
  a.y = y;
  a.ld_table = ld_table;
  a.ld_y = ld_y;
  a.tokens = tokens;
  a.vocab = static_cast<int32_t>(vocab);
  a.c = c;
  a.scale = scale;
  a.table_bf16 = table_type == MIQ_BF16;
  a.ids64 = id_type == MIQ_I64;
  a.y_bf16 = y_type == MIQ_BF16;
  return done(miq::launch_embed_fprop(a, static_cast<hipStream_t>(stream)));
}

int miq_embed_grad_workspace_size(int64_t vocab, int32_t c, int64_t tokens, size_t* bytes) {
  if (bytes == nullptr) return null("bytes pointer is NULL");
  const int st = check_embed_sizes(vocab, c, tokens);
  if (st != MIQ_OK) return st;
  *bytes = tokens == 0 || c == 0 || vocab == 0
               ? 0
               : miq::embed_grad_workspace_bytes(static_cast<int32_t>(vocab), c, static_cast<int32_t>(tokens));
  return MIQ_OK;
}

int miq_plan_embed_grad(int64_t vocab, int32_t c, int64_t tokens, int32_t plan[2]) {
  if (plan == nullptr) return null("plan pointer is NULL");
  const int st = check_embed_sizes(vocab, c, tokens);
  if (st != MIQ_OK) return st;
  plan[0] = plan[1] = 0;
  if (vocab > 0 && c > 0) {
    miq::plan_embed_grad(static_cast<int32_t>(vocab), c, static_cast<int32_t>(tokens), &plan[0], &plan[1]);
  }
  return MIQ_OK;
}

int miq_embed_grad(const void* dy, const void* ids, void* dtable, int64_t vocab, int32_t c, int64_t tokens,
                   int64_t ld_dy, int64_t ld_dtable, float scale, int32_t accumulate, int32_t dy_type, int32_t id_type,
                   int32_t dtable_type, void* workspace, size_t workspace_bytes, void* stream) {
  size_t need = 0;
  const int st = miq_embed_grad_workspace_size(vocab, c, tokens, &need);
  if (st != MIQ_OK) return st;
  if (!real_type(dy_type) || !real_type(dtable_type)) return bad("dy_type and dtable_type must be MIQ_F32 or MIQ_BF16");
  if (!id_type_ok(id_type)) return bad("id_type must be MIQ_I32 or MIQ_I64");
  if (accumulate != 0 && accumulate != 1) return bad("accumulate must be 0 or 1");
  if (!stride_ok(ld_dy, c) || !stride_ok(ld_dtable, c)) return bad("row distance is smaller than the row");
  if (vocab == 0 || c == 0 || (tokens == 0 && accumulate != 0)) return MIQ_OK;
  if (dtable == nullptr) return null("output pointer is NULL");
  if (tokens > 0 && (dy == nullptr || ids == nullptr)) return null("dy or ids pointer is NULL");
  if (need > 0 && workspace == nullptr) return null("workspace pointer is NULL");
  if (workspace_bytes < need) return bad("workspace is smaller than miq_embed_grad_workspace_size reports");
  if (!aligned(dy, size_of(dy_type)) || !aligned(dtable, size_of(dtable_type)) || !aligned(ids, size_of(id_type)) ||
      !aligned(workspace, 16)) {
    return bad("a pointer is not aligned to its element, or the workspace to 16 bytes");
  }
  miq::EmbedGradArgs a{};
  a.dy = dy;
  a.ids = ids;
  a.dtable = dtable;
  a.ws = workspace;
  a.ld_dy = ld_dy;
  a.ld_dtable = ld_dtable;
  a.tokens = static_cast<int32_t>(tokens);
  a.vocab = static_cast<int32_t>(vocab);
  a.c = c;
  a.scale = scale;
  a.accumulate = accumulate != 0;
  a.dy_bf16 = dy_type == MIQ_BF16;
  a.ids64 = id_type == MIQ_I64;
  a.dtable_bf16 = dtable_type == MIQ_BF16;
  return done(miq::launch_embed_grad(a, static_cast<hipStream_t>(stream)));
}

int miq_act8_fprop(const void* x, void* y, int8_t* codes, uint8_t* scales, int64_t rows, int32_t c, int64_t ld_x,
                   int64_t ld_y, int32_t act, int32_t gated, int32_t type, void* stream) {
  const int st = check_act8(rows, c, act, gated, type);
  if (st != MIQ_OK) return st;
  if (!stride_ok(ld_x, static_cast<int64_t>(c) * (1 + gated)) || (y != nullptr && !stride_ok(ld_y, c))) {
    return bad("row distance is smaller than the row");
  }
  if (rows == 0 || c == 0) return MIQ_OK;
  if (x == nullptr) return null("input pointer is NULL");
  if (codes == nullptr || scales == nullptr) return null("codes or scales pointer is NULL");
  if (!aligned(x, size_of(type)) || !aligned(y, size_of(type))) return bad("a pointer is not aligned to its element");
  miq::Act8Args a{};
  a.x = x;
  a.y = y;
  a.codes = codes;
  a.scales = scales;
  a.rows = rows;
  a.c = c;
  a.ld_x = ld_x;
  a.ld_y = ld_y;
  a.act = act;
  a.gated = gated != 0;
  a.bf16 = type == MIQ_BF16;
  return done(miq::launch_act8_fprop(a, static_cast<hipStream_t>(stream)));
}

int miq_act8_bprop(const void* dy, const int8_t* codes, const uint8_t* scales, void* dx, int64_t rows, int32_t c,
                   int64_t ld_dy, int64_t ld_dx, int32_t act, int32_t gated, int32_t type, void* stream) {
  const int st = check_act8(rows, c, act, gated, type);
  if (st != MIQ_OK) return st;
  if (!stride_ok(ld_dy, c) || !stride_ok(ld_dx, static_cast<int64_t>(c) * (1 + gated))) {
    return bad("row distance is smaller than the row");
  }
  if (rows == 0 || c == 0) return MIQ_OK;
  if (dy == nullptr) return null("dy pointer is NULL");
  if (codes == nullptr || scales == nullptr) return null("codes or scales pointer is NULL");
  if (dx == nullptr) return null("output pointer is NULL");
  if (!aligned(dy, size_of(type)) || !aligned(dx, size_of(type))) return bad("a pointer is not aligned to its element");
  miq::Act8Args a{};
  a.dy = dy;
  a.y = dx;
  a.codes = const_cast<int8_t*>(codes);  // read only by this pass
  a.scales = const_cast<uint8_t*>(scales);
  a.rows = rows;
  a.c = c;
  a.ld_dy = ld_dy;
  a.ld_y = ld_dx;
  a.act = act;
  a.gated = gated != 0;
  a.bf16 = type == MIQ_BF16;
  return done(miq::launch_act8_bprop(a, static_cast<hipStream_t>(stream)));
}

int miq_act8_expand(const int8_t* codes, const uint8_t* scales, void* y, int64_t rows, int32_t c, int64_t ld_y,
                    int32_t act, int32_t gated, int32_t type, void* stream) {
  const int st = check_act8(rows, c, act, gated, type);
  if (st != MIQ_OK) return st;
  if (!stride_ok(ld_y, c)) return bad("row distance is smaller than the row");
  if (rows == 0 || c == 0) return MIQ_OK;
  if (codes == nullptr || scales == nullptr) return null("codes or scales pointer is NULL");
  if (y == nullptr) return null("output pointer is NULL");
  if (!aligned(y, size_of(type))) return bad("a pointer is not aligned to its element");
  miq::Act8Args a{};
  a.y = y;
  a.codes = const_cast<int8_t*>(codes);  // read only by this pass
  a.scales = const_cast<uint8_t*>(scales);
  a.rows = rows;
  a.c = c;
  a.ld_y = ld_y;
  a.act = act;
  a.gated = gated != 0;
  a.bf16 = type == MIQ_BF16;
  return done(miq::launch_act8_expand(a, static_cast<hipStream_t>(stream)));
}

int miq_act8_grad_workspace_size(int64_t rows, int32_t c, int32_t k, int32_t dy_type, size_t* bytes) {
  if (bytes == nullptr) return null("bytes pointer is NULL");
  const int st = check_side(rows, c, k, dy_type);
  if (st != MIQ_OK) return st;
  *bytes = c == 0 || k == 0 ? 0 : miq::act8_grad_workspace_bytes(static_cast<int32_t>(rows), c, k, dy_type == MIQ_BF16);
  return MIQ_OK;
}

int miq_plan_act8_grad(int64_t rows, int32_t c, int32_t k, int32_t dy_type, int32_t plan[2]) {
  if (plan == nullptr) return null("plan pointer is NULL");
  const int st = check_side(rows, c, k, dy_type);
  if (st != MIQ_OK) return st;
  plan[0] = plan[1] = 0;
  if (c > 0 && k > 0) {
    miq::plan_act8_grad(static_cast<int32_t>(rows), c, k, dy_type == MIQ_BF16, &plan[0], &plan[1]);
  }
  return MIQ_OK;
}

int miq_act8_grad(const void* dy, const int8_t* codes, const uint8_t* scales, void* dw, int64_t rows, int32_t c,
                  int32_t k, int64_t ld_dy, int64_t ld_dw, int32_t accumulate, int32_t dy_type, int32_t dw_type,
                  void* workspace, size_t workspace_bytes, void* stream) {
  size_t need = 0;
  const int st = miq_act8_grad_workspace_size(rows, c, k, dy_type, &need);
  if (st != MIQ_OK) return st;
  if (dw_type != MIQ_F32 && !(dw_type == MIQ_BF16 && dy_type == MIQ_BF16)) {
    return bad("dw_type must be MIQ_F32, or MIQ_BF16 with a bf16 dy");
  }
  if (accumulate != 0 && accumulate != 1) return bad("accumulate must be 0 or 1");
  if (!stride_ok(ld_dy, k) || !stride_ok(ld_dw, c)) return bad("row distance is smaller than the row");
  if (c == 0 || k == 0 || (rows == 0 && accumulate != 0)) return MIQ_OK;
  if (dw == nullptr) return null("output pointer is NULL");
  if (rows > 0 && dy == nullptr) return null("dy pointer is NULL");
  if (rows > 0 && (codes == nullptr || scales == nullptr)) return null("codes or scales pointer is NULL");
  if (need > 0 && workspace == nullptr) return null("workspace pointer is NULL");
  if (workspace_bytes < need) return bad("workspace is smaller than miq_act8_grad_workspace_size reports");
  if (!aligned(dy, size_of(dy_type)) || !aligned(dw, size_of(dw_type)) || !aligned(workspace, 16)) {
    return bad("a pointer is not aligned to its element, or the workspace to 16 bytes");
  }
  miq::Act8GradArgs a{};
  a.dy = dy;
  a.codes = codes;
  a.scales = scales;
  a.dw = dw;
  a.ws = workspace;
  a.ld_dy = ld_dy;
  a.ld_dw = ld_dw;
  a.rows = static_cast<int32_t>(rows);
  a.c = c;
  a.k = k;
  a.accumulate = accumulate != 0;
  a.dy_bf16 = dy_type == MIQ_BF16;
  a.dw_bf16 = dw_type == MIQ_BF16;
  return done(miq::launch_act8_grad(a, static_cast<hipStream_t>(stream)));
}

}  // extern "C"
