// mx_moe_api.cpp - C ABI of the routed-experts operators: router, dispatch,
// combine, block-scaled FP8 (declared in include/mxfp4hip.h).
#include <hip/hip_runtime.h>

#include <cstdarg>
#include <cstdio>

#include "../../include/mxfp4hip.h"
#include "mx_block.h"

// Context internals (mx_api.cpp).
hipStream_t mx_ctx_stream(mx_ctx* c);
int mx_ctx_error(mx_ctx* c, int code, const char* message);
int mx_ctx_workspace(mx_ctx* c, size_t bytes, void** p);

namespace mx {

ExpertsLayout experts_layout(int T, int H, int I, int E, int topk) {
  const size_t n = (size_t)T * topk, used = n < (size_t)E ? n : E, few = (size_t)block_stream_most(E);
  auto blocks = [](int k) { return (size_t)((k + kQBlock - 1) / kQBlock); };
  ExpertsLayout l{};
  auto take = [&](size_t bytes) { const size_t o = l.total; l.total = (o + bytes + 255) / 256 * 256; return o; };
  l.xq = take((size_t)T * H);
  l.xs = take(T * blocks(H) * 4);
  l.rows = take(n * 4);
  l.src = take(n * 4);
  l.counts = take((size_t)E * 4);
  l.tiles = take((used + n / 16) * sizeof(RowTile));  // tiles have 16 rows at least
  l.n_tiles = take(4);
  l.hist = take(dispatch_ws_bytes((int)n, E));
  const size_t mids = n < few ? n : few;
  l.mid = take((mids > (size_t)topk ? mids : topk) * I * 4);  // (one token's slots are not split)
  l.mq = take(n * I);
  l.ms = take(n * blocks(I) * 4);
  l.y = take(n * H * 4);
  return l;
}

}  // namespace mx

namespace {

int fail(mx_ctx* c, int code, const char* fmt, ...) {
  char buf[256];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof buf, fmt, ap);
  va_end(ap);
  return mx_ctx_error(c, code, buf);
}

#define MX_RUN(ctx, expr)                                                                           \
  do {                                                                                              \
    const hipError_t e_ = (expr);                                                                   \
    if (e_ != hipSuccess) return fail(ctx, MX_EGPU, "%s failed: %s", #expr, hipGetErrorString(e_)); \
  } while (0)

bool is_aligned(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }
bool is_float(int dtype) { return dtype == MX_DTYPE_F32 || dtype == MX_DTYPE_F16 || dtype == MX_DTYPE_BF16; }
size_t size_of(int dtype) { return dtype == MX_DTYPE_F32 ? 4 : 2; }
int blocks(int n) { return (n + mx::kQBlock - 1) / mx::kQBlock; }

// slots of a batch
int check_slots(mx_ctx* c, int tokens, int topk) {
  if (tokens < 0 || topk < 1 || topk > 64) return fail(c, MX_EINVAL, "MoE needs tokens >= 0 and topk in 1..64.");
  if ((long long)tokens * topk >= 1 << 26) return fail(c, MX_EINVAL, "MoE tokens x topk must be below 2^26.");
  return MX_OK;
}

int check_experts(mx_ctx* c, int experts) {
  if (experts < 1 || experts > mx::kMaxRouteExperts)
    return fail(c, MX_EINVAL, "MoE routing needs 1 to %d experts.", mx::kMaxRouteExperts);
  return MX_OK;
}

// mx_moe_block_forward of one token: its slots need no order, and its few rows are
// quantized where they are used.
int block_experts_of_one(mx_ctx* c, int H, int I, int E, int topk, const void* x, int dtype, const int32_t* ids,
                         const float* weights, const mx_mlp_weights* w, const void* add, void* out) {
  const mx::ExpertsLayout l = mx::experts_layout(1, H, I, E, topk);
  void* p = nullptr;
  if (int rc = mx_ctx_workspace(c, l.total, &p)) return rc;
  uint8_t* ws = static_cast<uint8_t*>(p);
  hipStream_t st = mx_ctx_stream(c);
  mx::BlockGemmArgs g{};
  g.m = topk;
  g.ids = ids;
  g.experts = E;
  g.splits = 1;
  g.raw = x;
  g.w0 = static_cast<const uint8_t*>(w->gate.data);
  g.w1 = static_cast<const uint8_t*>(w->up.data);
  g.s0 = static_cast<const float*>(w->gate.scales);
  g.s1 = static_cast<const float*>(w->up.scales);
  g.w_stride = (size_t)I * H;
  g.s_stride = (size_t)blocks(I) * blocks(H);
  g.c = ws + l.mid;
  g.n = I;
  g.k = H;
  MX_RUN(c, mx::launch_block_direct(dtype, g, st));
  g.raw = ws + l.mid;
  g.row_per_slot = 1;
  g.w0 = static_cast<const uint8_t*>(w->down.data);
  g.w1 = nullptr;
  g.s0 = static_cast<const float*>(w->down.scales);
  g.c = ws + l.y;
  g.n = H;
  g.k = I;
  MX_RUN(c, mx::launch_block_direct(MX_DTYPE_F32, g, st));
  const mx::CombineArgs b{ws + l.y, nullptr, weights, add, out, 1, topk, H, ids, E};
  MX_RUN(c, mx::launch_combine(MX_DTYPE_F32, dtype, b, st));
  return MX_OK;
}

// One pass of mx_moe_block_forward over T >= 1 tokens.
int block_experts(mx_ctx* c, int T, int H, int I, int E, int topk, const void* x, int dtype, const int32_t* ids,
                  const float* weights, const mx_mlp_weights* w, const void* add, void* out) {
  const int n = T * topk;
  // one tile height for both products, so that they share the list of tiles
  const int used = n < E ? n : E, tile_rows = mx::block_tile_rows(n, used, I, H, dtype, true), max_tiles = used + n / tile_rows;
  // Few rows write the middle in f32 first, more of them its codes alone.  The
  // experts' rows stay in f32 up to their weighted sum, however many: in f16 a row
  // may pass the largest number where the sum does not, and rows that nearly cancel
  // would leave their roundings.  (Rows of 16 bits take half the bytes: 4096 tokens,
  // top 8 of 64 x (7168, 2048), 1870 us instead of 2010; 256 tokens 567 and 575.)
  const bool few = mx::block_streams(tile_rows);
  const mx::ExpertsLayout l = mx::experts_layout(T, H, I, E, topk);
  void* p = nullptr;
  if (int rc = mx_ctx_workspace(c, l.total, &p)) return rc;
  uint8_t* ws = static_cast<uint8_t*>(p);
  hipStream_t st = mx_ctx_stream(c);
  mx::DispatchArgs d{ids, n, E, reinterpret_cast<int32_t*>(ws + l.counts), reinterpret_cast<int32_t*>(ws + l.rows),
                     reinterpret_cast<int32_t*>(ws + l.src), reinterpret_cast<mx::RowTile*>(ws + l.tiles),
                     reinterpret_cast<int32_t*>(ws + l.n_tiles), tile_rows, reinterpret_cast<int32_t*>(ws + l.hist)};
  MX_RUN(c, mx::launch_prepare(d, dtype, x, T, H, ws + l.xq, reinterpret_cast<float*>(ws + l.xs), st));
  mx::BlockGemmArgs g{};
  g.a = ws + l.xq;
  g.a_s = reinterpret_cast<float*>(ws + l.xs);
  g.a_rows = T;
  g.w0 = static_cast<const uint8_t*>(w->gate.data);
  g.w1 = static_cast<const uint8_t*>(w->up.data);
  g.s0 = static_cast<const float*>(w->gate.scales);
  g.s1 = static_cast<const float*>(w->up.scales);
  g.c = few ? ws + l.mid : ws + l.mq;
  g.c_s = reinterpret_cast<float*>(ws + l.ms);
  g.m = n;
  g.n = I;
  g.k = H;
  g.tiles = d.tiles;
  g.n_tiles = d.n_tiles;
  g.max_tiles = max_tiles;
  g.splits = 1;
  g.tile_rows = tile_rows;
  g.w_stride = (size_t)I * H;
  g.s_stride = (size_t)blocks(I) * blocks(H);
  g.src = d.src;
  g.src_div = topk;
  MX_RUN(c, mx::launch_block_gemm(MX_DTYPE_F32, g, st));
  if (few)
    MX_RUN(c, mx::launch_block_quantize(MX_DTYPE_F32, ws + l.mid, n, I, ws + l.mq, reinterpret_cast<float*>(ws + l.ms), st));
  g.a = ws + l.mq;
  g.a_s = reinterpret_cast<float*>(ws + l.ms);
  g.a_rows = n;
  g.w0 = static_cast<const uint8_t*>(w->down.data);
  g.w1 = nullptr;
  g.s0 = static_cast<const float*>(w->down.scales);
  g.c = ws + l.y;
  g.n = H;
  g.k = I;
  g.src = nullptr;
  g.fp8_cores = 1;
  MX_RUN(c, mx::launch_block_gemm(MX_DTYPE_F32, g, st));
  const mx::CombineArgs b{ws + l.y, d.rows, weights, add, out, T, topk, H, nullptr, 0};
  MX_RUN(c, mx::launch_combine(MX_DTYPE_F32, dtype, b, st));
  return MX_OK;
}

}  // namespace

extern "C" {

int mx_moe_route(mx_ctx* c, const mx_route_config* cfg, const void* logits, int logits_dtype, size_t logits_stride,
                 const float* bias, int32_t* ids, float* weights) {
  if (!c) return MX_EINVAL;
  if (!cfg) return fail(c, MX_EINVAL, "route config is null.");
  if (cfg->tokens > 0x7fffffffu || cfg->experts > 0x7fffffffu || cfg->topk > 64)
    return fail(c, MX_EINVAL, "route sizes are out of range.");
  const int T = (int)cfg->tokens, E = (int)cfg->experts, K = (int)cfg->topk;
  if (int rc = check_slots(c, T, K)) return rc;
  if (int rc = check_experts(c, E)) return rc;
  if (K > E) return fail(c, MX_EINVAL, "route topk %d is more than %d experts.", K, E);
  if (cfg->score != MX_ROUTE_SOFTMAX && cfg->score != MX_ROUTE_SIGMOID)
    return fail(c, MX_EINVAL, "Unknown route score %u.", cfg->score);
  if (!is_float(logits_dtype)) return fail(c, MX_EINVAL, "route logits must be f32, f16 or bf16.");
  const int G = cfg->groups > 1 ? (int)cfg->groups : 1;
  if (cfg->groups > (uint32_t)mx::kMaxRouteGroups || E % G)
    return fail(c, MX_EINVAL, "route groups must divide the experts and be at most %d.", mx::kMaxRouteGroups);
  if (G > 1) {
    if (cfg->topk_groups < 1 || cfg->topk_groups > (uint32_t)G)
      return fail(c, MX_EINVAL, "route topk_groups must be 1 to %d.", G);
    if (cfg->group_top != 1 && cfg->group_top != 2) return fail(c, MX_EINVAL, "route group_top must be 1 or 2.");
    if ((long)cfg->topk_groups * (E / G) < K)
      return fail(c, MX_EINVAL, "route topk is more than the experts of topk_groups groups.");
  }
  if (logits_stride && logits_stride < (size_t)E) return fail(c, MX_EINVAL, "route logits_stride is below the experts.");
  if (T == 0) return MX_OK;
  if (!logits || !ids || !weights) return fail(c, MX_EINVAL, "route buffers must not be null.");
  if (!is_aligned(logits, size_of(logits_dtype)) || !is_aligned(bias, 4) || !is_aligned(ids, 4) || !is_aligned(weights, 4))
    return fail(c, MX_EINVAL, "route buffers must be aligned to their elements.");
  const mx::RouteArgs a{logits, logits_stride ? logits_stride : (size_t)E, bias, ids, weights, T, E, K, G,
                        (int)cfg->topk_groups, (int)cfg->group_top, cfg->score == MX_ROUTE_SIGMOID,
                        cfg->renormalize != 0, cfg->scale};
  MX_RUN(c, mx::launch_route(logits_dtype, a, mx_ctx_stream(c)));
  return MX_OK;
}

int mx_moe_dispatch(mx_ctx* c, int tokens, int topk, int experts, const int32_t* ids, int32_t* counts, int32_t* rows,
                    const void* x, int dtype, int hidden, void* xs) {
  if (!c) return MX_EINVAL;
  if (int rc = check_slots(c, tokens, topk)) return rc;
  if (int rc = check_experts(c, experts)) return rc;
  if (!counts || (tokens && (!ids || !rows))) return fail(c, MX_EINVAL, "dispatch buffers must not be null.");
  if (!is_aligned(ids, 4) || !is_aligned(counts, 4) || !is_aligned(rows, 4))
    return fail(c, MX_EINVAL, "dispatch ids, counts and rows must be 4-byte aligned.");
  if (!x != !xs) return fail(c, MX_EINVAL, "dispatch takes both x and xs or neither.");
  if (x) {
    if (!is_float(dtype)) return fail(c, MX_EINVAL, "dispatch rows must be f32, f16 or bf16.");
    if (hidden < 1 || hidden >= mx::kMaxHidden)
      return fail(c, MX_EINVAL, "dispatch hidden must be positive and below %d.", mx::kMaxHidden);
    if (!is_aligned(x, size_of(dtype)) || !is_aligned(xs, size_of(dtype)))
      return fail(c, MX_EINVAL, "dispatch rows must be aligned to their elements.");
  }
  const int n = tokens * topk;
  void* ws = nullptr;
  if (int rc = mx_ctx_workspace(c, mx::dispatch_ws_bytes(n, experts), &ws)) return rc;
  mx::DispatchArgs a{};
  a.ids = ids;
  a.n = n;
  a.experts = experts;
  a.counts = counts;
  a.rows = rows;
  a.hist = static_cast<int32_t*>(ws);
  if (x && tokens) MX_RUN(c, mx::launch_dispatch_rows(a, topk, x, xs, (size_t)hidden * size_of(dtype), mx_ctx_stream(c)));
  else MX_RUN(c, mx::launch_dispatch(a, mx_ctx_stream(c)));
  return MX_OK;
}

int mx_moe_combine(mx_ctx* c, int tokens, int topk, int hidden, const void* y, int y_dtype, const int32_t* rows,
                   const float* weights, const void* add, void* out, int out_dtype) {
  if (!c) return MX_EINVAL;
  if (int rc = check_slots(c, tokens, topk)) return rc;
  if (hidden < 1 || hidden >= mx::kMaxHidden)
    return fail(c, MX_EINVAL, "combine hidden must be positive and below %d.", mx::kMaxHidden);
  if (!is_float(y_dtype) || !is_float(out_dtype)) return fail(c, MX_EINVAL, "combine rows must be f32, f16 or bf16.");
  if (tokens == 0) return MX_OK;
  if (!y || !rows || !weights || !out) return fail(c, MX_EINVAL, "combine buffers must not be null.");
  if (!is_aligned(y, size_of(y_dtype)) || !is_aligned(add, size_of(out_dtype)) || !is_aligned(out, size_of(out_dtype)) ||
      !is_aligned(rows, 4) || !is_aligned(weights, 4))
    return fail(c, MX_EINVAL, "combine buffers must be aligned to their elements.");
  const mx::CombineArgs a{y, rows, weights, add, out, tokens, topk, hidden, nullptr, 0};
  MX_RUN(c, mx::launch_combine(y_dtype, out_dtype, a, mx_ctx_stream(c)));
  return MX_OK;
}

int mx_block_quantize(mx_ctx* c, const void* src, int src_dtype, int rows, int k, uint8_t* q, float* scales) {
  if (!c) return MX_EINVAL;
  if (rows < 0 || k <= 0 || k % 16) return fail(c, MX_EINVAL, "block quantize needs rows >= 0 and k a positive multiple of 16.");
  if (k > mx::kMaxBlocks * mx::kQBlock) return fail(c, MX_EINVAL, "block quantize k is at most %d.", mx::kMaxBlocks * mx::kQBlock);
  if (rows >= mx::kMaxRows) return fail(c, MX_EINVAL, "block quantize rows must be below %d.", mx::kMaxRows);
  if (!is_float(src_dtype)) return fail(c, MX_EINVAL, "block quantize source must be f32, f16 or bf16.");
  if (rows == 0) return MX_OK;
  if (!src || !q || !scales || !is_aligned(src, 16) || !is_aligned(q, 16) || !is_aligned(scales, 4))
    return fail(c, MX_EINVAL, "block quantize buffers must be non-null, source and codes 16-byte and scales 4-byte aligned.");
  MX_RUN(c, mx::launch_block_quantize(src_dtype, src, rows, k, q, scales, mx_ctx_stream(c)));
  return MX_OK;
}

int mx_block_matmul(mx_ctx* c, const uint8_t* a, const float* a_scales, const uint8_t* b, const float* b_scales, void* out,
                    int c_dtype, int m, int n, int k) {
  if (!c) return MX_EINVAL;
  if (m < 0 || n <= 0 || k <= 0 || k % 16)
    return fail(c, MX_EINVAL, "block matmul needs m >= 0, n > 0 and k a positive multiple of 16.");
  if (k > mx::kMaxBlocks * mx::kQBlock) return fail(c, MX_EINVAL, "block matmul k is at most %d.", mx::kMaxBlocks * mx::kQBlock);
  if (m >= mx::kMaxRows || n >= mx::kMaxRows) return fail(c, MX_EINVAL, "block matmul m and n must be below %d.", mx::kMaxRows);
  if (!is_float(c_dtype)) return fail(c, MX_EINVAL, "block matmul C must be f32, f16 or bf16.");
  if (m == 0) return MX_OK;
  if (!a || !a_scales || !b || !b_scales || !out || !is_aligned(a, 16) || !is_aligned(b, 16) || !is_aligned(out, 16) ||
      !is_aligned(a_scales, 4) || !is_aligned(b_scales, 4))
    return fail(c, MX_EINVAL, "block matmul buffers must be non-null, codes and C 16-byte and scales 4-byte aligned.");
  mx::BlockGemmArgs g{};
  g.a = a;
  g.a_s = a_scales;
  g.a_rows = m;
  g.w0 = b;
  g.s0 = b_scales;
  g.c = out;
  g.m = m;
  g.n = n;
  g.k = k;
  g.tile_rows = mx::block_tile_rows(m, 1, n, k, c_dtype, false);
  g.splits = mx::block_splits(m, n, k, g.tile_rows);
  if (const size_t bytes = mx::block_split_bytes(m, n, k))
    if (int rc = mx_ctx_workspace(c, bytes, &g.part)) return rc;
  MX_RUN(c, mx::launch_block_gemm(c_dtype, g, mx_ctx_stream(c)));
  return MX_OK;
}

int mx_moe_block_forward(mx_ctx* c, const mx_mlp_config* cfg, int n_experts, int topk, const void* x, int dtype,
                         const int32_t* ids, const float* weights, const mx_mlp_weights* w, const void* add, void* out) {
  if (!c) return MX_EINVAL;
  if (!cfg) return fail(c, MX_EINVAL, "MLP config is null.");
  if (cfg->tokens > 0x7fffffffu || cfg->hidden > 0x7ffffff0u || cfg->intermediate > 0x7ffffff0u)
    return fail(c, MX_EINVAL, "MLP sizes are out of range.");
  const int T = (int)cfg->tokens, H = (int)cfg->hidden, I = (int)cfg->intermediate, E = n_experts;
  if (int rc = check_slots(c, T, topk)) return rc;
  if (int rc = check_experts(c, E)) return rc;
  if (H < 16 || I < 16 || H % 16 || I % 16)
    return fail(c, MX_EINVAL, "Block FP8 needs hidden and intermediate to be positive multiples of 16.");
  if (H > mx::kMaxBlocks * mx::kQBlock || I > mx::kMaxBlocks * mx::kQBlock)
    return fail(c, MX_EINVAL, "Block FP8 hidden and intermediate are at most %d.", mx::kMaxBlocks * mx::kQBlock);
  if (dtype != MX_DTYPE_F16 && dtype != MX_DTYPE_BF16) return fail(c, MX_EINVAL, "MoE rows must be f16 or bf16.");
  if (!w) return fail(c, MX_EINVAL, "MLP weight buffers must not be null.");
  const mx_qmatrix* mats[3] = {&w->gate, &w->up, &w->down};
  for (const mx_qmatrix* m : mats)
    if (!m->data || !m->scales || !is_aligned(m->data, 16) || !is_aligned(m->scales, 4))
      return fail(c, MX_EINVAL, "Block FP8 weights must be non-null, codes 16-byte and scales 4-byte aligned.");
  if (T == 0) return MX_OK;
  if (!x || !ids || !weights || !out) return fail(c, MX_EINVAL, "MoE buffers must not be null.");
  if (!is_aligned(x, 16) || !is_aligned(out, 16) || !is_aligned(add, 16) || !is_aligned(ids, 4) || !is_aligned(weights, 4))
    return fail(c, MX_EINVAL, "MoE rows must be 16-byte aligned, ids and weights 4-byte.");
  if (T == 1 && H <= mx::kMaxDirect && I <= mx::kMaxDirect)
    return block_experts_of_one(c, H, I, E, topk, x, dtype, ids, weights, w, add, out);
  // Larger batches in parts: a part's picked rows of x are addressed by 31 bits, and
  // half of that keeps the f32 rows of its slots to 4 GB a slot of a token.
  const int most = (int)(0x3fff0000u / (uint32_t)H);
  for (int t = 0; t < T; t += most) {
    const size_t row = (size_t)t * H * 2;
    const int rc = block_experts(c, T - t < most ? T - t : most, H, I, E, topk, static_cast<const uint8_t*>(x) + row, dtype,
                                 ids + (size_t)t * topk, weights + (size_t)t * topk, w,
                                 add ? static_cast<const uint8_t*>(add) + row : nullptr, static_cast<uint8_t*>(out) + row);
    if (rc) return rc;
  }
  return MX_OK;
}

}  // extern "C"
