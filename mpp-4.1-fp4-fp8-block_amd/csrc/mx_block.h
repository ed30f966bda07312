// mx_block.h - launchers of the routed-experts operators (mx_moe.hip,
// mx_block.hip), shared with the C-ABI layer.
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "../../include/mxfp4hip.h"

namespace mx {

constexpr int kQBlock = 128;         // values (of weights: rows too) of one block scale
constexpr int kMaxBlocks = 512;       // blocks of K in one product
constexpr int kMaxRows = 1 << 28;     // rows of a block-scaled matrix: a launch's grid holds 2^32 threads
constexpr int kMaxHidden = 1 << 28;   // values of an exchanged row: their place is an int
constexpr int kMaxDirect = 8192;      // values of a row that launch_block_direct quantizes
constexpr int kMaxRouteExperts = 512;
constexpr int kMaxRouteGroups = 64;

// ---- router and exchange (mx_moe.hip) ---------------------------------------
struct RouteArgs {
  const void* logits;
  size_t stride;                     // elements between the rows of logits
  const float* bias;                 // null: none
  int32_t* ids;
  float* weights;
  int tokens, experts, topk, groups, topk_groups, group_top;
  int sigmoid, renormalize;
  float scale;
};
hipError_t launch_route(int dtype, const RouteArgs& a, hipStream_t st);

// A run of rows of one expert: one row tile of a grouped product.
struct RowTile {
  int expert, row0, rows, pad;
};
struct DispatchArgs {
  const int32_t* ids;                // [tokens][topk]
  int n, experts;                    // n = tokens topk slots
  int32_t* counts;                   // [experts]
  int32_t* rows;                     // [n] slot -> row, -1: none
  int32_t* src;                      // [n] row -> slot; null: not wanted
  RowTile* tiles;                    // row tiles of tile_rows rows; null: not wanted
  int32_t* n_tiles;
  int tile_rows;
  int32_t* hist;                     // dispatch_ws_bytes
};
size_t dispatch_ws_bytes(int n, int experts);
hipError_t launch_dispatch(const DispatchArgs& a, hipStream_t st);
// and xs[rows[t][s]] = x[t]; row_bytes of any even size
hipError_t launch_dispatch_rows(const DispatchArgs& a, int topk, const void* x, void* xs, size_t row_bytes, hipStream_t st);
// and x (f16 or bf16) as launch_block_quantize does
hipError_t launch_prepare(const DispatchArgs& a, int dtype, const void* x, int rows, int k, uint8_t* q, float* scales,
                          hipStream_t st);

struct CombineArgs {
  const void* y;
  const int32_t* rows;
  const float* weights;
  const void* add;                   // null: none
  void* out;
  int tokens, topk, hidden;
  // rows null: the row of a slot is the slot, where its expert is one of `experts`
  const int32_t* ids;
  int experts;
};
hipError_t launch_combine(int y_dtype, int out_dtype, const CombineArgs& a, hipStream_t st);

// Workspace of mx_moe_block_forward: offsets of its parts, 256-byte aligned.  Every
// part takes no less for more tokens (or more of anything), whichever kernels run.
struct ExpertsLayout {
  size_t xq, xs;                     // [T][H] codes of x, [H / 128][T] scales
  size_t rows, src, counts, tiles, n_tiles, hist;
  size_t mid;                        // f32 middles, of as many slots as streams take
  size_t mq, ms;                     // [n][I] codes of the middle, [I / 128][n] scales
  size_t y;                          // f32 [n][H] experts' rows
  size_t total;
};
ExpertsLayout experts_layout(int T, int H, int I, int E, int topk);

// ---- block-scaled FP8 (mx_block.hip) ------------------------------------------
hipError_t launch_block_quantize(int dtype, const void* src, int rows, int k, uint8_t* q, float* scales,
                                 hipStream_t st);
hipError_t launch_block_quantize_weights(const float* w, int rows, int k, uint8_t* q, float* scales, hipStream_t st);

// C[m][n] = sum_kb a_s[kb][m] w_s[n / 128][kb] sum_{k in kb} a[m][k] w[n][k], or with
// w1 silu(C0) C1 of two such products.
struct BlockGemmArgs {
  const uint8_t* a;                  // E4M3 [a_rows][k]
  const float* a_s;                  // [k / 128][a_rows]
  int a_rows;
  const uint8_t *w0, *w1;            // E4M3 [n][k]; w1 null: no SwiGLU
  const float *s0, *s1;              // [n / 128][k / 128]
  void* c;                           // [m][n]; SwiGLU: E4M3 codes, and
  float* c_s;                        // their scales [n / 128][m]
  int m, n, k;
  int fp8_cores;                     // f32 results by tiles: the FP8 cores' sums will do
  int tile_rows;                     // block_tile_rows
  int splits;                        // parts of K (block_splits): more than one are summed from
  void* part;                        // f32 [splits][m][n]
  // grouped: row tiles of experts, whose weights lie w_stride and s_stride apart
  const RowTile* tiles;              // null: one matrix
  const int32_t* n_tiles;
  int max_tiles;
  size_t w_stride, s_stride;
  const int32_t* src;                // row -> slot, and
  int src_div;                       // slot / src_div = row of a (null: row of a = row)
  // one token's slots (launch_block_direct): the row is quantized where it is used
  const void* raw;                   // [k], or [m][k] with row_per_slot
  int row_per_slot;
  const int32_t* ids;                // [m] the slots' experts
  int experts;
};
// Activation rows of a tile for `rows` rows in `groups` matrices [n][k]: 16 or 32
// (weights streamed), 64, 128 (f32 results) or 256.
int block_tile_rows(long rows, int groups, int n, int k, int c_dtype, bool swiglu);
int block_splits(int m, int n, int k, int tile_rows);
// Bytes of the parts of any product of up to m rows: no less for more of m, n or k,
// so that a workspace of the largest product holds the others' (a call that grew it
// would free what a captured call still points at).
size_t block_split_bytes(int m, int n, int k);
// The product by tiles of g.tile_rows rows.  SwiGLU: streamed tiles write
// f32 [m][n] to c, larger ones E4M3 codes to c and their scales to c_s.
inline bool block_streams(int tile_rows) { return tile_rows <= 32; }
// The most rows in `groups` matrices that block_tile_rows gives to streams.
inline long block_stream_most(int groups) { return groups > 1 ? 20L * groups : 32; }
hipError_t launch_block_gemm(int c_dtype, const BlockGemmArgs& g, hipStream_t st);
hipError_t launch_block_stream(int c_dtype, const BlockGemmArgs& g, hipStream_t st);  // mx_block_stream.hip
// One token, k <= kMaxDirect: gate/up products of an f16 or bf16 row or the down
// product of its f32 middles, to f32.
hipError_t launch_block_direct(int raw_dtype, const BlockGemmArgs& g, hipStream_t st);
hipError_t launch_block_tile(int c_dtype, const BlockGemmArgs& g, hipStream_t st);    // mx_block_tile.hip

}  // namespace mx
