// mx_block_stream.hip - products of block-scaled FP8 weights with at most 32
// activation rows a tile: the weights stream from HBM to registers once.
//
// Bound: HBM.  A wave takes every W-th block of K of its workgroup's weight rows,
// straight to registers, in whole 128-byte lines (8 rows a load, the halves then
// exchanged between lanes); no wave waits for another before the final sum.  The
// products are f16 MFMAs of the widened codes, whose sums are f32: the matrix cores
// have time for that while the weights come in.  One token's 352 MB through 8 of 64
// experts: 43 us gate/up (5.5 TB/s) and 23 us down (5.1), where a copy reaches 4.9.
#include "mx_block.h"
#include "mx_block_device.h"

namespace mx {
namespace {

__device__ __align__(16) const uint8_t kZeros[16] = {};

// v with its lanes' halves of 16 exchanged where MASK has the lane's group of
// four: old elsewhere.
template <int MASK>
__device__ __forceinline__ v4i from_other_half(v4i old, v4i v) {
  v4i r;
#pragma unroll
  for (int i = 0; i < 4; i++) r[i] = __builtin_amdgcn_update_dpp(old[i], v[i], 0x128, 0xf, MASK, false);
  return r;
}

template <int NG, int TT>
struct Step {
  v4i w[NG][2], a[TT][2];
  float as[TT], ws[2];
};

// 16 NG weight rows (SwiGLU: half of them gate, half up) x 16 TT activation rows;
// W waves take every W-th 128-block of K, D blocks ahead.  XT >= 0: one token, whose
// slots are the row tiles; the workgroup quantizes its row (in XT) into LDS while
// its first weights are on their way.
template <int DT, bool DUAL, int NG, int W, int D, int TT, int XT>
__global__ __launch_bounds__(64 * W) void k_block_stream(BlockGemmArgs g) {
  constexpr int ND = DUAL ? 2 : 1, CH = 16 * NG / ND;  // channels of the workgroup
  constexpr bool RAW = XT >= 0;
  __shared__ float part[W][NG][16 * TT][17];
  __shared__ __attribute__((aligned(16))) uint8_t xq[RAW ? kMaxDirect : 16];
  __shared__ float xs[RAW ? kMaxDirect / kQBlock : 1];
  const int NT = (g.n + CH - 1) / CH;
  int row0 = blockIdx.x / NT * (16 * TT), rows = min(16 * TT, g.m - row0), expert = 0;
  // (the row's values are under way before the slot's expert is known)
  constexpr int RB = RAW ? kMaxDirect / kQBlock / (4 * W) : 1;
  float raw[RB][8];
  if constexpr (RAW) {
    row0 = blockIdx.x / NT;
    rows = 1;
    const size_t at = (size_t)(g.row_per_slot ? row0 : 0) * g.k;
#pragma unroll
    for (int i = 0; i < RB; i++) {
      const int c = (i * 64 * W + threadIdx.x) * 8;  // block i * 4 W + tid / 16
#pragma unroll
      for (int u = 0; u < 8; u++) raw[i][u] = 0.0f;
      if (c < g.k) load_n_as_f32<RAW ? XT : MX_DTYPE_F32, 8>(g.raw, at + c, raw[i]);
    }
    expert = g.ids[row0];
    if ((unsigned)expert >= (unsigned)g.experts) return;
  } else if (g.tiles) {
    const int rt = blockIdx.x / NT;
    const RowTile t = g.tiles[rt];  // (read beside the count: max_tiles are there)
    if (rt >= *g.n_tiles) return;
    row0 = t.row0;
    rows = t.rows;
    expert = t.expert;
  }
  const int n0 = blockIdx.x % NT * CH;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r16 = lane & 15, kq = lane >> 4;
  const int K = g.k, KB = (K + kQBlock - 1) / kQBlock;
  // A load covers 8 whole rows of 128 bytes: lane l has row l % 8 and chunk
  // 2 (l / 16) + (l / 8) % 2, and gets its own row's other chunk from the lane
  // half of 16 away.
  const int wchunk = 2 * kq + (r16 >> 3);
  const uint8_t* w[NG][2];
#pragma unroll
  for (int i = 0; i < NG; i++)
#pragma unroll
    for (int u = 0; u < 2; u++) {
      const int n = n0 + (i % (NG / ND)) * 16 + u * 8 + (r16 & 7);
      w[i][u] = (DUAL && i >= NG / 2 ? g.w1 : g.w0) + expert * g.w_stride + (size_t)min(n, g.n - 1) * K + wchunk * 16;
    }
  const uint8_t* a[TT];
  const float* as[TT];
#pragma unroll
  for (int t = 0; t < TT; t++) {
    const int row = row0 + min(t * 16 + r16, rows - 1), ar = RAW ? 0 : g.src ? g.src[row] / g.src_div : row;
    a[t] = g.a + (size_t)ar * K + kq * 32;
    as[t] = g.a_s + ar;
  }
  const size_t so = expert * g.s_stride + (size_t)(n0 / kQBlock) * KB;
  const float *s0 = g.s0 + so, *s1 = (DUAL ? g.s1 : g.s0) + so;
  const uint8_t* zeros = kZeros;
  asm volatile("" : "+v"(zeros));  // a value, not a constant: selects, where the compiler would branch

  auto load = [&](int kb, Step<NG, TT>& s) {
    const size_t o = (size_t)kb * kQBlock;
    const int left = K - kb * kQBlock;  // chunks past K are zero on both sides: what lies there may be NaN
    const bool win = wchunk * 16 < left;
#pragma unroll
    for (int i = 0; i < NG; i++)
#pragma unroll
      for (int u = 0; u < 2; u++) s.w[i][u] = *reinterpret_cast<const v4i*>(win ? w[i][u] + o : zeros);
    s.ws[0] = s0[kb];
    if constexpr (DUAL) s.ws[1] = s1[kb];
    if constexpr (RAW) return;
#pragma unroll
    for (int t = 0; t < TT; t++) {
#pragma unroll
      for (int u = 0; u < 2; u++) s.a[t][u] = *reinterpret_cast<const v4i*>(kq * 32 + u * 16 < left ? a[t] + o + u * 16 : zeros);
      s.as[t] = as[t][(size_t)kb * g.a_rows];
    }
  };
  v4f acc[NG][TT];
#pragma unroll
  for (int i = 0; i < NG; i++)
#pragma unroll
    for (int t = 0; t < TT; t++) acc[i][t] = v4f{0, 0, 0, 0};
  auto use = [&](int kb, const Step<NG, TT>& s) {
    v8h x[TT][4];
    float sc[TT][ND];
#pragma unroll
    for (int t = 0; t < TT; t++) {
#pragma unroll
      for (int u = 0; u < 2; u++) {
        const v4i codes = RAW ? *reinterpret_cast<const v4i*>(xq + kb * kQBlock + kq * 32 + u * 16) : s.a[t][u];
#pragma unroll
        for (int h = 0; h < 2; h++) x[t][2 * u + h] = fp8x8_to_f16<BK_E4M3>((uint32_t)codes[2 * h], (uint32_t)codes[2 * h + 1]);
      }
#pragma unroll
      for (int d = 0; d < ND; d++) sc[t][d] = (RAW ? xs[kb] : s.as[t]) * s.ws[d];
    }
#pragma unroll
    for (int i = 0; i < NG; i++) {
      // lanes of the lower half: row r16 of the first load; upper: of the second
      const v4i c[2] = {from_other_half<0xc>(s.w[i][0], s.w[i][1]), from_other_half<0x3>(s.w[i][1], s.w[i][0])};
      v8h wh[4];
#pragma unroll
      for (int u = 0; u < 2; u++)
#pragma unroll
        for (int h = 0; h < 2; h++) wh[2 * u + h] = fp8x8_to_f16<BK_E4M3>((uint32_t)c[u][2 * h], (uint32_t)c[u][2 * h + 1]);
#pragma unroll
      for (int t = 0; t < TT; t++) {
        v4f sum = {0, 0, 0, 0};
#pragma unroll
        for (int q = 0; q < 4; q++) sum = mfma_f16_16x16x32(wh[q], x[t][q], sum);
#pragma unroll
        for (int v = 0; v < 4; v++) acc[i][t][v] = fmaf(sum[v], sc[t][DUAL && i >= NG / 2 ? 1 : 0], acc[i][t][v]);
      }
    }
  };
  Step<NG, TT> st[D];
#pragma unroll
  for (int d = 0; d < D; d++)
    if (wave + W * d < KB) load(wave + W * d, st[d]);
  if constexpr (RAW) {
#pragma unroll
    for (int i = 0; i < RB; i++) {
      const int kb = i * 4 * W + (threadIdx.x >> 4);
      if (kb >= KB) break;
      const float sc = quantize_lanes16(raw[i], xq + kb * kQBlock + (threadIdx.x & 15) * 8);
      if ((threadIdx.x & 15) == 0) xs[kb] = sc;
    }
    __syncthreads();
  }
  for (int kb = wave; kb < KB; kb += W * D) {
#pragma unroll
    for (int d = 0; d < D; d++) {
      if (kb + W * d < KB) use(kb + W * d, st[d]);
      if (kb + W * (d + D) < KB) load(kb + W * (d + D), st[d]);
    }
  }
#pragma unroll
  for (int i = 0; i < NG; i++)
#pragma unroll
    for (int t = 0; t < TT; t++)
#pragma unroll
      for (int v = 0; v < 4; v++) part[wave][i][t * 16 + r16][kq * 4 + v] = acc[i][t][v];
  __syncthreads();
  // the waves' sums, in their order
  for (int o = threadIdx.x; o < rows * CH; o += 64 * W) {
    const int r = o / CH, c = o % CH;
    if (n0 + c >= g.n) continue;
    float x[ND];
#pragma unroll
    for (int d = 0; d < ND; d++) {
      const int i = c / 16 + d * (NG / 2);
      x[d] = part[0][i][r][c % 16];
#pragma unroll
      for (int w = 1; w < W; w++) x[d] += part[w][i][r][c % 16];
    }
    float y = x[0];
    if constexpr (DUAL) y = silu(y) * x[1];
    store_from_f32<DT>(g.c, (size_t)(row0 + r) * g.n + n0 + c, y);
  }
}

template <int DT, bool DUAL, int NG, int W, int D, int TT, int XT>
hipError_t launch_one(const BlockGemmArgs& g, hipStream_t st) {
  constexpr int CH = 16 * NG / (DUAL ? 2 : 1);
  const long tiles = (long)(XT >= 0 ? g.m : g.tiles ? g.max_tiles : (g.m + 16 * TT - 1) / (16 * TT)) * ((g.n + CH - 1) / CH);
  if (tiles > 0x7fffffffL) return hipErrorInvalidValue;
  hipLaunchKernelGGL((k_block_stream<DT, DUAL, NG, W, D, TT, XT>), dim3((unsigned)tiles), dim3(64 * W), 0, st, g);
  return hipGetLastError();
}

// 32 weight rows a workgroup of 4 waves.  Blocks under way in a wave: where K is
// short, one, and more waves on a CU (32 experts' 1408 -> 4096, 10 rows each: 37 us,
// 39 with two and 45 with three); past 4096 two (one token's gate and up products
// of 7168: 43, 47 with one).  One token, whose activations take no registers: three.
// Where the tiles leave CUs idle, 16 rows (with SwiGLU 32) and 8 waves: one row of
// 7552 -> 2560 12.9 -> 7.9 us, of 4096 -> 4096 8.7 -> 7.1, but of 4096 -> 14336 14.8
// -> 16.4.
template <int DT, bool DUAL, int TT, int XT>
hipError_t launch_shape(const BlockGemmArgs& g, hipStream_t st) {
  const long tiles = (long)(XT >= 0 ? g.m : g.tiles ? g.max_tiles : (g.m + 16 * TT - 1) / (16 * TT)) * ((g.n + 31) / 32);
  if constexpr (TT == 1) {
    if (tiles * (DUAL ? 2 : 1) < 256) return launch_one<DT, DUAL, DUAL ? 2 : 1, 8, 2, TT, XT>(g, st);
  }
  if constexpr (XT >= 0) return launch_one<DT, DUAL, 2, 4, 3, TT, XT>(g, st);
  else return g.k <= 32 * kQBlock ? launch_one<DT, DUAL, 2, 4, 1, TT, XT>(g, st) : launch_one<DT, DUAL, 2, 4, 2, TT, XT>(g, st);
}

template <int TT>
hipError_t launch_rows(int c_dtype, const BlockGemmArgs& g, hipStream_t st) {
  if (g.w1) return launch_shape<MX_DTYPE_F32, true, TT, -1>(g, st);
  switch (c_dtype) {
    case MX_DTYPE_F32: return launch_shape<MX_DTYPE_F32, false, TT, -1>(g, st);
    case MX_DTYPE_F16: return launch_shape<MX_DTYPE_F16, false, TT, -1>(g, st);
    case MX_DTYPE_BF16: return launch_shape<MX_DTYPE_BF16, false, TT, -1>(g, st);
  }
  return hipErrorInvalidValue;
}

}  // namespace

hipError_t launch_block_stream(int c_dtype, const BlockGemmArgs& g, hipStream_t st) {
  return g.tile_rows == 16 ? launch_rows<1>(c_dtype, g, st) : launch_rows<2>(c_dtype, g, st);
}

hipError_t launch_block_direct(int raw_dtype, const BlockGemmArgs& g, hipStream_t st) {
  switch (raw_dtype) {
    case MX_DTYPE_F32: return launch_shape<MX_DTYPE_F32, false, 1, MX_DTYPE_F32>(g, st);  // the middle
    case MX_DTYPE_F16: return launch_shape<MX_DTYPE_F32, true, 1, MX_DTYPE_F16>(g, st);
    case MX_DTYPE_BF16: return launch_shape<MX_DTYPE_F32, true, 1, MX_DTYPE_BF16>(g, st);
  }
  return hipErrorInvalidValue;
}

}  // namespace mx
