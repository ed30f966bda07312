// mx_block.hip - FP8 with one f32 scale per 128 values (weights: per 128 x 128):
// quantizers and products.
#include "mx_block.h"
#include "mx_convert.h"
#include "mx_device.h"

namespace mx {
namespace {

// Scale of 128 values of largest magnitude amax (bits; NaN and infinity are
// above every number): amax times the f32 nearest 1 / 448.
__device__ __forceinline__ float block_scale(uint32_t amax) {
  const float s = __builtin_bit_cast(float, amax) * (1.0f / 448.0f);
  return amax == 0 ? 1.0f : s < 1.17549435e-38f ? 1.17549435e-38f : s;
}

// Four values / s as E4M3 codes.  An IEEE division: a product with 1 / s would
// round some quotients to the other side of a tie.
__device__ __forceinline__ uint32_t e4m3x4(const float* v, float s) {
  v2s w = {0, 0};
  w = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(w, v[0] / s, v[1] / s, 1.0f, false);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(w, v[2] / s, v[3] / s, 1.0f, true);
  return __builtin_bit_cast(uint32_t, w);
}

// 16 lanes of 8 values a block; a workgroup takes 16 rows, so that their
// scales are written together.
template <int DT>
__global__ __launch_bounds__(256) void k_quantize(const void* src, int rows, int k, uint8_t* q, float* scales,
                                                  const int32_t* n_rows) {
  const int lane16 = threadIdx.x & 15, row = blockIdx.x * 16 + (threadIdx.x >> 4);
  if (row >= rows || (n_rows && row >= *n_rows)) return;
  const int kb = blockIdx.y, at = kb * kQBlock + lane16 * 8;
  float v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
  if (at < k) load_n_as_f32<DT, 8>(src, (size_t)row * k + at, v);
  uint32_t amax = 0;
#pragma unroll
  for (int u = 0; u < 8; u++) amax = max(amax, abs_bits(v[u]));
#pragma unroll
  for (int o = 8; o; o >>= 1) amax = max(amax, (uint32_t)__shfl_xor((int)amax, o));
  const float s = block_scale(amax);
  if (at < k) *reinterpret_cast<v2i*>(q + (size_t)row * k + at) = v2i{(int)e4m3x4(v, s), (int)e4m3x4(v + 4, s)};
  if (lane16 == 0) scales[(size_t)kb * rows + row] = s;
}

// One workgroup per 128 x 128 block, 64 values a thread.
__global__ __launch_bounds__(256) void k_quantize_weights(const float* w, int rows, int k, uint8_t* q, float* scales) {
  __shared__ uint32_t part[4];
  const int r0 = blockIdx.y * kQBlock, k0 = blockIdx.x * kQBlock;
  const int c = k0 + (threadIdx.x & 15) * 8;
  float v[8][8];
  uint32_t amax = 0;
#pragma unroll
  for (int i = 0; i < 8; i++) {
    const int r = r0 + i * 16 + (threadIdx.x >> 4);
#pragma unroll
    for (int u = 0; u < 8; u++) v[i][u] = 0.0f;
    if (r < rows && c < k) load_n_as_f32<MX_DTYPE_F32, 8>(w, (size_t)r * k + c, v[i]);
#pragma unroll
    for (int u = 0; u < 8; u++) amax = max(amax, abs_bits(v[i][u]));
  }
#pragma unroll
  for (int o = 32; o; o >>= 1) amax = max(amax, (uint32_t)__shfl_xor((int)amax, o));
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = amax;
  __syncthreads();
  const float s = block_scale(max(max(part[0], part[1]), max(part[2], part[3])));
#pragma unroll
  for (int i = 0; i < 8; i++) {
    const int r = r0 + i * 16 + (threadIdx.x >> 4);
    if (r < rows && c < k) *reinterpret_cast<v2i*>(q + (size_t)r * k + c) = v2i{(int)e4m3x4(v[i], s), (int)e4m3x4(v[i] + 4, s)};
  }
  if (threadIdx.x == 0) scales[(size_t)blockIdx.y * gridDim.x + blockIdx.x] = s;
}

// ---- product --------------------------------------------------------------------
// v_mfma_f32_16x16x128_f8f6f4 with unit scales sums one 128-block at a time; its
// sum, times the two block scales, is added in f32.  Weight rows are the
// MFMA's rows and activation rows its columns, so a lane has one activation
// scale and one weight scale for its four sums, and four neighbouring outputs.
// Both operands hold byte j of lane l as k = 32 (l / 16) + j of row l % 16: any
// order of k that they share gives the same sum.
__device__ __forceinline__ v4f mfma_fp8_16x16x128(v8i a, v8i b) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, v4f{0, 0, 0, 0}, 0, 0, 0, 127, 0, 127);
}

__device__ __forceinline__ v8i load_row32(const uint8_t* row, int k0, int k) {
  v8i r = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
  for (int u = 0; u < 2; u++)
    if (k0 + u * 16 < k) {
      const v4i x = *reinterpret_cast<const v4i*>(row + k0 + u * 16);
#pragma unroll
      for (int i = 0; i < 4; i++) r[u * 4 + i] = x[i];
    }
  return r;
}

// 64 x 64 outputs a workgroup: a wave has 16 weight rows (SwiGLU: of gate and
// of up) and 64 activation rows, read from global memory.
template <int DT, bool DUAL>
__global__ __launch_bounds__(256) void k_block_gemm(BlockGemmArgs g) {
  int row0 = blockIdx.y * 64, rows = min(64, g.m - row0), expert = 0;
  if (g.tiles) {
    if ((int)blockIdx.y >= *g.n_tiles) return;
    const RowTile t = g.tiles[blockIdx.y];
    row0 = t.row0;
    rows = t.rows;
    expert = t.expert;
  }
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r16 = lane & 15, kq = lane >> 4;
  const int n0 = blockIdx.x * 64 + wave * 16, n = min(n0 + r16, g.n - 1), kb_n = (g.k + kQBlock - 1) / kQBlock;
  const uint8_t* w[2] = {g.w0 + expert * g.w_stride + (size_t)n * g.k, g.w1 + expert * g.w_stride + (size_t)n * g.k};
  const size_t so = expert * g.s_stride + (size_t)(min(n0, g.n - 1) / kQBlock) * kb_n;
  const float* s[2] = {g.s0 + so, g.s1 + so};
  int ar[4];
#pragma unroll
  for (int t = 0; t < 4; t++) {
    const int r = row0 + min(t * 16 + r16, rows - 1);
    ar[t] = g.src ? g.src[r] / g.src_div : r;
  }
  v4f acc[2][4];
#pragma unroll
  for (int d = 0; d < 2; d++)
#pragma unroll
    for (int t = 0; t < 4; t++) acc[d][t] = v4f{0, 0, 0, 0};
  for (int kb = 0; kb < kb_n; kb++) {
    const int k0 = kb * kQBlock + kq * 32;
    v8i wf[2];
    wf[0] = load_row32(w[0], k0, g.k);
    if constexpr (DUAL) wf[1] = load_row32(w[1], k0, g.k);
#pragma unroll
    for (int t = 0; t < 4; t++) {
      if (t * 16 >= rows) break;
      const v8i x = load_row32(g.a + (size_t)ar[t] * g.k, k0, g.k);
      const float as = g.a_s[(size_t)kb * g.a_rows + ar[t]];
#pragma unroll
      for (int d = 0; d < (DUAL ? 2 : 1); d++) acc[d][t] += mfma_fp8_16x16x128(wf[d], x) * (as * s[d][kb]);
    }
  }
#pragma unroll
  for (int t = 0; t < 4; t++)
#pragma unroll
    for (int v = 0; v < 4; v++) {
      const int r = t * 16 + r16, c = n0 + kq * 4 + v;
      if (r >= rows || c >= g.n) continue;
      float x = acc[0][t][v];
      if constexpr (DUAL) x = silu(x) * acc[1][t][v];
      store_from_f32<DT>(g.c, (size_t)(row0 + r) * g.n + c, x);
    }
}

template <int DT>
hipError_t gemm_dt(const BlockGemmArgs& g, hipStream_t st) {
  const dim3 grid((g.n + 63) / 64, g.tiles ? g.max_tiles : (g.m + 63) / 64);
  if (g.w1) hipLaunchKernelGGL((k_block_gemm<DT, true>), grid, dim3(256), 0, st, g);
  else hipLaunchKernelGGL((k_block_gemm<DT, false>), grid, dim3(256), 0, st, g);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_block_quantize(int dtype, const void* src, int rows, int k, uint8_t* q, float* scales,
                                 const int32_t* n_rows, hipStream_t st) {
  const dim3 grid((rows + 15) / 16, (k + kQBlock - 1) / kQBlock);
  switch (dtype) {
    case MX_DTYPE_F32: hipLaunchKernelGGL((k_quantize<MX_DTYPE_F32>), grid, dim3(256), 0, st, src, rows, k, q, scales, n_rows); break;
    case MX_DTYPE_F16: hipLaunchKernelGGL((k_quantize<MX_DTYPE_F16>), grid, dim3(256), 0, st, src, rows, k, q, scales, n_rows); break;
    case MX_DTYPE_BF16: hipLaunchKernelGGL((k_quantize<MX_DTYPE_BF16>), grid, dim3(256), 0, st, src, rows, k, q, scales, n_rows); break;
    default: return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

hipError_t launch_block_quantize_weights(const float* w, int rows, int k, uint8_t* q, float* scales, hipStream_t st) {
  hipLaunchKernelGGL(k_quantize_weights, dim3((k + kQBlock - 1) / kQBlock, (rows + kQBlock - 1) / kQBlock), dim3(256), 0,
                     st, w, rows, k, q, scales);
  return hipGetLastError();
}

hipError_t launch_block_gemm(int c_dtype, const BlockGemmArgs& g, hipStream_t st) {
  switch (c_dtype) {
    case MX_DTYPE_F32: return gemm_dt<MX_DTYPE_F32>(g, st);
    case MX_DTYPE_F16: return gemm_dt<MX_DTYPE_F16>(g, st);
    case MX_DTYPE_BF16: return gemm_dt<MX_DTYPE_BF16>(g, st);
  }
  return hipErrorInvalidValue;
}

}  // namespace mx
