// mx_block_device.h - device helpers of the block-scaled FP8 kernels.
#pragma once

#include "mx_block.h"
#include "mx_convert.h"
#include "mx_device.h"
#include "mx_widen.h"

namespace mx {

// Scale of 128 values of largest magnitude amax (bits; NaN and infinity are
// above every number): amax times the f32 nearest 1 / 448.
__device__ __forceinline__ float block_scale(uint32_t amax) {
  const float s = __builtin_bit_cast(float, amax) * (1.0f / 448.0f);
  return amax == 0 ? 1.0f : s < 1.17549435e-38f ? 1.17549435e-38f : s;
}

// Four values / s as E4M3 codes.  An IEEE division: a product with 1 / s would
// round some quotients to the other side of a tie.
__device__ __forceinline__ uint32_t e4m3x4(v4f v, float s) {
  v2s w = {0, 0};
  w = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(w, v[0] / s, v[1] / s, 1.0f, false);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(w, v[2] / s, v[3] / s, 1.0f, true);
  return __builtin_bit_cast(uint32_t, w);
}

// 16 lanes quantize one block of a row, 8 values each (v: the lane's, 0 past the
// row); returns its scale, and writes the codes to q unless it is null.
__device__ __forceinline__ float quantize_lanes16(const float* v, uint8_t* q) {
  uint32_t amax = 0;
#pragma unroll
  for (int u = 0; u < 8; u++) amax = max(amax, abs_bits(v[u]));
#pragma unroll
  for (int o = 8; o; o >>= 1) amax = max(amax, (uint32_t)__shfl_xor((int)amax, o));
  const float s = block_scale(amax);
  if (q) *reinterpret_cast<v2i*>(q) = v2i{(int)e4m3x4(v4f{v[0], v[1], v[2], v[3]}, s), (int)e4m3x4(v4f{v[4], v[5], v[6], v[7]}, s)};
  return s;
}

template <int DT>
__device__ __forceinline__ void quantize_block(const void* src, int rows, int k, uint8_t* q, float* scales, int row, int kb) {
  const int c = kb * kQBlock + (threadIdx.x & 15) * 8;
  float v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
  if (c < k) load_n_as_f32<DT, 8>(src, (size_t)row * k + c, v);
  const float s = quantize_lanes16(v, c < k ? q + (size_t)row * k + c : nullptr);
  if ((threadIdx.x & 15) == 0) scales[(size_t)kb * rows + row] = s;
}

// The sum of one 128-block of 16 weight rows (the MFMA's rows) and 16 activation
// rows (its columns): a lane has one activation scale and one weight scale for
// its four sums, and four neighbouring outputs.  Both operands hold byte j of
// lane l as k = 32 (l / 16) + j of row l % 16: any order of k that they share
// gives the same sum.
__device__ __forceinline__ v4f mfma_fp8_16x16x128(v8i a, v8i b) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, v4f{0, 0, 0, 0}, 0, 0, 0, 127, 0, 127);
}

// 32 codes as four operands of the f16 MFMA, exactly.
__device__ __forceinline__ void widen4(const v8i& w, v8h* h) {
#pragma unroll
  for (int q = 0; q < 4; q++) h[q] = fp8x8_to_f16<BK_E4M3>((uint32_t)w[2 * q], (uint32_t)w[2 * q + 1]);
}

// `left` of four values, at any address of their type (rows of an odd length start
// anywhere)
template <int DT>
__device__ __forceinline__ void store4(void* p, size_t i, v4f v, int left) {
  if (left >= 4) {
    if constexpr (DT == MX_DTYPE_F32) {
      __builtin_memcpy(static_cast<float*>(p) + i, &v, 16);
    } else if constexpr (DT == MX_DTYPE_F16) {
      const v4h h{(_Float16)v[0], (_Float16)v[1], (_Float16)v[2], (_Float16)v[3]};
      __builtin_memcpy(static_cast<_Float16*>(p) + i, &h, 8);
    } else {
      const v4bf h{(__bf16)v[0], (__bf16)v[1], (__bf16)v[2], (__bf16)v[3]};
      __builtin_memcpy(static_cast<__bf16*>(p) + i, &h, 8);
    }
    return;
  }
#pragma unroll
  for (int u = 0; u < 4; u++)
    if (u < left) store_from_f32<DT>(p, i + u, v[u]);
}

}  // namespace mx
