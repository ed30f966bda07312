// mx_block.hip - FP8 with one f32 scale per 128 values (weights: per 128 x 128):
// quantizers and products.
#include "mx_block_device.h"

namespace mx {
namespace {

// Bound: HBM and L2 (34 MB of bf16 at 3.5 TB/s, read and written).  A workgroup
// takes one block of 16 rows, so that their scales are written together; four
// blocks a lane, all loaded first, measured 14.3 -> 17.4 us.
template <int DT>
__global__ __launch_bounds__(256) void k_quantize(const void* src, int rows, int k, uint8_t* q, float* scales) {
  const int row = blockIdx.x * 16 + (threadIdx.x >> 4);
  if (row < rows) quantize_block<DT>(src, rows, k, q, scales, row, blockIdx.y);
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
    if (r < rows && c < k) *reinterpret_cast<v2i*>(q + (size_t)r * k + c) = v2i{(int)e4m3x4(v4f{v[i][0], v[i][1], v[i][2], v[i][3]}, s), (int)e4m3x4(v4f{v[i][4], v[i][5], v[i][6], v[i][7]}, s)};
  }
  if (threadIdx.x == 0) scales[(size_t)blockIdx.y * gridDim.x + blockIdx.x] = s;
}

}  // namespace

hipError_t launch_block_quantize(int dtype, const void* src, int rows, int k, uint8_t* q, float* scales,
                                 hipStream_t st) {
  const dim3 grid((rows + 15) / 16, (k + kQBlock - 1) / kQBlock);
  switch (dtype) {
    case MX_DTYPE_F32: hipLaunchKernelGGL((k_quantize<MX_DTYPE_F32>), grid, dim3(256), 0, st, src, rows, k, q, scales); break;
    case MX_DTYPE_F16: hipLaunchKernelGGL((k_quantize<MX_DTYPE_F16>), grid, dim3(256), 0, st, src, rows, k, q, scales); break;
    case MX_DTYPE_BF16: hipLaunchKernelGGL((k_quantize<MX_DTYPE_BF16>), grid, dim3(256), 0, st, src, rows, k, q, scales); break;
    default: return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

hipError_t launch_block_quantize_weights(const float* w, int rows, int k, uint8_t* q, float* scales, hipStream_t st) {
  hipLaunchKernelGGL(k_quantize_weights, dim3((k + kQBlock - 1) / kQBlock, (rows + kQBlock - 1) / kQBlock), dim3(256), 0,
                     st, w, rows, k, q, scales);
  return hipGetLastError();
}

int block_tile_rows(long rows, int groups, int n, int c_dtype, bool swiglu) {
  const long each = (rows + groups - 1) / groups;
  if (each <= 16) return 16;
  // f32 results keep more bits than the FP8 matrix cores' sums hold
  if (!swiglu && c_dtype == MX_DTYPE_F32) return 64;
  const long tiles = groups * ((each + 255) / 256) * ((n + 255) / 256) * (swiglu ? 2 : 1);
  return each >= 160 && tiles >= 128 ? 256 : 64;
}

hipError_t launch_block_gemm(int c_dtype, const BlockGemmArgs& g, hipStream_t st) {
  return g.tile_rows == 16 ? launch_block_stream(c_dtype, g, st) : launch_block_tile(c_dtype, g, st);
}

}  // namespace mx
