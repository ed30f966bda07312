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

// Streamed tiles keep the weights' way from HBM busy and cost a fetch of the
// weights for each; the others cost rounds of the CUs by a stage's time, in us,
// as measured (a stage: one 128-block of K):
//   64 rows    0.41 a stage up to 256 tiles, 0.65 for two on a CU; in f16 0.8 and
//              1.25 (SwiGLU 0.85 and 1.2)
//   128 rows   1.8, f32 results only
//   256 rows   1.05, from half of the CUs on more (L2, and a lower clock), 1.5 for all
// 1645 rows of 7680 -> 9728: 191 us with 64 rows and 172 with 256; to f32, 1381 rows
// of 512 -> 6144 26 us with 64 rows and 31 with 128.  16 experts with 32 rows each
// run on 64-row tiles, which sum SwiGLU's products in f16, from 48 rows on on 256-row
// tiles, which read each expert's weights once.
int block_tile_rows(long rows, int groups, int n, int k, int c_dtype, bool swiglu) {
  const long each = (rows + groups - 1) / groups;
  if (groups > 1) {  // experts differ in rows: room for more than the mean
    if (each <= 6) return 16;
    if (each <= 20) return 32;  // (block_stream_most)
    if (swiglu) return each <= 48 ? 64 : 256;
  }
  if (each <= 16) return 16;
  // two fetches of small weights come from the cache
  if (each <= 32) return ((swiglu ? n * 2L : n) + 31) / 32 <= 192 ? 16 : 32;
  const bool f32 = !swiglu && c_dtype == MX_DTYPE_F32;
  const double kb = (k + kQBlock - 1) / kQBlock;
  auto rounds = [](long tiles, long at_once) { return (double)((tiles + at_once - 1) / at_once); };
  auto tiles = [&](long r, long c) { return groups * ((each + r - 1) / r) * ((n + c - 1) / c); };
  const long t64 = tiles(64, 128);
  const double us64 = t64 <= 256 ? kb * (swiglu ? 0.85 : f32 ? 0.8 : 0.41) + 6
                                 : rounds(t64, swiglu ? 256 : 512) * (kb * (swiglu ? 1.2 : f32 ? 1.25 : 0.65) + 5.5);
  if (f32) return rounds(tiles(128, 256), 256) * (kb * 1.8 + 9) < us64 ? 128 : 64;
  const long t256 = tiles(256, swiglu ? 128 : 256), last = t256 % 256;
  const double stage = t256 > 214 ? 1.5 : t256 > 150 ? 0.007 * (double)t256 : 1.05;
  // (after others, a last round for at most half of the CUs takes about half of one)
  return (t256 / 256 + (last == 0 ? 0 : last <= 128 && t256 > 256 ? 0.55 : 1)) * (kb * stage + 8) < us64 ? 256 : 64;
}

hipError_t launch_block_gemm(int c_dtype, const BlockGemmArgs& g, hipStream_t st) {
  return block_streams(g.tile_rows) ? launch_block_stream(c_dtype, g, st) : launch_block_tile(c_dtype, g, st);
}

}  // namespace mx
