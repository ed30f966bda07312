// mx_moe.hip - the router of a mixture of experts, and the exchange of rows
// between token order and expert order.
#include "mx_block_device.h"

namespace mx {
namespace {

// Tokens of one launch: a grid holds 2^32 threads in x, and a token takes up to 256.
constexpr int kMostTokens = 1 << 23;
size_t dtype_size(int dtype) { return dtype == MX_DTYPE_F32 ? 4 : 2; }

// ---- lanes ----------------------------------------------------------------------
// DPP: lane ^ 1, lane ^ 2, 7 - lane of 8, 15 - lane of 16.  After as many of them as
// log2(L), every lane of L has what the L lanes have together.
constexpr int kXor1 = 0xb1, kXor2 = 0x4e, kMirror8 = 0x141, kMirror16 = 0x140;
template <int CTRL>
__device__ __forceinline__ uint32_t dpp(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp((int)v, (int)v, CTRL, 0xf, 0xf, false);
}
template <int CTRL>
__device__ __forceinline__ float dpp(float v) { return __builtin_bit_cast(float, dpp<CTRL>(__builtin_bit_cast(uint32_t, v))); }
template <int CTRL>
__device__ __forceinline__ double dpp(double v) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  return __builtin_bit_cast(double, (uint64_t)dpp<CTRL>((uint32_t)(u >> 32)) << 32 | dpp<CTRL>((uint32_t)u));
}
template <class T>
__device__ __forceinline__ T lane_value(T v, int lane) {
  if constexpr (sizeof(T) == 8) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    return __builtin_bit_cast(T, (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(u >> 32), lane) << 32 |
                                     (uint32_t)__builtin_amdgcn_readlane((int)u, lane));
  } else {
    return __builtin_bit_cast(T, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), lane));
  }
}
// op over the wave's 64 lanes, as a uniform value
template <class T, class Op>
__device__ __forceinline__ T over_wave(T v, Op op) {
  v = op(v, dpp<kXor1>(v));
  v = op(v, dpp<kXor2>(v));
  v = op(v, dpp<kMirror8>(v));
  v = op(v, dpp<kMirror16>(v));
  return op(op(lane_value(v, 0), lane_value(v, 16)), op(lane_value(v, 32), lane_value(v, 48)));
}

// ---- router ---------------------------------------------------------------------
//
//   p = softmax(l) or 1 / (1 + e^-l), key = p + b, the best groups, the best k
//   keys; weight = p (/ the sum of the chosen p) * scale
//
// One wave a token, expert j * 64 + lane in register j.  The sum of a softmax is
// taken in f64 and rounded once, so that keys, and with them the choice, do not
// depend on the order of the sum.
//
// Bound: instructions, and at few tokens the launch.  The maximum of a wave by
// DPP and four lane reads, then the holder by one comparison a register, is a third
// of the instructions of a 64-bit (key, index) maximum by lane shuffles.

// Keys as integers of the same order; 0: not available.
__device__ __forceinline__ uint32_t ordered(float f) {
  const uint32_t u = __builtin_bit_cast(uint32_t, f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

template <int DT, int NP>
__global__ __launch_bounds__(256) void k_route(RouteArgs a) {
  __shared__ float keys[4][NP * 64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int t = blockIdx.x * 4 + wave;
  if (t >= a.tokens) return;
  const float kLow = -__builtin_inff(), kTop = 3.402823466e38f;
  const int E = a.experts;
  float v[NP], p[NP], key[NP];
#pragma unroll
  for (int j = 0; j < NP; j++) {
    const int e = j * 64 + lane;
    v[j] = e < E ? load_as_f32<DT>(a.logits, (size_t)t * a.stride + e) : kLow;
    key[j] = a.bias && e < E ? a.bias[e] : 0.0f;
  }
  float top = -kTop;
#pragma unroll
  for (int j = 0; j < NP; j++) {
    if (!(v[j] > kLow)) v[j] = kLow;  // NaN: masked
    v[j] = fminf(v[j], kTop);
    top = fmaxf(top, v[j]);
  }
  if (a.sigmoid) {
#pragma unroll
    for (int j = 0; j < NP; j++) p[j] = 1.0f / (1.0f + expf(-v[j]));
  } else {
    top = over_wave(top, [](float x, float y) { return fmaxf(x, y); });
    double sum = 0.0;
#pragma unroll
    for (int j = 0; j < NP; j++) {
      p[j] = v[j] > kLow ? expf(v[j] - top) : 0.0f;
      sum += (double)p[j];
    }
    const float s = (float)over_wave(sum, [](double x, double y) { return x + y; });
#pragma unroll
    for (int j = 0; j < NP; j++) p[j] = p[j] / s;
  }
#pragma unroll
  for (int j = 0; j < NP; j++) {
    key[j] = p[j] + key[j];
    if (!(v[j] > kLow) || !(key[j] > kLow)) key[j] = kLow;
  }
  if (a.groups > 1) {
    // L lanes a group; the first one keeps its score
    const int size = E / a.groups, L = 64 >> (32 - __builtin_clz(a.groups - 1)), sub = lane & (L - 1), grp = lane / L;
#pragma unroll
    for (int j = 0; j < NP; j++) keys[wave][j * 64 + lane] = key[j];
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    float b0 = kLow, b1 = kLow;
    if (grp < a.groups)
      for (int i = sub; i < size; i += L) {
        const float k = keys[wave][grp * size + i];
        b1 = fmaxf(b1, fminf(k, b0));
        b0 = fmaxf(b0, k);
      }
    auto join = [&](float o0, float o1) {
      b1 = fmaxf(fminf(b0, o0), fmaxf(b1, o1));
      b0 = fmaxf(b0, o0);
    };
    if (L >= 2) join(dpp<kXor1>(b0), dpp<kXor1>(b1));
    if (L >= 4) join(dpp<kXor2>(b0), dpp<kXor2>(b1));
    if (L >= 8) join(dpp<kMirror8>(b0), dpp<kMirror8>(b1));
    if (L >= 16) join(dpp<kMirror16>(b0), dpp<kMirror16>(b1));
    if (L >= 32) join(__shfl_xor(b0, 16), __shfl_xor(b1, 16));
    const float score = a.group_top == 2 && b1 > kLow ? b0 + b1 : b0;
    int rank = 0;
    for (int i = 0; i < a.groups; i++) {
      const float s = lane_value(score, i * L);
      rank += s > score || (s == score && i < grp);
    }
    const uint64_t kept = __ballot(grp < a.groups && rank < a.topk_groups);
    const float per = 1.0f / (float)size;  // (e + 0.5) / size is at least 0.5 / size from a whole number
#pragma unroll
    for (int j = 0; j < NP; j++) {
      const int e = j * 64 + lane, ge = (int)(((float)e + 0.5f) * per);
      if (e < E && !((kept >> (ge * L)) & 1)) key[j] = kLow;
    }
  }
  // best first; the lower index wins a tie
  uint32_t ord[NP];
#pragma unroll
  for (int j = 0; j < NP; j++) ord[j] = key[j] > kLow ? ordered(key[j]) : 0;
  float mine = 0.0f, total = 0.0f;
  int id = -1;
  for (int s = 0; s < a.topk; s++) {
    uint32_t best = ord[0];
#pragma unroll
    for (int j = 1; j < NP; j++) best = max(best, ord[j]);
    best = over_wave(best, [](uint32_t x, uint32_t y) { return x > y ? x : y; });
    if (!best) break;
    float w = 0.0f;
    int e = -1;
#pragma unroll
    for (int j = NP - 1; j >= 0; j--) {
      const uint64_t at = __ballot(ord[j] == best);
      if (at) {
        const int l = __builtin_ctzll(at);
        e = j * 64 + l;
        w = lane_value(p[j], l);
      }
    }
#pragma unroll
    for (int j = 0; j < NP; j++)
      if (j * 64 + lane == e) ord[j] = 0;
    total += w;
    if (lane == s) { mine = w; id = e; }
  }
  if (lane < a.topk) {
    float w = mine;
    if (a.renormalize) w = total > 0.0f ? w / total : 0.0f;
    a.ids[(size_t)t * a.topk + lane] = id;
    a.weights[(size_t)t * a.topk + lane] = id < 0 ? 0.0f : w * a.scale;
  }
}

template <int DT>
hipError_t route_dt(const RouteArgs& a, hipStream_t st) {
  const dim3 grid((a.tokens + 3) / 4);
  const int np = (a.experts + 63) / 64;
  if (np == 1) hipLaunchKernelGGL((k_route<DT, 1>), grid, dim3(256), 0, st, a);
  else if (np == 2) hipLaunchKernelGGL((k_route<DT, 2>), grid, dim3(256), 0, st, a);
  else if (np <= 4) hipLaunchKernelGGL((k_route<DT, 4>), grid, dim3(256), 0, st, a);
  else hipLaunchKernelGGL((k_route<DT, 8>), grid, dim3(256), 0, st, a);
  return hipGetLastError();
}

// ---- expert order -----------------------------------------------------------------
// A stable counting sort of the slots by expert.  A workgroup places kChunk slots:
// it needs the counts of all slots before and after them, which it takes from all
// ids where those are few (one launch; 32768 of them cost 2 us) and from a table of
// the chunks' counts, written by a launch of its own, where they are many.  A wave
// finds the slots of one expert among its 64 by nine ballots, one a bit; only
// integer counts are added by atomics, so the order of the rows is the slots'.
constexpr int kPlaceThreads = 1024, kPlaceWaves = kPlaceThreads / 64, kChunk = 4096, kPerWave = kChunk / kPlaceWaves;
constexpr int kCopies = 4;
constexpr int kMaxCounted = 16 * kChunk;  // ids that every workgroup counts itself

__device__ __forceinline__ int expert_of(const DispatchArgs& a, int i) {
  const int e = i < a.n ? a.ids[i] : -1;
  return (unsigned)e < (unsigned)a.experts ? e : -1;
}

__global__ __launch_bounds__(kPlaceThreads) void k_count(DispatchArgs a) {
  __shared__ int h[kMaxRouteExperts];
  for (int e = threadIdx.x; e < a.experts; e += kPlaceThreads) h[e] = 0;
  __syncthreads();
  for (int i = threadIdx.x; i < kChunk; i += kPlaceThreads) {
    const int e = expert_of(a, blockIdx.x * kChunk + i);
    if (e >= 0) atomicAdd(&h[e], 1);
  }
  __syncthreads();
  for (int e = threadIdx.x; e < a.experts; e += kPlaceThreads) a.hist[(size_t)blockIdx.x * a.experts + e] = h[e];
}

// inclusive prefix sums of v over the workgroup's threads
__device__ __forceinline__ int scan_all(int v, int* part) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int u = __shfl_up(v, o);
    if (lane >= o) v += u;
  }
  if (lane == 63) part[wave] = v;
  __syncthreads();
  for (int w = 0; w < wave; w++) v += part[w];
  __syncthreads();
  return v;
}

struct PlaceShared {
  int at[kPlaceWaves][kMaxRouteExperts];  // next row of an expert, by wave
  int other[2][kCopies][kMaxRouteExperts];  // slots before the chunk, and after it
  int part[kPlaceWaves];
};

// chunk `chunk` of the slots, by kPlaceThreads threads
__device__ __forceinline__ void place(const DispatchArgs& a, int chunk, PlaceShared& s) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, E = a.experts;
  const int first = chunk * kChunk, mine0 = first + wave * kPerWave;
  for (int i = tid; i < kPlaceWaves * kMaxRouteExperts; i += kPlaceThreads) s.at[0][i] = 0;
  for (int i = tid; i < 2 * kCopies * kMaxRouteExperts; i += kPlaceThreads) s.other[0][0][i] = 0;
  __syncthreads();
  int mine[kPerWave / 64];
#pragma unroll
  for (int i = 0; i < kPerWave / 64; i++) mine[i] = expert_of(a, mine0 + i * 64 + lane);
  if (a.hist) {
    const int chunks = (a.n + kChunk - 1) / kChunk;
    if (tid < E)
      for (int c = 0; c < chunks; c++)
        if (c != chunk) s.other[c > chunk][0][tid] += a.hist[(size_t)c * E + tid];
  } else {
    // eight loads at a time; the lanes' counts are spread over copies, since lanes
    // that add to one word take turns
    constexpr int kAhead = 8;
    int* copy = s.other[0][tid & (kCopies - 1)];
    for (int i0 = tid; i0 < a.n; i0 += kAhead * kPlaceThreads) {
      int e[kAhead];
#pragma unroll
      for (int u = 0; u < kAhead; u++) e[u] = expert_of(a, i0 + u * kPlaceThreads);
#pragma unroll
      for (int u = 0; u < kAhead; u++) {
        const int c = (i0 + u * kPlaceThreads) / kChunk;
        if (e[u] >= 0 && c != chunk) atomicAdd(copy + (c > chunk ? kCopies * kMaxRouteExperts : 0) + e[u], 1);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < kPerWave / 64; i++)
    if (mine[i] >= 0) atomicAdd(&s.at[wave][mine[i]], 1);
  __syncthreads();
  int own = 0, before = 0, all = 0;
  if (tid < E) {
#pragma unroll
    for (int w = 0; w < kPlaceWaves; w++) own += s.at[w][tid];
    all = own;
#pragma unroll
    for (int c = 0; c < kCopies; c++) {
      before += s.other[0][c][tid];
      all += s.other[0][c][tid] + s.other[1][c][tid];
    }
  }
  const int start = scan_all(all, s.part) - all;
  if (chunk == 0) {
    if (tid < E) a.counts[tid] = all;
    if (a.tiles) {
      const int tiles = (all + a.tile_rows - 1) / a.tile_rows, end = scan_all(tiles, s.part);
      if (tid == kPlaceThreads - 1) *a.n_tiles = end;
      for (int i = 0; i < tiles; i++)
        a.tiles[end - tiles + i] = RowTile{tid, start + i * a.tile_rows, min(a.tile_rows, all - i * a.tile_rows), 0};
    }
  }
  if (tid < E) {
    int row = start + before;
#pragma unroll
    for (int w = 0; w < kPlaceWaves; w++) {
      const int c = s.at[w][tid];
      s.at[w][tid] = row;
      row += c;
    }
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kPerWave / 64; i++) {
    const int slot = mine0 + i * 64 + lane, e = mine[i];
    uint64_t same = __ballot(e >= 0);
#pragma unroll
    for (int b = 0; b < 9; b++) {
      const uint64_t m = __ballot((e >> b) & 1);
      same &= (e >> b) & 1 ? m : ~m;
    }
    int row = -1;
    if (e >= 0) {
      // the lowest of the lanes takes their rows; a wave's LDS operations keep
      // their order
      const int lead = __builtin_ctzll(same);
      int base = 0;
      if (lane == lead) base = atomicAdd(&s.at[wave][e], (int)__builtin_popcountll(same));
      row = __shfl(base, lead) + (int)__builtin_popcountll(same & ((1ull << lane) - 1));
      if (a.src) a.src[row] = slot;
    }
    if (slot < a.n) a.rows[slot] = row;
  }
}

__global__ __launch_bounds__(kPlaceThreads) void k_place(DispatchArgs a) {
  __shared__ PlaceShared s;
  place(a, blockIdx.x, s);
}

// The experts' order and the quantized rows of x, side by side in one launch.
template <int DT>
__global__ __launch_bounds__(kPlaceThreads) void k_prepare(DispatchArgs a, int chunks, const void* x, int rows, int k, uint8_t* q,
                                                           float* scales) {
  __shared__ PlaceShared s;
  if ((int)blockIdx.x < chunks) return place(a, blockIdx.x, s);
  // 64 blocks, those of neighbouring rows first
  const uint32_t at = (blockIdx.x - chunks) * (kPlaceThreads / 16) + (threadIdx.x >> 4);
  const int kb = (int)(at / (uint32_t)rows), row = (int)(at % (uint32_t)rows);
  if (kb * kQBlock < k) quantize_block<DT>(x, rows, k, q, scales, row, kb);
}

// 16 bytes at any even address, or the `left` that a row still has.
__device__ __forceinline__ void load16(const uint8_t* p, size_t left, v4i& v) {
  if (left >= 16) {
    __builtin_memcpy(&v, p, 16);
    return;
  }
  uint16_t h[8];
#pragma unroll
  for (int u = 0; u < 8; u++) h[u] = (size_t)u * 2 < left ? reinterpret_cast<const uint16_t*>(p)[u] : (uint16_t)0;
  __builtin_memcpy(&v, h, 16);
}
__device__ __forceinline__ void store16(uint8_t* p, size_t left, const v4i& v) {
  if (left >= 16) {
    __builtin_memcpy(p, &v, 16);
    return;
  }
  uint16_t h[8];
  __builtin_memcpy(h, &v, 16);
#pragma unroll
  for (int u = 0; u < 8; u++)
    if ((size_t)u * 2 < left) reinterpret_cast<uint16_t*>(p)[u] = h[u];
}

// A small batch's order and its rows in one launch: every token's workgroup
// counts the slots before its own by itself, one ballot for 64 ids and a slot.
// 64 tokens of 8 x 7168 f16: 9.6 us in two launches -> 6.1.
constexpr int kMaxSmall = 4096;

__global__ __launch_bounds__(256) void k_dispatch_small(DispatchArgs a, int topk, const uint8_t* x, uint8_t* xs, size_t row_bytes) {
  __shared__ int ids[kMaxSmall];
  __shared__ int part[4][64];
  __shared__ int h[kMaxRouteExperts];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, t = blockIdx.x;
  const size_t at0 = ((size_t)blockIdx.y * 256 + tid) * 16;
  v4i first = {0, 0, 0, 0};  // on its way while the rows are found
  if (at0 < row_bytes) load16(x + (size_t)t * row_bytes + at0, row_bytes - at0, first);
  for (int i = tid; i < a.n; i += 256) ids[i] = expert_of(a, i);
  const bool counts = t == 0 && blockIdx.y == 0;
  if (counts)
    for (int e = tid; e < a.experts; e += 256) h[e] = 0;
  __syncthreads();
  for (int s = 0; s < topk; s++) {
    const int at = t * topk + s, e = ids[at];
    int before = 0;
    for (int i = wave * 64; i < a.n; i += 256) {
      const int o = i + lane, v = o < a.n ? ids[o] : -1;
      before += (int)__builtin_popcountll(__ballot(v >= 0 && (v < e || (v == e && o < at))));
    }
    if (lane == 0) part[wave][s] = before;
  }
  if (counts)
    for (int i = tid; i < a.n; i += 256)
      if (ids[i] >= 0) atomicAdd(&h[ids[i]], 1);
  __syncthreads();
  if (counts)
    for (int e = tid; e < a.experts; e += 256) a.counts[e] = h[e];
  if (tid < topk) {
    const int row = ids[t * topk + tid] < 0 ? -1 : part[0][tid] + part[1][tid] + part[2][tid] + part[3][tid];
    part[0][tid] = row;
    if (blockIdx.y == 0) a.rows[t * topk + tid] = row;
  }
  __syncthreads();
  for (size_t i = at0; i < row_bytes; i += gridDim.y * 4096) {
    v4i v = first;
    if (i != at0) load16(x + (size_t)t * row_bytes + i, row_bytes - i, v);
    for (int s = 0; s < topk; s++) {
      const int r = part[0][s];
      if (r >= 0) store16(xs + (size_t)r * row_bytes + i, row_bytes - i, v);
    }
  }
}

// ---- rows out and back ---------------------------------------------------------------
__global__ __launch_bounds__(256) void k_gather(const uint8_t* x, const int32_t* rows, uint8_t* xs, int topk, size_t row_bytes) {
  const int t = blockIdx.x;
  const size_t i = ((size_t)blockIdx.y * 256 + threadIdx.x) * 16;
  if (i >= row_bytes) return;
  v4i v;
  load16(x + (size_t)t * row_bytes + i, row_bytes - i, v);
  for (int s = 0; s < topk; s++) {
    const int r = rows[(size_t)t * topk + s];
    if (r >= 0) store16(xs + (size_t)r * row_bytes + i, row_bytes - i, v);
  }
}

// 8 values a thread, at any address: rows of an odd length start anywhere (6276
// tokens of 5 x 1055 bf16: 50.7 us one by one -> 30.2).
template <int YT, int OT>
__global__ __launch_bounds__(256) void k_combine(CombineArgs a) {
  const int t = blockIdx.x, i = (blockIdx.y * 256 + threadIdx.x) * 8, left = a.hidden - i;
  if (left <= 0) return;
  float sum[8];
#pragma unroll
  for (int u = 0; u < 8; u++) sum[u] = 0.0f;
  if (a.add) load_some_as_f32<OT>(a.add, (size_t)t * a.hidden + i, left, sum);
  for (int s = 0; s < a.topk; s++) {
    const size_t at = (size_t)t * a.topk + s;
    const int r = a.rows ? a.rows[at] : (unsigned)a.ids[at] < (unsigned)a.experts ? (int)at : -1;
    if (r < 0) continue;
    const float w = a.weights[at];
    float y[8];
    load_some_as_f32<YT>(a.y, (size_t)r * a.hidden + i, left, y);
#pragma unroll
    for (int u = 0; u < 8; u++) sum[u] += w * y[u];
  }
  store_some_from_f32<OT>(a.out, (size_t)t * a.hidden + i, left, sum);
}

template <int YT, int OT>
hipError_t combine_dt(const CombineArgs& a, hipStream_t st) {
  const unsigned parts = ((unsigned)a.hidden + 2047) / 2048;
  for (int t = 0; t < a.tokens; t += kMostTokens) {
    CombineArgs p = a;
    p.tokens = a.tokens - t < kMostTokens ? a.tokens - t : kMostTokens;
    const size_t slot = (size_t)t * a.topk, out = (size_t)t * a.hidden * dtype_size(OT);
    if (a.rows) p.rows += slot;  // (without, the slots of one token)
    p.weights += slot;
    p.out = static_cast<uint8_t*>(a.out) + out;
    if (a.add) p.add = static_cast<const uint8_t*>(a.add) + out;
    hipLaunchKernelGGL((k_combine<YT, OT>), dim3(p.tokens, parts), dim3(256), 0, st, p);
    if (hipError_t e = hipGetLastError()) return e;
  }
  return hipSuccess;
}

template <int YT>
hipError_t combine_y(int out_dtype, const CombineArgs& a, hipStream_t st) {
  switch (out_dtype) {
    case MX_DTYPE_F32: return combine_dt<YT, MX_DTYPE_F32>(a, st);
    case MX_DTYPE_F16: return combine_dt<YT, MX_DTYPE_F16>(a, st);
    case MX_DTYPE_BF16: return combine_dt<YT, MX_DTYPE_BF16>(a, st);
  }
  return hipErrorInvalidValue;
}

}  // namespace

static hipError_t route_part(int dtype, const RouteArgs& a, hipStream_t st) {
  switch (dtype) {
    case MX_DTYPE_F32: return route_dt<MX_DTYPE_F32>(a, st);
    case MX_DTYPE_F16: return route_dt<MX_DTYPE_F16>(a, st);
    case MX_DTYPE_BF16: return route_dt<MX_DTYPE_BF16>(a, st);
  }
  return hipErrorInvalidValue;
}

hipError_t launch_route(int dtype, const RouteArgs& a, hipStream_t st) {
  for (int t = 0; t < a.tokens; t += kMostTokens) {
    RouteArgs p = a;
    p.tokens = a.tokens - t < kMostTokens ? a.tokens - t : kMostTokens;
    p.logits = static_cast<const uint8_t*>(a.logits) + (size_t)t * a.stride * dtype_size(dtype);
    p.ids += (size_t)t * a.topk;
    p.weights += (size_t)t * a.topk;
    if (hipError_t e = route_part(dtype, p, st)) return e;
  }
  return hipSuccess;
}

static int chunks_of(int n) { return n > 0 ? (n + kChunk - 1) / kChunk : 1; }
size_t dispatch_ws_bytes(int n, int experts) { return n > kMaxCounted ? (size_t)chunks_of(n) * experts * 4 : 0; }

static hipError_t count_many(DispatchArgs& a, hipStream_t st) {
  if (a.n <= kMaxCounted) {
    a.hist = nullptr;
    return hipSuccess;
  }
  hipLaunchKernelGGL(k_count, dim3(chunks_of(a.n)), dim3(kPlaceThreads), 0, st, a);
  return hipGetLastError();
}

hipError_t launch_dispatch(const DispatchArgs& a0, hipStream_t st) {
  DispatchArgs a = a0;
  if (hipError_t e = count_many(a, st)) return e;
  hipLaunchKernelGGL(k_place, dim3(chunks_of(a.n)), dim3(kPlaceThreads), 0, st, a);
  return hipGetLastError();
}

hipError_t launch_prepare(const DispatchArgs& a0, int dtype, const void* x, int rows, int k, uint8_t* q, float* scales,
                          hipStream_t st) {
  DispatchArgs a = a0;
  if (hipError_t e = count_many(a, st)) return e;
  const int chunks = chunks_of(a.n);
  const long groups = (long)rows * ((k + kQBlock - 1) / kQBlock), per = kPlaceThreads / 16;
  if (groups > 0x7fffffffL) return hipErrorInvalidValue;
  const dim3 grid((unsigned)(chunks + (groups + per - 1) / per));
  if (dtype == MX_DTYPE_F16) hipLaunchKernelGGL((k_prepare<MX_DTYPE_F16>), grid, dim3(kPlaceThreads), 0, st, a, chunks, x, rows, k, q, scales);
  else hipLaunchKernelGGL((k_prepare<MX_DTYPE_BF16>), grid, dim3(kPlaceThreads), 0, st, a, chunks, x, rows, k, q, scales);
  return hipGetLastError();
}

hipError_t launch_dispatch_rows(const DispatchArgs& a, int topk, const void* x, void* xs, size_t row_bytes, hipStream_t st) {
  const int tokens = a.n / topk;
  const bool small = a.n <= kMaxSmall && (long)a.n * topk <= 8 * kMaxSmall;
  if (!small)
    if (hipError_t e = launch_dispatch(a, st)) return e;
  const uint8_t* from = static_cast<const uint8_t*>(x);
  uint8_t* to = static_cast<uint8_t*>(xs);
  const unsigned parts = (unsigned)((row_bytes + 4095) / 4096);
  // (in one launch few tokens' rows are split over workgroups, many's are not: each
  // counts the slots for itself)
  if (small) {
    hipLaunchKernelGGL(k_dispatch_small, dim3(tokens, tokens >= 256 ? 1 : parts), dim3(256), 0, st, a, topk, from, to, row_bytes);
    return hipGetLastError();
  }
  for (int t = 0; t < tokens; t += kMostTokens) {
    hipLaunchKernelGGL(k_gather, dim3(tokens - t < kMostTokens ? tokens - t : kMostTokens, parts), dim3(256), 0, st,
                       from + (size_t)t * row_bytes, a.rows + (size_t)t * topk, to, topk, row_bytes);
    if (hipError_t e = hipGetLastError()) return e;
  }
  return hipSuccess;
}

hipError_t launch_combine(int y_dtype, int out_dtype, const CombineArgs& a, hipStream_t st) {
  switch (y_dtype) {
    case MX_DTYPE_F32: return combine_y<MX_DTYPE_F32>(out_dtype, a, st);
    case MX_DTYPE_F16: return combine_y<MX_DTYPE_F16>(out_dtype, a, st);
    case MX_DTYPE_BF16: return combine_y<MX_DTYPE_BF16>(out_dtype, a, st);
  }
  return hipErrorInvalidValue;
}

}  // namespace mx
