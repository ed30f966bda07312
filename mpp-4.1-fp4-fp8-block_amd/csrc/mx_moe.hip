// mx_moe.hip - the router of a mixture of experts, and the exchange of rows
// between token order and expert order.
#include "mx_block.h"
#include "mx_convert.h"
#include "mx_device.h"

namespace mx {
namespace {

// ---- router ---------------------------------------------------------------------
//
//   p = softmax(l) or 1 / (1 + e^-l), key = p + b, the best groups, the best k
//   keys; weight = p (/ the sum of the chosen p) * scale
//
// One wave a token, expert j * 64 + lane in register j.  The sum of a softmax is
// taken in f64 and rounded once, so that keys, and with them the choice, do not
// depend on the order of the sum.
__device__ __forceinline__ uint32_t ordered(float f) {
  const uint32_t u = __builtin_bit_cast(uint32_t, f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

template <int DT, int NP>
__global__ __launch_bounds__(256) void k_route(RouteArgs a) {
  __shared__ float keys[4][NP * 64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int t = blockIdx.x * 4 + wave;
  if (t >= a.tokens) return;
  const float kLow = -__builtin_inff(), kTop = 3.402823466e38f;
  const int E = a.experts;
  float v[NP], p[NP], key[NP];
  float top = -kTop;
#pragma unroll
  for (int j = 0; j < NP; j++) {
    const int e = j * 64 + lane;
    v[j] = e < E ? load_as_f32<DT>(a.logits, (size_t)t * a.stride + e) : kLow;
    if (!(v[j] > kLow)) v[j] = kLow;  // NaN: masked
    v[j] = fminf(v[j], kTop);
    top = fmaxf(top, v[j]);
  }
  if (a.sigmoid) {
#pragma unroll
    for (int j = 0; j < NP; j++) p[j] = 1.0f / (1.0f + expf(-v[j]));
  } else {
#pragma unroll
    for (int o = 32; o; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
    double sum = 0.0;
#pragma unroll
    for (int j = 0; j < NP; j++) {
      p[j] = v[j] > kLow ? expf(v[j] - top) : 0.0f;
      sum += (double)p[j];
    }
#pragma unroll
    for (int o = 32; o; o >>= 1) sum += __shfl_xor(sum, o);
    const float s = (float)sum;
#pragma unroll
    for (int j = 0; j < NP; j++) p[j] = p[j] / s;
  }
#pragma unroll
  for (int j = 0; j < NP; j++) {
    const int e = j * 64 + lane;
    key[j] = a.bias && e < E ? p[j] + a.bias[e] : p[j];
    if (!(v[j] > kLow) || !(key[j] > kLow)) key[j] = kLow;
  }
  if (a.groups > 1) {
    const int size = E / a.groups;
#pragma unroll
    for (int j = 0; j < NP; j++) keys[wave][j * 64 + lane] = key[j];
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    float b0 = kLow, b1 = kLow;
    if (lane < a.groups)
      for (int i = 0; i < size; i++) {
        const float k = keys[wave][lane * size + i];
        b1 = fmaxf(b1, fminf(k, b0));
        b0 = fmaxf(b0, k);
      }
    const float score = a.group_top == 2 && b1 > kLow ? b0 + b1 : b0;
    int rank = 0;
    for (int i = 0; i < a.groups; i++) {
      const float s = __shfl(score, i);
      rank += s > score || (s == score && i < lane);
    }
    const uint64_t kept = __ballot(lane < a.groups && rank < a.topk_groups);
#pragma unroll
    for (int j = 0; j < NP; j++) {
      const int e = j * 64 + lane;
      if (e < E && !((kept >> (e / size)) & 1)) key[j] = kLow;
    }
  }
  // best first; the lower index wins a tie
  float mine = 0.0f, total = 0.0f;
  int id = -1;
  for (int s = 0; s < a.topk; s++) {
    uint64_t best = 0;
#pragma unroll
    for (int j = 0; j < NP; j++) {
      const uint64_t c = key[j] > kLow ? (uint64_t)ordered(key[j]) << 32 | (uint32_t)(0xffff - (j * 64 + lane)) : 0;
      best = c > best ? c : best;
    }
#pragma unroll
    for (int o = 32; o; o >>= 1) {
      const uint64_t c = __shfl_xor((unsigned long long)best, o);
      best = c > best ? c : best;
    }
    if (!best) break;
    const int e = 0xffff - (int)(best & 0xffffffffu);
    float w = 0.0f;
#pragma unroll
    for (int j = 0; j < NP; j++)
      if (j == e >> 6) w = p[j];
    w = __shfl(w, e & 63);
#pragma unroll
    for (int j = 0; j < NP; j++)
      if (j * 64 + lane == e) key[j] = kLow;
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
// A stable counting sort of the slots by expert, in chunks of kChunk slots: the
// chunks' histograms, then every chunk adds up those before it and gives its
// slots their rows.  A wave finds the slots of one expert among its 64 by nine
// ballots, one a bit; only integer counts are added by atomics, so the order
// of the rows is the slots'.
constexpr int kChunk = 2048, kPerWave = kChunk / 4;

__device__ __forceinline__ int expert_of(const DispatchArgs& a, int i) {
  const int e = i < a.n ? a.ids[i] : -1;
  return (unsigned)e < (unsigned)a.experts ? e : -1;
}

__global__ __launch_bounds__(256) void k_count(DispatchArgs a) {
  __shared__ int h[kMaxRouteExperts];
  for (int e = threadIdx.x; e < a.experts; e += 256) h[e] = 0;
  __syncthreads();
  for (int i = threadIdx.x; i < kChunk; i += 256) {
    const int e = expert_of(a, blockIdx.x * kChunk + i);
    if (e >= 0) atomicAdd(&h[e], 1);
  }
  __syncthreads();
  for (int e = threadIdx.x; e < a.experts; e += 256) a.hist[(size_t)blockIdx.x * a.experts + e] = h[e];
}

// inclusive prefix sums of v over the workgroup's 256 threads
__device__ __forceinline__ int scan256(int v, int* part) {
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

__global__ __launch_bounds__(256) void k_place(DispatchArgs a, int chunks) {
  __shared__ int at[4][kMaxRouteExperts];   // next row of an expert, by wave
  __shared__ int part[4];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, E = a.experts;
  const int first = blockIdx.x * kChunk + wave * kPerWave;
  for (int i = tid; i < 4 * kMaxRouteExperts; i += 256) at[0][i] = 0;
  __syncthreads();
  int mine[kPerWave / 64];
#pragma unroll
  for (int i = 0; i < kPerWave / 64; i++) {
    mine[i] = expert_of(a, first + i * 64 + lane);
    if (mine[i] >= 0) atomicAdd(&at[wave][mine[i]], 1);
  }
  __syncthreads();
  // experts 2 tid and 2 tid + 1
  int before[2] = {0, 0}, all[2] = {0, 0};
#pragma unroll
  for (int u = 0; u < 2; u++) {
    const int e = 2 * tid + u;
    if (e >= E) continue;
    if (chunks == 1) {
      all[u] = at[0][e] + at[1][e] + at[2][e] + at[3][e];
    } else {
      for (int c = 0; c < chunks; c++) {
        const int h = a.hist[(size_t)c * E + e];
        all[u] += h;
        if (c < (int)blockIdx.x) before[u] += h;
      }
    }
  }
  const int incl = scan256(all[0] + all[1], part);
  const int start[2] = {incl - all[0] - all[1], incl - all[1]};
  if (blockIdx.x == 0) {
    int tiles[2] = {0, 0};
#pragma unroll
    for (int u = 0; u < 2; u++)
      if (2 * tid + u < E) {
        a.counts[2 * tid + u] = all[u];
        if (a.tiles) tiles[u] = (all[u] + a.tile_rows - 1) / a.tile_rows;
      }
    if (a.tiles) {
      const int ti = scan256(tiles[0] + tiles[1], part);
      if (tid == 255) *a.n_tiles = ti;
      int next = ti - tiles[0] - tiles[1];
#pragma unroll
      for (int u = 0; u < 2; u++)
        for (int i = 0; i < tiles[u]; i++)
          a.tiles[next++] = RowTile{2 * tid + u, start[u] + i * a.tile_rows, min(a.tile_rows, all[u] - i * a.tile_rows), 0};
    }
  }
#pragma unroll
  for (int u = 0; u < 2; u++) {
    const int e = 2 * tid + u;
    if (e >= E) continue;
    int row = start[u] + before[u];
#pragma unroll
    for (int w = 0; w < 4; w++) {
      const int c = at[w][e];
      at[w][e] = row;
      row += c;
    }
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kPerWave / 64; i++) {
    const int slot = first + i * 64 + lane, e = mine[i];
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
      if (lane == lead) base = atomicAdd(&at[wave][e], (int)__builtin_popcountll(same));
      row = __shfl(base, lead) + (int)__builtin_popcountll(same & ((1ull << lane) - 1));
      if (a.src) a.src[row] = slot;
    }
    if (slot < a.n) a.rows[slot] = row;
  }
}

// ---- rows out and back ---------------------------------------------------------------
template <typename V>
__global__ __launch_bounds__(256) void k_gather(const V* x, const int32_t* rows, V* xs, int topk, int len) {
  const int t = blockIdx.x, i = blockIdx.y * 256 + threadIdx.x;
  if (i >= len) return;
  const V v = x[(size_t)t * len + i];
  for (int s = 0; s < topk; s++) {
    const int r = rows[(size_t)t * topk + s];
    if (r >= 0) xs[(size_t)r * len + i] = v;
  }
}

template <int YT, int OT, int N>
__global__ __launch_bounds__(256) void k_combine(CombineArgs a) {
  const int t = blockIdx.x, i = (blockIdx.y * 256 + threadIdx.x) * N;
  if (i >= a.hidden) return;
  float sum[N];
  if (a.add) load_n_as_f32<OT, N>(a.add, (size_t)t * a.hidden + i, sum);
  else {
#pragma unroll
    for (int u = 0; u < N; u++) sum[u] = 0.0f;
  }
  for (int s = 0; s < a.topk; s++) {
    const int r = a.rows[(size_t)t * a.topk + s];
    if (r < 0) continue;
    const float w = a.weights[(size_t)t * a.topk + s];
    float y[N];
    load_n_as_f32<YT, N>(a.y, (size_t)r * a.hidden + i, y);
#pragma unroll
    for (int u = 0; u < N; u++) sum[u] += w * y[u];
  }
  store_n_from_f32<OT, N>(a.out, (size_t)t * a.hidden + i, sum);
}

template <int YT, int OT>
hipError_t combine_dt(const CombineArgs& a, hipStream_t st) {
  const uintptr_t p = reinterpret_cast<uintptr_t>(a.y) | reinterpret_cast<uintptr_t>(a.add) | reinterpret_cast<uintptr_t>(a.out);
  if (a.hidden % 8 == 0 && p % 16 == 0)
    hipLaunchKernelGGL((k_combine<YT, OT, 8>), dim3(a.tokens, (a.hidden + 2047) / 2048), dim3(256), 0, st, a);
  else
    hipLaunchKernelGGL((k_combine<YT, OT, 1>), dim3(a.tokens, (a.hidden + 255) / 256), dim3(256), 0, st, a);
  return hipGetLastError();
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

hipError_t launch_route(int dtype, const RouteArgs& a, hipStream_t st) {
  switch (dtype) {
    case MX_DTYPE_F32: return route_dt<MX_DTYPE_F32>(a, st);
    case MX_DTYPE_F16: return route_dt<MX_DTYPE_F16>(a, st);
    case MX_DTYPE_BF16: return route_dt<MX_DTYPE_BF16>(a, st);
  }
  return hipErrorInvalidValue;
}

static int chunks_of(int n) { return (n + kChunk - 1) / kChunk; }
size_t dispatch_ws_bytes(int n, int experts) { return chunks_of(n) > 1 ? (size_t)chunks_of(n) * experts * 4 : 0; }

hipError_t launch_dispatch(const DispatchArgs& a, hipStream_t st) {
  const int chunks = chunks_of(a.n);
  if (chunks > 1) hipLaunchKernelGGL(k_count, dim3(chunks), dim3(256), 0, st, a);
  hipLaunchKernelGGL(k_place, dim3(chunks > 0 ? chunks : 1), dim3(256), 0, st, a, chunks > 0 ? chunks : 1);
  return hipGetLastError();
}

hipError_t launch_gather(const void* x, const int32_t* rows, void* xs, int tokens, int topk, size_t row_bytes,
                         hipStream_t st) {
  const uintptr_t p = reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(xs);
  auto go = [&](auto v) {
    using V = decltype(v);
    const int len = (int)(row_bytes / sizeof(V));
    hipLaunchKernelGGL((k_gather<V>), dim3(tokens, (len + 255) / 256), dim3(256), 0, st, static_cast<const V*>(x), rows,
                       static_cast<V*>(xs), topk, len);
  };
  if (row_bytes % 16 == 0 && p % 16 == 0) go(v4i{});
  else if (row_bytes % 4 == 0 && p % 4 == 0) go(uint32_t{});
  else go(uint16_t{});
  return hipGetLastError();
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
