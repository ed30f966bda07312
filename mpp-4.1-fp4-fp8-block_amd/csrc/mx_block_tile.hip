// mx_block_tile.hip - tile products of block-scaled FP8 matrices.
//
//   C[m][n] = sum_kb a_s[kb][m] w_s[n / 128][kb] sum_{k in kb} A[m][k] W[n][k]
//
// A stage is one 128-block of K: its sum comes from one MFMA of 16 x 16 x 128 with
// unit scales and is added, times the two block scales, in f32.  Weight rows are
// the MFMA's rows and activation rows its columns, so that a lane has one
// activation scale and one weight scale for its four sums, which are neighbouring
// outputs: 4 FMAs for each MFMA, issued beneath it.
//
// Bound of the 256 x 256 tiles: the matrix cores and the work beside them, which
// the clock pays for too.  By counters 8192^3 takes 455 to 467 us with the cores busy
// 60 % of it at 1.9 to 2.0 GHz (2.4 without products), 4096 rows of 4096 -> 14336 231
// us (2.1 PFLOP/s; library products of 8192^3 with one scale 2.6) and 49 % at 2.0.
// Beside the MFMAs are
//   L2 -> LDS    64 KB a stage for 8.4 MFLOP; an XCD's CUs take neighbouring tiles
//                (loads of 8192^3 without products 371 -> 297 us)
//   LDS read     24 KB a wave and stage, without bank conflicts
//   waits        one barrier a stage, with the loads, the scaling and the next
//                stage's fragments spread over the products
// (the three together 280 -> 255 us for the 4096 rows).  Where K is short a tile's
// ends count more than the clock: experts' rows of 2048 -> 7168 keep the cores busy
// 31 % at 2.3 GHz.  Workgroups that go on to a next tile over the end of their last
// one gain 2 % there (665 -> 654 us), less in gate/up (1098 -> 1091, where SwiGLU then
// spills 30 registers) and nothing for the 4096 rows (246.6 -> 246.9): not kept.
//
// The cores align eight neighbouring products to the largest and cut what lies
// 2^-13 below its power of two, before they add in f32: about 1.3e-5 of a sum of
// normally distributed values, far below a 16-bit result's rounding and the
// format's own 2^-4.  f32 results, and the sums before SwiGLU on 64-row tiles, whose
// time is the weights' way from HBM, widen the codes to f16 instead (WIDE), whose
// products add in f32: about 1e-7 of the sum, for half the rate.  A product that
// adds to the one before it starts 54 cycles after it, where one that does not
// starts after 16: four sums are kept going at once (1024 rows of 8192 -> 2048 to
// f32: 60 -> 56 us).
#include <type_traits>

#include "mx_block.h"
#include "mx_block_device.h"
#include "mx_convert.h"
#include "mx_device.h"
#include "mx_dma.h"
#include "mx_widen.h"

namespace mx {
namespace {

constexpr int kCUs = 256;           // of an MI355X, 32 in each of 8 XCDs
constexpr int kPast = 0x7fffff00;  // past every resource's range
constexpr int lgkm0_vm(int n) { return (n & 15) | ((n >> 4) << 14) | (7 << 4); }
// The resource from `offset` bytes on, of those that it has.  (An instruction's scalar
// offset would not be checked against the range.)
__device__ __forceinline__ v4i rsrc_from(v4i rsrc, int offset) {
  const uint64_t a = ((uint64_t)(uint32_t)rsrc[1] << 32 | (uint32_t)rsrc[0]) + (uint32_t)offset;
  return v4i{(int)(uint32_t)a, (int)(uint32_t)(a >> 32), rsrc[2] - offset, rsrc[3]};
}
__device__ __forceinline__ void dma4(const void* src, void* lds) { __builtin_amdgcn_global_load_lds(src, lds, 4, 0, 0); }

// The 64 banks hold two rows of 128 bytes.  A 16-byte read takes its lanes in
// groups of 16: lanes 0-3, 12-15, 20-27 and 4-11, 16-19, 28-31, and the same 32
// on.  Lane l reads chunk 2 (l / 16) + h of row l % 16, so a group has every row
// once, rows 4 to 11 with a chunk 2 further (or nearer) than the others; with
// this key its reads go to 16 places that are all different (the counter of bank
// conflicts went from 4 a read to 0).
__device__ __forceinline__ int place_key(int r) { return (r >> 1 & 1) | (r >> 3 & 1) * 6; }

// TN weight rows (SwiGLU: TN / 2 of gate and the same of up) x TM activation
// rows, by WN x WM waves, over K (or one of g.splits parts) in stages of one
// 128-block, NS of them in LDS.  (With room for two of the waves on a SIMD the
// compiler leaves the sums out of AGPRs, which the scaling cannot read.)
template <int DT, bool DUAL, int TN, int TM, int WN, int WM, int NS, bool WIDE>
__global__ __launch_bounds__(64 * WN * WM, 2) void k_block_tile(BlockGemmArgs g) {
  constexpr int NW = WN * WM, CN = TN / WN, CM = TM / WM, NI = CN / 16, MJ = CM / 16;
  constexpr int SLOT = (TN + TM) * kQBlock, NDMA = (TN + TM) / 8 / NW, PER = NDMA + 1;
  constexpr int ND = DUAL ? 2 : 1;  // weight scales of a wave
  static_assert((TN + TM) / 8 % NW == 0 && TM % 64 == 0, "whole instructions");
  static_assert(TN / ND <= kQBlock || !DUAL, "one block of mid channels");
  __shared__ __attribute__((aligned(16))) uint8_t r0[SLOT];
  __shared__ __attribute__((aligned(16))) uint8_t r1[SLOT];
  __shared__ __attribute__((aligned(16))) uint8_t r2[NS > 2 ? SLOT : 16];
  __shared__ __attribute__((aligned(16))) float a0[TM];
  __shared__ __attribute__((aligned(16))) float a1[TM];
  __shared__ __attribute__((aligned(16))) float a2[NS > 2 ? TM : 4];
  __shared__ float wsl[2][kMaxBlocks];
  __shared__ float amax_l[DUAL ? WN : 1][DUAL ? TM : 1];

  const int NT = (g.n + TN / ND - 1) / (TN / ND), MT = g.tiles ? *g.n_tiles : (g.m + TM - 1) / TM;
  // An XCD takes a run of neighbouring tiles, 8 weight tiles by all row tiles: its
  // 32 CUs then work on about 8 weight and 4 row tiles and fetch each once.
  const int total = MT * NT * g.splits, per = (total + 7) / 8;
  int mine = blockIdx.x >> 3, half = 0;  // of the XCD's run
  // A last round for at most half of the CUs: its tiles go to two workgroups each.
  const int rest = TM == 256 ? per % (kCUs / 8) : 0;
  const bool halves = rest && rest <= kCUs / 16 && mine >= per - rest;
  if (halves) {
    half = (mine - (per - rest)) & 1;
    mine = per - rest + (mine - (per - rest)) / 2;
  }
  const int at = (blockIdx.x & 7) * per + mine;
  if (mine >= per || at >= total) return;
  const int sp = at / (MT * NT), tile = at % (MT * NT);
  const int grp = tile / (8 * MT), in = tile % (8 * MT), gw = min(8, NT - grp * 8);
  const int rt = in / gw, n0 = (grp * 8 + in % gw) * (TN / ND);
  int row0 = rt * TM, rows = min(TM, g.m - row0), expert = 0;
  if (g.tiles) {
    const RowTile t = g.tiles[rt];
    row0 = t.row0;
    rows = t.rows;
    expert = t.expert;
  }
  if (halves) {
    row0 += half * (TM / 2);
    rows = min(TM / 2, rows - half * (TM / 2));
    if (rows <= 0) return;
  }
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), wn = wave % WN, wm = wave / WN;
  // this part's blocks of K: KB from kb0 on
  const int K = g.k, KA = (K + kQBlock - 1) / kQBlock, kb0 = sp * KA / g.splits, KB = (sp + 1) * KA / g.splits - kb0;

  // their scales of the weights
  const size_t so = expert * g.s_stride;
  for (int i = tid; i < KB; i += 64 * NW) {
#pragma unroll
    for (int d = 0; d < 2; d++) {
      // SwiGLU: gate and up; else the tile's two blocks of weight rows
      const int nb = n0 / kQBlock + (DUAL ? 0 : d);
      const float* s = (DUAL && d ? g.s1 : g.s0) + so;
      wsl[d][i] = s[(size_t)min(nb, (g.n - 1) / kQBlock) * KA + kb0 + i];
    }
  }

  // DMA: an instruction moves 8 rows of 128 bytes, 16-byte chunk c of row r to
  // place c ^ place_key(r).
  // Through buffer resources of the tile's rows (of a whole batch whose rows are
  // picked), with the row in the lane's offset: what lies past them reads as zero.
  // So do chunks past K, on both sides: what lies there may be NaN.
  const int skip = kb0 * kQBlock, tail = min(kQBlock, K - skip - (KB - 1) * kQBlock) / 16;  // chunks of the last block
  const int chunk = (lane & 7) ^ place_key((wave & 1) * 8 + (lane >> 3));
  static_assert(NW % 2 == 0, "a wave's groups of 8 rows are all even or all odd");
  constexpr int TW = TN / ND, QW = TN / 8 / NW, QA = NDMA - QW;  // weight rows of a matrix; instructions of a wave
  static_assert(QW % ND == 0 && TN / 8 % NW == 0, "whole instructions");
  // wave w moves weight rows (q NW + w) 8 ..: with SwiGLU, the first half of q gate
  const uint32_t wrange = (uint32_t)min(TW, g.n - n0) * (uint32_t)K - skip;
  const size_t wo = expert * g.w_stride + (size_t)n0 * K + skip;
  const v4i wrs0 = rsrc_of<true>(g.w0 + wo, wrange), wrs1 = rsrc_of<true>((DUAL ? g.w1 : g.w0) + wo, wrange);
  constexpr int QM = QW / ND;  // instructions of a matrix
  int woff[QM];
#pragma unroll
  for (int q = 0; q < QM; q++) woff[q] = ((q * NW + wave) * 8 + (lane >> 3)) * K + chunk * 16;
  const v4i ars = rsrc_of<true>((g.src ? g.a : g.a + (size_t)row0 * K) + skip, (uint32_t)(g.src ? g.a_rows : rows) * (uint32_t)K - skip);
  int aoff[QA];
#pragma unroll
  for (int q = 0; q < QA; q++) {
    const int r = (q * NW + wave) * 8 + (lane >> 3), ra = min(r, rows - 1);
    aoff[q] = r < rows ? (g.src ? g.src[row0 + ra] / g.src_div : ra) * K + chunk * 16 : kPast;
  }
  const int srow = row0 + min((wave * 64) % TM + lane, rows - 1);
  const float* ssrc = g.a_s + (size_t)kb0 * g.a_rows + (g.src ? g.src[srow] / g.src_div : srow);
  auto slot = [&](auto u) -> uint8_t* {
    constexpr int U = decltype(u)::value % NS;
    if constexpr (U == 0) return r0;
    else if constexpr (U == 1) return r1;
    else return r2;
  };
  auto aslot = [&](auto u) -> float* {
    constexpr int U = decltype(u)::value % NS;
    if constexpr (U == 0) return a0;
    else if constexpr (U == 1) return a1;
    else return a2;
  };
  // A stage's loads in four parts, so that no wave waits long to issue them.
  constexpr int PARTS = 4;
  auto issue = [&](int k, auto u, int p) __attribute__((always_inline)) {
    uint8_t* s = slot(u);
    // (no branch: the compiler would move products past it)
    const bool zero = (k >= KB) | ((k == KB - 1) & (chunk >= tail));
    const int ko = min(k, KB - 1) * kQBlock;
#pragma unroll
    for (int q = p * QW / PARTS; q < (p + 1) * QW / PARTS; q++)
      buffer_dma16(rsrc_from(q >= QM ? wrs1 : wrs0, ko), s + (q * NW + wave) * 1024, zero ? kPast : woff[q % QM]);
#pragma unroll
    for (int q = p * QA / PARTS; q < (p + 1) * QA / PARTS; q++)
      buffer_dma16(rsrc_from(ars, ko), s + TN * 128 + (q * NW + wave) * 1024, zero ? kPast : aoff[q]);
    if (p == PARTS - 1) dma4(ssrc + (size_t)min(k, KB - 1) * g.a_rows, aslot(u) + (wave * 64) % TM);
  };
  auto issue_all = [&](int k, auto u) {
#pragma unroll
    for (int p = 0; p < PARTS; p++) issue(k, u, p);
  };

  using I0 = std::integral_constant<int, 0>;
  using I1 = std::integral_constant<int, 1>;
  using I2 = std::integral_constant<int, 2>;
  issue_all(0, I0{});
  if constexpr (NS > 2) issue_all(1, I1{});
  issue(NS - 1, std::integral_constant<int, NS - 1>{}, 0);
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_s_waitcnt(lgkm0_vm((NS - 2) * PER + QW / PARTS + QA / PARTS));
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_sched_barrier(0);
  const int wblk = DUAL ? 0 : (wn * CN) / kQBlock;

  // The rest with as many columns as have rows (the waves' registers are those of
  // the whole tile).
  auto body = [&](auto columns) __attribute__((always_inline)) {
  constexpr int MC = decltype(columns)::value;
  static_assert(MC % 2 == 0 && MC >= PARTS, "columns alternate, and hold a stage's parts");
  // fragments: lane l has bytes [32 (l / 16), +32) of row l % 16.  Wave wm takes
  // every WM-th run of 16 activation rows, so that the waves of a tile with few
  // rows are left with equally many.
  auto arow = [&](int j) { return (j * WM + wm) * 16; };
  int here = lane;
  asm volatile("" : "+v"(here));  // (a value of this body: the bodies' common parts are not worked out before them)
  const int r16 = here & 15, kq = here >> 4;
  const int sw = place_key(r16), off0 = r16 * 128 + (((2 * kq) ^ sw) << 4), off1 = r16 * 128 + (((2 * kq + 1) ^ sw) << 4);
  auto wrow = [&](int i) { return DUAL ? (i < NI / 2 ? wn * (CN / 2) + i * 16 : TN / 2 + wn * (CN / 2) + (i - NI / 2) * 16) : wn * CN + i * 16; };
  auto frag = [&](const uint8_t* s, int row) __attribute__((always_inline)) -> v8i {
    const v4i lo = *reinterpret_cast<const v4i*>(s + row * 128 + off0), hi = *reinterpret_cast<const v4i*>(s + row * 128 + off1);
    return v8i{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
  };

  v4f acc[NI][MC];
#pragma unroll
  for (int i = 0; i < NI; i++)
#pragma unroll
    for (int j = 0; j < MC; j++) acc[i][j] = v4f{0, 0, 0, 0};


  // The sums of column j are scaled and added while column j + 1 is multiplied
  // (t, sc).  Over the products of a stage's last column, past the barrier that
  // ends its reads, go the next stage's first column and weight fragments (each
  // after the last use of its registers) and the first loads into the slot; the
  // other loads over the stage's first columns.  (Columns two ahead measured the
  // same where they fit the registers, and spill here.)
  v8i wf[NI], af[2];
  v8h wh[WIDE ? NI : 1][4];
  constexpr int CH = WIDE && NI < 4 && NW == 4 ? 2 : 1;  // sums of a product's K quarters
  v4f t[NI], t1[CH > 1 ? NI : 1];
  float sc[2][ND], av[2], ws[ND];
  auto column = [&](auto u, int j) __attribute__((always_inline)) {
    af[j & 1] = frag(slot(u) + TN * 128, arow(j));
    av[j & 1] = aslot(u)[arow(j) + r16];
  };
  auto weights = [&](auto u, int i) __attribute__((always_inline)) { wf[i] = frag(slot(u), wrow(i)); };
  auto block_scales = [&](int k) {
#pragma unroll
    for (int d = 0; d < ND; d++) ws[d] = wsl[DUAL ? d : wblk][min(k, KB - 1)];
  };
  auto add = [&](int i, int j) __attribute__((always_inline)) {  // column j's sums
#pragma unroll
    for (int v = 0; v < 4; v++) acc[i][j][v] = fmaf(CH > 1 ? t[i][v] + t1[i][v] : t[i][v], sc[j & 1][DUAL && i >= NI / 2 ? 1 : 0], acc[i][j][v]);
  };
#pragma unroll
  for (int i = 0; i < NI; i++) {
    t[i] = v4f{0, 0, 0, 0};
    if (CH > 1) t1[i] = v4f{0, 0, 0, 0};
  }
#pragma unroll
  for (int d = 0; d < ND; d++) sc[1][d] = 0.0f;
  column(I0{}, 0);
  block_scales(0);
#pragma unroll
  for (int i = 0; i < NI; i++) weights(I0{}, i);

  auto stage = [&](int k, auto u) __attribute__((always_inline)) {
    constexpr int U = decltype(u)::value;
    using Next = std::integral_constant<int, (U + 1) % NS>;
    using Last = std::integral_constant<int, (U + NS - 1) % NS>;
    if constexpr (WIDE) {
#pragma unroll
      for (int i = 0; i < NI; i++) widen4(wf[i], wh[i]);
    }
#pragma unroll
    for (int j = 0; j < MC; j++) {
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int d = 0; d < ND; d++) sc[j & 1][d] = av[j & 1] * ws[d];
      if (j == MC - 1) {
        // the stage's fragments are in registers and the next stage has landed
        __builtin_amdgcn_s_waitcnt(lgkm0_vm((NS - 2) * PER));
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_sched_barrier(0);
        column(Next{}, 0);
        block_scales(k + 1);
        issue(k + NS, u, 0);
      } else {
        column(u, j + 1);
        if (j + 1 < PARTS) issue(k + NS - 1, Last{}, j + 1);
      }
      v8h xh[4];
      if constexpr (WIDE) widen4(af[j & 1], xh);
      if constexpr (WIDE) {
        // A quarter of K for all weight rows in turn, and with few of them two sums of
        // each: a product waits for the end of the one that it adds to.
#pragma unroll
        for (int q = 0; q < 4; q++)
#pragma unroll
          for (int i = 0; i < NI; i++) {
            if (q == 0) add(i, (j + MC - 1) % MC);
            v4f& sum = q % CH ? t1[i] : t[i];
            sum = mfma_f16_16x16x32(wh[i][q], xh[q], q < CH ? v4f{0, 0, 0, 0} : sum);
            if (j == MC - 1 && q == 0) weights(Next{}, i);
          }
      } else {
#pragma unroll
        for (int i = 0; i < NI; i++) {
          add(i, (j + MC - 1) % MC);
          t[i] = mfma_fp8_16x16x128(wf[i], af[j & 1]);
          if (j == MC - 1) weights(Next{}, i);
        }
      }
#pragma unroll
      for (int i = 0; i < (WIDE ? 4 : 1) * NI; i++) {
        __builtin_amdgcn_sched_group_barrier(0x2, 5, 0);
        __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
        if (j == MC - 1) __builtin_amdgcn_sched_group_barrier(0x100, 3, 0);
        else __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x20, 1, 0);
      }
    }
    __builtin_amdgcn_sched_barrier(0);
  };
  int k = 0;
  for (; k + NS <= KB; k += NS) {
    stage(k, I0{});
    stage(k + 1, I1{});
    if constexpr (NS > 2) stage(k + 2, I2{});
  }
  if (k < KB) {
    stage(k, I0{});
    if constexpr (NS > 2) {
      if (k + 1 < KB) stage(k + 1, I1{});
    }
  }
  __builtin_amdgcn_s_waitcnt(lgkm0_vm(0));
#pragma unroll
  for (int i = 0; i < NI; i++) add(i, MC - 1);
  if constexpr (DUAL) {
    // silu(gate) up, then one scale per row and its 128 channels
#pragma unroll
    for (int j = 0; j < MC; j++) {
      uint32_t amax = 0;
#pragma unroll
      for (int i = 0; i < NI / 2; i++)
#pragma unroll
        for (int v = 0; v < 4; v++) {
          const int c = n0 + wrow(i) + kq * 4 + v;
          const float x = c < g.n ? silu(acc[i][j][v]) * acc[i + NI / 2][j][v] : 0.0f;
          acc[i][j][v] = x;
          amax = max(amax, abs_bits(x));
        }
      amax = max(amax, (uint32_t)__shfl_xor((int)amax, 16));
      amax = max(amax, (uint32_t)__shfl_xor((int)amax, 32));
      if (kq == 0) amax_l[wn][arow(j) + r16] = __builtin_bit_cast(float, amax);
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < MC; j++) {
      const int r = arow(j) + r16;
      if (r >= rows) continue;
      uint32_t amax = 0;
#pragma unroll
      for (int w = 0; w < WN; w++) amax = max(amax, __builtin_bit_cast(uint32_t, amax_l[w][r]));
      const float s = block_scale(amax);
      if (wn == 0 && kq == 0) g.c_s[(size_t)(n0 / kQBlock) * g.m + row0 + r] = s;
#pragma unroll
      for (int i = 0; i < NI / 2; i++) {
        const int c = n0 + wrow(i) + kq * 4;
        if (c < g.n) *reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(g.c) + (size_t)(row0 + r) * g.n + c) = e4m3x4(acc[i][j], s);
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < MC; j++) {
      const int r = arow(j) + r16;
      if (r >= rows) continue;
#pragma unroll
      for (int i = 0; i < NI; i++) {
        const int c = n0 + wrow(i) + kq * 4;
        store4<DT>(g.c, ((size_t)sp * g.m + row0 + r) * g.n + c, acc[i][j], g.n - c);
      }
    }
  }
  };
  if constexpr (MJ == 8) {
    if (rows <= 4 * 16 * WM) return body(std::integral_constant<int, 4>{});
    if (rows <= 6 * 16 * WM) return body(std::integral_constant<int, 6>{});
  }
  body(std::integral_constant<int, MJ>{});
}

// Sums of a product's parts, in their order.
template <int DT, int N>
__global__ __launch_bounds__(256) void k_block_join(const float* part, size_t len, int splits, void* c) {
  const size_t i = ((size_t)blockIdx.x * 256 + threadIdx.x) * N;
  if (i >= len) return;
  float sum[N], v[N];
  load_n_as_f32<MX_DTYPE_F32, N>(part, i, sum);
  for (int s = 1; s < splits; s++) {
    load_n_as_f32<MX_DTYPE_F32, N>(part, s * len + i, v);
#pragma unroll
    for (int u = 0; u < N; u++) sum[u] += v[u];
  }
  store_n_from_f32<DT, N>(c, i, sum);
}

template <int DT, bool DUAL, int TN, int TM, int WN, int WM, int NS, bool WIDE>
hipError_t launch_one(const BlockGemmArgs& g, hipStream_t st) {
  const int nt = (g.n + TN / (DUAL ? 2 : 1) - 1) / (TN / (DUAL ? 2 : 1));
  const long tiles = (long)(g.tiles ? g.max_tiles : (g.m + TM - 1) / TM) * nt * g.splits;
  if (tiles > 0x7fffff00L) return hipErrorInvalidValue;
  const unsigned grid = (unsigned)((tiles + 7) / 8 * 8) + (TM == 256 ? kCUs / 2 : 0);  // (room for the halved tiles)
  hipLaunchKernelGGL((k_block_tile<DT, DUAL, TN, TM, WN, WM, NS, WIDE>), dim3(grid), dim3(64 * WN * WM), 0, st, g);
  return hipGetLastError();
}

template <int DT>
hipError_t store_tiles(const BlockGemmArgs& g, hipStream_t st) {
  // f32 results keep more bits than the FP8 matrix cores' sums hold, but for rows
  // that are rounded to 16 bits after a last sum
  constexpr bool WIDE = DT == MX_DTYPE_F32;
  if (WIDE && g.fp8_cores)
    return g.tile_rows == 256 ? launch_one<DT, false, 256, 256, 4, 2, 2, false>(g, st) : launch_one<DT, false, 128, 64, 4, 1, 3, false>(g, st);
  if constexpr (WIDE) {
    if (g.tile_rows == 128) return launch_one<DT, false, 256, 128, 4, 2, 3, true>(g, st);
  } else {
    if (g.tile_rows == 256) return launch_one<DT, false, 256, 256, 4, 2, 2, false>(g, st);
  }
  if (g.splits == 1) return launch_one<DT, false, 128, 64, 4, 1, 3, WIDE>(g, st);
  BlockGemmArgs p = g;
  p.c = g.part;
  if (hipError_t e = launch_one<MX_DTYPE_F32, false, 128, 64, 4, 1, 3, WIDE>(p, st)) return e;
  const size_t len = (size_t)g.m * g.n;
  const float* part = static_cast<const float*>(g.part);
  if (len % 8 == 0) hipLaunchKernelGGL((k_block_join<DT, 8>), dim3((unsigned)((len / 8 + 255) / 256)), dim3(256), 0, st, part, len, g.splits, g.c);
  else hipLaunchKernelGGL((k_block_join<DT, 1>), dim3((unsigned)((len + 255) / 256)), dim3(256), 0, st, part, len, g.splits, g.c);
  return hipGetLastError();
}

}  // namespace

// Parts of K for a dense product by 64-row tiles that would leave half of the CUs
// idle: about a workgroup a CU, each with four blocks at least.  The parts' sum
// costs a launch (3.5 us): 46 rows of 3968 -> 1221 17.5 us in one part and 10.4 in
// seven, 300 rows of 4096 -> 4096 (160 tiles) 19.9 in one and 19.6 in two.
int block_splits(int m, int n, int k, int tile_rows) {
  if (tile_rows != 64) return 1;
  const long tiles = (long)((m + 63) / 64) * ((n + 127) / 128);
  if (tiles >= 128) return 1;
  const long s = 256 / tiles, most = (k + kQBlock - 1) / kQBlock / 4;
  return (int)(s < most ? s : most > 1 ? most : 1);
}

// At most 256 tiles' f32 sums, and one part for every four blocks of K.
size_t block_split_bytes(int m, int n, int k) {
  const long parts = (k + kQBlock - 1) / kQBlock / 4;
  const double all = 4.0 * parts * m * n, tiles = 4.0 * 256 * 64 * 128;
  return m <= 32 || parts <= 1 ? 0 : (size_t)(all < tiles ? all : tiles);
}

hipError_t launch_block_tile(int c_dtype, const BlockGemmArgs& g, hipStream_t st) {
  if (g.w1)
    return g.tile_rows == 256 ? launch_one<MX_DTYPE_F32, true, 256, 256, 4, 2, 2, false>(g, st)
                              : launch_one<MX_DTYPE_F32, true, 256, 64, 8, 1, 3, true>(g, st);
  switch (c_dtype) {
    case MX_DTYPE_F32: return store_tiles<MX_DTYPE_F32>(g, st);
    case MX_DTYPE_F16: return store_tiles<MX_DTYPE_F16>(g, st);
    case MX_DTYPE_BF16: return store_tiles<MX_DTYPE_BF16>(g, st);
  }
  return hipErrorInvalidValue;
}

}  // namespace mx
