// Products over microscaled operands: y[M, N] = x^[M, K] . W[N, K]^T (+ s . h . B^T) (+ bias), x^ in mxfp8 or mxfp4, W in
// mxfp4, on v_mfma_scale_f32_32x32x64_f8f6f4, which multiplies the codes and applies both blocks' scales (fp32 sums).
//
// Operand order of that instruction (lane l: row l % 32, half h = l / 32), found by comparing with products in 64 bits:
//   fp4: 16 bytes, indices 32 h .. 32 h + 31 of the 64-wide step; fp8: two pieces of 16 bytes, indices 16 h .. and 32 + 16 h ..
//   scale: the byte of block h of the step, selected from a dword; result: column l % 32 of the second operand, rows
//   8 (v / 4) + 4 h + v % 4 of the first.
// The weight is the first operand, so a lane holds four consecutive outputs of one row of y.
//
// Workgroup: WM x WN waves, a wave computes TM x TN tiles of 32 x 32, k-step 128.  Codes go HBM -> LDS by direct loads of 16
// bytes per lane into a ring of three stages, scales likewise, one 16-byte piece per row and 512 contraction indices, into
// a ring of two; nothing but LDS reads and matrix instructions is left in the waves.  One barrier per step.
#include <algorithm>
#include <type_traits>

#include "group.h"
#include "mx_math.h"

namespace ttamd {
namespace {

typedef int v8i __attribute__((ext_vector_type(8)));
typedef float v16f __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4_t __attribute__((ext_vector_type(4)));

#define TT_LDS_PTR(p) ((__attribute__((address_space(3))) void*)(p))

struct MxGemmArgs {
  const uint8_t* xc;   // [M, Kp] or [M, Kp / 2]: codes of the input, rows padded to 128 elements
  const uint8_t* xp;   // its scales, [groups][M][16]
  const uint8_t* wc;   // [N, K / 2]
  const uint8_t* wp;   // [groups][N][16]
  const uint16_t* h;   // [M, ldh] or null: adapter activation
  const uint16_t* lb;  // [N, rank]
  const uint16_t* bias;
  uint16_t* y;         // [M, N]
  float* part;         // [slices][M][N] or null
  float lscale;
  int M, N, K, Kp, rank, ldh;
  int tiles_m, tiles_n, slices, steps_per_slice;  // steps of 128, a multiple of 4 per slice
};

template <int WM, int WN, int TM, int TN, bool F8>
struct MxTile {
  static constexpr int kThreads = 64 * WM * WN;
  static constexpr int BM = 32 * WM * TM, BN = 32 * WN * TN;
  static constexpr int kRowA = F8 ? 128 : 64, kRowW = 64;  // bytes of a row per step
  static constexpr int kA = BM * kRowA, kW = BN * kRowW, kStage = kA + kW;
  static constexpr int kStages = 3;
  static constexpr int kScales = (BM + BN) * 16;
  static constexpr int kRings = kStages * kStage + 2 * kScales;
  static constexpr int kLoadsA = kA / (kThreads * 16), kLoadsW = kW / (kThreads * 16);
  static constexpr int kScaleWaves = (BM + BN) / 64;  // waves' worth of scale pieces
  static constexpr int kLoadsS = (kScaleWaves + WM * WN - 1) / (WM * WN);
  static constexpr int kPitch = 64 * TN + 16;  // bytes of a row of a wave's output band in LDS
  static constexpr int kBands = WM * WN * 32 * TM * kPitch;
  static constexpr int kLds = kRings > kBands ? kRings : kBands;
  static_assert(kA % (kThreads * 16) == 0 && kW % (kThreads * 16) == 0, "whole loads");
  static_assert(kLds <= 160 * 1024, "LDS of a CU");
};

template <int WM, int WN, int TM, int TN, bool F8>
__global__ __launch_bounds__(64 * WM * WN) void mx_gemm_kernel(const MxGemmArgs g) {
#if defined(__HIP_DEVICE_COMPILE__)
  using T = MxTile<WM, WN, TM, TN, F8>;
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  const int lane = threadIdx.x & 63, l31 = lane & 31, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave % WM, wn = wave / WM;

  // workgroups go to the eight XCDs in turn: each takes a contiguous share of the tiles, in bands of eight row tiles so
  // that the tiles in flight on one XCD share rows and columns in its L2
  int tile_m, tile_n, slice;
  {
    const int tiles = g.tiles_m * g.tiles_n, total = (int)gridDim.x;
    int id = (int)blockIdx.x;
    const int q = total >> 3, rem = total & 7, xcd = id & 7, k = id >> 3;
    id = xcd * q + (xcd < rem ? xcd : rem) + k;
    slice = id / tiles;
    id -= slice * tiles;
    const int band = 8 * g.tiles_n, b = id / band, in = id - b * band;
    const int rows = g.tiles_m - 8 * b < 8 ? g.tiles_m - 8 * b : 8;
    tile_m = 8 * b + in % rows;
    tile_n = in / rows;
  }
  const int m0 = tile_m * T::BM, n0 = tile_n * T::BN;
  const int nk_all = g.Kp >> 7;
  const int k_begin = slice * g.steps_per_slice;
  const int k_end = k_begin + g.steps_per_slice < nk_all ? k_begin + g.steps_per_slice : nk_all;

  // ---- sources of the direct loads.  A stage's rows lie in LDS one after the other; the 16-byte pieces of a row are
  //      permuted by the row (on the address side) so that the 32 rows a wave reads at one piece index spread over the banks
  const uint32_t lds0 = (uint32_t)(uintptr_t)TT_LDS_PTR(smem);
  const int ldx = F8 ? g.Kp : g.Kp >> 1, ldw = g.K >> 1;
  const char* const xbase = reinterpret_cast<const char*>(g.xc) + (int64_t)m0 * ldx;
  const char* const wbase = reinterpret_cast<const char*>(g.wc) + (int64_t)n0 * ldw;
  uint32_t a_off[T::kLoadsA], w_off[T::kLoadsW], w_over[T::kLoadsW];
#pragma unroll
  for (int i = 0; i < T::kLoadsA; ++i) {
    const int slot = (wave * T::kLoadsA + i) * 64 + lane;  // 16-byte slot of the stage
    const int row = F8 ? slot >> 3 : slot >> 2;
    const int piece = F8 ? (slot & 7) ^ ((row >> 1) & 7) : (slot & 3) ^ ((row >> 2) & 3);
    const int r = m0 + row < g.M ? row : g.M - 1 - m0;
    a_off[i] = (uint32_t)r * (uint32_t)ldx + 16u * piece;
  }
  // the weight's rows are not padded: in a last step that reaches past their end the piece before it is read instead
  // (the input's codes are zero there)
#pragma unroll
  for (int i = 0; i < T::kLoadsW; ++i) {
    const int slot = (wave * T::kLoadsW + i) * 64 + lane;
    const int row = slot >> 2, piece = (slot & 3) ^ ((row >> 2) & 3);
    const int r = n0 + row < g.N ? row : g.N - 1 - n0;
    w_off[i] = (uint32_t)r * (uint32_t)ldw + 16u * piece;
    const int end = (nk_all - 1) * 64 + 16 * piece + 16;
    w_over[i] = end > ldw ? (uint32_t)(end - ldw) : 0u;
  }
  // scale pieces: wave w loads rows [64 w, + 64) of the tile's BM input rows and BN weight rows, in rounds of all waves
  const char* s_src[T::kLoadsS];
  int64_t s_step[T::kLoadsS];
  bool s_mine[T::kLoadsS];
#pragma unroll
  for (int i = 0; i < T::kLoadsS; ++i) {
    const int sw = wave + i * WM * WN, row = sw * 64 + lane;
    s_mine[i] = sw < T::kScaleWaves;
    if (sw * 64 < T::BM) {
      const int r = m0 + row < g.M ? m0 + row : g.M - 1;
      s_src[i] = reinterpret_cast<const char*>(g.xp) + (int64_t)r * 16;
      s_step[i] = (int64_t)g.M * 16;
    } else {
      const int r = n0 + row - T::BM < g.N ? n0 + row - T::BM : g.N - 1;
      s_src[i] = reinterpret_cast<const char*>(g.wp) + (int64_t)r * 16;
      s_step[i] = (int64_t)g.N * 16;
    }
  }
  auto dma = [&](uint32_t off, const char* base, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(base), "s"(lds) : "memory", "m0");
  };
  auto issue = [&](int kt, int stage) {  // past the end: the last step again, so that the number of loads in flight is known
    const bool last = kt >= nk_all - 1;
    kt = kt < nk_all ? kt : nk_all - 1;
    const uint32_t sa = lds0 + stage * T::kStage;
    const char* xb = xbase + (int64_t)kt * T::kRowA;
    const char* wb = wbase + (int64_t)kt * T::kRowW;
#pragma unroll
    for (int i = 0; i < T::kLoadsA; ++i) dma(a_off[i], xb, sa + (wave * T::kLoadsA + i) * 1024);
#pragma unroll
    for (int i = 0; i < T::kLoadsW; ++i) {
      // unsigned wrap-around of the 32-bit offset is avoided: over <= 48 is taken off the piece's own offset
      dma(last ? w_off[i] + (uint32_t)((kt * T::kRowW)) - w_over[i] : w_off[i], last ? wbase : wb, sa + T::kA + (wave * T::kLoadsW + i) * 1024);
    }
  };
  const int groups = (nk_all + 3) >> 2;
  auto issue_scales = [&](int grp, int ring) {
    grp = grp < groups ? grp : groups - 1;
#pragma unroll
    for (int i = 0; i < T::kLoadsS; ++i) {
      if (s_mine[i] || T::kLoadsS == 1) {
        const uint32_t dst = lds0 + T::kStages * T::kStage + ring * T::kScales + (wave + i * WM * WN) * 1024;
        if (s_mine[i])
          asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(s_src[i] + grp * s_step[i]), "s"(dst) : "memory", "m0");
      }
    }
  };

  v16f acc[TN][TM];
#pragma unroll
  for (int j = 0; j < TN; ++j)
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int v = 0; v < 16; ++v) acc[j][i][v] = 0.f;

  // operand reads: piece p of row r of the input at a_rd + 32 i rows, of the weight at w_rd + 32 j rows
  const int ar = 32 * TM * wm + l31, wr = 32 * TN * wn + l31;
  int a_rd[4], w_rd[2];
#pragma unroll
  for (int p = 0; p < 4; ++p)  // F8: pieces 4 c + h and 4 c + 2 + h of sub-step c; fp4: piece 2 c + h
    a_rd[p] = F8 ? ar * 128 + (((2 * p + half) ^ ((ar >> 1) & 7)) << 4) : ar * 64 + ((((2 * p + half) & 3) ^ ((ar >> 2) & 3)) << 4);
#pragma unroll
  for (int p = 0; p < 2; ++p) w_rd[p] = T::kA + wr * 64 + (((2 * p + half) ^ ((wr >> 2) & 3)) << 4);
  const int s_rd = T::kStages * T::kStage + 8 * half;

  mx_u32x2 sx[TM], sw[TN];
  auto read_scales = [&](int ring) {
    const char* p = smem + s_rd + ring * T::kScales;
#pragma unroll
    for (int i = 0; i < TM; ++i) sx[i] = *reinterpret_cast<const mx_u32x2*>(p + (ar + 32 * i) * 16);
#pragma unroll
    for (int j = 0; j < TN; ++j) sw[j] = *reinterpret_cast<const mx_u32x2*>(p + (T::BM + wr + 32 * j) * 16);
  };
  auto load4 = [&](const char* p, v8i& v, int at) {
    const mx_u32x4 q = *reinterpret_cast<const mx_u32x4*>(p);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[at + e] = (int)q[e];
  };
  // step S of a group of four (S picks the scales' byte)
  auto step = [&](int stage, auto which) {
    constexpr int S = decltype(which)::value;
    const char* st = smem + stage * T::kStage;
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      v8i xf[TM] = {}, wf[TN] = {};
#pragma unroll
      for (int i = 0; i < TM; ++i) {
        if constexpr (F8) {
          load4(st + a_rd[2 * c] + i * 32 * 128, xf[i], 0);
          load4(st + a_rd[2 * c + 1] + i * 32 * 128, xf[i], 4);
        } else {
          load4(st + a_rd[c] + i * 32 * 64, xf[i], 0);
        }
      }
#pragma unroll
      for (int j = 0; j < TN; ++j) load4(st + w_rd[c] + j * 32 * 64, wf[j], 0);
      constexpr int kDword = S >> 1;
#pragma unroll
      for (int j = 0; j < TN; ++j)
#pragma unroll
        for (int i = 0; i < TM; ++i) {
          // byte 2 (S % 2) + c of the dword: the selects are immediates
          if (c == 0)
            acc[j][i] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(wf[j], xf[i], acc[j][i], 4, F8 ? 0 : 4, 2 * (S & 1), sw[j][kDword],
                                                                       2 * (S & 1), sx[i][kDword]);
          else
            acc[j][i] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(wf[j], xf[i], acc[j][i], 4, F8 ? 0 : 4, 2 * (S & 1) + 1, sw[j][kDword],
                                                                       2 * (S & 1) + 1, sx[i][kDword]);
        }
    }
  };

  // ---- pipeline.  Loads of a wave complete in order.  At step t a wave waits until what it requested for step t has
  //      landed, passes the barrier (everybody's has, and everybody is done with step t - 1), requests step t + 2 into the
  //      stage of step t - 1, and computes.  Program order: scales 0, stage 0, stage 1; step t: (t % 4 == 0: the next
  //      group's scales,) stage t + 2.  Newer than stage t at step t's wait are the loads of stage t + 1; scales requested in
  //      between are waited for with it, three steps before they are read.
  constexpr int kStageLoads = T::kLoadsA + T::kLoadsW;
  auto wait_for = [&]() {
    // lgkmcnt: this wave's reads of step t - 1 are complete before another wave's loads may overwrite them
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(kStageLoads) : "memory");
  };
  using I0 = std::integral_constant<int, 0>;
  using I1 = std::integral_constant<int, 1>;
  using I2 = std::integral_constant<int, 2>;
  using I3 = std::integral_constant<int, 3>;
  int stage = 0, ring = 0;
  auto next = [&]() { stage = stage == 2 ? 0 : stage + 1; };
  auto two_on = [&]() { return stage == 0 ? 2 : stage - 1; };
  issue_scales(k_begin >> 2, 0);
  issue(k_begin, 0);
  issue(k_begin + 1, 1);
  for (int t = k_begin; t < k_end; t += 4) {
    wait_for();
    issue_scales((t >> 2) + 1, ring ^ 1);
    issue(t + 2, two_on());
    read_scales(ring);
    step(stage, I0{});
    next();
    if (t + 1 >= k_end) break;
    wait_for();
    issue(t + 3, two_on());
    step(stage, I1{});
    next();
    if (t + 2 >= k_end) break;
    wait_for();
    issue(t + 4, two_on());
    step(stage, I2{});
    next();
    if (t + 3 >= k_end) break;
    wait_for();
    issue(t + 5, two_on());
    step(stage, I3{});
    next();
    ring ^= 1;
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the requests past the end

  // ---- adapter: s . h . B^T as further contraction steps of 16 ranks, the scale rounded into h's side
  if (g.rank > 0 && slice == 0) {
    for (int r0 = 0; r0 < g.rank; r0 += 16) {
      const int r = r0 + 8 * half;
      bf16x8_t hx[TM], bw[TN];
#pragma unroll
      for (int i = 0; i < TM; ++i) {
        int row = m0 + ar + 32 * i;
        row = row < g.M ? row : g.M - 1;
        bf16x8_t v = {};
        if (r < g.rank) v = *reinterpret_cast<const bf16x8_t*>(g.h + (int64_t)row * g.ldh + r);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = (__bf16)((float)v[e] * g.lscale);
        hx[i] = v;
      }
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        int row = n0 + wr + 32 * j;
        row = row < g.N ? row : g.N - 1;
        bf16x8_t v = {};
        if (r < g.rank) v = *reinterpret_cast<const bf16x8_t*>(g.lb + (int64_t)row * g.rank + r);
        bw[j] = v;
      }
#pragma unroll
      for (int j = 0; j < TN; ++j)
#pragma unroll
        for (int i = 0; i < TM; ++i) acc[j][i] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(bw[j], hx[i], acc[j][i], 0, 0, 0);
    }
  }

  if (g.slices > 1) {
    // fp32 sums of this slice, rounded and finished by the sum of the slices
    float* out = g.part + (int64_t)slice * g.M * g.N;
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      const int row = m0 + ar + 32 * i;
      if (row >= g.M) continue;
#pragma unroll
      for (int j = 0; j < TN; ++j)
#pragma unroll
        for (int v = 0; v < 16; ++v) {
          const int col = n0 + 32 * TN * wn + 32 * j + 8 * (v >> 2) + 4 * half + (v & 3);
          if (col < g.N) out[(int64_t)row * g.N + col] = acc[j][i][v];
        }
    }
    return;
  }
  // ---- the wave's band [32 TM rows][32 TN columns] goes through LDS so that whole row segments are stored
  __syncthreads();
  char* band = smem + wave * (32 * TM * T::kPitch);
#pragma unroll
  for (int j = 0; j < TN; ++j) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int col = n0 + 32 * TN * wn + 32 * j + 8 * q + 4 * half;
      float b[4] = {0.f, 0.f, 0.f, 0.f};
      if (g.bias) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (col + e < g.N) b[e] = __builtin_bit_cast(float, (uint32_t)g.bias[col + e] << 16);
      }
#pragma unroll
      for (int i = 0; i < TM; ++i) {
        bf16x4_t o;
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = (__bf16)(acc[j][i][4 * q + e] + b[e]);
        *reinterpret_cast<bf16x4_t*>(band + (l31 + 32 * i) * T::kPitch + (32 * j + 8 * q + 4 * half) * 2) = o;
      }
    }
  }
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // only this wave reads its band
  const int col0 = n0 + 32 * TN * wn, row_first = m0 + 32 * TM * wm;
  if ((g.N & 7) == 0) {
    constexpr int kPer = 4 * TN;  // 16-byte pieces of a row
    constexpr int kRows = 64 / kPer;
#pragma unroll
    for (int r = 0; r < 32 * TM; r += kRows) {
      const int rr = r + lane / kPer, c = 8 * (lane % kPer);
      const mx_u32x4 v = *reinterpret_cast<const mx_u32x4*>(band + rr * T::kPitch + 2 * c);
      if (row_first + rr < g.M && col0 + c < g.N) *reinterpret_cast<mx_u32x4*>(g.y + (int64_t)(row_first + rr) * g.N + col0 + c) = v;
    }
  } else {
    for (int r = 0; r < 32 * TM; ++r) {
      if (row_first + r >= g.M) break;
#pragma unroll
      for (int c = lane; c < 32 * TN; c += 64) {
        const uint16_t v = *reinterpret_cast<const uint16_t*>(band + r * T::kPitch + 2 * c);
        if (col0 + c < g.N) g.y[(int64_t)(row_first + r) * g.N + col0 + c] = v;
      }
    }
  }
#endif
}

// y = bf16(sum of the slices in order + bias)
__global__ __launch_bounds__(256) void mx_sum_slices_kernel(const float* __restrict__ part, const uint16_t* __restrict__ bias,
                                                            uint16_t* __restrict__ y, int64_t numel, int N, int slices) {
  const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
  if (i >= numel) return;
  float s[4] = {0.f, 0.f, 0.f, 0.f};
  const int n = numel - i < 4 ? (int)(numel - i) : 4;
  if (n == 4 && (numel & 3) == 0) {
    typedef float f32x4 __attribute__((ext_vector_type(4)));
    for (int k = 0; k < slices; ++k) {
      const f32x4 v = *reinterpret_cast<const f32x4*>(part + (int64_t)k * numel + i);
#pragma unroll
      for (int e = 0; e < 4; ++e) s[e] += v[e];
    }
  } else {
    for (int k = 0; k < slices; ++k)
      for (int e = 0; e < n; ++e) s[e] += part[(int64_t)k * numel + i + e];
  }
  for (int e = 0; e < n; ++e) {
    const float b = bias ? __builtin_bit_cast(float, (uint32_t)bias[(i + e) % N] << 16) : 0.f;
    y[i + e] = __builtin_bit_cast(uint16_t, (__bf16)(s[e] + b));
  }
}

using TileL8 = MxTile<4, 2, 2, 4, true>;
using TileL4 = MxTile<4, 2, 2, 4, false>;
using TileS8 = MxTile<2, 2, 2, 2, true>;
using TileS4 = MxTile<2, 2, 2, 2, false>;

struct MxPlan {
  bool large;
  int slices, steps_per_slice;
};

MxPlan plan_mx(int64_t M, int64_t N, int64_t K) {
  const int64_t steps = mx_padded_k(K) / 128, big = ((M + 255) / 256) * ((N + 255) / 256);
  if (big >= 192) return MxPlan{true, 1, (int)((steps + 3) / 4 * 4)};
  const int64_t tiles = ((M + 127) / 128) * ((N + 127) / 128);
  const int64_t groups = (steps + 3) / 4;
  int64_t slices = 512 / tiles;
  slices = std::max<int64_t>(1, std::min({slices, groups / 2, int64_t(16)}));
  const int64_t per = (groups + slices - 1) / slices;
  return MxPlan{false, (int)((groups + per - 1) / per), (int)(4 * per)};
}

template <int WM, int WN, int TM, int TN, bool F8>
int launch_mx(MxGemmArgs& g, hipStream_t s) {
  using T = MxTile<WM, WN, TM, TN, F8>;
  g.tiles_m = (g.M + T::BM - 1) / T::BM;
  g.tiles_n = (g.N + T::BN - 1) / T::BN;
  // the LDS limit is a per-device attribute of the function (a race only repeats the call)
  static bool attr_set[64] = {};
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) dev = -1;
  if (dev < 0 || !attr_set[dev]) {
    hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(&mx_gemm_kernel<WM, WN, TM, TN, F8>), hipFuncAttributeMaxDynamicSharedMemorySize, T::kLds);
    if (e != hipSuccess) return fail(TTAMD_ELAUNCH, "mx_gemm: cannot reserve %d bytes of LDS: %s", T::kLds, hipGetErrorString(e));
    if (dev >= 0) attr_set[dev] = true;
  }
  const int64_t blocks = (int64_t)g.tiles_m * g.tiles_n * g.slices;
  if (blocks >= (int64_t(1) << 31)) return fail(TTAMD_EUNSUPPORTED, "mx_gemm: M=%d N=%d are too large for one launch", g.M, g.N);
  mx_gemm_kernel<WM, WN, TM, TN, F8><<<dim3((unsigned)blocks), dim3(T::kThreads), T::kLds, s>>>(g);
  return check_launch("mx_gemm");
}

size_t align256(size_t v) { return (v + 255) & ~size_t(255); }

}  // namespace

size_t mx_operand_bytes(int64_t M, int64_t K, int fmt) {
  const int64_t Kp = mx_padded_k(K);
  return align256((size_t)M * (fmt == TTAMD_MXFP4 ? Kp / 2 : Kp));
}

size_t mx_gemm_part_bytes(int64_t M, int64_t N, int64_t K) {
  const MxPlan p = plan_mx(M, N, K);
  return p.slices > 1 ? align256((size_t)p.slices * M * N * sizeof(float)) : 0;
}

int run_mx_gemm(const MxProduct& q, int64_t M, int64_t N, int64_t K, int fmt, float* part, hipStream_t s) {
  const MxPlan p = plan_mx(M, N, K);
  MxGemmArgs g = {};
  g.xc = q.x_codes; g.xp = q.x_pieces; g.wc = q.w_codes; g.wp = q.w_pieces;
  g.h = q.h; g.lb = q.lora_b; g.bias = q.bias; g.y = q.y;
  g.lscale = q.lscale;
  g.M = (int)M; g.N = (int)N; g.K = (int)K; g.Kp = (int)mx_padded_k(K);
  g.rank = q.rank; g.ldh = q.ldh;
  g.slices = p.slices; g.steps_per_slice = p.steps_per_slice;
  g.part = part;
  TT_REQUIRE(p.slices == 1 || part, "mx_gemm: no room for the slices of the contraction");
  int rc;
  if (fmt == TTAMD_MXFP8)
    rc = p.large ? launch_mx<4, 2, 2, 4, true>(g, s) : launch_mx<2, 2, 2, 2, true>(g, s);
  else
    rc = p.large ? launch_mx<4, 2, 2, 4, false>(g, s) : launch_mx<2, 2, 2, 2, false>(g, s);
  if (rc || p.slices == 1) return rc;
  const int64_t numel = M * N;
  mx_sum_slices_kernel<<<dim3((unsigned)((numel + 1023) / 1024)), dim3(256), 0, s>>>(part, q.bias, q.y, numel, (int)N, p.slices);
  return check_launch("mx_sum_slices");
}

int check_mx_product(const char* who, int64_t M, int64_t N, int64_t K) {
  TT_REQUIRE(M > 0 && N > 0 && K > 0 && K % kMxBlock == 0, "%s: bad shape M=%lld N=%lld K=%lld (K is a multiple of 32)", who, (long long)M, (long long)N, (long long)K);
  if (!(M < (1 << 30) && N < (1 << 30) && K < (1 << 23))) return fail(TTAMD_EUNSUPPORTED, "%s: M=%lld N=%lld K=%lld are too large", who, (long long)M, (long long)N, (long long)K);
  return TTAMD_OK;
}

}  // namespace ttamd

using namespace ttamd;

extern "C" size_t ttamd_mx_linear_workspace_bytes(int64_t M, int64_t N, int64_t K, int activation_format) {
  if (M <= 0 || N <= 0 || K <= 0 || K % kMxBlock) return 0;
  return mx_operand_bytes(M, K, activation_format) + align256(mx_piece_bytes(M, K)) + align256(mx_piece_bytes(N, K)) + mx_gemm_part_bytes(M, N, K);
}

extern "C" int ttamd_mx_linear_bf16(const void* x, int activation_format, const uint8_t* w_codes, const uint8_t* w_scales, const void* bias,
                                    void* y, int64_t M, int64_t N, int64_t K, void* workspace, size_t workspace_bytes, void* stream) {
  if (int rc = check_mx_product("mx_linear", M, N, K)) return rc;
  TT_REQUIRE(activation_format == TTAMD_MXFP4 || activation_format == TTAMD_MXFP8, "mx_linear: unknown format code %d", activation_format);
  TT_REQUIRE(x && w_codes && w_scales && y && aligned16(x) && aligned16(w_codes) && aligned16(w_scales) && aligned16(y) &&
                 (reinterpret_cast<uintptr_t>(bias) & 1u) == 0,
             "mx_linear: pointers must be non-null and 16-byte aligned");
  const size_t need = ttamd_mx_linear_workspace_bytes(M, N, K, activation_format);
  if (workspace_bytes < need || !workspace || !aligned16(workspace))
    return fail(TTAMD_EWORKSPACE, "mx_linear: needs %zu bytes of 16-byte aligned workspace, got %zu", need, workspace_bytes);
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  char* w = reinterpret_cast<char*>(workspace);
  MxProduct q = {};
  uint8_t* xc = reinterpret_cast<uint8_t*>(w);
  w += mx_operand_bytes(M, K, activation_format);
  uint8_t* xp = reinterpret_cast<uint8_t*>(w);
  w += align256(mx_piece_bytes(M, K));
  uint8_t* wp = reinterpret_cast<uint8_t*>(w);
  w += align256(mx_piece_bytes(N, K));
  if (int rc = run_mx_quantize_operand(x, M, K, activation_format, xc, xp, &w_scales, &N, &wp, 1, s)) return rc;
  q.x_codes = xc; q.x_pieces = xp; q.w_codes = w_codes; q.w_pieces = wp;
  q.bias = reinterpret_cast<const uint16_t*>(bias);
  q.y = reinterpret_cast<uint16_t*>(y);
  return run_mx_gemm(q, M, N, K, activation_format, reinterpret_cast<float*>(w), s);
}
