// Products over microscaled operands: y[M, N] = x^[M, K] . W[N, K]^T (+ s . h . B^T) (+ bias), x^ in mxfp8 or mxfp4, W in
// mxfp4, on v_mfma_scale_f32_16x16x128_f8f6f4, which multiplies the codes and applies both blocks' scales.  Sums: fp32 over
// fp4 x fp4 products; of fp8 x fp4 ones each eight neighbours (contraction indices 8 i .. 8 i + 7) are added first, and what lies
// below 2^-13 of the largest of them is dropped (one large and one small product: 2^-13 arrives, 2^-14 does not; in another eight,
// of the same block or not, 2^-23 arrives).
//
// Operand order of that instruction (lane l: row l % 16, quarter q = l / 16), found by comparing with products in 64 bits:
//   fp4: 16 bytes, indices 32 q .. 32 q + 31 of the 128-wide step; fp8: two pieces of 16 bytes, indices 16 q .. and 64 + 16 q ..
//   scale: the lowest byte of a register, that of block q of the step; result: column l % 16 of the second operand, rows
//   4 q + v of the first.
// The weight is the first operand, so a lane holds four consecutive outputs of one row of y.  The 16 x 16 x 128 shape and not
// 32 x 32 x 64: this part is limited by power under matrix load, and loops of nothing but these instructions on random
// operands run at 4.0 against 3.3 PFLOP/s (fp8 x fp4) and 7.3 against 6.1 (fp4 x fp4).
//
// Workgroup: WM x WN waves, a wave computes TM x TN tiles of 16 x 16, k-step 128.  Codes go HBM -> LDS by direct loads of 16
// bytes per lane into a ring of three stages, scales likewise, one 16-byte piece per row and 512 contraction indices, into
// a ring of two; nothing but LDS reads and matrix instructions is left in the waves.  One barrier per step.  The kernel is
// persistent: a workgroup's items follow each other in one pipeline.
#include <algorithm>
#include <type_traits>

#include "group.h"
#include "mx_math.h"

namespace ttamd {
namespace {

typedef int v8i __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4_t __attribute__((ext_vector_type(4)));

#define TT_INLINE __attribute__((always_inline))
#define TT_LDS_PTR(p) ((__attribute__((address_space(3))) void*)(p))

struct MxGemmMember {
  const uint8_t* wc;   // [N, K / 2]
  const uint8_t* wp;   // [groups][N][16]
  const uint16_t* h;   // [M, ldh] or null: adapter activation
  const uint16_t* lb;  // [N, rank]
  const uint16_t* bias;
  uint16_t* y;         // [M, N]
  float lscale;
  int N, rank, tile_end;  // its column tiles end there among all members'
};
struct MxGemmArgs {
  const uint8_t* xc;   // [M, Kp] or [M, Kp / 2]: codes of the input, rows padded to 256 elements
  const uint8_t* xp;   // its scales, [groups][M][16]
  MxGemmMember m[kMxWeights];
  float* part;         // [slices][M][N] or null
  int n, M, K, Kp, ldh;
  int tiles_m, tiles_n, slices, steps_per_slice;  // steps of 128, a multiple of 4 per slice
};

constexpr int kCUs = 256;

template <int WM, int WN, int TM, int TN, bool F8>
struct MxTile {
  static constexpr int kThreads = 64 * WM * WN;
  static constexpr int BM = 16 * WM * TM, BN = 16 * WN * TN;
  static constexpr int kRowA = F8 ? 128 : 64, kRowW = 64;  // bytes of a row per step
  static constexpr int kA = BM * kRowA, kW = BN * kRowW, kStage = kA + kW;
  static constexpr int kStages = 3;
  static constexpr int kScales = (BM + BN) * 16;
  static constexpr int kLds = kStages * kStage + 2 * kScales;
  static constexpr int kPerCU = kLds <= 40 * 1024 ? 4 : kLds <= 53 * 1024 ? 3 : kLds <= 80 * 1024 ? 2 : 1;  // workgroups that a CU's LDS holds
  static constexpr int kLoadsA = kA / (kThreads * 16), kLoadsW = kW / (kThreads * 16);
  static constexpr int kScaleWaves = (BM + BN) / 64;  // waves' worth of scale pieces
  static constexpr int kLoadsS = (kScaleWaves + WM * WN - 1) / (WM * WN);
  static constexpr int kStores = TM * TN / 2;         // of a wave's whole tile
  static_assert(kA % (kThreads * 16) == 0 && kW % (kThreads * 16) == 0 && (BM + BN) % 64 == 0, "whole loads");
  static_assert(kLds <= 160 * 1024, "LDS of a CU");
  static_assert(TN % 2 == 0, "two halves of a step");
};

// eight outputs of a row; rows of an odd length start anywhere
struct __attribute__((packed, aligned(2))) MxStore16 {
  uint32_t d[4];
};

// f(integral_constant<A>), .. f(integral_constant<B - 1>)
template <int A, int B, typename F>
__device__ __forceinline__ void for_range(F&& f) {
  if constexpr (A < B) {
    f(std::integral_constant<int, A>{});
    for_range<A + 1, B>(f);
  }
}

// GROUP: several weights' tiles in one launch (whole contractions)
template <int WM, int WN, int TM, int TN, bool F8, bool GROUP>
__global__ __launch_bounds__(512) void mx_gemm_kernel(const MxGemmArgs g) {
#if defined(__HIP_DEVICE_COMPILE__)
  using T = MxTile<WM, WN, TM, TN, F8>;
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  const int lane = threadIdx.x & 63, r16 = lane & 15, quarter = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave % WM, wn = wave / WM;
  const int nk_all = g.Kp >> 7;

  // Work items are (slice, tile).  In a round every workgroup takes one; the workgroups of an XCD (they go to the eight XCDs
  // in turn) take consecutive items, and items walk the tiles in bands of eight row tiles, so that the tiles in flight on
  // one XCD share rows and columns in its L2.  The last round is spread over the XCDs evenly.
  const int tiles = g.tiles_m * g.tiles_n, total = tiles * g.slices, grid = (int)gridDim.x;
  const int xcd = (int)blockIdx.x & 7, place = (int)blockIdx.x >> 3;
  auto item_of = [&](int round) TT_INLINE {  // -1: none
    const int begin = round * grid, cnt = total - begin < grid ? total - begin : grid;
    if (cnt <= 0) return -1;
    const int q = cnt >> 3, rem = cnt & 7, share = q + (xcd < rem ? 1 : 0);
    return place < share ? begin + xcd * q + (xcd < rem ? xcd : rem) + place : -1;
  };
  struct Item {
    int m0, n0, k_begin, k_end, slice, mem;
  };
  // divisions are worked out in vector registers: their results go back to scalar ones
  auto uniform = [](int v) TT_INLINE { return __builtin_amdgcn_readfirstlane(v); };
  auto decode = [&](int id) TT_INLINE {
    Item w;
    w.slice = uniform(id / tiles);
    id -= w.slice * tiles;
    const int band = 8 * g.tiles_n, b = uniform(id / band), in = id - b * band;
    const int rows = g.tiles_m - 8 * b < 8 ? g.tiles_m - 8 * b : 8, across = uniform(in / rows);
    w.m0 = (8 * b + in - across * rows) * T::BM;
    w.mem = 0;
    int before = 0;
    if constexpr (GROUP) {
#pragma unroll
      for (int q = 0; q < kMxWeights - 1; ++q)
        if (q < g.n - 1 && across >= g.m[q].tile_end) {
          w.mem = q + 1;
          before = g.m[q].tile_end;
        }
    }
    w.n0 = (across - before) * T::BN;
    w.k_begin = w.slice * g.steps_per_slice;
    w.k_end = w.k_begin + g.steps_per_slice < nk_all ? w.k_begin + g.steps_per_slice : nk_all;
    return w;
  };

  // ---- the requesting side: which step of which item is requested next.  A stage's rows lie in LDS one after the other;
  //      the 16-byte pieces of a row are permuted by the row (on the address side) so that the rows a wave reads at one
  //      piece index spread over the banks.  Buffer loads: the uniform part of an address is in scalar registers with the
  //      number of bytes from there to the operand's end, and what lies past it (rows beyond M or N, a last weight row's
  //      end, everything behind the last item) is not read.  A weight row that ends inside a step is followed by the next
  //      row's codes: the input's are zero there.
  const uint32_t lds0 = (uint32_t)(uintptr_t)TT_LDS_PTR(smem);
  const int ldx = F8 ? g.Kp : g.Kp >> 1, ldw = g.K >> 1;
  constexpr int kRowsA = F8 ? 8 : 16;  // rows of an instruction (64 pieces): 128 or 64 bytes each
  typedef int v4i __attribute__((ext_vector_type(4)));
  auto dma = [&](uint32_t off, const uint8_t* base, int bytes, uint32_t lds) TT_INLINE {
    const uint64_t p = (uint64_t)(uintptr_t)base;
    const v4i srd = {uniform((int)(uint32_t)p), uniform((int)((p >> 32) & 0xffff)), uniform(bytes > 0 ? bytes : 0), 0x00027000};
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds" ::"v"(off), "s"(srd), "s"(lds) : "memory", "m0");
  };
  // what a lane number is turned into outside the loop over steps is worked out again where it is used: kept, it would take
  // the registers that the sums need
  auto fresh = [](int v) TT_INLINE {
    asm volatile("" : "+v"(v));
    return v;
  };
  // A lane's offsets from an instruction's first row.  Piece p of a row lies at p ^ (row / 2) % 8 (rows of 128 bytes; odd
  // instructions: + 4) or p ^ 2 (row / 8) % 2 (64 bytes): a 16-byte read serves lanes 0 - 3, 12 - 15, 20 - 27 and lanes 4 - 11,
  // 16 - 19, 28 - 31 of each half wave at a time, and with these permutations their pieces fall on different banks
  const uint32_t w_off = (uint32_t)(lane >> 2) * (uint32_t)ldw + 16u * (uint32_t)((lane & 3) ^ 2 * (lane >> 5));
  const uint32_t a_off = F8 ? (uint32_t)(lane >> 3) * (uint32_t)ldx + 16u * (uint32_t)((lane & 7) ^ (lane >> 4))
                            : (uint32_t)(lane >> 2) * (uint32_t)ldx + 16u * (uint32_t)((lane & 3) ^ 2 * (lane >> 5));
  static_assert(T::kLoadsA % 2 == 0 || !F8, "the parity of an instruction is that of i");
  int p_round = 0, p_k = 0, p_end = 0, p_stage = 0, p_ring = 0, p_m0 = 0, p_n0 = 0;
  const uint8_t *p_x = nullptr, *p_w = nullptr;  // the tile's first rows at step p_k,
  int p_xn = 0, p_wn = 0;                        // and the bytes from there to the operands' ends, as far as a tile reaches
  bool p_more = false;
  const uint8_t* p_wp = nullptr;  // the weight's scales and rows
  int p_N = 0;
  auto open = [&](int id) TT_INLINE {
    p_more = id >= 0;
    const Item w = decode(p_more ? id : 0);
    p_k = w.k_begin;
    p_end = w.k_end;
    p_m0 = w.m0;
    p_n0 = w.n0;
    p_x = g.xc + (int64_t)w.m0 * ldx + w.k_begin * T::kRowA;
    p_N = g.m[w.mem].N;
    p_wp = g.m[w.mem].wp;
    p_w = g.m[w.mem].wc + (int64_t)w.n0 * ldw + w.k_begin * T::kRowW;
    // requests behind the last item read nothing: the number in flight stays what the waits assume
    p_xn = p_more ? (g.M - w.m0 < T::BM + 1 ? g.M - w.m0 : T::BM + 1) * ldx - w.k_begin * T::kRowA : 0;
    p_wn = p_more ? (p_N - w.n0 < T::BN + 1 ? p_N - w.n0 : T::BN + 1) * ldw - w.k_begin * T::kRowW : 0;
  };
  // load i of the next step's operands
  auto request = [&](auto i_) TT_INLINE {
    constexpr int i = decltype(i_)::value;
    const uint32_t st = lds0 + p_stage * T::kStage;
    if constexpr (i < T::kLoadsA) {
      const int q = wave * T::kLoadsA + i;
      dma(((uint32_t)fresh((int)a_off) ^ (F8 && (i & 1) ? 64u : 0u)) + (uint32_t)(q * kRowsA) * (uint32_t)ldx, p_x, p_xn, st + q * 1024);
    } else {
      const int q = wave * T::kLoadsW + i - T::kLoadsA;
      dma((uint32_t)fresh((int)w_off) + (uint32_t)(q * 16) * (uint32_t)ldw, p_w, p_wn, st + T::kA + q * 1024);
    }
  };
  // on to the step after it; at the first step of a group of four its scales are requested (waves in turn: 64 rows each of
  // the tile's BM input rows and BN weight rows)
  auto request_scales = [&]() TT_INLINE {
    if ((p_k & 3) == 0 && p_more) {
#pragma unroll
      for (int i = 0; i < T::kLoadsS; ++i) {
        const int sw = wave + i * WM * WN;
        if (sw < T::kScaleWaves) {
          const bool of_x = sw * 64 < T::BM;
          const int rows = of_x ? g.M : p_N, first = of_x ? p_m0 + 64 * sw : p_n0 + 64 * sw - T::BM;
          dma(16u * (uint32_t)fresh(threadIdx.x & 63), (of_x ? g.xp : p_wp) + ((int64_t)(p_k >> 2) * rows + first) * 16,
              (rows - first < 64 ? rows - first : 64) * 16,
              lds0 + T::kStages * T::kStage + p_ring * T::kScales + sw * 1024);
        }
      }
      p_ring ^= 1;
    }
  };
  auto advance = [&]() TT_INLINE {
    p_x += T::kRowA;
    p_w += T::kRowW;
    p_xn -= T::kRowA;
    p_wn -= T::kRowW;
    p_stage = p_stage == 2 ? 0 : p_stage + 1;
    if (++p_k == p_end) open(item_of(++p_round));
  };

  int round = 0, id = item_of(0);
  if (id < 0) return;
  Item it = decode(id);
  open(id);

  v4f acc[TN][TM];
  auto clear = [&]() TT_INLINE {
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
      for (int i = 0; i < TM; ++i) acc[j][i] = v4f{0.f, 0.f, 0.f, 0.f};
  };

  // operand reads: pieces of rows ar + 16 i of the input and wr + 16 j of the weight (16 rows on, the permutation repeats)
  const int ar = 16 * TM * wm + r16, wr = 16 * TN * wn + r16;
  const int a_rd0 = F8 ? ar * 128 + ((quarter ^ ((ar >> 1) & 7)) << 4) : ar * 64 + ((quarter ^ 2 * ((ar >> 3) & 1)) << 4);
  const int a_rd1 = ar * 128 + (((4 + quarter) ^ ((ar >> 1) & 7)) << 4);
  const int w_rd = T::kA + wr * 64 + ((quarter ^ 2 * ((wr >> 3) & 1)) << 4);
  const int s_rd = T::kStages * T::kStage + 4 * quarter;

  // Scales: a dword per tile holds four steps, the current pair's in its low half; it is shifted from pair to pair.
  // Operands: the input's of a step, each tile's replaced by the next step's as soon as it has been multiplied for the last
  // time, and the weight's of two half steps (the first and the last TN / 2 of its tiles).
  constexpr int TH = TN / 2;
  uint32_t sx[TM], sw[TN];
  v4i xf[TM][F8 ? 2 : 1], wf[2][TH];
  auto read_scales = [&](int ring) TT_INLINE {
    const char* p = smem + s_rd + ring * T::kScales;
#pragma unroll
    for (int i = 0; i < TM; ++i) sx[i] = *reinterpret_cast<const uint32_t*>(p + (ar + 16 * i) * 16);
#pragma unroll
    for (int j = 0; j < TN; ++j) sw[j] = *reinterpret_cast<const uint32_t*>(p + (T::BM + wr + 16 * j) * 16);
  };
  auto shift_scales = [&]() TT_INLINE {
#pragma unroll
    for (int i = 0; i < TM; ++i) sx[i] >>= 16;
#pragma unroll
    for (int j = 0; j < TN; ++j) sw[j] >>= 16;
  };
  auto load4 = [&](const char* p) TT_INLINE { return *reinterpret_cast<const v4i*>(p); };
  auto read_x = [&](int stage, int i) TT_INLINE {
    const char* st = smem + stage * T::kStage;
    xf[i][0] = load4(st + a_rd0 + i * 16 * T::kRowA);
    if constexpr (F8) xf[i][1] = load4(st + a_rd1 + i * 16 * T::kRowA);
  };
  auto read_w = [&](int stage, auto half_, int j) TT_INLINE {
    constexpr int c = decltype(half_)::value;
    wf[c][j] = load4(smem + stage * T::kStage + w_rd + (TH * c + j) * 16 * 64);
  };
  // fp4 operands take four of the eight registers
  auto wide = [&](v4i lo, v4i hi) TT_INLINE { return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7); };
  // after_tile(i): what else the wave does while the matrix cores work, one share after each of the input's tiles
  auto multiply = [&](auto step_, auto half_, auto after_tile) TT_INLINE {
    constexpr int S = decltype(step_)::value, c = decltype(half_)::value;
    __builtin_amdgcn_sched_barrier(0);
    for_range<0, TM>([&](auto i_) TT_INLINE {
      constexpr int i = decltype(i_)::value;
      __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int j = 0; j < TH; ++j)
        acc[TH * c + j][i] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wide(wf[c][j], wf[c][j]), wide(xf[i][0], xf[i][F8 ? 1 : 0]),
                                                                             acc[TH * c + j][i], 4, F8 ? 0 : 4, S, (int)sw[TH * c + j], S, (int)sx[i]);
      __builtin_amdgcn_s_setprio(0);
      __builtin_amdgcn_sched_barrier(0);
      after_tile(i_);
      __builtin_amdgcn_sched_barrier(0);
    });
    // the products stay in front of what follows: the compiler would sink them behind the next barrier, into the block where
    // their sums are used next
#pragma unroll
    for (int j = 0; j < TH; ++j)
#pragma unroll
      for (int i = 0; i < TM; ++i) asm volatile("" : "+v"(acc[TH * c + j][i]));
    __builtin_amdgcn_sched_barrier(0);
  };

  // ---- what becomes of an item's sums
  auto finish = [&]() TT_INLINE {
    const int lane = fresh(threadIdx.x & 63), r16 = lane & 15, quarter = lane >> 4, ar = 16 * TM * wm + r16;
    const MxGemmMember& w = g.m[GROUP ? it.mem : 0];
    const int N = w.N;
    if (!GROUP && g.slices > 1) {
      // fp32 sums of this slice, rounded and finished by the sum of the slices
      float* out = g.part + (int64_t)it.slice * g.M * N;
#pragma unroll
      for (int i = 0; i < TM; ++i) {
        const int row = it.m0 + ar + 16 * i;
        if (row >= g.M) continue;
#pragma unroll
        for (int j = 0; j < TN; ++j) {
          const int col = it.n0 + 16 * (TN * wn + j) + 4 * quarter;
          float* p = out + (int64_t)row * N + col;
          if ((N & 3) == 0) {
            if (col < N) *reinterpret_cast<v4f*>(p) = acc[j][i];
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (col + e < N) p[e] = acc[j][i][e];
          }
        }
      }
      return;
    }
    // Two neighbouring tiles' outputs change places between neighbouring quarters: a lane of quarter q then holds the eight
    // outputs 8 (q / 2) .. of tile j + q % 2 in its row
#pragma unroll
    for (int j = 0; j < TN; j += 2) {
      asm volatile("" ::: "memory");  // one pair of tiles after the other: all of them at once do not fit the registers
      const int n0 = it.n0 + 16 * (TN * wn + j);
      float b[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      if (w.bias) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {  // before the exchange: four of each tile
          const int n = n0 + 16 * (e >> 2) + 4 * quarter + (e & 3);
          b[e] = n < N ? __builtin_bit_cast(float, (uint32_t)w.bias[n] << 16) : 0.f;
        }
      }
      const int col = n0 + 16 * (quarter & 1) + 8 * (quarter >> 1);
#pragma unroll
      for (int i = 0; i < TM; ++i) {
        uint32_t d[4];  // pairs of outputs of tile j in d[0], d[1], of tile j + 1 in d[2], d[3]
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          mx_bf16x2 o;
          o.x = (__bf16)(acc[j + (e >> 1)][i][2 * (e & 1)] + b[2 * e]);
          o.y = (__bf16)(acc[j + (e >> 1)][i][2 * (e & 1) + 1] + b[2 * e + 1]);
          d[e] = __builtin_bit_cast(uint32_t, o);
        }
        const auto s0 = __builtin_amdgcn_permlane16_swap(d[0], d[2], false, false);
        const auto s1 = __builtin_amdgcn_permlane16_swap(d[1], d[3], false, false);
        MxStore16 o;
        o.d[0] = s0[0]; o.d[1] = s1[0]; o.d[2] = s0[1]; o.d[3] = s1[1];
        const int row = it.m0 + ar + 16 * i;
        uint16_t* y = w.y + (int64_t)row * N + col;
        if (row < g.M && col + 8 <= N) {
          *reinterpret_cast<MxStore16*>(y) = o;
        } else if (row < g.M) {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (col + e < N) y[e] = (uint16_t)(o.d[e >> 1] >> (16 * (e & 1)));
        }
      }
    }
  };
  // adapter: s . h . B^T as further contraction steps of 32 ranks.  s . h goes in as the sum of two bf16 numbers, 16 bits of it:
  // rounded to one it is a second rounding of h (no error for a factor that is a power of two, up to half a step for others)
  auto adapt = [&]() TT_INLINE {
    const int lane = fresh(threadIdx.x & 63), r16 = lane & 15, quarter = lane >> 4, ar = 16 * TM * wm + r16, wr = 16 * TN * wn + r16;
    const MxGemmMember& w = g.m[GROUP ? it.mem : 0];
    const int rank = w.rank, N = w.N;
    for (int r0 = 0; r0 < rank; r0 += 32) {
      const int r = r0 + 8 * quarter;
      bf16x8_t hx[TM], hx_low[TM];
#pragma unroll
      for (int i = 0; i < TM; ++i) {
        int row = it.m0 + ar + 16 * i;
        row = row < g.M ? row : g.M - 1;
        bf16x8_t v = {};
        if (r < rank) v = *reinterpret_cast<const bf16x8_t*>(w.h + (int64_t)row * g.ldh + r);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float f = (float)v[e] * w.lscale;
          hx[i][e] = (__bf16)f;
          hx_low[i][e] = (__bf16)(__builtin_fabsf(f) < 0x1p127f ? f - (float)hx[i][e] : 0.f);  // infinities stay what they are
        }
      }
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        asm volatile("" ::: "memory");  // half of the weight's tiles at a time
        bf16x8_t bw[TH];
#pragma unroll
        for (int j = 0; j < TH; ++j) {
          int row = it.n0 + wr + 16 * (TH * c + j);
          row = row < N ? row : N - 1;
          bf16x8_t v = {};
          if (r < rank) v = *reinterpret_cast<const bf16x8_t*>(w.lb + (int64_t)row * rank + r);
          bw[j] = v;
        }
#pragma unroll
        for (int j = 0; j < TH; ++j)
#pragma unroll
          for (int i = 0; i < TM; ++i) {
            acc[TH * c + j][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(bw[j], hx[i], acc[TH * c + j][i], 0, 0, 0);
            acc[TH * c + j][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(bw[j], hx_low[i], acc[TH * c + j][i], 0, 0, 0);
          }
      }
    }
  };

  // ---- pipeline over the steps of all of the workgroup's items.  While the matrix cores work on the first half of the
  //      weight's tiles of step t a wave reads the second half from LDS; then it waits until what it requested for step
  //      t + 1 has landed, passes the barrier (everybody's has, and everybody's reads of step t are complete), requests step
  //      t + 3 into the stage of step t, and reads the input and the weight's first half of step t + 1 while the second half
  //      of step t is multiplied.  An item's outputs are stored while the next one's first steps are on their way.
  //      Memory operations of a wave complete in order.  Newer than stage t + 1 at step t's wait are the loads of stage
  //      t + 2 (scales requested in between are waited for with it) and, in the first two steps of an item, the stores of
  //      the item before: a whole tile's are counted, others are waited for.
  constexpr int kStageLoads = T::kLoadsA + T::kLoadsW;
  using I0 = std::integral_constant<int, 0>;
  using I1 = std::integral_constant<int, 1>;
  int stage = 0, ring = 0, stored = 0;  // stored: steps for which whole-tile stores may still be in flight
  for (int t = 0; t < 3; ++t) {
    request_scales();
    for_range<0, kStageLoads>(request);
    advance();
  }
  asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"(2 * kStageLoads) : "memory");
  auto begin_item = [&]() TT_INLINE {
    read_scales(ring);
    for_range<0, TM>([&](auto i) TT_INLINE { read_x(stage, i); });
    for_range<0, TH>([&](auto j) TT_INLINE { read_w(stage, I0{}, j); });
    clear();
  };
  begin_item();
  auto step = [&](auto step_) TT_INLINE {
    multiply(step_, I0{}, [&](auto i_) TT_INLINE {  // shares of TH weight tiles
      constexpr int i = decltype(i_)::value;
      for_range<TH * i / TM, TH*(i + 1) / TM>([&](auto j) TT_INLINE { read_w(stage, I1{}, j); });
    });
    if (stored > 0)
      asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(kStageLoads + T::kStores) : "memory");
    else
      asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(kStageLoads) : "memory");
    --stored;
    request_scales();
    stage = stage == 2 ? 0 : stage + 1;
    multiply(step_, I1{}, [&](auto i_) TT_INLINE {
      constexpr int i = decltype(i_)::value;
      read_x(stage, i);
      for_range<TH * i / TM, TH*(i + 1) / TM>([&](auto j) TT_INLINE { read_w(stage, I0{}, j); });
      for_range<kStageLoads * i / TM, kStageLoads*(i + 1) / TM>(request);
    });
    advance();
  };
  for (;;) {
    for (int t = it.k_begin;; t += 2) {  // the input's rows are padded to whole pairs of steps by zeros
      step(I0{});
      step(I1{});
      if (t + 2 >= it.k_end) break;
      if ((t & 2) != 0) {
        ring ^= 1;
        read_scales(ring);
      } else {
        shift_scales();
      }
    }
    if (g.m[GROUP ? it.mem : 0].rank > 0 && it.slice == 0) adapt();
    finish();
    id = item_of(++round);
    if (id < 0) break;
    stored = g.slices == 1 && it.m0 + T::BM <= g.M && it.n0 + T::BN <= g.m[GROUP ? it.mem : 0].N ? 2 : 0;
    it = decode(id);
    ring ^= 1;
    begin_item();  // once more what the last step has read: held through the end of an item it would take its registers
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
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

// Which tile a product runs on and how often its contraction is cut.  The times, in us, of `waves` work items per CU of
// `steps` steps each (d + e * waves per step once several share a CU, `alone` for a single one), fitted to 70 shapes of 64 -
// 3000 rows, 1024 - 14336 outputs and 2048 - 14336 contraction indices on both input formats; the model's choice was
// the best of all 20 of them in the median and within 11 % of it everywhere.  Both sides of some borders, us, fp8 inputs:
// 64 x 14336 x 4096 64-wide tiles 13.0, 64 x 128 15.4, 128-wide 21; 333 x 4096 x 4096 64 x 128 15.8, 64-wide 16.5, 128-wide
// 20.8; 2000 x 4096 x 4096 128-wide 33, 256-wide 46; 3000 x 14336 x 4096 256-wide 138, 128-wide 161; 64 x 4096 x 14336 64-wide
// in four slices 16.0, in two 22.8, whole 37.
struct MxShape {
  int bm, bn;
  float alone, d, e, item, launch;
};
constexpr MxShape kShapes[2][4] = {
    {{256, 256, 0.76f, 0.f, 0.76f, 7.f, 4.f}, {128, 128, 0.44f, 0.f, 0.315f, 1.2f, 4.5f}, {64, 128, 0.36f, 0.f, 0.225f, 0.6f, 4.f}, {64, 64, 0.28f, 0.08f, 0.13f, 0.4f, 3.5f}},
    {{256, 256, 1.1f, 0.f, 1.1f, 8.f, 4.f}, {128, 128, 0.53f, 0.f, 0.41f, 1.2f, 4.5f}, {64, 128, 0.385f, 0.f, 0.2625f, 0.6f, 4.f}, {64, 64, 0.29f, 0.165f, 0.122f, 0.4f, 3.5f}}};

struct MxPlan {
  int shape, slices, steps_per_slice;
  float time;
};

// n weights over the same input in one launch: whole contractions
MxPlan plan_mx(int64_t M, const int64_t* N, int n, int64_t K, int fmt) {
  const int64_t steps = mx_padded_k(K) / 128, groups = (steps + 3) / 4;
  MxPlan best = {0, 1, (int)(4 * groups), 1e30f};
  for (int shape = 0; shape < 4; ++shape) {
    const MxShape& t = kShapes[fmt == TTAMD_MXFP8][shape];
    int64_t tiles = 0;
    for (int i = 0; i < n; ++i) tiles += ((M + t.bm - 1) / t.bm) * ((N[i] + t.bn - 1) / t.bn);
    for (int64_t slices = 1; slices <= (n == 1 ? 16 : 1) && slices <= groups; slices *= 2) {
      const int64_t per = (groups + slices - 1) / slices;
      // partial sums of rows of an odd length are stored element by element; 256 MB of them would not pay anywhere
      if (slices > 1 && (N[0] % 4 || slices * M * N[0] > (int64_t(1) << 26))) break;
      if ((groups + per - 1) / per != slices) continue;
      const float waves = (float)((tiles * slices + kCUs - 1) / kCUs), k = (float)std::min(steps, 4 * per);
      const float step = waves > 1.f ? std::max(t.alone, t.d + t.e * waves) : t.alone;
      float time = t.launch + t.item * waves + k * step;
      if (slices > 1) time += 3.2f + (float)(slices * M * N[0]) * (4.f / 3e6f);
      if (time < best.time) best = MxPlan{shape, (int)slices, (int)(4 * per), time};
    }
  }
  return best;
}
MxPlan plan_mx(int64_t M, int64_t N, int64_t K, int fmt) { return plan_mx(M, &N, 1, K, fmt); }

template <int WM, int WN, int TM, int TN, bool F8, bool GROUP>
int launch_mx(MxGemmArgs& g, hipStream_t s) {
  using T = MxTile<WM, WN, TM, TN, F8>;
  g.tiles_m = (g.M + T::BM - 1) / T::BM;
  g.tiles_n = 0;
  for (int i = 0; i < g.n; ++i) g.m[i].tile_end = g.tiles_n += (g.m[i].N + T::BN - 1) / T::BN;
  // the LDS limit is a per-device attribute of the function (a race only repeats the call)
  static bool attr_set[64] = {};
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) dev = -1;
  if (dev < 0 || !attr_set[dev]) {
    hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(&mx_gemm_kernel<WM, WN, TM, TN, F8, GROUP>), hipFuncAttributeMaxDynamicSharedMemorySize, T::kLds);
    if (e != hipSuccess) return fail(TTAMD_ELAUNCH, "mx_gemm: cannot reserve %d bytes of LDS: %s", T::kLds, hipGetErrorString(e));
    if (dev >= 0) attr_set[dev] = true;
  }
  const int64_t items = (int64_t)g.tiles_m * g.tiles_n * g.slices;
  if (items >= (int64_t(1) << 30)) return fail(TTAMD_EUNSUPPORTED, "mx_gemm: %lld tiles are too many for one launch", (long long)items);
  const int64_t grid = std::min<int64_t>((items + 7) / 8 * 8, kCUs * T::kPerCU);
  mx_gemm_kernel<WM, WN, TM, TN, F8, GROUP><<<dim3((unsigned)grid), dim3(T::kThreads), T::kLds, s>>>(g);
  return check_launch("mx_gemm");
}

size_t align256(size_t v) { return (v + 255) & ~size_t(255); }

}  // namespace

size_t mx_operand_bytes(int64_t M, int64_t K, int fmt) {
  const int64_t Kp = mx_padded_k(K);
  return align256((size_t)M * (fmt == TTAMD_MXFP4 ? Kp / 2 : Kp));
}

size_t mx_gemm_part_bytes(int64_t M, int64_t N, int64_t K, int fmt) {
  const MxPlan p = plan_mx(M, N, K, fmt);
  return p.slices > 1 ? align256((size_t)p.slices * M * N * sizeof(float)) : 0;
}

namespace {
template <bool F8, bool GROUP>
int launch_shape(int shape, MxGemmArgs& g, hipStream_t s) {
  switch (shape) {
    case 0: return launch_mx<4, 2, 4, 8, F8, GROUP>(g, s);
    case 1: return launch_mx<2, 2, 4, 4, F8, GROUP>(g, s);
    case 2: return launch_mx<1, 4, 4, 2, F8, GROUP>(g, s);
    default: return launch_mx<2, 2, 2, 2, F8, GROUP>(g, s);
  }
}

MxGemmArgs gemm_args(const MxProduct* q, int n, int64_t M, const int64_t* N, int64_t K, const MxPlan& p, float* part) {
  MxGemmArgs g = {};
  g.xc = q[0].x_codes; g.xp = q[0].x_pieces;
  for (int i = 0; i < n; ++i) g.m[i] = MxGemmMember{q[i].w_codes, q[i].w_pieces, q[i].h, q[i].lora_b, q[i].bias, q[i].y, q[i].lscale, (int)N[i], q[i].rank, 0};
  g.n = n;
  g.M = (int)M; g.K = (int)K; g.Kp = (int)mx_padded_k(K); g.ldh = q[0].ldh;
  g.slices = p.slices; g.steps_per_slice = p.steps_per_slice;
  g.part = part;
  return g;
}
}  // namespace

int run_mx_gemm(const MxProduct& q, int64_t M, int64_t N, int64_t K, int fmt, float* part, hipStream_t s) {
  const MxPlan p = plan_mx(M, N, K, fmt);
  MxGemmArgs g = gemm_args(&q, 1, M, &N, K, p, part);
  TT_REQUIRE(p.slices == 1 || part, "mx_gemm: no room for the slices of the contraction");
  const int rc = fmt == TTAMD_MXFP8 ? launch_shape<true, false>(p.shape, g, s) : launch_shape<false, false>(p.shape, g, s);
  if (rc || p.slices == 1) return rc;
  return run_mx_sum_slices(part, q.bias, q.y, M * N, (int)N, p.slices, s);
}

// Weights over the same mxfp8 input: one launch for all where the model gives it less time than one for each (1500 x 4096 -> 4096,
// 1024 and 1024 52.9 us against 71.4 in three; 8192 x 4096 -> twice 14336 831 against 820, both within a run's spread).
int run_mx_gemm_group(const MxProduct* q, int n, int64_t M, const int64_t* N, int64_t K, float* part, hipStream_t s) {
  float each = 0.f;
  for (int i = 0; i < n; ++i) each += plan_mx(M, N[i], K, TTAMD_MXFP8).time;
  const MxPlan p = plan_mx(M, N, n, K, TTAMD_MXFP8);
  if (n > 1 && p.time < each) {
    MxGemmArgs g = gemm_args(q, n, M, N, K, p, nullptr);
    return launch_shape<true, true>(p.shape, g, s);
  }
  for (int i = 0; i < n; ++i)
    if (int rc = run_mx_gemm(q[i], M, N[i], K, TTAMD_MXFP8, part, s)) return rc;
  return TTAMD_OK;
}

int run_mx_sum_slices(const float* part, const uint16_t* bias, uint16_t* y, int64_t numel, int N, int slices, hipStream_t s) {
  mx_sum_slices_kernel<<<dim3((unsigned)((numel + 1023) / 1024)), dim3(256), 0, s>>>(part, bias, y, numel, N, slices);
  return check_launch("mx_sum_slices");
}

int check_mx_product(const char* who, int64_t M, int64_t N, int64_t K) {
  TT_REQUIRE(M > 0 && N > 0 && K > 0 && K % kMxBlock == 0, "%s: bad shape M=%lld N=%lld K=%lld (K is a multiple of 32)", who, (long long)M, (long long)N, (long long)K);
  if (!(M < (1 << 30) && N < (1 << 30) && K < (1 << 22))) return fail(TTAMD_EUNSUPPORTED, "%s: M=%lld N=%lld K=%lld are too large", who, (long long)M, (long long)N, (long long)K);
  return TTAMD_OK;
}

}  // namespace ttamd

using namespace ttamd;

extern "C" size_t ttamd_mx_linear_workspace_bytes(int64_t M, int64_t N, int64_t K, int activation_format) {
  if (M <= 0 || N <= 0 || K <= 0 || K % kMxBlock || mx_few_quantises(M, K)) return 0;
  if (mx_few_applies(M, N)) return mx_operand_bytes(M, K, activation_format) + align256(mx_piece_bytes(M, K));
  return mx_operand_bytes(M, K, activation_format) + align256(mx_piece_bytes(M, K)) + align256(mx_piece_bytes(N, K)) + mx_gemm_part_bytes(M, N, K, activation_format);
}

extern "C" int ttamd_mx_linear_bf16(const void* x, int activation_format, const uint8_t* w_codes, const uint8_t* w_scales, const void* bias,
                                    void* y, int64_t M, int64_t N, int64_t K, void* workspace, size_t workspace_bytes, void* stream) {
  if (int rc = check_mx_product("mx_linear", M, N, K)) return rc;
  TT_REQUIRE(activation_format == TTAMD_MXFP4 || activation_format == TTAMD_MXFP8, "mx_linear: unknown format code %d", activation_format);
  TT_REQUIRE(x && w_codes && w_scales && y && aligned16(x) && aligned16(w_codes) && aligned16(w_scales) && aligned16(y) &&
                 (reinterpret_cast<uintptr_t>(bias) & 1u) == 0,
             "mx_linear: pointers must be non-null and 16-byte aligned");
  const size_t need = ttamd_mx_linear_workspace_bytes(M, N, K, activation_format);
  if (need > 0 && (workspace_bytes < need || !workspace || !aligned16(workspace)))
    return fail(TTAMD_EWORKSPACE, "mx_linear: needs %zu bytes of 16-byte aligned workspace, got %zu", need, workspace_bytes);
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (mx_few_quantises(M, K)) return run_mx_few(x, nullptr, nullptr, w_codes, w_scales, bias, y, M, N, K, activation_format, s);
  char* w = reinterpret_cast<char*>(workspace);
  MxProduct q = {};
  uint8_t* xc = reinterpret_cast<uint8_t*>(w);
  w += mx_operand_bytes(M, K, activation_format);
  uint8_t* xp = reinterpret_cast<uint8_t*>(w);
  w += align256(mx_piece_bytes(M, K));
  if (mx_few_applies(M, N)) {
    if (int rc = run_mx_quantize_operand(x, M, K, activation_format, xc, xp, nullptr, nullptr, nullptr, 0, s)) return rc;
    return run_mx_few(nullptr, xc, xp, w_codes, w_scales, bias, y, M, N, K, activation_format, s);
  }
  uint8_t* wp = reinterpret_cast<uint8_t*>(w);
  w += align256(mx_piece_bytes(N, K));
  if (int rc = run_mx_quantize_operand(x, M, K, activation_format, xc, xp, &w_scales, &N, &wp, 1, s)) return rc;
  q.x_codes = xc; q.x_pieces = xp; q.w_codes = w_codes; q.w_pieces = wp;
  q.bias = reinterpret_cast<const uint16_t*>(bias);
  q.y = reinterpret_cast<uint16_t*>(y);
  return run_mx_gemm(q, M, N, K, activation_format, reinterpret_cast<float*>(w), s);
}
