// Grad-input of frozen mxfp4 linears with a common input, for up to some thousand tokens without a dense copy of the
// weights:
//
//     gx[M, K] = sum_i gy_i[M, N_i] . W_i[N_i, K]  +  gh[M, R] . A[R, K]      (fp32 sums, one rounding)
//
// A weight's blocks run along K and the contraction runs along N, so the scales cannot be the matrix instruction's: the codes
// are expanded to bf16 (exactly: two significant bits times a power of two) on their way through LDS and the product runs on
// v_mfma_f32_16x16x32_bf16.  Workgroup: 8 waves, tile BM x 128 (BM 64, 128 or 256: the weight's share of a step is the same),
// step 64 of the contraction.  gy, codes and scales go HBM -> LDS by direct loads into a ring of five stages (three at 256
// rows); in step t the workgroup expands the weight rows of step t + 1 (a thread one half block) into one of two buffers and
// multiplies those of step t, read transposed (ds_read_b64_tr_b16).  One barrier per step, and all that a step reads from LDS
// is asked for right behind it, before the requests for memory: read, request, expand and multiply one after the other took
// 0.88 us a step of 128 rows instead of 0.73.  The contraction is cut into slices where the tiles do not fill the chip.  Bound:
// LDS and the way through it; the products alone would take 0.2 - 0.9 us a step.
#include "group.h"
#include "mx_math.h"

namespace ttamd {
namespace {

typedef float v4f __attribute__((ext_vector_type(4)));
typedef int v4i __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef short s16x4_t __attribute__((ext_vector_type(4)));
typedef short s16x8_t __attribute__((ext_vector_type(8)));

#define TT_LDS_PTR(p) ((__attribute__((address_space(3))) void*)(p))

struct MxDxArgs {
  const uint16_t* gy[kGroupMax];    // [M, N]
  const uint8_t* codes[kGroupMax];  // [N, K / 2]
  const uint8_t* scales[kGroupMax]; // [N, K / 32]
  int n[kGroupMax];
  const uint16_t* gh;               // [M, ldgh], the members' ranks side by side
  const uint16_t* la[kGroupMax];    // [rank, K]
  int rank_end[kGroupMax];
  uint16_t* gx;
  float* part;                      // [slices][M][K] or null
  int members, M, K, ldgh, steps, tiles_m, tiles_c, slices, steps_per_slice;
};

constexpr int kBC = 128, kStep = 64;
constexpr int kPitch = 2 * kBC + 32;  // four consecutive rows of a transposing read fall on disjoint banks
template <int BM>
struct MxDxTile {
  static constexpr int kGy = BM * 128, kCodes = kStep * kBC / 2, kScales = 8 * 256;  // of a stage, in bytes
  static constexpr int kStage = kGy + kCodes + kScales;
  static constexpr int kStages = BM <= 128 ? 5 : 3;  // what LDS holds
  static constexpr int kExpanded = kStep * kPitch;
  static constexpr int kLds = kStages * kStage + 2 * kExpanded;
  static constexpr int kLoadsGy = kGy / 8192;  // per wave
  static constexpr int kWavesM = BM / 64, kWavesC = 8 / kWavesM, TC = kBC / 16 / kWavesC;
  static_assert(kLds <= 160 * 1024, "LDS of a CU");
};

template <int BM>
__global__ __launch_bounds__(512) void mx_dx_kernel(const MxDxArgs g) {
#if defined(__HIP_DEVICE_COMPILE__)
  using T = MxDxTile<BM>;
  constexpr int TC = T::TC, TM = 4, kStages = T::kStages;
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  const int lane = threadIdx.x & 63, r16 = lane & 15, quarter = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave % T::kWavesM, wc = wave / T::kWavesM;
  auto uniform = [](int v) { return __builtin_amdgcn_readfirstlane(v); };
  // column tiles of the same rows and slice next to each other, rows of the same columns on the same XCD's turn
  int id = (int)blockIdx.x;
  const int slice = uniform(id / (g.tiles_m * g.tiles_c));
  id -= slice * g.tiles_m * g.tiles_c;
  const int tile_c = uniform(id / g.tiles_m), tile_m = id - tile_c * g.tiles_m;
  const int m0 = tile_m * BM, c0 = tile_c * kBC;
  const int s_begin = slice * g.steps_per_slice;
  const int s_end = s_begin + g.steps_per_slice < g.steps ? s_begin + g.steps_per_slice : g.steps;

  // ---- requests.  Buffer loads: rows beyond M and steps beyond the slice read zeros (a scale of zero is
  //      2^-127, and gy's rows are zero with it)
  const uint32_t lds0 = (uint32_t)(uintptr_t)TT_LDS_PTR(smem);
  auto dma16 = [&](uint32_t off, const void* base, int bytes, uint32_t lds) {
    const uint64_t p = (uint64_t)(uintptr_t)base;
    const v4i srd = {uniform((int)(uint32_t)p), uniform((int)((p >> 32) & 0xffff)), uniform(bytes > 0 ? bytes : 0), 0x00027000};
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds" ::"v"(off), "s"(srd), "s"(lds) : "memory", "m0");
  };
  auto dma4 = [&](uint32_t off, const void* base, int bytes, uint32_t lds) {
    const uint64_t p = (uint64_t)(uintptr_t)base;
    const v4i srd = {uniform((int)(uint32_t)p), uniform((int)((p >> 32) & 0xffff)), uniform(bytes > 0 ? bytes : 0), 0x00027000};
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_dword %0, %1, 0 offen lds" ::"v"(off), "s"(srd), "s"(lds) : "memory", "m0");
  };
  int p_step = s_begin, p_stage = 0, seg = 0, seg_begin = 0;  // the next step to request, and the member it lies in
  while (seg + 1 < g.members && p_step >= seg_begin + g.n[seg] / kStep) {
    seg_begin += g.n[seg] / kStep;
    ++seg;
  }
  // the member's addresses, read again only where the next member begins: a wait for the argument memory every step otherwise
  const uint16_t* gy_at;
  const uint8_t *codes_at, *scales_at;
  int N, n;  // row length and next column of gy
  auto enter = [&]() {
    N = g.n[seg];
    n = (p_step - seg_begin) * kStep;
    gy_at = g.gy[seg] + (int64_t)m0 * N;
    codes_at = g.codes[seg] + c0 / 2;
    scales_at = g.scales[seg] + c0 / 32;
  };
  enter();
  auto request = [&]() {
    const bool more = p_step < s_end;
    const uint32_t st = lds0 + p_stage * T::kStage;
    const int rows = g.M - m0 < BM ? g.M - m0 : BM;
    // gy: 8 rows of 128 bytes per instruction, piece p of a row at p ^ (row / 2) % 8
    const uint32_t off = (uint32_t)(lane >> 3) * (uint32_t)(2 * N) + 16u * (uint32_t)((lane & 7) ^ (lane >> 4));
#pragma unroll
    for (int i = 0; i < T::kLoadsGy; ++i) {
      const int q = wave * T::kLoadsGy + i;  // its parity flips the permutation's upper bit
      dma16((off ^ ((q & 1) ? 64u : 0u)) + (uint32_t)(q * 8) * (uint32_t)(2 * N), gy_at + n, more ? rows * 2 * N - 2 * n : 0,
            st + q * 1024);
    }
    // codes: 8 rows of 64 bytes per wave by its first 32 lanes; scales: a dword for each of its 8 rows (K is a multiple of kBC)
    const uint32_t c_off = (uint32_t)(8 * wave + (lane >> 2)) * (uint32_t)(g.K / 2) + 16u * (lane & 3);
    if (lane < 32)
      dma16(c_off, codes_at + (int64_t)n * (g.K / 2), more ? kStep * (g.K / 2) - c0 / 2 : 0, st + T::kGy + wave * 512);
    const uint32_t s_off = lane < 8 ? (uint32_t)(8 * wave + lane) * (uint32_t)(g.K / 32) : 0x7fffffffu;
    dma4(s_off, scales_at + (int64_t)n * (g.K / 32), more ? kStep * (g.K / 32) - c0 / 32 : 0, st + T::kGy + T::kCodes + wave * 256);
    p_stage = p_stage == kStages - 1 ? 0 : p_stage + 1;
    ++p_step;
    n += kStep;
    if (n >= N && seg + 1 < g.members) {
      seg_begin += N / kStep;
      ++seg;
      enter();
    }
  };

  // ---- expansion: thread t takes 16 elements of row t / 8: half t % 2 of block (t / 2) % 4
  const int e_row = threadIdx.x >> 3, e_part = threadIdx.x & 7;
  mx_u32x2 e_codes;
  uint32_t e_byte;
  auto expand_read = [&](int stage) {
    const char* st = smem + stage * T::kStage + T::kGy;
    e_codes = *reinterpret_cast<const mx_u32x2*>(st + e_row * 64 + 8 * e_part);
    e_byte = *reinterpret_cast<const uint8_t*>(st + T::kCodes + (e_row >> 3) * 256 + (e_row & 7) * 4 + (e_part >> 1));
  };
  auto expand_write = [&](int buffer) {
    const float s = mx_scale_value(e_byte == 255 ? 127u : e_byte);
    mx_u32x4 lo = mx_bf16_of_fp4(e_codes.x, s), hi = mx_bf16_of_fp4(e_codes.y, s);
    if (e_byte == 255) lo = hi = mx_u32x4{0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u};
    char* to = smem + kStages * T::kStage + buffer * T::kExpanded + e_row * kPitch + 32 * e_part;
    *reinterpret_cast<mx_u32x4*>(to) = lo;
    *reinterpret_cast<mx_u32x4*>(to + 16) = hi;
  };

  v4f acc[TC][TM];
#pragma unroll
  for (int j = 0; j < TC; ++j)
#pragma unroll
    for (int i = 0; i < TM; ++i) acc[j][i] = v4f{0.f, 0.f, 0.f, 0.f};

  const int ar = 64 * wm + r16;
  const int x_rd[2] = {ar * 128 + ((quarter ^ ((ar >> 1) & 7)) << 4), ar * 128 + (((4 + quarter) ^ ((ar >> 1) & 7)) << 4)};
  // a transposing read: lane i of quarter q points at row 8 q + i / 4 (+ 4), columns 4 (i % 4) .. + 3 of a 16-column block
  const int w_rd = kStages * T::kStage + (8 * quarter + (r16 >> 2)) * kPitch + 8 * (r16 & 3) + 2 * 16 * TC * wc;
  bf16x8_t xf[2][TM], wf[2][TC];  // operands of both halves of a step
  auto operands = [&](int stage, int buffer, int h) {
#pragma unroll
    for (int j = 0; j < TC; ++j) {
      const char* p = smem + w_rd + buffer * T::kExpanded + h * 32 * kPitch + j * 32;
      const s16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4_t*)(p));
      const s16x4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4_t*)(p + 4 * kPitch));
      const s16x8_t both = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
      wf[h][j] = __builtin_bit_cast(bf16x8_t, both);
    }
#pragma unroll
    for (int i = 0; i < TM; ++i) xf[h][i] = *reinterpret_cast<const bf16x8_t*>(smem + stage * T::kStage + x_rd[h] + i * 2048);
  };
  auto multiply = [&](int h) {
#pragma unroll
    for (int j = 0; j < TC; ++j)
#pragma unroll
      for (int i = 0; i < TM; ++i) acc[j][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wf[h][j], xf[h][i], acc[j][i], 0, 0, 0);
  };

  // ---- pipeline.  At step t a wave waits until what it requested for step t + 1 has landed and its own expansion of step t
  //      is in LDS, and passes the barrier: everybody's is, and everybody is done with step t - 1, whose stage takes the
  //      request of step t + 4 (five stages).  Newer than stage t + 1 are the loads of stages t + 2 and t + 3.
  constexpr int kLoads = T::kLoadsGy + 2;
  for (int i = 0; i < kStages - 1; ++i) request();
  asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"((kStages - 2) * kLoads) : "memory");
  expand_read(0);
  expand_write(0);
  int stage = 0;
  for (int t = s_begin; t < s_end; ++t) {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((kStages - 3) * kLoads) : "memory");
    const int next = stage == kStages - 1 ? 0 : stage + 1, buffer = (t - s_begin) & 1;
    expand_read(next);  // behind the last step: zeros
    operands(stage, buffer, 0);
    operands(stage, buffer, 1);
    request();
    expand_write(buffer ^ 1);
    multiply(0);
    multiply(1);
    stage = next;
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");

  // ---- adapters: 64 ranks as one more step, A's rows where the weight's were, gh from memory
  if (slice == 0 && g.ldgh > 0) {
    __syncthreads();
    const int r = threadIdx.x >> 3, part = threadIdx.x & 7;  // a thread copies 16 elements of row r of the members' stacked A
    int which = 0, first = 0;
    while (which + 1 < g.members && r >= g.rank_end[which]) first = g.rank_end[which++];
    mx_u32x4 lo = {0, 0, 0, 0}, hi = {0, 0, 0, 0};
    if (r < g.ldgh) {
      const mx_u32x4* p = reinterpret_cast<const mx_u32x4*>(g.la[which] + (int64_t)(r - first) * g.K + c0 + 16 * part);
      lo = p[0];
      hi = p[1];
    }
    char* to = smem + kStages * T::kStage + r * kPitch + 32 * part;
    *reinterpret_cast<mx_u32x4*>(to) = lo;
    *reinterpret_cast<mx_u32x4*>(to + 16) = hi;
    __syncthreads();
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (32 * h >= g.ldgh) break;
      bf16x8_t xf[TM];
#pragma unroll
      for (int i = 0; i < TM; ++i) {
        int row = m0 + ar + 16 * i;
        row = row < g.M ? row : g.M - 1;
        const int k = 32 * h + 8 * quarter;
        mx_u32x4 v = {0, 0, 0, 0};
        if (k < g.ldgh) v = *reinterpret_cast<const mx_u32x4*>(g.gh + (int64_t)row * g.ldgh + k);
        xf[i] = __builtin_bit_cast(bf16x8_t, v);
      }
#pragma unroll
      for (int j = 0; j < TC; ++j) {
        const char* p = smem + w_rd + h * 32 * kPitch + j * 32;
        const s16x4_t a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4_t*)(p));
        const s16x4_t b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4_t*)(p + 4 * kPitch));
        const s16x8_t both = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
        for (int i = 0; i < TM; ++i) acc[j][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, both), xf[i], acc[j][i], 0, 0, 0);
      }
    }
  }

  // ---- outputs: a lane holds columns 4 q .. + 3 of each 16-wide tile in its row
#pragma unroll
  for (int i = 0; i < TM; ++i) {
    const int row = m0 + ar + 16 * i;
    if (row >= g.M) continue;
    if (g.slices > 1) {
#pragma unroll
      for (int j = 0; j < TC; ++j) {
        const int c = c0 + 16 * (TC * wc + j) + 4 * quarter;
        *reinterpret_cast<v4f*>(g.part + ((int64_t)slice * g.M + row) * g.K + c) = acc[j][i];
      }
    } else {
#pragma unroll
      for (int j = 0; j < TC; ++j) {
        const int c = c0 + 16 * (TC * wc + j) + 4 * quarter;
        typedef __bf16 bf16x4_t __attribute__((ext_vector_type(4)));
        bf16x4_t o;
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = (__bf16)acc[j][i][e];
        *reinterpret_cast<bf16x4_t*>(g.gx + (int64_t)row * g.K + c) = o;
      }
    }
  }
#endif
}

struct MxDxPlan {
  int bm, slices, steps_per_slice;
  bool fused;  // else: the weights expanded to bf16 tiles in memory, and the dense product on them
};

// The fused kernel against the dense product on expanded weights, tile height and slices: the least of a fitted time in us
// (steps of 64; a workgroup fills a CU, so 256 run in one turn).  Fused, a turn's step takes 0.60 us at 64 rows, 0.73 at 128 and
// 1.0 at 256, however few CUs have work; slices write and read fp32 partial sums.  The dense product's 256-wide tiles take 0.92
// a step on a nearly idle chip and 1.42 on a full one, where power bounds them, and the expansion writes two bytes an element.
// Measured, fused against both of the others (us): 24 x 2048 -> 2048 10.6 / 39; 350 x 2048 -> 2048 17.9 / 38; 350 x 6144 ->
// 4096 39 / 103; 1024 x 6144 -> 4096 64 / 106; 1500 x 6144 -> 4096 98 / 112; 350 x 14336 -> 4096 70 / 229; 1024 x 14336 -> 4096
// 127 / 232; 350 x 4096 -> 14336 69 / 93, but 1024 134 / 120.
MxDxPlan plan_dx(int64_t M, int64_t n_total, int64_t K) {
  const int64_t steps = n_total / kStep;
  const int64_t dense_tiles = ((M + 255) / 256) * ((K + 255) / 256);
  const float fill = dense_tiles < 256 ? (float)dense_tiles / 256.f : 1.f;
  float best = 6.f + (float)((dense_tiles + 255) / 256) * (float)steps * (0.92f + 0.5f * fill * fill) + (float)n_total * (float)K * 4.6e-7f;
  MxDxPlan p = {0, 1, 0, false};
  if (K % kBC) return p;  // whole column tiles, whose rows of scales are dwords
  for (int bm = 64; bm <= 256; bm *= 2) {
    const int64_t tiles = ((M + bm - 1) / bm) * (K / kBC);
    for (int64_t slices = 1; slices <= 16; slices *= 2) {
      const int64_t per = (steps + slices - 1) / slices;
      if ((steps + per - 1) / per != slices) continue;
      if (slices > 1 && (per < 3 || slices * M * K > (int64_t(1) << 26))) break;
      float time = 3.f + (float)((tiles * slices + 255) / 256) * (float)per * (bm == 64 ? 0.60f : bm == 128 ? 0.73f : 1.0f);
      if (slices > 1) time += 3.f + (float)(slices * M * K) * 2e-6f;
      if (time < best) {
        best = time;
        p = MxDxPlan{bm, (int)slices, (int)per, true};
      }
    }
  }
  return p;
}

template <int BM>
int launch_dx(MxDxArgs& g, hipStream_t s) {
  using T = MxDxTile<BM>;
  static bool attr_set[64] = {};  // the LDS limit is a per-device attribute of the function (a race only repeats the call)
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) dev = -1;
  if (dev < 0 || !attr_set[dev]) {
    hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(&mx_dx_kernel<BM>), hipFuncAttributeMaxDynamicSharedMemorySize, T::kLds);
    if (e != hipSuccess) return fail(TTAMD_ELAUNCH, "mx_dx: cannot reserve %d bytes of LDS: %s", T::kLds, hipGetErrorString(e));
    if (dev >= 0) attr_set[dev] = true;
  }
  g.tiles_m = (g.M + BM - 1) / BM;
  g.tiles_c = g.K / kBC;
  mx_dx_kernel<BM><<<dim3((unsigned)(g.tiles_m * g.tiles_c * g.slices)), dim3(512), T::kLds, s>>>(g);
  return check_launch("mx_dx");
}

size_t align256(size_t v) { return (v + 255) & ~size_t(255); }

}  // namespace

bool mx_dx_fused(int64_t M, int64_t n_total, int64_t K) { return plan_dx(M, n_total, K).fused; }

size_t mx_dx_fused_bytes(int64_t M, int64_t n_total, int64_t K) {
  const MxDxPlan p = plan_dx(M, n_total, K);
  return p.slices > 1 ? align256((size_t)p.slices * M * K * sizeof(float)) : 0;
}

int run_mx_dx(const GroupDx& d, const uint8_t* const* codes, const uint8_t* const* scales, const void* gh_cat, void* gx, float* part, hipStream_t s) {
  MxDxArgs g = {};
  int64_t n_total = 0;
  g.members = d.n;
  for (int i = 0; i < d.n; ++i) {
    g.gy[i] = d.gy[i];
    g.codes[i] = codes[i];
    g.scales[i] = scales[i];
    g.n[i] = (int)d.N[i];
    g.la[i] = d.lora_a[i];
    g.rank_end[i] = d.r_off[i + 1];
    n_total += d.N[i];
  }
  const MxDxPlan p = plan_dx(d.M, n_total, d.K);
  TT_REQUIRE(p.fused && d.K % kBC == 0, "mx_dx: K (%lld) is taken in whole column tiles of %d", (long long)d.K, kBC);
  g.gh = reinterpret_cast<const uint16_t*>(gh_cat);
  g.gx = reinterpret_cast<uint16_t*>(gx);
  g.part = part;
  g.M = (int)d.M; g.K = (int)d.K; g.ldgh = d.r_off[d.n]; g.steps = (int)(n_total / kStep);
  g.slices = p.slices; g.steps_per_slice = p.steps_per_slice;
  TT_REQUIRE(p.slices == 1 || part, "mx_dx: no room for the slices of the contraction");
  const int rc = p.bm == 64 ? launch_dx<64>(g, s) : p.bm == 128 ? launch_dx<128>(g, s) : launch_dx<256>(g, s);
  return rc || p.slices == 1 ? rc : run_mx_sum_slices(part, nullptr, g.gx, d.M * d.K, (int)d.K, p.slices, s);
}

}  // namespace ttamd
