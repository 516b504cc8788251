// Microscaled tensors: a bf16 / fp32 tensor into blocks of 32 with a shared power-of-two scale (mxfp4, mxfp8) and back.
// (The format is the OCP one, scales rounded down.)
//
//     e = max(floor(log2(max |v|)) - emax, -127),  code = RNE(v / 2^e) saturated,  value = code * 2^e
//
// Every step is exact but the one rounding, so any correct implementation gives the same bits.  Bound: HBM.  Four lanes
// share a block: a lane loads eight elements as one or two 16-byte pieces (a wave's loads are contiguous), takes their
// largest magnitude on the bit patterns, meets its three neighbours by quad permutes, and converts with gfx950's scaled
// conversions (two elements per instruction).  One workgroup covers kChunks * 256 pieces so that each thread has that many
// loads in flight.
#include "mx_math.h"

namespace ttamd {
namespace {

constexpr int kChunks = 4;  // pieces of eight elements per thread

struct OperandWeights {  // weights whose scales the quantise launch of an input lays out for the product
  const uint8_t* scales[kMxWeights];
  uint8_t* pieces[kMxWeights];
  int64_t rows[kMxWeights];
  int blk_end[kMxWeights];
  int n;
};

__device__ __forceinline__ uint32_t umax(uint32_t a, uint32_t b) { return a > b ? a : b; }

// largest biased exponent of eight elements
struct Bf16x8 {
  mx_u32x4 v;
  __device__ __forceinline__ void load(const void* p, int64_t i) { v = reinterpret_cast<const mx_u32x4*>(p)[i]; }
  __device__ __forceinline__ void clear() { v = mx_u32x4{0, 0, 0, 0}; }
  __device__ __forceinline__ uint32_t exponent() const { return mx_bf16_exponent(v); }
};
struct F32x8 {
  float v[8];
  __device__ __forceinline__ void load(const void* p, int64_t i) {
    typedef float f32x4 __attribute__((ext_vector_type(4)));
    const f32x4 a = reinterpret_cast<const f32x4*>(p)[2 * i], b = reinterpret_cast<const f32x4*>(p)[2 * i + 1];
#pragma unroll
    for (int q = 0; q < 4; ++q) { v[q] = a[q]; v[4 + q] = b[q]; }
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int q = 0; q < 8; ++q) v[q] = 0.f;
  }
  __device__ __forceinline__ uint32_t exponent() const {
    uint32_t m = 0;
#pragma unroll
    for (int q = 0; q < 8; ++q) m = umax(m, __builtin_bit_cast(uint32_t, v[q]) & 0x7fffffffu);
    return m >> 23;
  }
};

#if defined(__HIP_DEVICE_COMPILE__)
// codes of one piece (zeros for a block of NaN) and the block's scale byte
template <int FMT, typename V>
__device__ __forceinline__ mx_u32x2 encode(const V& e, uint32_t& byte) {
  byte = mx_scale_byte(mx_quad_max(e.exponent()), FMT);
  const float s = mx_scale_value(byte == 255 ? 127u : byte);
  mx_u32x2 c = {0, 0};
  if constexpr (FMT == TTAMD_MXFP4)
    c.x = mx_pack4(e.v, s);
  else
    c = mx_pack8(e.v, s);
  if (byte == 255) c = mx_u32x2{0, 0};
  return c;
}
template <int FMT>
__device__ __forceinline__ void store_codes(uint8_t* codes, int64_t piece, mx_u32x2 c) {
  if constexpr (FMT == TTAMD_MXFP4)
    reinterpret_cast<uint32_t*>(codes)[piece] = c.x;
  else
    reinterpret_cast<mx_u32x2*>(codes)[piece] = c;
}
// One workgroup's share of the weights' scales in the product's layout: a thread one piece of 16, a wave four pieces of each of
// 16 rows: it reads 64 bytes of a row and writes 256 bytes of a group.
__device__ __forceinline__ void lay_out_scales(int blk, int K, const OperandWeights& w) {
  int which = 0;
#pragma unroll
  for (int q = 0; q < kMxWeights - 1; ++q)
    if (q < w.n - 1 && blk >= w.blk_end[q]) which = q + 1;
  if (which) blk -= w.blk_end[which - 1];
  const int nb = K / kMxBlock, groups = (nb + 15) >> 4, quads = (groups + 3) >> 2;
  const int64_t wave = (int64_t)blk * (blockDim.x >> 6) + (threadIdx.x >> 6), rows = w.rows[which];
  const int lane = threadIdx.x & 63;
  const int64_t row = wave / quads * 16 + (lane & 15);
  const int g = (int)(wave % quads) * 4 + (lane >> 4);
  if (row >= rows || g >= groups) return;
  const uint8_t* src = w.scales[which] + row * nb + 16 * g;
  mx_u32x4 d = {0, 0, 0, 0};
  if ((nb & 15) == 0) {
    d = *reinterpret_cast<const mx_u32x4*>(src);
  } else {
#pragma unroll
    for (int q = 0; q < 16; ++q) {  // no load within a branch, or they wait for each other
      const int left = nb - 16 * g;
      const uint32_t byte = src[q < left ? q : left - 1];
      d[q >> 2] |= (q < left ? byte : 0u) << (8 * (q & 3));
    }
  }
  // byte 4 s + q -> byte 4 q + s
  const uint32_t t0 = __builtin_amdgcn_perm(d.y, d.x, 0x05010400u), t1 = __builtin_amdgcn_perm(d.y, d.x, 0x07030602u);
  const uint32_t u0 = __builtin_amdgcn_perm(d.w, d.z, 0x05010400u), u1 = __builtin_amdgcn_perm(d.w, d.z, 0x07030602u);
  const mx_u32x4 o = {__builtin_amdgcn_perm(u0, t0, 0x05040100u), __builtin_amdgcn_perm(u0, t0, 0x07060302u),
                      __builtin_amdgcn_perm(u1, t1, 0x05040100u), __builtin_amdgcn_perm(u1, t1, 0x07060302u)};
  reinterpret_cast<mx_u32x4*>(w.pieces[which])[(int64_t)g * rows + row] = o;
}
#endif

template <typename V, int FMT>
__global__ __launch_bounds__(256) void mx_quantize_kernel(const void* __restrict__ x, int64_t pieces, uint8_t* __restrict__ codes,
                                                          uint8_t* __restrict__ scales) {
#if defined(__HIP_DEVICE_COMPILE__)
  mx_saturate_fp8();
  const int64_t p0 = (int64_t)blockIdx.x * (256 * kChunks) + threadIdx.x;
  V e[kChunks];
#pragma unroll
  for (int u = 0; u < kChunks; ++u) {
    e[u].clear();
    if (p0 + 256 * u < pieces) e[u].load(x, p0 + 256 * u);
  }
#pragma unroll
  for (int u = 0; u < kChunks; ++u) {
    const int64_t p = p0 + 256 * u;  // pieces is a multiple of 4: a block's four lanes are all in or all out
    uint32_t byte;
    const mx_u32x2 c = encode<FMT>(e[u], byte);
    if (p >= pieces) continue;
    store_codes<FMT>(codes, p, c);
    if ((threadIdx.x & 3) == 0) scales[p >> 2] = (uint8_t)byte;
  }
#endif
}

// An input for the products: codes with the row padded to 256 elements by zeros, scales in the products' own layout, and -
// workgroups past the input's - the weights' scales in that layout (17 / 32 of a byte per element is all there is of a
// weight, a sixteenth of it scales: their copy costs a launch more than it costs time).
template <int FMT>
__global__ __launch_bounds__(256) void mx_quantize_operand_kernel(const void* __restrict__ x, int64_t M, int K, int Kp,
                                                                  uint8_t* __restrict__ codes, uint8_t* __restrict__ xp,
                                                                  int x_blocks, const OperandWeights w) {
#if defined(__HIP_DEVICE_COMPILE__)
  if ((int)blockIdx.x >= x_blocks) return lay_out_scales((int)blockIdx.x - x_blocks, K, w);
  mx_saturate_fp8();
  const uint32_t per_row = (uint32_t)Kp >> 3, real = (uint32_t)K >> 3;
  const int64_t c0 = (int64_t)blockIdx.x * (256 * kChunks);
  const int64_t row0 = c0 / per_row;
  const uint32_t rem = (uint32_t)(c0 - row0 * per_row) + threadIdx.x;
  Bf16x8 e[kChunks];
  int64_t row[kChunks];
  uint32_t col[kChunks];
#pragma unroll
  for (int u = 0; u < kChunks; ++u) {
    const uint32_t t = rem + 256 * u, r = t / per_row;
    row[u] = row0 + r;
    col[u] = t - r * per_row;
    e[u].clear();
    if (row[u] < M && col[u] < real) e[u].load(x, row[u] * real + col[u]);
  }
#pragma unroll
  for (int u = 0; u < kChunks; ++u) {
    uint32_t byte;
    const mx_u32x2 c = encode<FMT>(e[u], byte);
    if (row[u] >= M) continue;
    store_codes<FMT>(codes, row[u] * per_row + col[u], c);
    const uint32_t blk = col[u] >> 2;
    if ((threadIdx.x & 3) == 0) xp[((int64_t)(blk >> 4) * M + row[u]) * 16 + mx_piece_byte(blk & 15)] = (uint8_t)byte;
  }
#endif
}

template <int FMT, bool F32>
__global__ __launch_bounds__(256) void mx_dequantize_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales,
                                                            int64_t pieces, void* __restrict__ out) {
#if defined(__HIP_DEVICE_COMPILE__)
  const int64_t p0 = (int64_t)blockIdx.x * (256 * kChunks) + threadIdx.x;
  mx_u32x2 c[kChunks];
  uint32_t b[kChunks];
#pragma unroll
  for (int u = 0; u < kChunks; ++u) {
    const int64_t p = p0 + 256 * u;
    c[u] = mx_u32x2{0, 0};
    b[u] = 0;
    if (p >= pieces) continue;
    if constexpr (FMT == TTAMD_MXFP4)
      c[u].x = reinterpret_cast<const uint32_t*>(codes)[p];
    else
      c[u] = reinterpret_cast<const mx_u32x2*>(codes)[p];
    b[u] = scales[p >> 2];
  }
#pragma unroll
  for (int u = 0; u < kChunks; ++u) {
    const int64_t p = p0 + 256 * u;
    if (p >= pieces) continue;
    // the conversion takes a scale's exponent only: a block of NaN is written as such
    const float s = mx_scale_value(b[u] == 255 ? 127u : b[u]);
    if constexpr (F32) {
      float v[8];
      if constexpr (FMT == TTAMD_MXFP4)
        mx_f32_of_fp4(c[u].x, s, v);
      else
        mx_f32_of_fp8(c[u], s, v);
      typedef float f32x4 __attribute__((ext_vector_type(4)));
      f32x4 lo, hi;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        lo[q] = b[u] == 255 ? __builtin_bit_cast(float, 0x7fc00000u) : v[q];
        hi[q] = b[u] == 255 ? __builtin_bit_cast(float, 0x7fc00000u) : v[4 + q];
      }
      reinterpret_cast<f32x4*>(out)[2 * p] = lo;
      reinterpret_cast<f32x4*>(out)[2 * p + 1] = hi;
    } else {
      mx_u32x4 o;
      if constexpr (FMT == TTAMD_MXFP4)
        o = mx_bf16_of_fp4(c[u].x, s);
      else
        o = mx_bf16_of_fp8(c[u], s);
      if (b[u] == 255) o = mx_u32x4{0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u};
      reinterpret_cast<mx_u32x4*>(out)[p] = o;
    }
  }
#endif
}

// The same for the input of adapter linears, with h = bf16(x^ . A^T) (A the members' rank x K matrices one below the other) from
// the registers that hold x^.  Workgroup: 16 rows; its 8 waves take the row in turns of 256 elements and add up in LDS, in a
// fixed order.  Lane l holds row l % 16, elements 8 (l / 16) .. + 7 of each block: the four lanes of a block meet by lane-quarter
// swaps, and the codes, taken back to bf16, are operands of v_mfma_f32_16x16x32_bf16 as they lie.  (A lane with whole blocks
// needs no neighbour, but its 16-byte loads lie 64 bytes apart: 137 us instead of 132 at 8192 x 14336, rank 16.)  Bound: HBM,
// beside some 600 vector instructions a turn and A, which every 16 rows read again from L2: 103 us at that size behind other work.
constexpr int kHiddenWaves = 8, kHiddenTurn = 256;
struct HiddenMembers {
  const uint16_t* la[kMxWeights];  // [rank, K]
  int r_end[kMxWeights];
  int n;
};
#if defined(__HIP_DEVICE_COMPILE__)
// the larger of each half over both sides of a lane swap of a value with itself
template <typename P>
__device__ __forceinline__ uint32_t max_u16x2(P swapped) {
  typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
  const uint32_t a = swapped[0], b = swapped[1];
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, a), __builtin_bit_cast(u16x2, b)));
}
#endif
// The next turn's x is asked for before this one's codes are stored, its share of A behind the products that read this one's,
// and codes leave by way of LDS as 256 bytes of a row: 109 -> 89 us at 8192 x 14336 rank 16 with x in the caches (4.0 TB/s).
// Up to 16 ranks half of A's share at a time leaves registers for two workgroups on a CU (8192 x 2048 17.2 -> 13.6 us, 8192 x 4096
// 28.2 -> 25.0, at 14336 level); with 32 they spill (8192 x 4096 34.9 -> 36.4).
template <int RT>  // groups of 16 ranks
__global__ __launch_bounds__(64 * kHiddenWaves) __attribute__((amdgpu_waves_per_eu(RT == 1 ? 4 : 2, RT == 1 ? 4 : 2))) void mx_quantize_hidden_kernel(const uint16_t* __restrict__ x, int64_t M, int K, int Kp,
                                                                              uint8_t* __restrict__ codes, uint8_t* __restrict__ xp,
                                                                              const HiddenMembers a, uint16_t* __restrict__ h,
                                                                              float* __restrict__ part, int slices, int k_slice, int x_blocks,
                                                                              const OperandWeights w) {
#if defined(__HIP_DEVICE_COMPILE__)
  typedef float f32x4 __attribute__((ext_vector_type(4)));
  typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
  if ((int)blockIdx.x >= x_blocks) return lay_out_scales((int)blockIdx.x - x_blocks, K, w);
  constexpr int kPitch = kHiddenTurn + 32;  // of a row of codes on their way out: its lanes' eight bytes on disjoint banks
  constexpr int kWaveLds = (16 * kPitch + 1023) / 1024 * 1024;
  static_assert(kWaveLds >= 1024 * RT, "the sums reuse the memory");
  __shared__ __attribute__((aligned(16))) char lds[kHiddenWaves * kWaveLds];
  const int lane = threadIdx.x & 63, r16 = lane & 15, quarter = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t tile = blockIdx.x / slices, row = tile * 16 + r16;
  const int slice = (int)(blockIdx.x - tile * slices), k_end = (slice + 1) * k_slice < Kp ? (slice + 1) * k_slice : Kp;
  const bool live = row < M;
  const int ranks = a.r_end[a.n - 1];
  const uint16_t* la[RT];  // lane's rank of each group; beyond the last one it computes what nobody stores
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    int r = 16 * t + r16;
    r = r < ranks ? r : 0;
    int which = 0;
#pragma unroll
    for (int q = 0; q < kMxWeights - 1; ++q)
      if (q < a.n - 1 && r >= a.r_end[q]) which = q + 1;
    la[t] = a.la[which] + (int64_t)(r - (which ? a.r_end[which - 1] : 0)) * K;
  }
  f32x4 acc[RT];
#pragma unroll
  for (int t = 0; t < RT; ++t) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};

  constexpr int kAhead = RT == 1 ? 4 : 8;  // blocks whose share of A is in registers
  mx_u32x4 v[8], b[RT][kAhead];  // of block j this lane's quarter
  auto load_x = [&](int k0) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      v[j] = mx_u32x4{0, 0, 0, 0};
      if (live && k0 + 32 * j < K) v[j] = *reinterpret_cast<const mx_u32x4*>(x + row * K + k0 + 32 * j + 8 * quarter);
    }
  };
  auto load_a = [&](int k0) {
#pragma unroll
    for (int t = 0; t < RT; ++t)
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        b[t][j] = mx_u32x4{0, 0, 0, 0};
        if (k0 + 32 * j < K) b[t][j] = *reinterpret_cast<const mx_u32x4*>(la[t] + k0 + 32 * j + 8 * quarter);
      }
  };
  char* out = lds + wave * kWaveLds;
  int k0 = slice * k_slice + kHiddenTurn * wave;
  if (k0 < k_end) {
    load_x(k0);
    load_a(k0);
  }
  for (; k0 < k_end; k0 += kHiddenTurn * kHiddenWaves) {
    const int next = k0 + kHiddenTurn * kHiddenWaves;
    // conversions saturate between the two settings of the mode; the pins hold them there
    mx_saturate_fp8();
    uint32_t byte[8];
    mx_u32x2 c[8];
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
      asm volatile("" : "+v"(v[j]), "+v"(v[j + 1]));
      uint32_t e = mx_bf16_exponent(v[j]) | mx_bf16_exponent(v[j + 1]) << 16;  // of both blocks, met across the lane quarters
      e = max_u16x2(__builtin_amdgcn_permlane32_swap(e, e, false, false));
      e = max_u16x2(__builtin_amdgcn_permlane16_swap(e, e, false, false));
#pragma unroll
      for (int i = j; i < j + 2; ++i) {
        byte[i] = mx_scale_byte(i == j ? e & 0xffffu : e >> 16, TTAMD_MXFP8);
        c[i] = mx_pack8(v[i], mx_scale_value(byte[i] == 255 ? 127u : byte[i]));
        if (byte[i] == 255) c[i] = mx_u32x2{0, 0};
        asm volatile("" : "+v"(c[i]));
      }
    }
    mx_saturate_fp8(false);
    if (next < k_end) load_x(next);
    // codes by way of LDS (a wave's own, whose accesses go in order), so that they leave as 256 bytes of a row
#pragma unroll
    for (int j = 0; j < 8; ++j) *reinterpret_cast<mx_u32x2*>(out + r16 * kPitch + 32 * j + 8 * quarter) = c[j];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const mx_u32x4 piece = *reinterpret_cast<const mx_u32x4*>(out + (4 * i + quarter) * kPitch + 16 * r16);
      const int64_t to = tile * 16 + 4 * i + quarter;
      if (to < M) *reinterpret_cast<mx_u32x4*>(codes + to * Kp + k0 + 16 * r16) = piece;  // Kp is a multiple of 256
    }
    if (live) {
      uint32_t two = byte[0] | byte[4] << 8;  // blocks q and 4 + q lie next to each other in the piece
#pragma unroll
      for (int q = 1; q < 4; ++q) two = quarter == q ? byte[q] | byte[4 + q] << 8 : two;
      *reinterpret_cast<uint16_t*>(xp + ((int64_t)(k0 >> 9) * M + row) * 16 + 4 * quarter + 2 * ((k0 >> 8) & 1)) = (uint16_t)two;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      mx_u32x4 e = mx_bf16_of_fp8(c[j], mx_scale_value(byte[j] == 255 ? 127u : byte[j]));
      if (byte[j] == 255) e = mx_u32x4{0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u};
#pragma unroll
      for (int t = 0; t < RT; ++t)
        acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, e), __builtin_bit_cast(bf16x8, b[t][j % kAhead]), acc[t], 0, 0, 0);
      if (kAhead < 8 && j == kAhead - 1) load_a(k0 + 32 * kAhead);
    }
    if (next < k_end) load_a(next);
  }
  f32x4 (*sums)[kWaveLds / 1024][64] = reinterpret_cast<f32x4 (*)[kWaveLds / 1024][64]>(lds);
  __syncthreads();  // the codes' places are free
#pragma unroll
  for (int t = 0; t < RT; ++t) sums[wave][t][lane] = acc[t];
  __syncthreads();
  // lane l's element v of group t: row 4 (l / 16) + v, rank 16 t + l % 16
  for (int i = threadIdx.x; i < RT * 256; i += 64 * kHiddenWaves) {
    const int l = i & 63, e = (i >> 6) & 3, t = i >> 8;
    float s = 0.f;
#pragma unroll
    for (int q = 0; q < kHiddenWaves; ++q) s += sums[q][t][l][e];
    const int64_t to = tile * 16 + 4 * (l >> 4) + e;
    const int r = 16 * t + (l & 15);
    if (to >= M || r >= ranks) continue;
    if (slices > 1)
      part[(slice * M + to) * ranks + r] = s;
    else
      h[to * ranks + r] = __builtin_bit_cast(uint16_t, (__bf16)s);
  }
#endif
}

// The mxfp4 weight [N, K] as bf16 in the operand order of the dense GEMM's forward tiles, tiled[N / 16][K / 32][64 lanes][8]
// (its grad-input launch reads those through transposing LDS loads).  A thread takes the 32 contraction indices of one
// block and writes the four 16-byte operands they make; a workgroup takes 16 rows x 16 blocks.  Bound: HBM, 2.53 bytes per
// element, written in pieces of 16 x 16 bytes.
__global__ __launch_bounds__(256) void mx_expand_tiles_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales,
                                                              int nk, char* __restrict__ tiles) {
#if defined(__HIP_DEVICE_COMPILE__)
  const int T = blockIdx.x, r = threadIdx.x & 15;
  const int t = 16 * (int)blockIdx.y + (int)(threadIdx.x >> 4);
  if (t >= nk) return;
  const int64_t blk = (int64_t)(16 * T + r) * nk + t;
  const mx_u32x4 cd = reinterpret_cast<const mx_u32x4*>(codes)[blk];
  const uint32_t b = scales[blk];
  const float s = mx_scale_value(b == 255 ? 127u : b);
  char* piece = tiles + ((int64_t)T * nk + t) * 1024;
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    mx_u32x4 o = mx_bf16_of_fp4(cd[g], s);
    if (b == 255) o = mx_u32x4{0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u};
    *reinterpret_cast<mx_u32x4*>(piece + (16 * g + r) * 16) = o;
  }
#endif
}

int64_t blocks_of(int64_t pieces) { return (pieces + 256 * kChunks - 1) / (256 * kChunks); }

int check_codec(const char* who, int dtype, int64_t rows, int64_t K, int format) {
  TT_REQUIRE(dtype == TTAMD_BF16 || dtype == TTAMD_F32, "%s: unknown dtype code %d", who, dtype);
  TT_REQUIRE(format == TTAMD_MXFP4 || format == TTAMD_MXFP8, "%s: unknown format code %d", who, format);
  TT_REQUIRE(rows >= 0 && K > 0 && K % kMxBlock == 0, "%s: K (%lld) must be a positive multiple of 32 (rows %lld)", who, (long long)K, (long long)rows);
  if (rows > 0 && K > (int64_t(1) << 40) / rows) return fail(TTAMD_EUNSUPPORTED, "%s: %lld x %lld elements are too many for one launch", who, (long long)rows, (long long)K);
  return TTAMD_OK;
}

}  // namespace

namespace {
// the weights whose scales a launch lays out, `threads` pieces to a workgroup; their workgroups
int64_t operand_weights(OperandWeights& w, const uint8_t* const* scales, const int64_t* rows, uint8_t* const* pieces, int n, int64_t K, int threads) {
  w = OperandWeights{};
  w.n = n;
  int64_t blocks = 0;
  for (int i = 0; i < n; ++i) {
    w.scales[i] = scales[i];
    w.pieces[i] = pieces[i];
    w.rows[i] = rows[i];
    blocks += ((rows[i] + 15) / 16 * ((mx_groups(K) + 3) / 4) * 64 + threads - 1) / threads;
    w.blk_end[i] = (int)blocks;
  }
  return blocks;
}
}  // namespace

int run_mx_quantize_operand(const void* x, int64_t M, int64_t K, int fmt, uint8_t* codes, uint8_t* pieces, const uint8_t* const* w_scales,
                            const int64_t* w_rows, uint8_t* const* w_pieces, int n_weights, hipStream_t s) {
  OperandWeights w;
  const int64_t Kp = mx_padded_k(K), xb = blocks_of(M * (Kp / 8)), wb = operand_weights(w, w_scales, w_rows, w_pieces, n_weights, K, 256);
  if (xb + wb >= (int64_t(1) << 31)) return fail(TTAMD_EUNSUPPORTED, "mx_quantize_operand: M=%lld K=%lld are too large for one launch", (long long)M, (long long)K);
  if (fmt == TTAMD_MXFP4)
    mx_quantize_operand_kernel<TTAMD_MXFP4><<<dim3((unsigned)(xb + wb)), dim3(256), 0, s>>>(x, M, (int)K, (int)Kp, codes, pieces, (int)xb, w);
  else
    mx_quantize_operand_kernel<TTAMD_MXFP8><<<dim3((unsigned)(xb + wb)), dim3(256), 0, s>>>(x, M, (int)K, (int)Kp, codes, pieces, (int)xb, w);
  return check_launch("mx_quantize_operand");
}

namespace {
struct HiddenPlan {
  int slices, k_slice;
};
// A workgroup's round (its eight waves a turn each, 2048 elements of 16 rows) takes 1.9 us and 1.7 more per 16 ranks, what a CU
// takes in of such loads; with few rows the rounds are dealt to several workgroups where that saves more than the launch that
// adds their sums (5 us).  Measured without and with (us): 350 x 14336 rank 16 30.3 / 11.6, rank 64 66.6 / 17.6; 1500 x 14336
// rank 16 32.1 / 23.2; 24 x 4096 rank 64 21.8 / 14.5.
HiddenPlan plan_hidden(int64_t M, int64_t K, int ranks) {
  const int64_t round = kHiddenTurn * kHiddenWaves, rounds = (mx_padded_k(K) + round - 1) / round, tiles = (M + 15) / 16;
  HiddenPlan p = {1, (int)(rounds * round)};
  const int64_t most = 256 / tiles < rounds ? 256 / tiles : rounds;
  if (most < 2) return p;
  const int64_t per = (rounds + most - 1) / most;
  if ((float)(rounds - per) * (1.9f + 1.7f * (float)((ranks + 15) / 16)) > 5.f) p = HiddenPlan{(int)((rounds + per - 1) / per), (int)(per * round)};
  return p;
}
}  // namespace
size_t mx_hidden_part_bytes(int64_t M, int64_t K, int ranks) {
  const HiddenPlan p = plan_hidden(M, K, ranks);
  return p.slices > 1 ? (size_t)p.slices * M * ranks * sizeof(float) : 0;
}
int run_mx_quantize_hidden(const void* x, int64_t M, int64_t K, uint8_t* codes, uint8_t* pieces, const uint16_t* const* lora_a, const int* r_off, int n,
                           uint16_t* h_cat, float* part, const uint8_t* const* w_scales, const int64_t* w_rows, uint8_t* const* w_pieces, hipStream_t s) {
  OperandWeights w;
  HiddenMembers a = {};
  a.n = n;
  for (int i = 0; i < n; ++i) {
    a.la[i] = lora_a[i];
    a.r_end[i] = r_off[i + 1];
  }
  const HiddenPlan p = plan_hidden(M, K, r_off[n]);
  TT_REQUIRE(p.slices == 1 || part, "mx_quantize_hidden: no room for the slices of the contraction");
  const int64_t xb = (M + 15) / 16 * p.slices, wb = operand_weights(w, w_scales, w_rows, w_pieces, n, K, 64 * kHiddenWaves);
  if (xb + wb >= (int64_t(1) << 31)) return fail(TTAMD_EUNSUPPORTED, "mx_quantize_hidden: M=%lld K=%lld are too large for one launch", (long long)M, (long long)K);
  const dim3 grid((unsigned)(xb + wb)), block(64 * kHiddenWaves);
  const uint16_t* in = reinterpret_cast<const uint16_t*>(x);
  const int Kp = (int)mx_padded_k(K);
  switch ((r_off[n] + 15) / 16) {
    case 1: mx_quantize_hidden_kernel<1><<<grid, block, 0, s>>>(in, M, (int)K, Kp, codes, pieces, a, h_cat, part, p.slices, p.k_slice, (int)xb, w); break;
    case 2: mx_quantize_hidden_kernel<2><<<grid, block, 0, s>>>(in, M, (int)K, Kp, codes, pieces, a, h_cat, part, p.slices, p.k_slice, (int)xb, w); break;
    case 3: mx_quantize_hidden_kernel<3><<<grid, block, 0, s>>>(in, M, (int)K, Kp, codes, pieces, a, h_cat, part, p.slices, p.k_slice, (int)xb, w); break;
    default: mx_quantize_hidden_kernel<4><<<grid, block, 0, s>>>(in, M, (int)K, Kp, codes, pieces, a, h_cat, part, p.slices, p.k_slice, (int)xb, w); break;
  }
  if (int rc = check_launch("mx_quantize_hidden")) return rc;
  return p.slices == 1 ? TTAMD_OK : run_mx_sum_slices(part, nullptr, h_cat, M * r_off[n], r_off[n], p.slices, s);
}
int run_mx_expand_tiles(const uint8_t* codes, const uint8_t* scales, int64_t N, int64_t K, void* tiles, hipStream_t s) {
  const int64_t nk = K / 32;
  if (N / 16 >= (int64_t(1) << 31) || (nk + 15) / 16 > 65535) return fail(TTAMD_EUNSUPPORTED, "mx_expand_tiles: weight too large");
  mx_expand_tiles_kernel<<<dim3((unsigned)(N / 16), (unsigned)((nk + 15) / 16)), dim3(256), 0, s>>>(codes, scales, (int)nk, (char*)tiles);
  return check_launch("mx_expand_tiles");
}

}  // namespace ttamd

using namespace ttamd;

extern "C" int ttamd_mx_quantize(const void* x, int dtype, int64_t rows, int64_t K, int format, uint8_t* codes, uint8_t* scales, void* stream) {
  if (int rc = check_codec("mx_quantize", dtype, rows, K, format)) return rc;
  if (rows == 0) return TTAMD_OK;
  TT_REQUIRE(x && codes && scales && aligned16(x) && aligned16(codes), "mx_quantize: pointers must be non-null, x and codes 16-byte aligned");
  const int64_t pieces = rows * (K / 8);
  const dim3 grid((unsigned)blocks_of(pieces)), block(256);
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (dtype == TTAMD_BF16 && format == TTAMD_MXFP4) mx_quantize_kernel<Bf16x8, TTAMD_MXFP4><<<grid, block, 0, s>>>(x, pieces, codes, scales);
  else if (dtype == TTAMD_BF16) mx_quantize_kernel<Bf16x8, TTAMD_MXFP8><<<grid, block, 0, s>>>(x, pieces, codes, scales);
  else if (format == TTAMD_MXFP4) mx_quantize_kernel<F32x8, TTAMD_MXFP4><<<grid, block, 0, s>>>(x, pieces, codes, scales);
  else mx_quantize_kernel<F32x8, TTAMD_MXFP8><<<grid, block, 0, s>>>(x, pieces, codes, scales);
  return check_launch("mx_quantize");
}

extern "C" int ttamd_mx_dequantize(const uint8_t* codes, const uint8_t* scales, int format, int64_t rows, int64_t K, int dtype, void* out,
                                   void* stream) {
  if (int rc = check_codec("mx_dequantize", dtype, rows, K, format)) return rc;
  if (rows == 0) return TTAMD_OK;
  TT_REQUIRE(codes && scales && out && aligned16(codes) && aligned16(out), "mx_dequantize: pointers must be non-null, codes and out 16-byte aligned");
  const int64_t pieces = rows * (K / 8);
  const dim3 grid((unsigned)blocks_of(pieces)), block(256);
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (dtype == TTAMD_F32 && format == TTAMD_MXFP4) mx_dequantize_kernel<TTAMD_MXFP4, true><<<grid, block, 0, s>>>(codes, scales, pieces, out);
  else if (dtype == TTAMD_F32) mx_dequantize_kernel<TTAMD_MXFP8, true><<<grid, block, 0, s>>>(codes, scales, pieces, out);
  else if (format == TTAMD_MXFP4) mx_dequantize_kernel<TTAMD_MXFP4, false><<<grid, block, 0, s>>>(codes, scales, pieces, out);
  else mx_dequantize_kernel<TTAMD_MXFP8, false><<<grid, block, 0, s>>>(codes, scales, pieces, out);
  return check_launch("mx_dequantize");
}
