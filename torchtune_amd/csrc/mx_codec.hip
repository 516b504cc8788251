// Microscaled tensors: a bf16 / fp32 tensor into blocks of 32 with a shared power-of-two scale (mxfp4, mxfp8) and back.
// (torchtune trains over such weights through torchao's MX prototypes; the format is the OCP one, scales rounded down.)
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
  if ((int)blockIdx.x >= x_blocks) {
    int blk = (int)blockIdx.x - x_blocks, which = 0;
#pragma unroll
    for (int q = 0; q < kMxWeights - 1; ++q)
      if (q < w.n - 1 && blk >= w.blk_end[q]) which = q + 1;
    if (which) blk -= w.blk_end[which - 1];
    const int nb = K / kMxBlock, groups = (nb + 15) >> 4;
    const int64_t i = (int64_t)blk * 256 + threadIdx.x, rows = w.rows[which];
    const int64_t row = i / groups;
    const int g = (int)(i - row * groups);
    if (row >= rows) return;
    const uint8_t* src = w.scales[which] + row * nb + 16 * g;
    mx_u32x4 d = {0, 0, 0, 0};
    if ((nb & 15) == 0) {
      d = *reinterpret_cast<const mx_u32x4*>(src);
    } else {
#pragma unroll
      for (int q = 0; q < 16; ++q)
        if (16 * g + q < nb) d[q >> 2] |= (uint32_t)src[q] << (8 * (q & 3));
    }
    // byte 4 s + q -> byte 4 q + s
    const uint32_t t0 = __builtin_amdgcn_perm(d.y, d.x, 0x05010400u), t1 = __builtin_amdgcn_perm(d.y, d.x, 0x07030602u);
    const uint32_t u0 = __builtin_amdgcn_perm(d.w, d.z, 0x05010400u), u1 = __builtin_amdgcn_perm(d.w, d.z, 0x07030602u);
    const mx_u32x4 o = {__builtin_amdgcn_perm(u0, t0, 0x05040100u), __builtin_amdgcn_perm(u0, t0, 0x07060302u),
                        __builtin_amdgcn_perm(u1, t1, 0x05040100u), __builtin_amdgcn_perm(u1, t1, 0x07060302u)};
    reinterpret_cast<mx_u32x4*>(w.pieces[which])[(int64_t)g * rows + row] = o;
    return;
  }
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

// The kept 8-bit input (rows padded, scales in pieces) as bf16 [M, K].
__global__ __launch_bounds__(256) void mx_dequantize_operand_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ xp,
                                                                    int64_t M, int K, int Kp, void* __restrict__ out) {
#if defined(__HIP_DEVICE_COMPILE__)
  const uint32_t per_row = (uint32_t)K >> 3;
  const int64_t c0 = (int64_t)blockIdx.x * (256 * kChunks);
  const int64_t row0 = c0 / per_row;
  const uint32_t rem = (uint32_t)(c0 - row0 * per_row) + threadIdx.x;
#pragma unroll
  for (int u = 0; u < kChunks; ++u) {
    const uint32_t t = rem + 256 * u, r = t / per_row, col = t - r * per_row;
    const int64_t row = row0 + r;
    if (row >= M) continue;
    const uint32_t blk = col >> 2;
    const mx_u32x2 c = *reinterpret_cast<const mx_u32x2*>(codes + row * Kp + 8 * col);
    const uint32_t b = xp[((int64_t)(blk >> 4) * M + row) * 16 + mx_piece_byte(blk & 15)];
    mx_u32x4 o = mx_bf16_of_fp8(c, mx_scale_value(b == 255 ? 127u : b));
    if (b == 255) o = mx_u32x4{0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u};
    reinterpret_cast<mx_u32x4*>(out)[row * per_row + col] = o;
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

int run_mx_quantize_operand(const void* x, int64_t M, int64_t K, int fmt, uint8_t* codes, uint8_t* pieces, const uint8_t* const* w_scales,
                            const int64_t* w_rows, uint8_t* const* w_pieces, int n_weights, hipStream_t s) {
  const int64_t Kp = mx_padded_k(K), xb = blocks_of(M * (Kp / 8));
  OperandWeights w = {};
  w.n = n_weights;
  int64_t wb = 0;
  for (int i = 0; i < n_weights; ++i) {
    w.scales[i] = w_scales[i];
    w.pieces[i] = w_pieces[i];
    w.rows[i] = w_rows[i];
    wb += (w_rows[i] * mx_groups(K) + 255) / 256;
    w.blk_end[i] = (int)wb;
  }
  if (xb + wb >= (int64_t(1) << 31)) return fail(TTAMD_EUNSUPPORTED, "mx_quantize_operand: M=%lld K=%lld are too large for one launch", (long long)M, (long long)K);
  if (fmt == TTAMD_MXFP4)
    mx_quantize_operand_kernel<TTAMD_MXFP4><<<dim3((unsigned)(xb + wb)), dim3(256), 0, s>>>(x, M, (int)K, (int)Kp, codes, pieces, (int)xb, w);
  else
    mx_quantize_operand_kernel<TTAMD_MXFP8><<<dim3((unsigned)(xb + wb)), dim3(256), 0, s>>>(x, M, (int)K, (int)Kp, codes, pieces, (int)xb, w);
  return check_launch("mx_quantize_operand");
}

int run_mx_dequantize_operand(const uint8_t* codes, const uint8_t* pieces, int64_t M, int64_t K, void* out, hipStream_t s) {
  const int64_t blocks = blocks_of(M * (K / 8));
  if (blocks >= (int64_t(1) << 31)) return fail(TTAMD_EUNSUPPORTED, "mx_dequantize_operand: M=%lld K=%lld are too large for one launch", (long long)M, (long long)K);
  mx_dequantize_operand_kernel<<<dim3((unsigned)blocks), dim3(256), 0, s>>>(codes, pieces, M, (int)K, (int)mx_padded_k(K), out);
  return check_launch("mx_dequantize_operand");
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
