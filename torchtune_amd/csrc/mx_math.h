// Microscaled (MX) blocks: 32 consecutive elements of a row share one power-of-two scale, stored as its biased exponent
// (E8M0: byte s stands for 2^(s - 127), 255 for NaN); the elements are fp4 (e2m1: two per byte, the earlier one in the low
// half) or fp8 (e4m3).  The conversions are gfx950's own instructions, which scale, round to nearest even and - fp4 always,
// fp8 with MODE.FP16_OVFL set - saturate (compared exhaustively over bf16 against round-half-even of x / 2^e).
#pragma once
#include "common.h"

namespace ttamd {

constexpr int kMxBlock = 32;
constexpr int kMxWeights = TTAMD_GROUP_MAX;  // most weights that one call multiplies an input with
constexpr int kMxGroup = 512;  // contraction indices of one 16-byte piece of scales in the product's own layout

__host__ __device__ constexpr int mx_emax(int fmt) { return fmt == TTAMD_MXFP4 ? 2 : 8; }

typedef uint32_t mx_u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t mx_u32x2 __attribute__((ext_vector_type(2)));
typedef float mx_f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 mx_bf16x2 __attribute__((ext_vector_type(2)));
typedef short mx_s16x2 __attribute__((ext_vector_type(2)));

// 2^(s - 127) for a scale byte s <= 254; NaN for 255
__device__ __forceinline__ float mx_scale_value(uint32_t s) {
  return __builtin_bit_cast(float, s == 0 ? 0x00400000u : (s == 255 ? 0x7fc00000u : s << 23));
}

// The scale byte of a block whose largest magnitude has the biased float exponent E (bits 30..23; 0 for zeros and
// subnormals): 2^(floor(log2(amax)) - emax), not below 2^-127.  A block with an infinity or a NaN is all NaN.
__device__ __forceinline__ uint32_t mx_scale_byte(uint32_t E, int fmt) {
  const uint32_t em = (uint32_t)mx_emax(fmt);
  return E == 255 ? 255u : (E > em ? E - em : 0u);
}

// fp8 conversions saturate instead of giving NaN from here to the end of the wave
__device__ __forceinline__ void mx_saturate_fp8() {
#if defined(__HIP_DEVICE_COMPILE__)
  __builtin_amdgcn_s_setreg(1 | (23 << 6), 1);  // hwreg(MODE), bit 23: FP16_OVFL
#endif
}

#if defined(__HIP_DEVICE_COMPILE__)
__device__ __forceinline__ mx_bf16x2 mx_pair(uint32_t v) { return __builtin_bit_cast(mx_bf16x2, v); }
// eight elements, as four packed bf16 pairs / as floats, into fp4 (one dword) or fp8 (two)
__device__ __forceinline__ uint32_t mx_pack4(const mx_u32x4& v, float s) {
  uint32_t o = 0;
  o = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(o, mx_pair(v.x), s, 0);
  o = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(o, mx_pair(v.y), s, 1);
  o = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(o, mx_pair(v.z), s, 2);
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(o, mx_pair(v.w), s, 3);
}
__device__ __forceinline__ uint32_t mx_pack4(const float (&v)[8], float s) {
  uint32_t o = 0;
  o = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(o, v[0], v[1], s, 0);
  o = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(o, v[2], v[3], s, 1);
  o = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(o, v[4], v[5], s, 2);
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(o, v[6], v[7], s, 3);
}
__device__ __forceinline__ mx_u32x2 mx_pack8(const mx_u32x4& v, float s) {
  mx_s16x2 a = {0, 0}, b = {0, 0};
  a = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(a, mx_pair(v.x), s, false);
  a = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(a, mx_pair(v.y), s, true);
  b = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(b, mx_pair(v.z), s, false);
  b = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(b, mx_pair(v.w), s, true);
  return mx_u32x2{__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b)};
}
__device__ __forceinline__ mx_u32x2 mx_pack8(const float (&v)[8], float s) {
  mx_s16x2 a = {0, 0}, b = {0, 0};
  a = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(a, v[0], v[1], s, false);
  a = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(a, v[2], v[3], s, true);
  b = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(b, v[4], v[5], s, false);
  b = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(b, v[6], v[7], s, true);
  return mx_u32x2{__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b)};
}

// the four bf16 pairs of one dword of fp4 codes / two dwords of fp8 codes (exact above bf16's subnormals)
__device__ __forceinline__ mx_u32x4 mx_bf16_of_fp4(uint32_t c, float s) {
  mx_u32x4 o;
  o.x = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 0));
  o.y = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 1));
  o.z = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 2));
  o.w = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 3));
  return o;
}
__device__ __forceinline__ mx_u32x4 mx_bf16_of_fp8(mx_u32x2 c, float s) {
  mx_u32x4 o;
  o.x = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c.x, s, false));
  o.y = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c.x, s, true));
  o.z = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c.y, s, false));
  o.w = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c.y, s, true));
  return o;
}
__device__ __forceinline__ void mx_f32_of_fp4(uint32_t c, float s, float (&o)[8]) {
  const mx_f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, 1);
  const mx_f32x2 d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, 2), e = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, 3);
  o[0] = a.x; o[1] = a.y; o[2] = b.x; o[3] = b.y; o[4] = d.x; o[5] = d.y; o[6] = e.x; o[7] = e.y;
}
__device__ __forceinline__ void mx_f32_of_fp8(mx_u32x2 c, float s, float (&o)[8]) {
  const mx_f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(c.x, s, false), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(c.x, s, true);
  const mx_f32x2 d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(c.y, s, false), e = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(c.y, s, true);
  o[0] = a.x; o[1] = a.y; o[2] = b.x; o[3] = b.y; o[4] = d.x; o[5] = d.y; o[6] = e.x; o[7] = e.y;
}
#endif

// ---------------------------------------------------------------------------------------------------
// The products' own layout of scales.  Of each row the 16 scale bytes of 512 contraction indices (16 blocks) form one
// piece, and the pieces of all rows for the same 512 indices lie one after the other: [K / 512 rounded up][rows][16].
// v_mfma_scale_f32_32x32x64 takes the scale of block 2 c + h of a 64-wide step from lane half h, so byte 8 h + c of a piece
// holds block 2 c + h: a lane finds the eight scales of its half side by side, and picks one by the instruction's byte
// select.  Blocks past the end of a row have scale byte 0 (2^-127): whatever codes meet there add less than 2^-149.
// ---------------------------------------------------------------------------------------------------
__host__ __device__ constexpr int64_t mx_groups(int64_t K) { return (K + kMxGroup - 1) / kMxGroup; }
__host__ __device__ constexpr int64_t mx_piece_bytes(int64_t rows, int64_t K) { return mx_groups(K) * rows * 16; }
__device__ __forceinline__ int mx_piece_byte(int block_in_group) { return 8 * (block_in_group & 1) + (block_in_group >> 1); }
__host__ __device__ constexpr int64_t mx_padded_k(int64_t K) { return (K + 127) / 128 * 128; }

// Internal entry points shared by the translation units
struct MxProduct {
  const uint8_t *x_codes, *x_pieces;  // rows padded to mx_padded_k(K) elements, scales in pieces
  const uint8_t *w_codes, *w_pieces;  // [N, K / 2], scales in pieces
  const uint16_t* h;                  // adapter activation [M, ldh] (rank columns of it), or null with rank 0
  const uint16_t* lora_b;             // [N, rank]
  const uint16_t* bias;               // [N] or null
  uint16_t* y;                        // [M, N]
  float lscale;
  int rank, ldh;
};
size_t mx_operand_bytes(int64_t M, int64_t K, int fmt);  // codes of an input with padded rows
size_t mx_gemm_part_bytes(int64_t M, int64_t N, int64_t K);
int run_mx_gemm(const MxProduct& q, int64_t M, int64_t N, int64_t K, int fmt, float* part, hipStream_t s);
int check_mx_product(const char* who, int64_t M, int64_t N, int64_t K);
int run_mx_quantize_operand(const void* x, int64_t M, int64_t K, int fmt, uint8_t* codes, uint8_t* pieces, const uint8_t* const* w_scales,
                            const int64_t* w_rows, uint8_t* const* w_pieces, int n_weights, hipStream_t s);
int run_mx_dequantize_operand(const uint8_t* codes, const uint8_t* pieces, int64_t M, int64_t K, void* out, hipStream_t s);
int run_mx_expand_tiles(const uint8_t* codes, const uint8_t* scales, int64_t N, int64_t K, void* tiles, hipStream_t s);

}  // namespace ttamd
