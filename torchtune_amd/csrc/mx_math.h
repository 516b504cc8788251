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

// fp8 conversions saturate instead of giving NaN from here on.  Switched off again in waves that go on to multiply: the mode
// also takes the NaN out of what they compute.
__device__ __forceinline__ void mx_saturate_fp8(bool on = true) {
#if defined(__HIP_DEVICE_COMPILE__)
  __builtin_amdgcn_s_setreg(1 | (23 << 6), on ? 1 : 0);  // hwreg(MODE), bit 23: FP16_OVFL
#endif
}

// largest biased exponent of eight bf16
__device__ __forceinline__ uint32_t mx_bf16_exponent(const mx_u32x4& v) {
  typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
  u16x2 m = {0, 0};
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const uint32_t mag = v[q] & 0x7fff7fffu;
    m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, mag));
  }
  return (uint32_t)(m.x > m.y ? m.x : m.y) >> 7;
}

#if defined(__HIP_DEVICE_COMPILE__)
// the largest of four neighbouring lanes' values
__device__ __forceinline__ uint32_t mx_quad_max(uint32_t v) {
  uint32_t o = (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0xb1, 0xf, 0xf, true);  // lanes 1 0 3 2
  v = v > o ? v : o;
  o = (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x4e, 0xf, 0xf, true);           // lanes 2 3 0 1
  return v > o ? v : o;
}
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

// the four bf16 pairs of one dword of fp4 codes / two dwords of fp8 codes: exact, or among bf16's subnormals rounded once
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
// v_mfma_scale_f32_16x16x128 takes the scale of block q of a 128-wide step from lane quarter q, so byte 4 q + s of a piece
// holds block 4 s + q: a lane finds the scales of its four steps in one dword.  Blocks past the end of a row have scale byte 0
// (2^-127), and the input's codes are zero there.
// ---------------------------------------------------------------------------------------------------
__host__ __device__ constexpr int64_t mx_groups(int64_t K) { return (K + kMxGroup - 1) / kMxGroup; }
__host__ __device__ constexpr int64_t mx_piece_bytes(int64_t rows, int64_t K) { return mx_groups(K) * rows * 16; }
__device__ __forceinline__ int mx_piece_byte(int block_in_group) { return 4 * (block_in_group & 3) + (block_in_group >> 2); }
__host__ __device__ constexpr int64_t mx_padded_k(int64_t K) { return (K + 255) / 256 * 256; }  // rows of codes: whole pairs of steps

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
size_t mx_gemm_part_bytes(int64_t M, int64_t N, int64_t K, int fmt);
int run_mx_gemm(const MxProduct& q, int64_t M, int64_t N, int64_t K, int fmt, float* part, hipStream_t s);
int run_mx_gemm_group(const MxProduct* q, int n, int64_t M, const int64_t* N, int64_t K, float* part, hipStream_t s);
bool mx_few_applies(int64_t M, int64_t N);    // the product of so few tokens streams the weight (mx_few.hip)
bool mx_few_quantises(int64_t M, int64_t K);  // and quantises its input by itself
int run_mx_few(const void* x, const uint8_t* x_codes, const uint8_t* x_pieces, const uint8_t* w_codes, const uint8_t* w_scales, const void* bias,
               void* y, int64_t M, int64_t N, int64_t K, int fmt, hipStream_t s);
int run_mx_sum_slices(const float* part, const uint16_t* bias, uint16_t* y, int64_t numel, int N, int slices, hipStream_t s);
struct GroupDx;
bool mx_dx_fused(int64_t M, int64_t n_total, int64_t K);  // the grad-input expands the weights on their way through LDS (mx_dx.hip)
size_t mx_dx_fused_bytes(int64_t M, int64_t n_total, int64_t K);
int run_mx_dx(const GroupDx& d, const uint8_t* const* codes, const uint8_t* const* scales, const void* gh_cat, void* gx, float* part, hipStream_t s);
int check_mx_product(const char* who, int64_t M, int64_t N, int64_t K);
int run_mx_quantize_operand(const void* x, int64_t M, int64_t K, int fmt, uint8_t* codes, uint8_t* pieces, const uint8_t* const* w_scales,
                            const int64_t* w_rows, uint8_t* const* w_pieces, int n_weights, hipStream_t s);
size_t mx_hidden_part_bytes(int64_t M, int64_t K, int ranks);
int run_mx_quantize_hidden(const void* x, int64_t M, int64_t K, uint8_t* codes, uint8_t* pieces, const uint16_t* const* lora_a, const int* r_off, int n,
                           uint16_t* h_cat, float* part, const uint8_t* const* w_scales, const int64_t* w_rows, uint8_t* const* w_pieces, hipStream_t s);
int run_mx_expand_tiles(const uint8_t* codes, const uint8_t* scales, int64_t N, int64_t K, void* tiles, hipStream_t s);

}  // namespace ttamd
