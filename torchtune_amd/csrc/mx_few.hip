// x^[M, K] . W[N, K]^T for a handful of tokens (generation, M <= 16): the packed weight is streamed once, straight from HBM
// into the operand registers of v_mfma_scale_f32_16x16x128_f8f6f4, so what bounds the call is 17 / 32 byte per weight
// element and the latency of one dependent chain load -> product -> sum.
//
// Operand order of that instruction (lane l: row l % 16, quarter q = l / 16): fp4: 16 bytes, indices 32 q .. + 31 of the
// 128-wide step; fp8: two pieces of 16 bytes, indices 16 q .. and 64 + 16 q ..; scale: that of block q of the step.  Result:
// column l % 16 of the second operand (a token), rows 4 q + v of the first (outputs).
//
// A workgroup computes 16 RN outputs of up to 16 tokens; each of its waves takes a stretch of the contraction, and their sums
// meet in LDS, in wave order.  A few thousand input elements (kFewOwnElements) are quantised by every workgroup again, into
// LDS, while its first weights are on their way: a launch of its own costs more than the rest of the call.  Above, the codes
// of a quantise launch are read: quantising in the waves costs more vector instructions than the loads leave room for (one
// token, 14336 x 4096: 12.6 us with the conversions at each product).  Lanes of tokens past the last repeat it; their sums
// are not stored.
#include "mx_math.h"

namespace ttamd {
namespace {

typedef int v8i __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));

struct MxFewArgs {
  const uint16_t* x;    // [M, K]                         (PRE false)
  const uint8_t* xc;    // [M, Kp] or [M, Kp / 2], padded (PRE)
  const uint8_t* xp;    // its scales in pieces           (PRE)
  const uint8_t* wc;    // [N, K / 2]
  const uint8_t* ws;    // [N, K / 32]
  const uint16_t* bias;
  uint16_t* y;
  int M, N, K, Kp;
};

constexpr int kFewWaves = 8;
// steps whose loads a wave has in flight at once
constexpr int few_unroll(int rn, bool pre) { return pre || rn == 2 ? 4 : 8; }

template <int FMT, int RN, bool PRE>
__global__ __launch_bounds__(64 * kFewWaves) void mx_few_kernel(const MxFewArgs g) {
#if defined(__HIP_DEVICE_COMPILE__)
  constexpr int kUnroll = few_unroll(RN, PRE);
  constexpr bool F8 = FMT == TTAMD_MXFP8;
  constexpr int kPieces = F8 ? 2 : 1;  // 16-byte pieces of a token's codes per lane and step
  extern __shared__ __attribute__((aligned(16))) char smem[];  // sums [waves][RN][4][64]; before, PRE false, the input's codes
  float* const red = reinterpret_cast<float*>(smem);
  const int lane = threadIdx.x & 63, r16 = lane & 15, q = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = (int)blockDim.x >> 6;
  const int n0 = (int)blockIdx.x * 16 * RN;
  const int nb = g.K >> 5, steps = (nb + 3) >> 2;
  const int per = (steps + waves - 1) / waves, s_begin = wave * per, s_end = s_begin + per < steps ? s_begin + per : steps;

  // the weight rows' 32-bit offsets from the workgroup's first row
  const uint8_t* const wbase = g.wc + (int64_t)n0 * (g.K >> 1);
  const uint8_t* const sbase = g.ws + (int64_t)n0 * nb;
  uint32_t woff[RN], soff[RN];
#pragma unroll
  for (int j = 0; j < RN; ++j) {
    const int n = n0 + 16 * j + r16 < g.N ? 16 * j + r16 : g.N - 1 - n0;
    woff[j] = (uint32_t)n * (uint32_t)(g.K >> 1);
    soff[j] = (uint32_t)n * (uint32_t)nb;
  }
  mx_u32x4 w[kUnroll][RN];
  uint32_t wsc[kUnroll][RN];
  auto fetch = [&](int s0) {
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      if (s0 + u < s_end) {
        int blk = 4 * (s0 + u) + q;
        blk = blk < nb ? blk : nb - 1;  // past the end of the row: the input's codes are zero there
#pragma unroll
        for (int j = 0; j < RN; ++j) {
          w[u][j] = *reinterpret_cast<const mx_u32x4*>(wbase + (woff[j] + 16u * blk));
          wsc[u][j] = sbase[soff[j] + blk];
        }
      }
    }
  };
  fetch(s_begin);

  const int pitch = F8 ? g.Kp + 16 : (g.Kp >> 1) + 16;  // LDS rows of codes
  char* const own_scales = smem + g.M * pitch;          // [M][Kp / 32]
  if constexpr (!PRE) {
    mx_saturate_fp8();
    const int per_row = g.Kp >> 3, real = g.K >> 3;
    for (int i = threadIdx.x; i < g.M * per_row; i += (int)blockDim.x) {  // per_row is a multiple of 16: whole blocks per four lanes
      const int m = i / per_row, c = i - m * per_row;
      mx_u32x4 v = {0, 0, 0, 0};
      if (c < real) v = reinterpret_cast<const mx_u32x4*>(g.x)[(int64_t)m * real + c];
      const uint32_t byte = mx_scale_byte(mx_quad_max(mx_bf16_exponent(v)), FMT);
      const float s = mx_scale_value(byte == 255 ? 127u : byte);
      if constexpr (F8)
        *reinterpret_cast<mx_u32x2*>(smem + m * pitch + 8 * c) = byte == 255 ? mx_u32x2{0, 0} : mx_pack8(v, s);
      else
        *reinterpret_cast<uint32_t*>(smem + m * pitch + 4 * c) = byte == 255 ? 0u : mx_pack4(v, s);
      if ((c & 3) == 0) own_scales[m * (per_row >> 2) + (c >> 2)] = (char)byte;
    }
    mx_saturate_fp8(false);
    __syncthreads();
  }
  v4f acc[RN];
#pragma unroll
  for (int j = 0; j < RN; ++j) acc[j] = v4f{0.f, 0.f, 0.f, 0.f};
  const int row = r16 < g.M ? r16 : g.M - 1;

  for (int s0 = s_begin; s0 < s_end; s0 += kUnroll) {
    if (s0 > s_begin) fetch(s0);
    mx_u32x4 xr[PRE ? kUnroll : 1][kPieces];
    uint32_t xs[PRE ? kUnroll : 1];
    if constexpr (PRE) {
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        const int s = s0 + u;
        if (s >= s_end) break;
        const uint8_t* p = g.xc + ((uint32_t)row * (uint32_t)(F8 ? g.Kp : g.Kp >> 1) + (uint32_t)((F8 ? 128 : 64) * s + 16 * q));
#pragma unroll
        for (int e = 0; e < kPieces; ++e) xr[u][e] = *reinterpret_cast<const mx_u32x4*>(p + 64 * e);
        xs[u] = g.xp[((uint32_t)(s >> 2) * (uint32_t)g.M + (uint32_t)row) * 16u + mx_piece_byte(4 * (s & 3) + q)];
      }
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int s = s0 + u;
      if (s >= s_end) break;
      v8i xf = {};
      uint32_t xscale;
      if constexpr (PRE) {
        xscale = xs[u];
#pragma unroll
        for (int e = 0; e < kPieces; ++e)
#pragma unroll
          for (int d = 0; d < 4; ++d) xf[4 * e + d] = (int)xr[u][e][d];
      } else {
        xscale = (uint8_t)own_scales[row * (g.Kp >> 5) + 4 * s + q];
#pragma unroll
        for (int e = 0; e < kPieces; ++e) {
          const mx_u32x4 v = *reinterpret_cast<const mx_u32x4*>(smem + row * pitch + (F8 ? 128 : 64) * s + 16 * q + 64 * e);
#pragma unroll
          for (int d = 0; d < 4; ++d) xf[4 * e + d] = (int)v[d];
        }
      }
#pragma unroll
      for (int j = 0; j < RN; ++j) {
        v8i wf = {};
#pragma unroll
        for (int d = 0; d < 4; ++d) wf[d] = (int)w[u][j][d];
        acc[j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wf, xf, acc[j], 4, F8 ? 0 : 4, 0, (int)wsc[u][j], 0, (int)xscale);
      }
    }
  }
  if constexpr (!PRE) __syncthreads();  // the codes have been read
#pragma unroll
  for (int j = 0; j < RN; ++j)
#pragma unroll
    for (int v = 0; v < 4; ++v) red[((wave * RN + j) * 4 + v) * 64 + lane] = acc[j][v];
  __syncthreads();
  constexpr int kOut = RN * 256;
  for (int i = threadIdx.x; i < kOut; i += (int)blockDim.x) {
    const int n = i % (16 * RN), m = i / (16 * RN);  // outputs fastest: stores of a token are contiguous
    const int at = (((n >> 4) * 4 + (n & 3)) << 6) + 16 * ((n >> 2) & 3) + m;
    if (m >= g.M || n0 + n >= g.N) continue;
    float s = 0.f;
    for (int v = 0; v < waves; ++v) s += red[v * kOut + at];
    if (g.bias) s += __builtin_bit_cast(float, (uint32_t)g.bias[n0 + n] << 16);
    g.y[(int64_t)m * g.N + n0 + n] = __builtin_bit_cast(uint16_t, (__bf16)s);
  }
#endif
}

template <int FMT, int RN, bool PRE>
int launch_few(const MxFewArgs& g, hipStream_t s) {
  constexpr int kSums = kFewWaves * RN * 1024;
  const int codes = PRE ? 0 : g.M * (FMT == TTAMD_MXFP8 ? g.Kp + 16 : g.Kp / 2 + 16) + g.M * (g.Kp / 32);
  mx_few_kernel<FMT, RN, PRE><<<dim3((unsigned)((g.N + 16 * RN - 1) / (16 * RN))), dim3(64 * kFewWaves), codes > kSums ? codes : kSums, s>>>(g);
  return check_launch("mx_few");
}

template <int FMT>
int launch_few_tokens(const MxFewArgs& g, bool pre, bool two, hipStream_t s) {
  if (pre) return two ? launch_few<FMT, 2, true>(g, s) : launch_few<FMT, 1, true>(g, s);
  return two ? launch_few<FMT, 2, false>(g, s) : launch_few<FMT, 1, false>(g, s);
}

}  // namespace

// Up to 16 tokens where the outputs leave a workgroup of 16 or 32 of them enough to do, or where there is no launch for the
// input.  us, here / on 64-wide tiles: 16 x 4096 x 4096 6.5 / 10.4, 13 x 2048 x 8192 9.5 / 11.1, 16 x 14336 x 4096 15.5 / 13.0.
bool mx_few_applies(int64_t M, int64_t N) { return M <= 16 && N < 8192; }
// 16384 elements of eight bits are 16 KB of LDS and two to four pieces of eight for each of 512 threads to convert
bool mx_few_quantises(int64_t M, int64_t K) { return M <= 16 && M * K <= 16384; }

int run_mx_few(const void* x, const uint8_t* x_codes, const uint8_t* x_pieces, const uint8_t* w_codes, const uint8_t* w_scales, const void* bias,
               void* y, int64_t M, int64_t N, int64_t K, int fmt, hipStream_t s) {
  MxFewArgs g = {};
  g.x = reinterpret_cast<const uint16_t*>(x);
  g.xc = x_codes; g.xp = x_pieces; g.wc = w_codes; g.ws = w_scales;
  g.bias = reinterpret_cast<const uint16_t*>(bias);
  g.y = reinterpret_cast<uint16_t*>(y);
  g.M = (int)M; g.N = (int)N; g.K = (int)K; g.Kp = (int)mx_padded_k(K);
  // 32 outputs per workgroup halve what is read of the input, where that still leaves every CU a workgroup
  const bool two = N >= 32 * 256, pre = x_codes != nullptr;
  return fmt == TTAMD_MXFP8 ? launch_few_tokens<TTAMD_MXFP8>(g, pre, two, s) : launch_few_tokens<TTAMD_MXFP4>(g, pre, two, s);
}

}  // namespace ttamd
