// x^[M, K] . W[N, K]^T for a handful of tokens (generation, M <= 64): the packed weight is streamed once, straight from HBM
// into the operand registers of v_mfma_scale_f32_16x16x128_f8f6f4, so what bounds the call is 17 / 32 byte per weight
// element and the latency of one dependent chain load -> product -> sum.
//
// Operand order of that instruction (lane l: row l % 16, quarter q = l / 16): fp4: 16 bytes, indices 32 q .. + 31 of the
// 128-wide step; fp8: two pieces of 16 bytes, indices 16 q .. and 64 + 16 q ..; scale: that of block q of the step.  Result:
// column l % 16 of the second operand (a token), rows 4 q + v of the first (outputs).
//
// A workgroup computes 16 RN outputs of 16 MT tokens; each of its waves takes a stretch of the contraction, and their sums
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
constexpr int few_unroll(int mt, int rn, bool pre) { return pre ? (mt >= 3 ? 2 : 4) : (rn == 2 ? 4 : 8); }

template <int FMT, int MT, int RN, bool PRE>
__global__ __launch_bounds__(64 * kFewWaves) void mx_few_kernel(const MxFewArgs g) {
#if defined(__HIP_DEVICE_COMPILE__)
  constexpr int kUnroll = few_unroll(MT, RN, PRE);
  constexpr bool F8 = FMT == TTAMD_MXFP8;
  constexpr int kPieces = F8 ? 2 : 1;  // 16-byte pieces of a token's codes per lane and step
  extern __shared__ __attribute__((aligned(16))) char smem[];  // sums [waves][RN][MT][4][64]; before, PRE false, the input's codes
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
  v4f acc[RN][MT];
#pragma unroll
  for (int j = 0; j < RN; ++j)
#pragma unroll
    for (int t = 0; t < MT; ++t) acc[j][t] = v4f{0.f, 0.f, 0.f, 0.f};
  int row[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) row[t] = 16 * t + r16 < g.M ? 16 * t + r16 : g.M - 1;

  for (int s0 = s_begin; s0 < s_end; s0 += kUnroll) {
    if (s0 > s_begin) fetch(s0);
    mx_u32x4 xr[PRE ? kUnroll : 1][MT][kPieces];
    uint32_t xs[PRE ? kUnroll : 1][MT];
    if constexpr (PRE) {
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        const int s = s0 + u;
        if (s >= s_end) break;
#pragma unroll
        for (int t = 0; t < MT; ++t) {
          const uint8_t* p = g.xc + ((uint32_t)row[t] * (uint32_t)(F8 ? g.Kp : g.Kp >> 1) + (uint32_t)((F8 ? 128 : 64) * s + 16 * q));
#pragma unroll
          for (int e = 0; e < kPieces; ++e) xr[u][t][e] = *reinterpret_cast<const mx_u32x4*>(p + 64 * e);
          xs[u][t] = g.xp[((uint32_t)(s >> 2) * (uint32_t)g.M + (uint32_t)row[t]) * 16u + mx_piece_byte(4 * (s & 3) + q)];
        }
      }
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int s = s0 + u;
      if (s >= s_end) break;
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        v8i xf = {};
        uint32_t xscale;
        if constexpr (PRE) {
          xscale = xs[u][t];
#pragma unroll
          for (int e = 0; e < kPieces; ++e)
#pragma unroll
            for (int d = 0; d < 4; ++d) xf[4 * e + d] = (int)xr[u][t][e][d];
        } else {
          xscale = (uint8_t)own_scales[row[t] * (g.Kp >> 5) + 4 * s + q];
#pragma unroll
          for (int e = 0; e < kPieces; ++e) {
            const mx_u32x4 v = *reinterpret_cast<const mx_u32x4*>(smem + row[t] * pitch + (F8 ? 128 : 64) * s + 16 * q + 64 * e);
#pragma unroll
            for (int d = 0; d < 4; ++d) xf[4 * e + d] = (int)v[d];
          }
        }
#pragma unroll
        for (int j = 0; j < RN; ++j) {
          v8i wf = {};
#pragma unroll
          for (int d = 0; d < 4; ++d) wf[d] = (int)w[u][j][d];
          acc[j][t] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wf, xf, acc[j][t], 4, F8 ? 0 : 4, 0, (int)wsc[u][j], 0, (int)xscale);
        }
      }
    }
  }
  if constexpr (!PRE) __syncthreads();  // the codes have been read
#pragma unroll
  for (int j = 0; j < RN; ++j)
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int v = 0; v < 4; ++v) red[(((wave * RN + j) * MT + t) * 4 + v) * 64 + lane] = acc[j][t][v];
  __syncthreads();
  constexpr int kOut = RN * MT * 256;
  for (int i = threadIdx.x; i < kOut; i += (int)blockDim.x) {
    const int n = i % (16 * RN), m = i / (16 * RN);  // outputs fastest: stores of a token are contiguous
    const int at = ((((n >> 4) * MT + (m >> 4)) * 4 + (n & 3)) << 6) + 16 * ((n >> 2) & 3) + (m & 15);
    if (m >= g.M || n0 + n >= g.N) continue;
    float s = 0.f;
    for (int v = 0; v < waves; ++v) s += red[v * kOut + at];
    if (g.bias) s += __builtin_bit_cast(float, (uint32_t)g.bias[n0 + n] << 16);
    g.y[(int64_t)m * g.N + n0 + n] = __builtin_bit_cast(uint16_t, (__bf16)s);
  }
#endif
}

template <int FMT, int MT, int RN, bool PRE>
int launch_few(const MxFewArgs& g, int waves, hipStream_t s) {
  const int codes = PRE ? 0 : g.M * (FMT == TTAMD_MXFP8 ? g.Kp + 16 : g.Kp / 2 + 16) + g.M * (g.Kp / 32);
  const int sums = waves * RN * MT * 1024, lds = codes > sums ? codes : sums;
  static_assert(kFewWaves * RN * MT * 1024 <= 64 * 1024, "LDS without asking for more");
  mx_few_kernel<FMT, MT, RN, PRE><<<dim3((unsigned)((g.N + 16 * RN - 1) / (16 * RN))), dim3(64 * waves), lds, s>>>(g);
  return check_launch("mx_few");
}

template <int FMT, bool PRE>
int launch_few_tokens(const MxFewArgs& g, int rn, int waves, hipStream_t s) {
  if constexpr (!PRE) {
    return rn == 2 ? launch_few<FMT, 1, 2, false>(g, waves, s) : launch_few<FMT, 1, 1, false>(g, waves, s);
  } else {
    const int mt = (g.M + 15) / 16;
    if (rn == 2) return mt == 1 ? launch_few<FMT, 1, 2, true>(g, waves, s) : mt == 2 ? launch_few<FMT, 2, 2, true>(g, waves, s) : mt == 3 ? launch_few<FMT, 3, 2, true>(g, waves, s) : launch_few<FMT, 4, 2, true>(g, waves, s);
    return mt == 1 ? launch_few<FMT, 1, 1, true>(g, waves, s) : mt == 2 ? launch_few<FMT, 2, 1, true>(g, waves, s) : mt == 3 ? launch_few<FMT, 3, 1, true>(g, waves, s) : launch_few<FMT, 4, 1, true>(g, waves, s);
  }
}

}  // namespace

bool mx_few_applies(int64_t M) { return M <= 64; }
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
  const int rn = N >= 32 * 256 ? 2 : 1;
  const int waves = kFewWaves;
  const bool pre = x_codes != nullptr;
  if (fmt == TTAMD_MXFP8) return pre ? launch_few_tokens<TTAMD_MXFP8, true>(g, rn, waves, s) : launch_few_tokens<TTAMD_MXFP8, false>(g, rn, waves, s);
  return pre ? launch_few_tokens<TTAMD_MXFP4, true>(g, rn, waves, s) : launch_few_tokens<TTAMD_MXFP4, false>(g, rn, waves, s);
}

}  // namespace ttamd
