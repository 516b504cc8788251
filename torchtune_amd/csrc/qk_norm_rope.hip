// Queries and keys between their projections and the attention: the norm of every head and the rotation by the token's position
// in one pass, forward and backward.
//
//   r = 1 / sqrt(mean(x^2) + eps),  n = x r w   (without scales: n = x)
//   (a, b) -> (a cos - b sin, b cos + a sin) for the two elements a, b of n that frequency i turns: 2 i and 2 i + 1
//   (interleaved) or i and D / 2 + i (halves); cos and sin stand in row pos of the table, pos being the token's position on
//   the axis whose section holds i.
//   backward: g = the rotation by the negative angle of gy;  gw = sum over rows of g x r;  gx = r (g w - x r^2 mean(g w x)).
//
// Everything is computed in fp32 from the inputs and rounded once.  Nothing but the inputs is kept for the backward: the row is
// read there anyway, and its r costs less than reading one that was kept.
//
// Bound: HBM.  A row (one head of one token) belongs to G = 2^ceil(log2(D / 16)) neighbouring lanes, each with 16 of its elements:
// those that frequencies 8 j .. 8 j + 7 turn, so that a pair never leaves its lane and one piece of the table serves both pairings.
#include "row_vec.h"

namespace ttamd {
namespace {

struct Part {
  const void* x;
  const void* scale;
  const void* gy;
  void* out;
  int64_t xs[3], gs[3];  // of batch, token, head
  uint32_t heads;
};

struct RopeArgs {
  Part part[2];
  const float* cache;
  const int64_t* pos;
  int64_t ps[3];  // of axis, batch, token
  int64_t cache_rows;
  int end[3];  // first frequencies of the axes 1 .. 3
  int n_axes;
  uint32_t S, tokens;  // tokens = B * S
  int D, lanes, log_group;
  float eps;
};

template <bool INTER>
struct Pairs {  // element of the lane's sixteen
  static constexpr int first(int p) { return INTER ? 2 * p : p; }
  static constexpr int second(int p) { return INTER ? 2 * p + 1 : p + 8; }
};

// where a lane's two pieces of eight begin
template <bool INTER>
__device__ __forceinline__ int piece(int j, int which, int D) {
  return INTER ? 16 * j + 8 * which : 8 * j + (D >> 1) * which;
}

template <class T, bool INTER>
__device__ __forceinline__ void load16(const typename T::elem* p, int j, int D, bool active, float (&v)[16]) {
  float a[8], b[8];
  typename T::Raw ra = {}, rb = {};
  if (active) {
    ra = T::load_once(p + piece<INTER>(j, 0, D));
    rb = T::load_once(p + piece<INTER>(j, 1, D));
  }
  T::unpack(ra, a);
  T::unpack(rb, b);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    v[i] = a[i];
    v[8 + i] = b[i];
  }
}

template <class T, bool INTER>
__device__ __forceinline__ void store16(typename T::elem* p, int j, int D, const float (&v)[16]) {
  float a[8], b[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    a[i] = v[i];
    b[i] = v[8 + i];
  }
  T::store(p + piece<INTER>(j, 0, D), T::pack(a));
  T::store(p + piece<INTER>(j, 1, D), T::pack(b));
}

// cosines and sines of frequencies 8 j .. 8 j + 7 at token (b, s).  A position outside the table gives NaN and reads nothing.
__device__ __forceinline__ void angles(const RopeArgs& a, uint32_t b, uint32_t s, int j, bool active, float (&cs)[8], float (&sn)[8]) {
  const int half = a.D >> 1;
  if (a.n_axes <= 1) {  // uniform
    const int64_t pos = a.pos ? a.pos[b * a.ps[1] + s * a.ps[2]] : (int64_t)s;
    const bool inside = active && (uint64_t)pos < (uint64_t)a.cache_rows;
    const f32x4_at4_t* c = reinterpret_cast<const f32x4_at4_t*>(a.cache + (pos * half + 8 * j) * 2);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const float nan = __builtin_nanf("");
      f32x4_at4_t v = {nan, nan, nan, nan};
      if (inside) v = c[q];
      cs[2 * q] = v.x;
      sn[2 * q] = v.y;
      cs[2 * q + 1] = v.z;
      sn[2 * q + 1] = v.w;
    }
    return;
  }
  int64_t pos[4];
#pragma unroll
  for (int x = 0; x < 4; ++x) pos[x] = x < a.n_axes ? a.pos[x * a.ps[0] + b * a.ps[1] + s * a.ps[2]] : 0;
#pragma unroll
  for (int p = 0; p < 8; ++p) {
    const int i = 8 * j + p;
    const int64_t at = i < a.end[0] ? pos[0] : i < a.end[1] ? pos[1] : i < a.end[2] ? pos[2] : pos[3];
    typedef float f32x2_t __attribute__((ext_vector_type(2)));
    f32x2_t v = {__builtin_nanf(""), __builtin_nanf("")};
    if (active && (uint64_t)at < (uint64_t)a.cache_rows) v = *reinterpret_cast<const f32x2_t*>(a.cache + (at * half + i) * 2);
    cs[p] = v.x;
    sn[p] = v.y;
  }
}

// the sum over the 2^log_group lanes of a row, in every one of them
__device__ __forceinline__ float row_sum(float v, int log_group) {
  if (log_group > 0) v += row_partner<1>(v);
  if (log_group > 1) v += row_partner<2>(v);
  if (log_group > 2) v += row_partner<4>(v);
  if (log_group > 3) v += row_partner<8>(v);
  if (log_group > 4) v += __shfl_xor(v, 16, kWave);
  return v;
}

// 1 / sqrt: the hardware's is off by an ulp, which bf16 results do not show
template <class T>
__device__ __forceinline__ float inverse_root(float v) {
  return sizeof(typename T::elem) == 2 ? __builtin_amdgcn_rsqf(v) : 1.f / __builtin_sqrtf(v);
}

template <class T, bool NORM, bool INTER>
__global__ __launch_bounds__(256) void qk_norm_rope_fwd_kernel(const RopeArgs a) {
  typedef typename T::elem E;
  const uint32_t row = (uint32_t)(((uint64_t)blockIdx.x * 256 + threadIdx.x) >> a.log_group);
  const uint32_t H = a.part[0].heads + a.part[1].heads;
  if (row >= a.tokens * H) return;  // the lanes of a row leave together
  const int j = threadIdx.x & ((1 << a.log_group) - 1);
  const bool active = j < a.lanes;
  const uint32_t token = row / H, h = row - token * H, b = token / a.S, s = token - b * a.S;
  const bool key = h >= a.part[0].heads;
  const Part& part = a.part[key];
  const uint32_t head = key ? h - a.part[0].heads : h;
  float x[16], w[16], cs[8], sn[8];
  load16<T, INTER>(reinterpret_cast<const E*>(part.x) + b * part.xs[0] + s * part.xs[1] + head * part.xs[2], j, a.D, active, x);
  angles(a, b, s, j, active, cs, sn);
  if constexpr (NORM) {
    load16<T, INTER>(reinterpret_cast<const E*>(part.scale), j, a.D, active, w);
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) ss += x[i] * x[i];
    const float r = inverse_root<T>(row_sum(ss, a.log_group) / (float)a.D + a.eps);
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] = x[i] * r * w[i];
  }
  float o[16];
#pragma unroll
  for (int p = 0; p < 8; ++p) {
    const float u = x[Pairs<INTER>::first(p)], v = x[Pairs<INTER>::second(p)];
    o[Pairs<INTER>::first(p)] = u * cs[p] - v * sn[p];
    o[Pairs<INTER>::second(p)] = v * cs[p] + u * sn[p];
  }
  if (active) store16<T, INTER>(reinterpret_cast<E*>(part.out) + ((int64_t)token * part.heads + head) * a.D, j, a.D, o);
}

constexpr int kBwdGrid = 1024;  // workgroups of the backward with scale gradients; each leaves a row of partial sums per part

// GSCALE: a fixed number of workgroups walk the rows, first those of the queries, then those of the keys, and each lane sums the
// scale gradient of its elements over the rows that it sees; else there is a workgroup for every 256 / G rows.
template <class T, bool NORM, bool INTER, bool GSCALE>
__global__ __launch_bounds__(256) void qk_norm_rope_bwd_kernel(const RopeArgs a, float* __restrict__ partial) {
  typedef typename T::elem E;
  __shared__ float sums[GSCALE ? 512 : 1];
  const int G = 1 << a.log_group, j = threadIdx.x & (G - 1);
  const bool active = j < a.lanes;
  const uint32_t per_wg = 256u >> a.log_group;
#pragma unroll 1
  for (int which = 0; which < 2; ++which) {
    const Part& part = a.part[which];
    float w[16], gs[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) gs[i] = 0.f;
    if constexpr (NORM) {
      if (part.heads) load16<T, INTER>(reinterpret_cast<const E*>(part.scale), j, a.D, active, w);
    }
    const uint64_t rows = (uint64_t)a.tokens * part.heads;
    for (uint64_t row0 = (uint64_t)blockIdx.x * per_wg; row0 < rows; row0 += (uint64_t)gridDim.x * per_wg) {
      const uint32_t row = (uint32_t)row0 + (threadIdx.x >> a.log_group);
      if (row >= rows) continue;  // the lanes of a row together
      const uint32_t token = row / part.heads, head = row - token * part.heads, b = token / a.S, s = token - b * a.S;
      float gy[16], x[16], cs[8], sn[8], g[16];
      load16<T, INTER>(reinterpret_cast<const E*>(part.gy) + b * part.gs[0] + s * part.gs[1] + head * part.gs[2], j, a.D, active, gy);
      if constexpr (NORM)
        load16<T, INTER>(reinterpret_cast<const E*>(part.x) + b * part.xs[0] + s * part.xs[1] + head * part.xs[2], j, a.D, active, x);
      angles(a, b, s, j, active, cs, sn);
#pragma unroll
      for (int p = 0; p < 8; ++p) {
        const float u = gy[Pairs<INTER>::first(p)], v = gy[Pairs<INTER>::second(p)];
        g[Pairs<INTER>::first(p)] = u * cs[p] + v * sn[p];
        g[Pairs<INTER>::second(p)] = v * cs[p] - u * sn[p];
      }
      if constexpr (NORM) {
        float ss = 0.f, dot = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) ss += x[i] * x[i];
        const float r = inverse_root<T>(row_sum(ss, a.log_group) / (float)a.D + a.eps);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          if constexpr (GSCALE) gs[i] += active ? g[i] * x[i] * r : 0.f;  // idle lanes hold NaN angles
          g[i] *= w[i];
          dot += active ? g[i] * x[i] : 0.f;
        }
        const float c = row_sum(dot, a.log_group) / (float)a.D * r * r;
#pragma unroll
        for (int i = 0; i < 16; ++i) g[i] = r * (g[i] - x[i] * c);
      }
      if (active && part.out) store16<T, INTER>(reinterpret_cast<E*>(part.out) + (int64_t)row * a.D, j, a.D, g);
    }
    if constexpr (GSCALE) {
      // the lanes that hold the same elements meet in LDS, one row of the workgroup after another: a fixed order
      for (int r = 0; r < (int)per_wg; ++r) {
        __syncthreads();
        if ((int)(threadIdx.x >> a.log_group) != r || !active) continue;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          float* at = sums + piece<INTER>(j, i >> 3, a.D) + (i & 7);
          *at = r ? *at + gs[i] : gs[i];
        }
      }
      __syncthreads();
      for (int d = threadIdx.x; d < a.D; d += 256) partial[((int64_t)which * gridDim.x + blockIdx.x) * a.D + d] = sums[d];
    }
  }
}

// gscale[d] = sum over the workgroups' partial sums, in slices of a fixed order; blockIdx.y is the part
template <class T>
__global__ __launch_bounds__(1024) void qk_norm_rope_gscale_kernel(const float* __restrict__ partial, int n, int D, void* gq, void* gk) {
  typedef typename T::elem E;
  __shared__ float red[64][17];
  const int col = threadIdx.x & 15, slice = threadIdx.x >> 4, d = blockIdx.x * 16 + col;  // D % 16 == 0
  const int per = (n + 63) / 64, lo = slice * per, hi = min(lo + per, n);
  const float* p = partial + (int64_t)blockIdx.y * n * D + d;
  float s = 0.f;
#pragma unroll 4
  for (int w = lo; w < hi; ++w) s += p[(int64_t)w * D];
  red[slice][col] = s;
  __syncthreads();
  E* out = reinterpret_cast<E*>(blockIdx.y ? gk : gq);
  if (slice || !out) return;
  s = 0.f;
  for (int i = 0; i < 64; ++i) s += red[i][col];
  T::put(out + d, s);
}

int prepare(const char* who, RopeArgs& a, const ttamd_rope_heads* parts, const ttamd_rope_positions* at, int dtype, float eps, int64_t B,
            int64_t S, int64_t D, bool backward) {
  TT_REQUIRE(parts && at && at->cache, "%s: null pointer argument", who);
  TT_REQUIRE(dtype == TTAMD_BF16 || dtype == TTAMD_F32, "%s: unknown dtype code %d", who, dtype);
  TT_REQUIRE(B > 0 && S > 0 && D > 0 && D % 16 == 0 && D <= 512 && B < (int64_t(1) << 31) && S < (int64_t(1) << 31) &&
                 B * S < (int64_t(1) << 31),
             "%s: bad shape b=%lld s=%lld h_d=%lld (h_d must be a multiple of 16, at most 512)", who, (long long)B, (long long)S, (long long)D);
  int64_t heads = 0;
  const bool norm = parts[0].scale || parts[1].scale;
  for (int i = 0; i < 2; ++i) {
    const ttamd_rope_heads& p = parts[i];
    TT_REQUIRE(p.heads >= 0 && p.heads < (1 << 20), "%s: bad number of heads %lld", who, (long long)p.heads);
    heads += p.heads;
    Part& q = a.part[i];
    q = Part{};
    if (!p.heads) continue;
    TT_REQUIRE(backward ? (p.gy && (p.x || !norm) && (p.out || p.gscale)) : (p.x && p.out), "%s: null pointer argument", who);
    TT_REQUIRE(!norm || p.scale, "%s: scales for the queries and for the keys, or for neither", who);
    TT_REQUIRE(!p.gscale || norm, "%s: the gradient of a scale that is not there", who);
    q.x = p.x;
    q.scale = p.scale;
    q.gy = p.gy;
    q.out = p.out;
    q.heads = (uint32_t)p.heads;
    for (int d = 0; d < 3; ++d) {
      q.xs[d] = p.x_stride[d];
      q.gs[d] = p.gy_stride[d];
    }
  }
  TT_REQUIRE(heads > 0, "%s: no heads", who);
  TT_REQUIRE(B * S * heads < (int64_t(1) << 31), "%s: more than 2^31 heads of tokens", who);
  TT_REQUIRE((reinterpret_cast<uintptr_t>(at->cache) & 7u) == 0, "%s: the table must be 8-byte aligned", who);
  TT_REQUIRE(at->n_axes >= 1 && at->n_axes <= 4 && (at->n_axes == 1 || at->positions), "%s: positions of %d axes (1 to 4)", who, at->n_axes);
  TT_REQUIRE(at->cache_rows > 0 && (at->positions || at->cache_rows >= S), "%s: the table has %lld rows", who, (long long)at->cache_rows);
  int64_t sum = 0;
  for (int i = 0; i < 4; ++i) {
    TT_REQUIRE(at->n_axes == 1 || i >= at->n_axes || at->section[i] >= 0, "%s: a section of %d frequencies", who, at->section[i]);
    sum += at->n_axes > 1 && i < at->n_axes ? at->section[i] : 0;
    if (i < 3) a.end[i] = i + 1 < at->n_axes ? (int)sum : (int)D;
  }
  TT_REQUIRE(at->n_axes == 1 || sum == D / 2, "%s: the sections hold %lld frequencies, a head has %lld", who, (long long)sum, (long long)(D / 2));
  a.cache = at->cache;
  a.pos = at->positions;
  for (int d = 0; d < 3; ++d) a.ps[d] = at->stride[d];
  a.cache_rows = at->cache_rows;
  a.n_axes = at->n_axes;
  a.S = (uint32_t)S;
  a.tokens = (uint32_t)(B * S);
  a.D = (int)D;
  a.lanes = (int)(D / 16);
  a.log_group = 0;
  while ((1 << a.log_group) < a.lanes) ++a.log_group;
  a.eps = eps;
  return TTAMD_OK;
}

unsigned workgroups(int64_t rows, int log_group) { return (unsigned)(((rows << log_group) + 255) / 256); }

}  // namespace
}  // namespace ttamd

using namespace ttamd;

#define TT_ROPE_CALL(T, NORM_, INTER_, LAUNCH)  \
  if (NORM_) {                                  \
    if (INTER_) {                               \
      LAUNCH(T, true, true)                     \
    } else {                                    \
      LAUNCH(T, true, false)                    \
    }                                           \
  } else if (INTER_) {                          \
    LAUNCH(T, false, true)                      \
  } else {                                      \
    LAUNCH(T, false, false)                     \
  }

extern "C" int ttamd_qk_norm_rope_fwd(const ttamd_rope_heads* parts, const ttamd_rope_positions* at, int dtype, float eps, int64_t B,
                                      int64_t S, int64_t head_dim, void* stream) {
  RopeArgs a;
  if (int rc = prepare("qk_norm_rope_fwd", a, parts, at, dtype, eps, B, S, head_dim, false)) return rc;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  const dim3 grid(workgroups((int64_t)a.tokens * (a.part[0].heads + a.part[1].heads), a.log_group)), block(256);
  const bool norm = parts[0].scale || parts[1].scale;
#define TT_LAUNCH(T, N, I) qk_norm_rope_fwd_kernel<T, N, I><<<grid, block, 0, st>>>(a);
  if (dtype == TTAMD_BF16) {
    TT_ROPE_CALL(BF16, norm, at->interleaved, TT_LAUNCH)
  } else {
    TT_ROPE_CALL(F32, norm, at->interleaved, TT_LAUNCH)
  }
#undef TT_LAUNCH
  return check_launch("qk_norm_rope_fwd");
}

extern "C" size_t ttamd_qk_norm_rope_bwd_workspace_bytes(int64_t head_dim) {
  return head_dim > 0 ? (size_t)kBwdGrid * 2 * (size_t)head_dim * sizeof(float) : 0;
}

extern "C" int ttamd_qk_norm_rope_bwd(const ttamd_rope_heads* parts, const ttamd_rope_positions* at, int dtype, float eps, int64_t B,
                                      int64_t S, int64_t head_dim, void* workspace, size_t workspace_bytes, void* stream) {
  RopeArgs a;
  if (int rc = prepare("qk_norm_rope_bwd", a, parts, at, dtype, eps, B, S, head_dim, true)) return rc;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  const dim3 block(256);
  const bool norm = parts[0].scale || parts[1].scale;
  void* gq = parts[0].heads ? parts[0].gscale : nullptr;
  void* gk = parts[1].heads ? parts[1].gscale : nullptr;
  const unsigned most = workgroups((int64_t)a.tokens * (a.part[0].heads > a.part[1].heads ? a.part[0].heads : a.part[1].heads), a.log_group);
  if (gq || gk) {
    const size_t need = ttamd_qk_norm_rope_bwd_workspace_bytes(head_dim);
    TT_REQUIRE(workspace && aligned16(workspace), "qk_norm_rope_bwd: the gradients of the scales need a 16-byte aligned workspace");
    if (workspace_bytes < need) return fail(TTAMD_EWORKSPACE, "qk_norm_rope_bwd: workspace has %zu bytes, needs %zu", workspace_bytes, need);
    float* partial = reinterpret_cast<float*>(workspace);
    const dim3 grid(most < (unsigned)kBwdGrid ? most : (unsigned)kBwdGrid), sum_grid((unsigned)head_dim / 16, 2);
#define TT_LAUNCH(T, N, I) qk_norm_rope_bwd_kernel<T, true, I, true><<<grid, block, 0, st>>>(a, partial);
    if (dtype == TTAMD_BF16) {
      TT_ROPE_CALL(BF16, true, at->interleaved, TT_LAUNCH)
      qk_norm_rope_gscale_kernel<BF16><<<sum_grid, dim3(1024), 0, st>>>(partial, (int)grid.x, (int)head_dim, gq, gk);
    } else {
      TT_ROPE_CALL(F32, true, at->interleaved, TT_LAUNCH)
      qk_norm_rope_gscale_kernel<F32><<<sum_grid, dim3(1024), 0, st>>>(partial, (int)grid.x, (int)head_dim, gq, gk);
    }
#undef TT_LAUNCH
  } else {
    const dim3 grid(most);
#define TT_LAUNCH(T, N, I) qk_norm_rope_bwd_kernel<T, N, I, false><<<grid, block, 0, st>>>(a, nullptr);
    if (dtype == TTAMD_BF16) {
      TT_ROPE_CALL(BF16, norm, at->interleaved, TT_LAUNCH)
    } else {
      TT_ROPE_CALL(F32, norm, at->interleaved, TT_LAUNCH)
    }
#undef TT_LAUNCH
  }
  return check_launch("qk_norm_rope_bwd");
}
