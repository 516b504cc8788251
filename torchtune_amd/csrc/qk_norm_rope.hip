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
// Bound: HBM.  A row (one head of one token) belongs to G = 8, 16, 32 or 64 neighbouring lanes, each with eight of its elements,
// which are whole pairs.  8192 tokens of 32 + 8 heads of 128 in bf16: forward 31 us (168 MB, 5.4 TB/s), backward with the gradients of
// the scales 48 us (252 MB, 5.2 TB/s) and 4 us for their sums.  With sixteen elements a lane 36 and 74 us (100 - 150 registers).
#include "row_vec.h"

namespace ttamd {
namespace {

// Workgroups of the backward with scale gradients (one more after rounding): five on a CU, as many as their registers let in.  48 us
// at the size above; 51 with 1024, 52 with 2048, which leave a last round of few.
constexpr int kBwdGrid = 1280;

struct Part {
  const void* x;
  const void* scale;
  const void* gy;
  void* out;
  int64_t xs[3], gs[3];  // of batch, token, head
  uint32_t heads;
  uint32_t units;  // pieces of a token's heads
  uint32_t wgs;    // workgroups
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
  uint32_t some;  // heads in a unit
  int D, lanes, log_group;
  float eps, inv_D;
};

// A lane's eight elements: 8 j .. 8 j + 7, or four of the head's first half and four of its second, 4 j .. 4 j + 3 and
// D / 2 + 4 j ..  The latter where a pair is made of both halves, and for fp32, whose lanes then write whole lines together.
// Pair p of a lane is elements first(p) and second(p) of the eight, and turned by `frequency`.
template <class T, bool INTER>
struct Lane {
  typedef typename T::elem E;
  static constexpr bool split = !INTER || sizeof(E) == 4;
  static constexpr int first(int p) { return INTER ? 2 * p : p; }
  static constexpr int second(int p) { return INTER ? 2 * p + 1 : p + 4; }
  static __device__ __forceinline__ int element(int j, int e, int D) { return split ? 4 * j + (e & 3) + (e >> 2) * (D >> 1) : 8 * j + e; }
  static __device__ __forceinline__ int frequency(int j, int p, int D) {
    return split && INTER ? 2 * j + (p & 1) + (p >> 1) * (D >> 2) : 4 * j + p;
  }
  typename T::Raw raw;
  __device__ __forceinline__ void load(const E* p, int j, int D, bool active) {
    raw = typename T::Raw{};
    if (!active) return;
    if constexpr (split)
      raw = T::join(T::load4_once(p + 4 * j), T::load4_once(p + 4 * j + (D >> 1)));
    else
      raw = T::load_once(p + 8 * j);
  }
  __device__ __forceinline__ void unpack(float (&v)[8]) const { T::unpack(raw, v); }
  static __device__ __forceinline__ void store(E* p, int j, int D, const float (&v)[8]) {
    const typename T::Raw r = T::pack(v);
    if constexpr (split) {
      T::store4(p + 4 * j, T::low(r));
      T::store4(p + 4 * j + (D >> 1), T::high(r));
    } else {
      T::store(p + 8 * j, r);
    }
  }
};

// cosines and sines of a lane's four pairs at token (b, s).  A position outside the table gives NaN and reads nothing.
template <class L>
__device__ __forceinline__ void angles(const RopeArgs& a, uint32_t b, uint32_t s, int j, bool active, float (&cs)[4], float (&sn)[4]) {
  const int half = a.D >> 1;
  const float nan = __builtin_nanf("");
  if (a.n_axes <= 1) {  // uniform
    const int64_t pos = a.pos ? a.pos[b * a.ps[1] + s * a.ps[2]] : (int64_t)s;
    const bool inside = active && (uint64_t)pos < (uint64_t)a.cache_rows;
    const float* c = a.cache + pos * half * 2;
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      f32x4_at4_t v = {nan, nan, nan, nan};
      if (inside) v = *reinterpret_cast<const f32x4_at4_t*>(c + 2 * L::frequency(j, 2 * q, a.D));
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
  for (int p = 0; p < 4; ++p) {
    const int i = L::frequency(j, p, a.D);
    const int64_t at = i < a.end[0] ? pos[0] : i < a.end[1] ? pos[1] : i < a.end[2] ? pos[2] : pos[3];
    typedef float f32x2_t __attribute__((ext_vector_type(2)));
    f32x2_t v = {nan, nan};
    if (active && (uint64_t)at < (uint64_t)a.cache_rows) v = *reinterpret_cast<const f32x2_t*>(a.cache + (at * half + i) * 2);
    cs[p] = v.x;
    sn[p] = v.y;
  }
}

// the sum over the 2^LOG lanes of a row, in every one of them
template <int LOG>
__device__ __forceinline__ float row_sum(float v) {
  v += row_partner<1>(v);
  v += row_partner<2>(v);
  v += row_partner<4>(v);
  if constexpr (LOG > 3) v += row_partner<8>(v);
  if constexpr (LOG > 4) v += __shfl_xor(v, 16, kWave);
  if constexpr (LOG > 5) v += __shfl_xor(v, 32, kWave);
  return v;
}

// 1 / sqrt: the hardware's is off by an ulp, which bf16 results do not show
template <class T>
__device__ __forceinline__ float inverse_root(float v) {
  return sizeof(typename T::elem) == 2 ? __builtin_amdgcn_rsqf(v) : 1.f / __builtin_sqrtf(v);
}

// What a group of lanes works on: every units-th head of one token, one after another, so that the angles are read once for them
// and the next head is on its way while one is worked on.  Neighbouring groups work on neighbouring heads.
struct Unit {
  uint32_t token, b, s, head;
  __device__ __forceinline__ Unit(const RopeArgs& a, const Part& part, uint32_t u) {
    token = u / part.units;
    head = u - token * part.units;
    b = token / a.S;
    s = token - b * a.S;
  }
};

template <class T, int LOG, bool NORM, bool INTER>
__global__ __launch_bounds__(256) void qk_norm_rope_fwd_kernel(const RopeArgs a) {
  typedef typename T::elem E;
  typedef Lane<T, INTER> L;
  const int j = threadIdx.x & ((1 << LOG) - 1);
  const bool active = j < a.lanes, key = blockIdx.x >= a.part[0].wgs;
  const Part& part = a.part[key];  // uniform
  const uint32_t u = (uint32_t)(((uint64_t)(blockIdx.x - (key ? a.part[0].wgs : 0)) * 256 + threadIdx.x) >> LOG);
  if (u >= a.tokens * part.units) return;  // the lanes of a group leave together
  Unit at(a, part, u);
  const E* x = reinterpret_cast<const E*>(part.x) + at.b * part.xs[0] + at.s * part.xs[1] + at.head * part.xs[2];
  E* out = reinterpret_cast<E*>(part.out) + ((int64_t)at.token * part.heads + at.head) * a.D;
  L row;
  row.load(x, j, a.D, active);
  float w[8], cs[4], sn[4];
  angles<L>(a, at.b, at.s, j, active, cs, sn);
  if constexpr (NORM) {
    L scale;
    scale.load(reinterpret_cast<const E*>(part.scale), j, a.D, active);
    scale.unpack(w);
  }
  const int64_t step = part.units * part.xs[2], out_step = (int64_t)part.units * a.D;
  for (uint32_t h = at.head; h < part.heads; h += part.units, x += step, out += out_step) {
    float v[8], o[8];
    row.unpack(v);
    if (h + part.units < part.heads) row.load(x + step, j, a.D, active);
    if constexpr (NORM) {
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) ss = __builtin_fmaf(v[i], v[i], ss);
      const float r = inverse_root<T>(row_sum<LOG>(ss) * a.inv_D + a.eps);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = v[i] * r * w[i];
    }
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      const float c = v[L::first(p)], d = v[L::second(p)];
      o[L::first(p)] = c * cs[p] - d * sn[p];
      o[L::second(p)] = d * cs[p] + c * sn[p];
    }
    if (active) L::store(out, j, a.D, o);
  }
}

// GSCALE: a workgroup walks units of its part with a stride of the part's workgroups, and each lane sums the scale gradient of its
// elements over all that it sees; else there is a workgroup for every 256 / G units.
template <class T, int LOG, bool NORM, bool INTER, bool GSCALE>
__global__ __launch_bounds__(256) void qk_norm_rope_bwd_kernel(const RopeArgs a, float* __restrict__ partial) {
  typedef typename T::elem E;
  typedef Lane<T, INTER> L;
  __shared__ float sums[GSCALE ? 512 : 1];
  const int G = 1 << LOG, j = threadIdx.x & (G - 1);
  const bool active = j < a.lanes, key = blockIdx.x >= a.part[0].wgs;
  const uint32_t per_wg = 256u >> LOG;
  const Part& part = a.part[key];  // uniform
  float w[8], gs[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) gs[i] = 0.f;
  if constexpr (NORM) {
    L scale;
    scale.load(reinterpret_cast<const E*>(part.scale), j, a.D, active);
    scale.unpack(w);
  }
  const uint64_t units = (uint64_t)a.tokens * part.units;
  const int64_t g_step = part.units * part.gs[2], x_step = part.units * part.xs[2], out_step = (int64_t)part.units * a.D;
  for (uint64_t u = (uint64_t)(blockIdx.x - (key ? a.part[0].wgs : 0)) * per_wg + (threadIdx.x >> LOG); u < units;
       u += (uint64_t)part.wgs * per_wg) {  // the lanes of a group together
    const Unit at(a, part, (uint32_t)u);
    const E* gyp = reinterpret_cast<const E*>(part.gy) + at.b * part.gs[0] + at.s * part.gs[1] + at.head * part.gs[2];
    const E* xp = reinterpret_cast<const E*>(part.x) + at.b * part.xs[0] + at.s * part.xs[1] + at.head * part.xs[2];
    E* out = reinterpret_cast<E*>(part.out) + ((int64_t)at.token * part.heads + at.head) * a.D;
    L gy_row, x_row;
    gy_row.load(gyp, j, a.D, active);
    if constexpr (NORM) x_row.load(xp, j, a.D, active);
    float cs[4], sn[4];
    angles<L>(a, at.b, at.s, j, active, cs, sn);
    for (uint32_t h = at.head; h < part.heads; h += part.units, gyp += g_step, xp += x_step, out += out_step) {
      float gy[8], x[8], g[8];
      gy_row.unpack(gy);
      if constexpr (NORM) x_row.unpack(x);
      if (h + part.units < part.heads) {
        gy_row.load(gyp + g_step, j, a.D, active);
        if constexpr (NORM) x_row.load(xp + x_step, j, a.D, active);
      }
#pragma unroll
      for (int p = 0; p < 4; ++p) {
        const float c = gy[L::first(p)], d = gy[L::second(p)];
        g[L::first(p)] = c * cs[p] + d * sn[p];
        g[L::second(p)] = d * cs[p] - c * sn[p];
      }
      if constexpr (NORM) {
        float ss = 0.f, dot = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) ss = __builtin_fmaf(x[i], x[i], ss);
        const float r = inverse_root<T>(row_sum<LOG>(ss) * a.inv_D + a.eps);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float gx = g[i] * x[i];  // an idle lane's angles are NaN; it adds nothing to the row and keeps its sums to itself
          if constexpr (GSCALE) gs[i] = __builtin_fmaf(gx, r, gs[i]);
          g[i] *= w[i];
          dot = __builtin_fmaf(gx, w[i], dot);
        }
        const float c = row_sum<LOG>(active ? dot : 0.f) * a.inv_D * r * r;
#pragma unroll
        for (int i = 0; i < 8; ++i) g[i] = r * __builtin_fmaf(-c, x[i], g[i]);
      }
      if (active && part.out) L::store(out, j, a.D, g);
    }
  }
  if constexpr (GSCALE) {
    // the lanes that hold the same elements meet in LDS, one group of the workgroup after another: a fixed order
    for (int r = 0; r < (int)per_wg; ++r) {
      __syncthreads();
      if ((int)(threadIdx.x >> LOG) != r || !active) continue;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float* at = sums + L::element(j, i, a.D);
        *at = r ? *at + gs[i] : gs[i];
      }
    }
    __syncthreads();
    for (int d = threadIdx.x; d < a.D; d += 256) partial[(int64_t)blockIdx.x * a.D + d] = sums[d];
  }
}

// gscale[d] = sum over the partial sums of the part's workgroups, in slices of a fixed order; blockIdx.y is the part
template <class T>
__global__ __launch_bounds__(1024) void qk_norm_rope_gscale_kernel(const float* __restrict__ partial, int nq, int nk, int D, void* gq, void* gk) {
  typedef typename T::elem E;
  __shared__ float red[64][17];
  const int col = threadIdx.x & 15, slice = threadIdx.x >> 4, d = blockIdx.x * 16 + col;  // D % 16 == 0
  const int n = blockIdx.y ? nk : nq, per = (n + 63) / 64, lo = slice * per, hi = min(lo + per, n);
  const float* p = partial + (int64_t)(blockIdx.y ? nq : 0) * D + d;
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

unsigned workgroups(int64_t units, int log_group) { return (unsigned)(((units << log_group) + 255) / 256); }

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
    for (const void* ptr : {p.x, p.scale, p.gy, (const void*)p.out, (const void*)p.gscale})
      TT_REQUIRE(reinterpret_cast<uintptr_t>(ptr) % (dtype == TTAMD_BF16 ? 2 : 4) == 0, "%s: misaligned pointer argument", who);
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
  a.lanes = (int)(D / 8);
  a.log_group = 3;
  while ((1 << a.log_group) < a.lanes) ++a.log_group;
  a.eps = eps;
  a.inv_D = (float)(1.0 / (double)D);
  // As many heads in a unit, up to four, as leave lanes for four waves on every SIMD of the chip.  At the size above the forward takes
  // 39 us with one, 31.5 with two, 31 with four, 34 with eight.
  a.some = 4;
  while (a.some > 1 && ((B * S * heads) << a.log_group) < (int64_t)a.some * 4 * 1024 * kWave) a.some >>= 1;
  for (Part& q : a.part) {
    q.units = (q.heads + a.some - 1) / a.some;
    q.wgs = workgroups((int64_t)a.tokens * q.units, a.log_group);
  }
  return TTAMD_OK;
}

}  // namespace
}  // namespace ttamd

using namespace ttamd;

// LAUNCH(type, log of a row's lanes, norm, interleaved) with what the call asks for
#define TT_ROPE_LANES(T, N, I, LAUNCH) \
  switch (a.log_group) {               \
    case 3: LAUNCH(T, 3, N, I); break; \
    case 4: LAUNCH(T, 4, N, I); break; \
    case 5: LAUNCH(T, 5, N, I); break; \
    default: LAUNCH(T, 6, N, I);       \
  }
#define TT_ROPE_PAIRS(T, N, LAUNCH)           \
  if (at->interleaved) {                      \
    TT_ROPE_LANES(T, N, true, LAUNCH)         \
  } else {                                    \
    TT_ROPE_LANES(T, N, false, LAUNCH)        \
  }
#define TT_ROPE_CALL(N, LAUNCH)               \
  if (dtype == TTAMD_BF16) {                  \
    TT_ROPE_PAIRS(BF16, N, LAUNCH)            \
  } else {                                    \
    TT_ROPE_PAIRS(F32, N, LAUNCH)             \
  }

extern "C" int ttamd_qk_norm_rope_fwd(const ttamd_rope_heads* parts, const ttamd_rope_positions* at, int dtype, float eps, int64_t B,
                                      int64_t S, int64_t head_dim, void* stream) {
  RopeArgs a;
  if (int rc = prepare("qk_norm_rope_fwd", a, parts, at, dtype, eps, B, S, head_dim, false)) return rc;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  const dim3 grid(a.part[0].wgs + a.part[1].wgs), block(256);
  const bool norm = parts[0].scale || parts[1].scale;
#define TT_LAUNCH(T, L, N, I) qk_norm_rope_fwd_kernel<T, L, N, I><<<grid, block, 0, st>>>(a)
  if (norm) {
    TT_ROPE_CALL(true, TT_LAUNCH)
  } else {
    TT_ROPE_CALL(false, TT_LAUNCH)
  }
#undef TT_LAUNCH
  return check_launch("qk_norm_rope_fwd");
}

extern "C" size_t ttamd_qk_norm_rope_bwd_workspace_bytes(int64_t head_dim) {
  return head_dim > 0 ? (size_t)(kBwdGrid + 1) * (size_t)head_dim * sizeof(float) : 0;
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
  if (gq || gk) {
    const size_t need = ttamd_qk_norm_rope_bwd_workspace_bytes(head_dim);
    TT_REQUIRE(workspace && aligned16(workspace), "qk_norm_rope_bwd: the gradients of the scales need a 16-byte aligned workspace");
    if (workspace_bytes < need) return fail(TTAMD_EWORKSPACE, "qk_norm_rope_bwd: workspace has %zu bytes, needs %zu", workspace_bytes, need);
    float* partial = reinterpret_cast<float*>(workspace);
    // the parts share the workgroups so that each takes as many rounds
    const unsigned rounds = (a.part[0].wgs + a.part[1].wgs + kBwdGrid - 1) / kBwdGrid;
    for (Part& p : a.part) p.wgs = (p.wgs + rounds - 1) / rounds;
    const int nq = (int)a.part[0].wgs, nk = (int)a.part[1].wgs;
    const dim3 grid(nq + nk), sum_grid((unsigned)head_dim / 16, 2);
#define TT_LAUNCH(T, L, N, I) qk_norm_rope_bwd_kernel<T, L, N, I, true><<<grid, block, 0, st>>>(a, partial)
    TT_ROPE_CALL(true, TT_LAUNCH)
#undef TT_LAUNCH
    if (dtype == TTAMD_BF16)
      qk_norm_rope_gscale_kernel<BF16><<<sum_grid, dim3(1024), 0, st>>>(partial, nq, nk, (int)head_dim, gq, gk);
    else
      qk_norm_rope_gscale_kernel<F32><<<sum_grid, dim3(1024), 0, st>>>(partial, nq, nk, (int)head_dim, gq, gk);
  } else {
    const dim3 grid(a.part[0].wgs + a.part[1].wgs);
#define TT_LAUNCH(T, L, N, I) qk_norm_rope_bwd_kernel<T, L, N, I, false><<<grid, block, 0, st>>>(a, nullptr)
    if (norm) {
      TT_ROPE_CALL(true, TT_LAUNCH)
    } else {
      TT_ROPE_CALL(false, TT_LAUNCH)
    }
#undef TT_LAUNCH
  }
  return check_launch("qk_norm_rope_bwd");
}
