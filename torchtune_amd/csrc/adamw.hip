// One AdamW step over many tensors, with the moments in 32 bits or in 8.
//
//   m' = b1 m + (1 - b1) g;  v' = b2 v + (1 - b2) g g;  p' = p (1 - lr wd) - rate (m' / (sqrt(v') root + eps))
//   rate = lr / (1 - b1^t), root = 1 / sqrt(1 - b2^t), formed on the host in 64 bits
//
// in fp32, every product and sum rounded by itself.  Bound: HBM, 22 bytes an element of a bf16 parameter with 32-bit states and 10
// with 8-bit ones.
//
// One launch covers up to 240 tensors: their addresses travel in the kernel's arguments (they may change from step to step),
// their sizes and places in the state buffers stand in a table on the GPU (they do not).  A workgroup takes 4096 elements of one
// tensor, which the chunk map names.
//
// 8 bits: 128 elements, 16 lanes of 8, share an exponent, so that finding it takes four moves within a row of lanes.  A code is
// the top of the fp32 number itself, exponent and 3 (m) or 4 (v) bits of mantissa, relative to the block's exponent: writing and
// reading it are additions and shifts, and what a number is held as does not depend on its neighbours while it is in range.
#include "row_vec.h"

namespace ttamd {
namespace {

constexpr int kChunk = TTAMD_ADAMW_CHUNK, kBlock = TTAMD_ADAMW_BLOCK;

// two rounds of multiplication and shift over a sequence with the golden ratio's step
TT_HD uint32_t spread(uint32_t x) {
  x ^= x >> 16;
  x *= 0x6A09E667u;
  x ^= x >> 15;
  x *= 0xBB67AE85u;
  return x ^ (x >> 16);
}
constexpr uint32_t kStep = 0x9E3779B9u;
TT_HD uint32_t number_of(uint32_t key, int64_t element) {
  return spread((uint32_t)element * kStep + key + (uint32_t)((uint64_t)element >> 32) * 0x85EBCA6Bu);
}

struct Scalars {
  float b1, c1, b2, c2, keep, rate, root, eps;
};

struct StepArgs {
  ttamd_adamw_states st;
  Scalars c;
  uint64_t seed_step;  // of the keys, see key_of
  uint32_t first, first_chunk;
  struct {
    void* p;
    const void* g;
  } t[TTAMD_ADAMW_TENSORS];
};
static_assert(sizeof(StepArgs) <= 4096, "kernel arguments");

TT_HD uint64_t key_base(int64_t seed, int64_t step) {
  return (uint64_t)seed * 0x9E3779B97F4A7C15ull + (uint64_t)step * 0xBF58476D1CE4E5B9ull + 0x6A09E667F3BCC909ull;
}
TT_HD uint32_t key_of(uint64_t base, uint32_t tensor) {
  uint64_t z = base + (uint64_t)tensor * 0x94D049BB133111EBull;
  z = (z ^ (z >> 32)) * 0xD6E8FEB86659FD93ull;
  z = (z ^ (z >> 32)) * 0xD6E8FEB86659FD93ull;
  return (uint32_t)(z ^ (z >> 32));
}

__device__ __forceinline__ uint32_t row_max(uint32_t v) {  // of sixteen lanes
  v = max(v, row_partner<1>(v));
  v = max(v, row_partner<2>(v));
  v = max(v, row_partner<4>(v));
  return max(v, row_partner<8>(v));
}

typedef uint32_t u32x2_at1_t __attribute__((ext_vector_type(2), aligned(1)));

// Eight elements from element `at` of n: whole where they are there, one by one at the end.
template <class T>
__device__ __forceinline__ void load8(const typename T::elem* p, int64_t at, int64_t n, float (&v)[8]) {
  if (at + 8 <= n) {
    T::unpack(T::load_once(p + at), v);
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = at + i < n ? T::get(p + at + i) : 0.f;
}
template <class T>
__device__ __forceinline__ void store8(typename T::elem* p, int64_t at, int64_t n, const float (&v)[8]) {
  if (at + 8 <= n) {
    T::store(p + at, T::pack(v));
    return;
  }
  for (int i = 0; i < 8; ++i)
    if (at + i < n) T::put(p + at + i, v[i]);
}
__device__ __forceinline__ void load_codes(const uint8_t* p, int64_t at, int64_t n, uint32_t (&c)[2]) {
  if (at + 8 <= n) {
    const u32x2_at1_t v = *reinterpret_cast<const u32x2_at1_t*>(p + at);
    c[0] = v.x;
    c[1] = v.y;
    return;
  }
  c[0] = c[1] = 0;
  for (int i = 0; i < 8; ++i)
    if (at + i < n) c[i >> 2] |= (uint32_t)p[at + i] << (8 * (i & 3));
}
__device__ __forceinline__ void store_codes(uint8_t* p, int64_t at, int64_t n, const uint32_t (&c)[2]) {
  if (at + 8 <= n) {
    *reinterpret_cast<u32x2_at1_t*>(p + at) = u32x2_at1_t{c[0], c[1]};
    return;
  }
  for (int i = 0; i < 8; ++i)
    if (at + i < n) p[at + i] = (uint8_t)(c[i >> 2] >> (8 * (i & 3)));
}

template <bool FIRST>
struct Code {  // FIRST: a sign and three bits of mantissa; else four
  static constexpr int mantissa = FIRST ? 3 : 4, drop = 23 - mantissa;
  static __device__ __forceinline__ float value(uint32_t c, uint32_t base) {
    const uint32_t size = FIRST ? c & 127u : c;
    const uint32_t bits = size ? (size + base) << drop : 0u;
    return bits_f32(FIRST ? bits | (c & 128u) << 24 : bits);
  }
  // the number's top bits after `r` (16 bits) has decided which way they are rounded
  static __device__ __forceinline__ uint32_t top(float x, uint32_t r) {
    const uint32_t size = min(f32_bits(x) & 0x7fffffffu, 0x7f800000u);
    return (size + (r << (drop - 16)) + (1u << (drop - 17))) >> drop;
  }
  static __device__ __forceinline__ uint32_t base(uint32_t exponent) { return (exponent - 15u) << mantissa; }
  static __device__ __forceinline__ uint32_t exponent(uint32_t largest_top) { return max(largest_top >> mantissa, 16u); }
  static __device__ __forceinline__ uint32_t code(uint32_t top, float x, uint32_t base) {
    const int c = (int)top - (int)base;
    if (FIRST) return c < 1 ? 0u : (uint32_t)c | ((f32_bits(x) >> 24) & 128u);
    return f32_bits(x) << 1 == 0u ? 0u : (uint32_t)max(c, 1);
  }
};

template <class T, bool EIGHT, bool ROUND>
__global__ __launch_bounds__(256) void adamw_step_kernel(const StepArgs a) {
  typedef typename T::elem E;
  const uint32_t chunk = a.first_chunk + blockIdx.x, tensor = a.st.chunk_map[chunk];
  const ttamd_adamw_place place = a.st.layout[tensor];
  E* p = reinterpret_cast<E*>(a.t[tensor - a.first].p);
  const E* g = reinterpret_cast<const E*>(a.t[tensor - a.first].g);
  const int64_t n = place.numel, start = (int64_t)(chunk - place.first_chunk) * kChunk;
  uint32_t key = 0;
  if constexpr (EIGHT || ROUND) key = key_of(a.seed_step, place.number);
#pragma unroll
  for (int piece = 0; piece < kChunk / 2048; ++piece) {
    const int64_t at = start + piece * 2048 + 8 * threadIdx.x;
    const bool any = at < n;  // lanes behind the end stay for the row maxima
    float pv[8], gv[8], m[8], v[8];
    load8<T>(p, at, n, pv);
    load8<T>(g, at, n, gv);
    const int64_t block = place.block + at / kBlock;
    if constexpr (EIGHT) {
      uint32_t mc[2], vc[2], em = 16, ev = 16;
      load_codes(reinterpret_cast<const uint8_t*>(a.st.exp_avg) + place.offset, at, n, mc);
      load_codes(reinterpret_cast<const uint8_t*>(a.st.exp_avg_sq) + place.offset, at, n, vc);
      if (any) {
        em = a.st.exp_avg_exponent[block];
        ev = a.st.exp_avg_sq_exponent[block];
      }
      const uint32_t bm = Code<true>::base(em), bv = Code<false>::base(ev);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        m[i] = Code<true>::value((mc[i >> 2] >> (8 * (i & 3))) & 255u, bm);
        v[i] = Code<false>::value((vc[i >> 2] >> (8 * (i & 3))) & 255u, bv);
      }
    } else {
      load8<F32>(reinterpret_cast<const float*>(a.st.exp_avg) + place.offset, at, n, m);
      load8<F32>(reinterpret_cast<const float*>(a.st.exp_avg_sq) + place.offset, at, n, v);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      m[i] = m[i] * a.c.b1 + gv[i] * a.c.c1;
      v[i] = v[i] * a.c.b2 + (gv[i] * gv[i]) * a.c.c2;
      pv[i] = pv[i] * a.c.keep - a.c.rate * (m[i] / (__builtin_sqrtf(v[i]) * a.c.root + a.c.eps));
    }
    uint32_t r[8];
    if constexpr (EIGHT || ROUND) {
      const uint32_t x0 = (uint32_t)at * kStep + key + (uint32_t)((uint64_t)at >> 32) * 0x85EBCA6Bu;
#pragma unroll
      for (int i = 0; i < 8; ++i) r[i] = spread(x0 + i * kStep);
    }
    if constexpr (ROUND) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t b = f32_bits(pv[i]);
        // NaN and infinity as they are
        pv[i] = (b & 0x7f800000u) == 0x7f800000u ? pv[i] : bits_f32((b + (r[i] & 0xffffu)) & 0xffff0000u);
      }
    }
    store8<T>(p, at, n, pv);
    if constexpr (EIGHT) {
      uint32_t mt[8], vt[8], mm = 0, vm = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        mt[i] = Code<true>::top(m[i], r[i] & 0xffffu);
        vt[i] = Code<false>::top(v[i], r[i] >> 16);
        if (at + i < n) {
          mm = max(mm, mt[i]);
          vm = max(vm, vt[i]);
        }
      }
      const uint32_t em = Code<true>::exponent(row_max(mm)), ev = Code<false>::exponent(row_max(vm));
      const uint32_t bm = Code<true>::base(em), bv = Code<false>::base(ev);
      uint32_t mc[2] = {0, 0}, vc[2] = {0, 0};
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        mc[i >> 2] |= Code<true>::code(mt[i], m[i], bm) << (8 * (i & 3));
        vc[i >> 2] |= Code<false>::code(vt[i], v[i], bv) << (8 * (i & 3));
      }
      store_codes(reinterpret_cast<uint8_t*>(a.st.exp_avg) + place.offset, at, n, mc);
      store_codes(reinterpret_cast<uint8_t*>(a.st.exp_avg_sq) + place.offset, at, n, vc);
      if (any && (threadIdx.x & 15) == 0) {
        a.st.exp_avg_exponent[block] = (uint8_t)em;
        a.st.exp_avg_sq_exponent[block] = (uint8_t)ev;
      }
    } else {
      store8<F32>(reinterpret_cast<float*>(a.st.exp_avg) + place.offset, at, n, m);
      store8<F32>(reinterpret_cast<float*>(a.st.exp_avg_sq) + place.offset, at, n, v);
    }
  }
}

__global__ __launch_bounds__(256) void adamw_moments_kernel(const ttamd_adamw_states st, uint16_t* __restrict__ exp_avg,
                                                            uint16_t* __restrict__ exp_avg_sq) {
  const uint32_t chunk = blockIdx.x;
  const ttamd_adamw_place place = st.layout[st.chunk_map[chunk]];
  const int64_t n = place.numel, start = (int64_t)(chunk - place.first_chunk) * kChunk;
#pragma unroll
  for (int piece = 0; piece < kChunk / 2048; ++piece) {
    const int64_t at = start + piece * 2048 + 8 * threadIdx.x;
    if (at >= n) continue;
    const int64_t block = place.block + at / kBlock;
    uint32_t mc[2], vc[2];
    load_codes(reinterpret_cast<const uint8_t*>(st.exp_avg) + place.offset, at, n, mc);
    load_codes(reinterpret_cast<const uint8_t*>(st.exp_avg_sq) + place.offset, at, n, vc);
    const uint32_t bm = Code<true>::base(st.exp_avg_exponent[block]), bv = Code<false>::base(st.exp_avg_sq_exponent[block]);
    float m[8], v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      m[i] = Code<true>::value((mc[i >> 2] >> (8 * (i & 3))) & 255u, bm);
      v[i] = Code<false>::value((vc[i >> 2] >> (8 * (i & 3))) & 255u, bv);
    }
    store8<BF16>(exp_avg + place.offset, at, n, m);
    store8<BF16>(exp_avg_sq + place.offset, at, n, v);
  }
}

int check_states(const char* who, const ttamd_adamw_states* s) {
  TT_REQUIRE(s && s->layout && s->chunk_map && s->exp_avg && s->exp_avg_sq, "%s: null pointer argument", who);
  TT_REQUIRE(s->state_bits == 32 || s->state_bits == 8, "%s: states of %d bits (8 or 32)", who, s->state_bits);
  TT_REQUIRE(s->state_bits == 32 || (s->exp_avg_exponent && s->exp_avg_sq_exponent), "%s: null pointer argument", who);
  return TTAMD_OK;
}

}  // namespace
}  // namespace ttamd

using namespace ttamd;

extern "C" uint32_t ttamd_adamw_key(int64_t seed, int64_t step, uint32_t tensor) { return key_of(key_base(seed, step), tensor); }
extern "C" uint32_t ttamd_adamw_number(uint32_t key, int64_t element) { return number_of(key, element); }

extern "C" int ttamd_adamw_step(void* const* params, const void* const* grads, int n, int dtype, const ttamd_adamw_states* states,
                                uint32_t first, uint32_t first_chunk, uint32_t n_chunks, const ttamd_adamw_scalars* s, void* stream) {
  TT_REQUIRE(params && grads && s, "adamw_step: null pointer argument");
  if (int rc = check_states("adamw_step", states)) return rc;
  TT_REQUIRE(dtype == TTAMD_BF16 || dtype == TTAMD_F32, "adamw_step: unknown dtype code %d", dtype);
  TT_REQUIRE(n > 0 && n <= TTAMD_ADAMW_TENSORS, "adamw_step: %d tensors (1 to %d)", n, TTAMD_ADAMW_TENSORS);
  TT_REQUIRE(n_chunks > 0 && n_chunks < (1u << 31), "adamw_step: %u chunks", n_chunks);
  TT_REQUIRE(s->step >= 1, "adamw_step: step %lld (counted from 1)", (long long)s->step);
  TT_REQUIRE(s->beta1 >= 0 && s->beta1 < 1 && s->beta2 >= 0 && s->beta2 < 1 && s->eps >= 0, "adamw_step: betas %g, %g and eps %g", s->beta1,
             s->beta2, s->eps);
  TT_REQUIRE(!s->stochastic || dtype == TTAMD_BF16, "adamw_step: stochastic rounding is for bf16 parameters");
  StepArgs a;
  a.st = *states;
  a.seed_step = key_base(s->seed, s->step);
  a.first = first;
  a.first_chunk = first_chunk;
  for (int i = 0; i < n; ++i) {
    TT_REQUIRE(params[i] && grads[i], "adamw_step: null pointer argument");
    a.t[i].p = params[i];
    a.t[i].g = grads[i];
  }
  for (int i = n; i < TTAMD_ADAMW_TENSORS; ++i) a.t[i] = {nullptr, nullptr};
  a.c = {(float)s->beta1, (float)(1 - s->beta1), (float)s->beta2, (float)(1 - s->beta2), (float)(1 - s->lr * s->weight_decay),
         (float)(s->lr / (1 - __builtin_pow(s->beta1, (double)s->step))), (float)(1 / __builtin_sqrt(1 - __builtin_pow(s->beta2, (double)s->step))),
         (float)s->eps};
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  const dim3 grid(n_chunks), block(256);
  const bool eight = states->state_bits == 8;
  if (dtype == TTAMD_F32) {
    if (eight)
      adamw_step_kernel<F32, true, false><<<grid, block, 0, st>>>(a);
    else
      adamw_step_kernel<F32, false, false><<<grid, block, 0, st>>>(a);
  } else if (eight) {
    if (s->stochastic)
      adamw_step_kernel<BF16, true, true><<<grid, block, 0, st>>>(a);
    else
      adamw_step_kernel<BF16, true, false><<<grid, block, 0, st>>>(a);
  } else if (s->stochastic) {
    adamw_step_kernel<BF16, false, true><<<grid, block, 0, st>>>(a);
  } else {
    adamw_step_kernel<BF16, false, false><<<grid, block, 0, st>>>(a);
  }
  return check_launch("adamw_step");
}

extern "C" int ttamd_adamw_moments_bf16(const ttamd_adamw_states* states, uint32_t n_chunks, void* exp_avg, void* exp_avg_sq, void* stream) {
  if (int rc = check_states("adamw_moments", states)) return rc;
  TT_REQUIRE(states->state_bits == 8, "adamw_moments: states of %d bits", states->state_bits);
  TT_REQUIRE(exp_avg && exp_avg_sq && n_chunks > 0 && n_chunks < (1u << 31), "adamw_moments: bad argument");
  adamw_moments_kernel<<<dim3(n_chunks), dim3(256), 0, reinterpret_cast<hipStream_t>(stream)>>>(
      *states, reinterpret_cast<uint16_t*>(exp_avg), reinterpret_cast<uint16_t*>(exp_avg_sq));
  return check_launch("adamw_moments");
}
