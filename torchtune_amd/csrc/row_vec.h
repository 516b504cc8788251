// Eight neighbouring elements of a row as floats, whatever the row's type and wherever it begins: an element's own alignment is
// enough (global memory takes wide accesses at any element; rows of odd lengths and views begin anywhere).
#pragma once
#include "common.h"
#include "nf4_math.h"

namespace ttamd {

typedef uint32_t u32x4_at2_t __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u32x2_at2_t __attribute__((ext_vector_type(2), aligned(2)));
typedef float f32x4_at4_t __attribute__((ext_vector_type(4), aligned(4)));

__device__ __forceinline__ uint32_t bf16_pair(float lo, float hi) {
  typedef __bf16 pair_t __attribute__((ext_vector_type(2)));
  pair_t v;
  v.x = (__bf16)lo;
  v.y = (__bf16)hi;
  return __builtin_bit_cast(uint32_t, v);
}

// BF16 and F32 name the element types: `Raw` is how eight of them arrive, `unpack` makes floats of them.
struct BF16 {
  typedef uint16_t elem;
  typedef u32x4_at2_t Raw;
  static __device__ __forceinline__ Raw load(const elem* p) { return *reinterpret_cast<const Raw*>(p); }
  static __device__ __forceinline__ Raw load_once(const elem* p) { return __builtin_nontemporal_load(reinterpret_cast<const Raw*>(p)); }
  static __device__ __forceinline__ void unpack(const Raw& r, float (&v)[8]) {
#pragma unroll
    for (int d = 0; d < 4; ++d) {
      v[2 * d] = bits_f32(r[d] << 16);
      v[2 * d + 1] = bits_f32(r[d] & 0xffff0000u);
    }
  }
  static __device__ __forceinline__ float get(const elem* p) { return bf16_bits_to_f32(*p); }
  static __device__ __forceinline__ void put(elem* p, float v) { *p = (uint16_t)bf16_pair(v, v); }
  static __device__ __forceinline__ Raw pack(const float (&v)[8]) {
    return Raw{bf16_pair(v[0], v[1]), bf16_pair(v[2], v[3]), bf16_pair(v[4], v[5]), bf16_pair(v[6], v[7])};
  }
  static __device__ __forceinline__ void store(elem* p, const Raw& r) { __builtin_nontemporal_store(r, reinterpret_cast<Raw*>(p)); }
  // four neighbours
  typedef u32x2_at2_t Raw4;
  static __device__ __forceinline__ Raw4 load4_once(const elem* p) { return __builtin_nontemporal_load(reinterpret_cast<const Raw4*>(p)); }
  static __device__ __forceinline__ void store4(elem* p, const Raw4& r) { __builtin_nontemporal_store(r, reinterpret_cast<Raw4*>(p)); }
  static __device__ __forceinline__ Raw join(const Raw4& a, const Raw4& b) { return Raw{a.x, a.y, b.x, b.y}; }
  static __device__ __forceinline__ Raw4 low(const Raw& r) { return Raw4{r.x, r.y}; }
  static __device__ __forceinline__ Raw4 high(const Raw& r) { return Raw4{r.z, r.w}; }
};

struct F32 {
  typedef float elem;
  struct Raw {
    f32x4_at4_t a, b;
  };
  static __device__ __forceinline__ Raw load(const elem* p) {
    const f32x4_at4_t* q = reinterpret_cast<const f32x4_at4_t*>(p);
    return Raw{q[0], q[1]};
  }
  static __device__ __forceinline__ Raw load_once(const elem* p) {
    const f32x4_at4_t* q = reinterpret_cast<const f32x4_at4_t*>(p);
    return Raw{__builtin_nontemporal_load(q), __builtin_nontemporal_load(q + 1)};
  }
  static __device__ __forceinline__ void unpack(const Raw& r, float (&v)[8]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[i] = r.a[i];
      v[4 + i] = r.b[i];
    }
  }
  static __device__ __forceinline__ float get(const elem* p) { return *p; }
  static __device__ __forceinline__ void put(elem* p, float v) { *p = v; }
  static __device__ __forceinline__ Raw pack(const float (&v)[8]) {
    return Raw{f32x4_at4_t{v[0], v[1], v[2], v[3]}, f32x4_at4_t{v[4], v[5], v[6], v[7]}};
  }
  static __device__ __forceinline__ void store(elem* p, const Raw& r) {
    // two halves of 32 bytes: the cache has to put neighbouring lanes' together
    f32x4_at4_t* q = reinterpret_cast<f32x4_at4_t*>(p);
    q[0] = r.a;
    q[1] = r.b;
  }
  typedef f32x4_at4_t Raw4;
  static __device__ __forceinline__ Raw4 load4_once(const elem* p) { return __builtin_nontemporal_load(reinterpret_cast<const Raw4*>(p)); }
  static __device__ __forceinline__ void store4(elem* p, const Raw4& r) { __builtin_nontemporal_store(r, reinterpret_cast<Raw4*>(p)); }
  static __device__ __forceinline__ Raw join(const Raw4& a, const Raw4& b) { return Raw{a, b}; }
  static __device__ __forceinline__ Raw4 low(const Raw& r) { return r.a; }
  static __device__ __forceinline__ Raw4 high(const Raw& r) { return r.b; }
};

// A lane's counterpart in a row of sixteen: inside a quad by one and by two, then mirrored in eight and in sixteen (quad
// permutations and row mirrors are moves of the vector ALU, not of LDS).  After the steps before it all lanes of the
// smaller group hold the same value, so that the mirror is as good as an exchange.
template <int STEP>
__device__ __forceinline__ uint32_t row_partner(uint32_t v) {
  constexpr int ctrl = STEP == 1 ? 0xB1 : STEP == 2 ? 0x4E : STEP == 4 ? 0x141 : 0x140;
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, ctrl, 0xf, 0xf, true);
}
template <int STEP>
__device__ __forceinline__ float row_partner(float v) {
  return bits_f32(row_partner<STEP>(f32_bits(v)));
}

}  // namespace ttamd
