// Log probabilities of given tokens, the entropy of each row and its largest log probabilities, and the gradient of the first two.
//
//   z = x / temperature;  m = max x;  d_j = (x_j - m) / temperature;  s = sum e^d_j;  u = sum e^d_j d_j
//   log p_j = d_j - ln s;  H = ln s - u / s
//   grad x_j = ( sum_t g_t [j = token t] - p_j sum_t g_t - gH p_j (log p_j + H) ) / temperature
//
// Forward: one pass over the logits with a running maximum, sum and weighted sum per thread, in fp32 and powers of two.  While the
// row streams, a thread shifts by M = fp32(c x_max), c = log2(e) / temperature, so that an element costs one fused multiply-add and
// one exp2; the sums are moved from M to c m at the end, so that nothing of M's rounding is left in them.
// Backward: the logits again, with m, s and H of each row kept from the forward (16 bytes a row instead of a second tensor of logits).
//
// Bound: HBM, closely followed by the vector ALU in the forward over bf16: at 6 TB/s a compute unit takes about 5 elements a
// cycle, which leaves twelve lane operations for each, and exp2 alone takes four.  2048 x 128256 in bf16 with the entropy: forward
// 95 us (525 MB, 5.5 TB/s), backward 163 us (1.05 GB, 6.4 TB/s); 700 x 50257 in fp32, rows at odd places: 24 and 47 us (5.9 and 6.0).
//
// The largest elements come from the same pass: a number that k maxima of disjoint sets of elements reach is no larger than the k-th
// largest element, so that only threads whose maximum reaches it (a few more than k) look at their elements again; what they find is
// ranked by counting.  An element and its place are one 64-bit number (larger value first, of equal values the earlier place), so
// that the result does not depend on the order in which candidates are found.
#include "row_vec.h"

namespace ttamd {
namespace {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kLowest = -3.4028234663852886e38f;
constexpr int kTopMax = 64;        // most alternatives
constexpr int kSegmentsMax = 64;   // of a row

struct LogitArgs {
  const void* logits;
  int64_t outer, inner;  // strides of row / n_inner and row % n_inner, in elements
  uint32_t rows, n_inner, V;
  uint32_t segments, segment;  // of a row, and elements in each (a multiple of 8)
  const int64_t* tokens;
  int64_t ignore_index;
  int n_tokens, top;
  float c;        // log2(e) / temperature
  float inv_temp;
  float* logprobs;
  float* entropy;
  float* top_logprobs;
  int64_t* top_tokens;
  float* stats;             // [rows, 4]: m, 1 / s, log2 s, H; or null
  float* part;              // [rows, segments, 4]
  uint64_t* part_top;       // [rows, segments, top]
};

// larger number: larger value, then earlier place.  NaN counts as -inf, as it does for the maxima.
__device__ __forceinline__ uint32_t ordered(float v) {
  const uint32_t b = f32_bits(v != v ? -__builtin_inff() : v + 0.f);  // -0 is 0
  return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float from_ordered(uint32_t k) { return bits_f32((k & 0x80000000u) ? k ^ 0x80000000u : ~k); }
__device__ __forceinline__ uint64_t candidate(float v, uint32_t at) { return ((uint64_t)ordered(v) << 32) | (0xffffffffu - at); }

// over the wave, in every lane: each row of sixteen by moves of the vector ALU, then one lane of each
__device__ __forceinline__ float lane_of(float v, int lane) { return bits_f32((uint32_t)__builtin_amdgcn_readlane((int)f32_bits(v), lane)); }
__device__ __forceinline__ float wave_max(float v) {
  v = __builtin_fmaxf(v, row_partner<1>(v));
  v = __builtin_fmaxf(v, row_partner<2>(v));
  v = __builtin_fmaxf(v, row_partner<4>(v));
  v = __builtin_fmaxf(v, row_partner<8>(v));
  return __builtin_fmaxf(__builtin_fmaxf(lane_of(v, 0), lane_of(v, 16)), __builtin_fmaxf(lane_of(v, 32), lane_of(v, 48)));
}
__device__ __forceinline__ float wave_add(float v) {
  v += row_partner<1>(v);
  v += row_partner<2>(v);
  v += row_partner<4>(v);
  v += row_partner<8>(v);
  return (lane_of(v, 0) + lane_of(v, 16)) + (lane_of(v, 32) + lane_of(v, 48));
}

// what a thread knows of the elements it has seen: largest x; sums shifted by M = fp32(c max), a finite number
struct Running {
  float max = -__builtin_inff(), M = kLowest, s = 0.f, u = 0.f;
};
__device__ __forceinline__ float shift(float max, float c) { return __builtin_amdgcn_fmed3f(max * c, kLowest, -kLowest); }

template <bool ENT>
__device__ __forceinline__ void add(Running& r, const float* v, int n, float c) {
  float top = r.max;
#pragma unroll
  for (int i = 0; i < n; ++i) top = __builtin_fmaxf(top, v[i]);
  const float M = shift(top, c), d = r.M - M, f = __builtin_amdgcn_exp2f(d);
  if constexpr (ENT) r.u = f * (r.u + r.s * __builtin_fmaxf(d, -1e30f));
  r.s *= f;
  r.max = top;
  r.M = M;
#pragma unroll
  for (int i = 0; i < n; ++i) {
    const float y = __builtin_fmaf(v[i], c, -M), e = __builtin_amdgcn_exp2f(y);
    r.s += e;
    if constexpr (ENT) r.u = __builtin_fmaf(e, __builtin_fmaxf(y, -200.f), r.u);  // e is 0 below
  }
}

// (max, s, u) of two sets of elements as one
template <bool ENT>
__device__ __forceinline__ void shift_to(Running& r, float max, float c) {
  const float M = shift(max, c), d = r.M - M, f = __builtin_amdgcn_exp2f(d);
  if constexpr (ENT) r.u = f * (r.u + r.s * __builtin_fmaxf(d, -1e30f));
  r.s *= f;
  r.max = max;
  r.M = M;
}

// over the workgroup, in every thread
template <int NT, bool ENT>
__device__ __forceinline__ void meet(Running& r, float c, float (*lds)[3]) {
  const int wave = threadIdx.x >> 6;
  shift_to<ENT>(r, wave_max(r.max), c);
  r.s = wave_add(r.s);
  if constexpr (ENT) r.u = wave_add(r.u);
  if constexpr (NT == 64) return;
  if ((threadIdx.x & 63) == 0) {
    lds[wave][0] = r.max;
    lds[wave][1] = r.s;
    lds[wave][2] = r.u;
  }
  __syncthreads();
  float max = lds[0][0];
#pragma unroll
  for (int w = 1; w < NT / 64; ++w) max = __builtin_fmaxf(max, lds[w][0]);
  Running all;
  all.max = max;
  all.M = shift(max, c);
#pragma unroll
  for (int w = 0; w < NT / 64; ++w) {
    Running one;
    one.max = lds[w][0];
    one.M = shift(one.max, c);
    one.s = lds[w][1];
    one.u = lds[w][2];
    shift_to<ENT>(one, max, c);
    all.s += one.s;
    all.u += one.u;
  }
  r = all;
}

// Eight elements of the row from `at`; what lies behind the end counts as -inf.
template <class T>
__device__ __forceinline__ void fetch(const typename T::elem* x, uint32_t at, uint32_t end, float (&v)[8]) {
  if (at + 8 <= end) {
    T::unpack(T::load(x + at), v);
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = at + i < end ? T::get(x + at + i) : -__builtin_inff();
}

// A bound that k of the wave's numbers, N a lane, reach: the k-th largest, by halving, of as many bits as a T has.  The wave counts
// with its lane masks.
template <class T, int N>
__device__ __forceinline__ uint32_t kth_bound(const uint32_t (&mine)[N], int k) {
  constexpr uint32_t kLast = sizeof(typename T::elem) == 2 ? 1u << 16 : 1u;
  uint32_t bound = 0;
#pragma unroll 1
  for (uint32_t bit = 1u << 31; bit >= kLast; bit >>= 1) {
    const uint32_t trial = bound | bit;
    int count = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) count += __popcll(__ballot(mine[i] >= trial));
    if (count >= k) bound = trial;
  }
  return bound;
}

constexpr int kRankAhead = 8;

template <int NT>
struct TopScratch {
  static constexpr int kCandidates = 4 * NT;  // found in a workgroup before the exact search takes over
  uint64_t found[kCandidates + kRankAhead];
  uint64_t best[kTopMax];
  uint32_t keys[NT];
  uint32_t count, bound;
  uint64_t wave_best[NT / kWave];
};

// found[0 .. n) -> the k largest, in order, in best (0 where there are fewer)
template <int NT>
__device__ __forceinline__ void rank(TopScratch<NT>& t, int n, int k) {
  for (int i = threadIdx.x; i < k; i += NT) t.best[i] = 0;
  if (threadIdx.x < kRankAhead) t.found[n + threadIdx.x] = 0;
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += NT) {
    const uint64_t mine = t.found[i];
    int above = 0;
    for (int q = 0; q < n; q += kRankAhead) {
#pragma unroll
      for (int e = 0; e < kRankAhead; ++e) above += t.found[q + e] > mine;
    }
    if (above < k) t.best[above] = mine;
  }
  __syncthreads();
}

// The k largest elements of [lo, hi) of a row, in t.best.  mine: the largest of the elements this thread has seen, which are
// the pieces of eight lo + 8 (threadIdx.x + NT i); largest: that of all threads.
template <class T, int NT>
__device__ void find_top(TopScratch<NT>& t, const typename T::elem* x, uint32_t lo, uint32_t hi, float mine, float largest, int k) {
  const uint32_t key = ordered(mine);
  if (threadIdx.x == 0) t.count = 0;
  uint32_t bound = ordered(largest);
  if (k > 1) {
    // k maxima that reach the bound hold k elements that do.  Of n maxima (of threads, or of the threads of one lane of all waves)
    // about n ln(n / (n - k)) elements reach it: from 64 maxima 24 for k = 20, but 97 for k = 50 against 56 from 256.
    constexpr int N = NT / kWave;
    t.keys[threadIdx.x] = key;
    __syncthreads();
    if (threadIdx.x < kWave) {
      uint32_t maxima[N], group[1] = {0};
#pragma unroll
      for (int w = 0; w < N; ++w) {
        maxima[w] = t.keys[threadIdx.x + kWave * w];
        group[0] = max(group[0], maxima[w]);
      }
      const uint32_t b = k <= 24 ? kth_bound<T>(group, k) : kth_bound<T>(maxima, k);
      if (threadIdx.x == 0) t.bound = b;
    }
    __syncthreads();
    bound = t.bound;
  } else {
    __syncthreads();
  }
  const float least = bound <= ordered(-__builtin_inff()) ? -__builtin_inff() : from_ordered(bound);
  auto look = [&](const float(&v)[8], uint32_t at) {
    float top = v[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) top = __builtin_fmaxf(top, v[i]);
    if (!(top >= least)) return;
    uint32_t some = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) some += v[i] >= least && at + i < hi;
    uint32_t slot = atomicAdd(&t.count, some);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (!(v[i] >= least && at + i < hi)) continue;
      if (slot < t.kCandidates) t.found[slot] = candidate(v[i], at + i);
      ++slot;
    }
  };
  // What this costs is the number of times that a wave waits for memory, with four loads under way: each thread that reaches the
  // bound for itself, or all lanes for one such thread after another, a piece each.
  constexpr int kAhead = 4;
  const uint32_t lane = threadIdx.x & 63, pieces = (hi - lo + 8 * NT - 1) / (8 * NT);
  uint64_t todo = __ballot(key >= bound);
  if ((uint32_t)__popcll(todo) * ((pieces + 63) / 64) < pieces) {  // uniform
    while (todo) {
      uint32_t first[kAhead];
#pragma unroll
      for (int q = 0; q < kAhead; ++q) {
        first[q] = todo ? lo + 8 * ((threadIdx.x & ~63u) + (uint32_t)__builtin_ctzll(todo)) : hi;
        todo &= todo - 1;
      }
      for (uint32_t piece = lane; piece < pieces + lane; piece += kWave) {
        typename T::Raw raw[kAhead];
#pragma unroll
        for (int q = 0; q < kAhead; ++q) {
          const uint32_t at = first[q] + 8 * NT * piece;
          raw[q] = typename T::Raw{};
          if (at + 8 <= hi) raw[q] = T::load(x + at);
        }
#pragma unroll
        for (int q = 0; q < kAhead; ++q) {
          const uint32_t at = first[q] + 8 * NT * piece;
          if (at >= hi) continue;
          float v[8];
          if (at + 8 <= hi)
            T::unpack(raw[q], v);
          else
            fetch<T>(x, at, hi, v);
          look(v, at);
        }
      }
    }
  } else if (key >= bound) {
    uint32_t at = lo + 8 * threadIdx.x;
    for (; at + 8 * NT * (kAhead - 1) + 8 <= hi; at += 8 * NT * kAhead) {
      typename T::Raw raw[kAhead];
#pragma unroll
      for (int q = 0; q < kAhead; ++q) raw[q] = T::load(x + at + 8 * NT * q);
#pragma unroll
      for (int q = 0; q < kAhead; ++q) {
        float v[8];
        T::unpack(raw[q], v);
        look(v, at + 8 * NT * q);
      }
    }
    for (; at < hi; at += 8 * NT) {
      float v[8];
      fetch<T>(x, at, hi, v);
      look(v, at);
    }
  }
  __syncthreads();
  const uint32_t n = t.count;
  if (n <= t.kCandidates) {  // uniform
    rank<NT>(t, (int)n, k);
    return;
  }
  // Many equal elements at the bound (a row that is masked but for a few, an even distribution): the largest below the one
  // found before, k times.
  uint64_t last = ~0ull;
  for (int i = 0; i < k; ++i) {
    uint64_t best = 0;
    for (uint32_t at = lo + 8 * threadIdx.x; at < hi; at += 8 * NT) {
      float v[8];
      fetch<T>(x, at, hi, v);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint64_t one = at + e < hi ? candidate(v[e], at + e) : 0;
        if (one < last && one > best) best = one;
      }
    }
#pragma unroll
    for (int off = 1; off < kWave; off <<= 1) {
      const uint64_t other = __shfl_xor(best, off, kWave);
      best = other > best ? other : best;
    }
    __syncthreads();
    if ((threadIdx.x & 63) == 0) t.wave_best[threadIdx.x >> 6] = best;
    __syncthreads();
    best = t.wave_best[0];
#pragma unroll
    for (int w = 1; w < NT / 64; ++w) best = t.wave_best[w] > best ? t.wave_best[w] : best;
    if (threadIdx.x == 0) t.best[i] = best;
    last = best;
  }
  __syncthreads();
}

// The first given token of a thread with its logit, asked for before the row is read: two reads that depend on each other.
template <class T>
struct Given {
  int64_t token = 0;
  float x = 0.f;
  bool valid = false;
  __device__ __forceinline__ void read(const LogitArgs& a, uint32_t row, const typename T::elem* logits, int i) {
    if (i >= a.n_tokens) return;
    token = a.tokens[(int64_t)row * a.n_tokens + i];
    valid = (uint64_t)token < a.V;  // any other place gives NaN and reads nothing
    if (valid) x = T::get(logits + token);
  }
};

// What is written for a row from its maximum and sums; every thread has them.
template <class T, int NT, bool ENT>
__device__ void finish(const LogitArgs& a, uint32_t row, const typename T::elem* x, Running r, Given<T> given, const TopScratch<NT>* t, float (*lds)[3]) {
  float s, u;
  const float rest = r.s > 0.f ? __builtin_fmaf(r.max, a.c, -r.M) : 0.f;  // what M's rounding left of the largest exponent
  const bool whole = r.s > 0.f && r.s < __builtin_inff() && __builtin_fabsf(r.u) < __builtin_inff() && __builtin_fabsf(rest) < 64.f;
  if (__builtin_fabsf(r.max) < __builtin_inff() && !whole) {
    // c x overflows or is too coarse (a row masked with the lowest value of its type, logits beyond 1e9): the differences are not.
    float ps = 0.f, pu = 0.f;
    for (uint32_t j = threadIdx.x; j < a.V; j += NT) {
      const float y = (T::get(x + j) - r.max) * a.c, e = __builtin_amdgcn_exp2f(y);
      ps += e;
      pu += e * __builtin_fmaxf(y, -200.f);
    }
    ps = wave_add(ps);
    pu = wave_add(pu);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) {
      lds[threadIdx.x >> 6][0] = ps;
      lds[threadIdx.x >> 6][1] = pu;
    }
    __syncthreads();
    s = u = 0.f;
    for (int w = 0; w < NT / 64; ++w) {
      s += lds[w][0];
      u += lds[w][1];
    }
  } else {
    // from M to c m: y' = y - rest, so e' = e 2^-rest
    const float f = __builtin_amdgcn_exp2f(-rest);
    s = r.s * f;
    u = f * (r.u - rest * r.s);
  }
  const bool empty = s == 0.f;  // nothing but -inf: no token has a probability
  const float log2s = empty ? 0.f : __builtin_amdgcn_logf(s), inv = empty ? 0.f : 1.f / s, m = empty ? 0.f : r.max;
  const float H = empty ? 0.f : (log2s - u * inv) * kLn2, lse = log2s * kLn2;
  if (threadIdx.x == 0) {
    if (a.entropy) a.entropy[row] = H;
    if (a.stats) {
      float* st = a.stats + 4 * (int64_t)row;
      st[0] = m;
      st[1] = inv;
      st[2] = log2s;
      st[3] = H;
    }
  }
  const float none = -__builtin_inff();
  for (int i = threadIdx.x; i < a.n_tokens; i += NT) {
    if (i >= NT) given.read(a, row, x, i);
    float lp = given.valid ? empty ? none : (given.x - m) * a.inv_temp - lse : __builtin_nanf("");
    if (given.token == a.ignore_index) lp = 0.f;
    a.logprobs[(int64_t)row * a.n_tokens + i] = lp;
  }
  for (int i = threadIdx.x; i < a.top; i += NT) {
    const uint64_t best = t->best[i];
    const uint32_t place = min(0xffffffffu - (uint32_t)best, a.V - 1);
    const float v = from_ordered((uint32_t)(best >> 32));  // in a row with a NaN, lse is one
    a.top_logprobs[(int64_t)row * a.top + i] = empty ? none : (v - m) * a.inv_temp - lse;
    a.top_tokens[(int64_t)row * a.top + i] = (int64_t)place;
  }
}

template <class T>
__device__ __forceinline__ const typename T::elem* row_of(const LogitArgs& a, uint32_t row) {
  const uint32_t o = row / a.n_inner;
  return reinterpret_cast<const typename T::elem*>(a.logits) + (int64_t)o * a.outer + (int64_t)(row - o * a.n_inner) * a.inner;
}

// A workgroup per row, or per segment of a row where there are few rows.
template <class T, int NT, bool ENT, bool TOP>
__global__ __launch_bounds__(NT) void token_logprobs_fwd_kernel(const LogitArgs a) {
  typedef typename T::elem E;
  __shared__ float lds[NT / 64][3];
  __shared__ char scratch[TOP ? sizeof(TopScratch<NT>) : 8] __attribute__((aligned(8)));
  TopScratch<NT>* top = reinterpret_cast<TopScratch<NT>*>(scratch);
  const uint32_t row = blockIdx.x / a.segments, seg = blockIdx.x - row * a.segments;
  const E* x = row_of<T>(a, row);
  const uint32_t lo = seg * a.segment, hi = min(lo + a.segment, a.V);
  Given<T> given;
  if (a.segments == 1) given.read(a, row, x, threadIdx.x);
  Running r;
  uint32_t at = lo + 8 * threadIdx.x;
  // two pieces of eight at a time: the maximum is moved once for sixteen elements
  for (; at + 8 * NT + 8 <= hi; at += 16 * NT) {
    float v[16];
    const typename T::Raw p = T::load(x + at), q = T::load(x + at + 8 * NT);
    T::unpack(p, *reinterpret_cast<float(*)[8]>(v));
    T::unpack(q, *reinterpret_cast<float(*)[8]>(v + 8));
    add<ENT>(r, v, 16, a.c);
  }
  for (; at < hi; at += 8 * NT) {
    float v[8];
    fetch<T>(x, at, hi, v);
    add<ENT>(r, v, 8, a.c);
  }
  const float mine = r.max;
  meet<NT, ENT>(r, a.c, lds);
  if constexpr (TOP) find_top<T, NT>(top[0], x, lo, hi, mine, r.max, a.top);
  if (a.segments == 1) {
    finish<T, NT, ENT>(a, row, x, r, given, top, lds);
    return;
  }
  if (threadIdx.x == 0) {
    float* p = a.part + 4 * (int64_t)blockIdx.x;
    p[0] = r.max;
    p[1] = r.s;
    p[2] = r.u;
  }
  if constexpr (TOP) {
    for (int i = threadIdx.x; i < a.top; i += NT) a.part_top[(int64_t)blockIdx.x * a.top + i] = top[0].best[i];
  }
}

// The segments of a row as one: sums in the order of the segments, the largest of their largest.
template <class T, bool ENT, bool TOP>
__global__ __launch_bounds__(256) void token_logprobs_join_kernel(const LogitArgs a) {
  __shared__ float lds[4][3];
  __shared__ char scratch[TOP ? sizeof(TopScratch<256>) : 8] __attribute__((aligned(8)));
  TopScratch<256>* top = reinterpret_cast<TopScratch<256>*>(scratch);
  const uint32_t row = blockIdx.x;
  const typename T::elem* x = row_of<T>(a, row);
  const float* p = a.part + 4 * (int64_t)row * a.segments;
  Given<T> given;
  given.read(a, row, x, threadIdx.x);
  // segment of a lane, summed by the wave; all waves do the same
  Running r;
  const int lane = threadIdx.x & 63;
  if (lane < (int)a.segments) {
    r.max = p[4 * lane];
    r.M = shift(r.max, a.c);
    r.s = p[4 * lane + 1];
    r.u = ENT ? p[4 * lane + 2] : 0.f;
  }
  shift_to<ENT>(r, wave_max(r.max), a.c);
  r.s = wave_add(r.s);
  if constexpr (ENT) r.u = wave_add(r.u);
  if constexpr (TOP) {
    // a bound from the i-th largest of every segment: k / i segments that reach it hold k elements that do
    const int k = a.top, n = (int)a.segments;
    const int i = (k + n - 1) / n, need = (k + i - 1) / i;
    const uint64_t* f = a.part_top + (int64_t)row * n * k;
    TopScratch<256>& t = top[0];
    static_assert(kSegmentsMax <= kWave, "a lane for each segment");
    if (threadIdx.x == 0) t.count = 0;
    const uint32_t reached[1] = {lane < n ? (uint32_t)(f[lane * k + i - 1] >> 32) : 0u};
    const uint32_t bound = kth_bound<T>(reached, need);  // in every wave
    __syncthreads();
    for (int q = threadIdx.x; q < n * k; q += 256) {
      const uint64_t one = f[q];
      if (one == 0 || (uint32_t)(one >> 32) < bound) continue;
      const uint32_t slot = atomicAdd(&t.count, 1u);
      if (slot < t.kCandidates) t.found[slot] = one;
    }
    __syncthreads();
    if (t.count <= t.kCandidates) {  // uniform
      rank<256>(t, (int)t.count, k);
    } else {
      // equal values: each segment's are in order, and the segments too, so that a place in the result is a count over them all
      for (int q = threadIdx.x; q < n * k; q += 256) {
        const uint64_t mine = f[q];
        int above = 0;
        for (int o = 0; o < n * k; ++o) above += f[o] > mine;
        if (mine && above < k) t.best[above] = mine;
      }
      __syncthreads();
    }
  }
  finish<T, 256, ENT>(a, row, x, r, given, top, lds);
}

constexpr int kBwdThreads = 256, kBwdPieces = 4;  // pieces of eight elements for each thread

struct GradArgs {
  LogitArgs f;
  const float* g_logprobs;  // [rows, n_tokens] or null
  const float* g_entropy;   // [rows] or null
  void* grad;               // [rows, V]
  uint32_t per_row;         // workgroups
};

template <class T, bool ENT>
__global__ __launch_bounds__(kBwdThreads) void token_logprobs_bwd_kernel(const GradArgs a) {
  typedef typename T::elem E;
  __shared__ float waves[kBwdThreads / 64];
  const LogitArgs& f = a.f;
  const uint32_t row = blockIdx.x / a.per_row, lo = (blockIdx.x - row * a.per_row) * (kBwdThreads * kBwdPieces * 8);
  const uint32_t hi = min(lo + kBwdThreads * kBwdPieces * 8, f.V);
  const E* x = row_of<T>(f, row);
  E* out = reinterpret_cast<E*>(a.grad) + (int64_t)row * f.V;
  const float m = f.stats[4 * (int64_t)row], inv = f.stats[4 * (int64_t)row + 1], log2s = f.stats[4 * (int64_t)row + 2],
              H = f.stats[4 * (int64_t)row + 3];
  // the sum of the row's incoming gradients: the same order in every workgroup of the row
  const int64_t* tokens = f.tokens + (int64_t)row * f.n_tokens;
  const float* g = a.g_logprobs ? a.g_logprobs + (int64_t)row * f.n_tokens : nullptr;
  float sum = 0.f;
  if (g) {
    if (f.n_tokens == 1) {
      sum = tokens[0] == f.ignore_index ? 0.f : g[0];
    } else {
      for (int i = threadIdx.x; i < f.n_tokens; i += kBwdThreads) sum += tokens[i] == f.ignore_index ? 0.f : g[i];
      sum = wave_add(sum);
      if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = sum;
      __syncthreads();
      sum = ((waves[0] + waves[1]) + waves[2]) + waves[3];
    }
  }
  const float gh = ENT ? a.g_entropy[row] : 0.f;
  // grad x_j = p_j (A + B y_j) with y in powers of two: log p = (y - log2 s) ln 2
  const float A = -(sum + gh * (H - log2s * kLn2)) * f.inv_temp, B = -gh * kLn2 * f.inv_temp;
  auto value = [&](float v) {
    const float y = (v - m) * f.c, p = __builtin_amdgcn_exp2f(y) * inv;
    return ENT ? p * __builtin_fmaf(B, __builtin_fmaxf(y, -200.f), A) : p * A;
  };
  const bool nothing = inv == 0.f || (A == 0.f && B == 0.f);  // uniform: ignored rows are not read
  // eight elements together, or in fp32 twice four, so that a wave writes whole lines
  constexpr bool split = sizeof(E) == 4;
  constexpr uint32_t kTile = 8 * kBwdThreads;
  const uint32_t first = split ? 4 * threadIdx.x : 8 * threadIdx.x;
  typename T::Raw raw[kBwdPieces];
#pragma unroll
  for (int i = 0; i < kBwdPieces; ++i) {
    const uint32_t tile = lo + kTile * i;
    raw[i] = typename T::Raw{};
    if (nothing || tile + kTile > hi) continue;  // uniform
    if constexpr (split)
      raw[i] = T::join(T::load4_once(x + tile + first), T::load4_once(x + tile + kTile / 2 + first));
    else
      raw[i] = T::load_once(x + tile + first);
  }
#pragma unroll
  for (int i = 0; i < kBwdPieces; ++i) {
    const uint32_t tile = lo + kTile * i;
    if (tile + kTile <= hi) {
      float v[8] = {};
      if (!nothing) {
        T::unpack(raw[i], v);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = value(v[e]);
      }
      const typename T::Raw r = T::pack(v);
      if constexpr (split) {
        T::store4(out + tile + first, T::low(r));
        T::store4(out + tile + kTile / 2 + first, T::high(r));
      } else {
        T::store(out + tile + first, r);
      }
    } else {  // the row's end
#pragma unroll
      for (int half = 0; half < (split ? 2 : 1); ++half) {
        const uint32_t at = tile + kTile / 2 * half + first, n = split ? 4 : 8;
        if (at + n <= hi) {
          float v[8] = {};
          if (!nothing) {
            if constexpr (split)
              T::unpack(T::join(T::load4_once(x + at), typename T::Raw4{}), v);
            else
              T::unpack(T::load_once(x + at), v);
#pragma unroll
            for (uint32_t e = 0; e < n; ++e) v[e] = value(v[e]);
          }
          if constexpr (split)
            T::store4(out + at, T::low(T::pack(v)));
          else
            T::store(out + at, T::pack(v));
        } else {
          for (uint32_t j = at; j < hi; ++j) T::put(out + j, nothing ? 0.f : value(T::get(x + j)));
        }
      }
    }
  }
  if (!g || inv == 0.f) return;
  // the given tokens' own elements once more, with what they receive; a token given twice adds up
  __syncthreads();
  for (int i = threadIdx.x; i < f.n_tokens; i += kBwdThreads) {
    const int64_t token = tokens[i];
    if (token == f.ignore_index || (uint64_t)token >= f.V || token < lo || token >= hi) continue;
    float own = 0.f;
    for (int q = 0; q < f.n_tokens; ++q) own += tokens[q] == token ? g[q] : 0.f;
    T::put(out + token, (nothing ? 0.f : value(T::get(x + token))) + own * f.inv_temp);
  }
}

// How many segments a row is cut into: where the rows alone leave compute units empty, pieces of at least 4096 elements.  One row of
// 128256 with 20 alternatives: 6.5 us for 31 workgroups and 4.4 for the one that joins them; 48 rows with five: 9.1 and 4.4.
uint32_t segments_of(int64_t rows, int64_t V) {
  const int64_t want = 1024 / rows, most = (V + 4095) / 4096;
  const int64_t n = want < most ? want : most;
  return (uint32_t)(n < 1 ? 1 : n > kSegmentsMax ? kSegmentsMax : n);
}

struct Work {
  uint32_t segments, segment;
  size_t part_top, bytes;
  Work(int64_t rows, int64_t V, int top) {
    segments = segments_of(rows, V);
    segment = (uint32_t)(((V + segments - 1) / segments + 7) / 8 * 8);
    segments = (uint32_t)((V + segment - 1) / segment);
    part_top = (size_t)rows * segments * 16;
    bytes = segments == 1 ? 0 : part_top + (size_t)rows * segments * top * 8;
  }
};

int prepare(const char* who, LogitArgs& a, const ttamd_logits* l, const int64_t* tokens, int64_t n_tokens, int64_t ignore_index,
            float temperature) {
  TT_REQUIRE(l && l->data && (tokens || n_tokens == 0), "%s: null pointer argument", who);
  TT_REQUIRE(l->dtype == TTAMD_BF16 || l->dtype == TTAMD_F32, "%s: unknown dtype code %d", who, l->dtype);
  TT_REQUIRE(reinterpret_cast<uintptr_t>(l->data) % (l->dtype == TTAMD_BF16 ? 2 : 4) == 0, "%s: misaligned pointer argument", who);
  TT_REQUIRE(l->rows > 0 && l->rows < (int64_t(1) << 31) && l->V > 0 && l->V < (int64_t(1) << 30) && l->n_inner > 0 && l->n_inner <= l->rows,
             "%s: bad shape rows=%lld V=%lld", who, (long long)l->rows, (long long)l->V);
  TT_REQUIRE(n_tokens >= 0 && n_tokens <= 65536, "%s: %lld tokens for a row", who, (long long)n_tokens);
  TT_REQUIRE(temperature > 0.f && temperature < __builtin_inff() && kLog2e / temperature < __builtin_inff(), "%s: temperature %g", who, (double)temperature);
  a = LogitArgs{};
  a.logits = l->data;
  a.outer = l->stride_outer;
  a.inner = l->stride_inner;
  a.rows = (uint32_t)l->rows;
  a.n_inner = (uint32_t)l->n_inner;
  a.V = (uint32_t)l->V;
  a.tokens = tokens;
  a.n_tokens = (int)n_tokens;
  a.ignore_index = ignore_index;
  a.c = (float)(1.4426950408889634 / (double)temperature);
  a.inv_temp = (float)(1.0 / (double)temperature);
  return TTAMD_OK;
}

template <class T, bool ENT, bool TOP>
void launch_fwd(const LogitArgs& a, hipStream_t st) {
  const dim3 grid(a.rows * a.segments);
  if (a.segments > 1) {
    token_logprobs_fwd_kernel<T, 256, ENT, TOP><<<grid, dim3(256), 0, st>>>(a);
    token_logprobs_join_kernel<T, ENT, TOP><<<dim3(a.rows), dim3(256), 0, st>>>(a);
  } else {
    // A wave for a row of few elements: 8000 x 1024 in 8.3 us (64 threads), 13.5 (256), 25.8 (512).  Above, 256: 1799 x 32064 in 26.2
    // (31.4 with 64, 27.5 with 512), 2048 x 128256 forward and backward in 258 (263 with 512, 260 with 1024).
    if (a.V <= 4096)
      token_logprobs_fwd_kernel<T, 64, ENT, TOP><<<grid, dim3(64), 0, st>>>(a);
    else
      token_logprobs_fwd_kernel<T, 256, ENT, TOP><<<grid, dim3(256), 0, st>>>(a);
  }
}

}  // namespace
}  // namespace ttamd

using namespace ttamd;

extern "C" size_t ttamd_token_logprobs_workspace_bytes(int64_t rows, int64_t V, int top) {
  if (rows <= 0 || rows >= (int64_t(1) << 31) || V <= 0 || V >= (int64_t(1) << 30) || top < 0 || top > kTopMax) return 0;
  return Work(rows, V, top).bytes;
}

extern "C" int ttamd_token_logprobs_fwd(const ttamd_logits* logits, const int64_t* tokens, int64_t n_tokens, int64_t ignore_index,
                                        float temperature, float* logprobs, float* entropy, int top, float* top_logprobs, int64_t* top_tokens,
                                        float* stats, void* workspace, size_t workspace_bytes, void* stream) {
  LogitArgs a;
  if (int rc = prepare("token_logprobs_fwd", a, logits, tokens, n_tokens, ignore_index, temperature)) return rc;
  TT_REQUIRE(logprobs || n_tokens == 0, "token_logprobs_fwd: null pointer argument");
  TT_REQUIRE(top >= 0 && top <= kTopMax && top <= logits->V, "token_logprobs_fwd: top (%d) must be at most %d and at most the vocabulary", top, kTopMax);
  TT_REQUIRE(top == 0 || (top_logprobs && top_tokens), "token_logprobs_fwd: null pointer argument");
  const Work w(logits->rows, logits->V, top);
  if (w.bytes) {
    TT_REQUIRE(workspace && aligned16(workspace), "token_logprobs_fwd: needs a 16-byte aligned workspace");
    if (workspace_bytes < w.bytes) return fail(TTAMD_EWORKSPACE, "token_logprobs_fwd: workspace has %zu bytes, needs %zu", workspace_bytes, w.bytes);
  }
  a.segments = w.segments;
  a.segment = w.segment;
  a.part = reinterpret_cast<float*>(workspace);
  a.part_top = w.bytes ? reinterpret_cast<uint64_t*>(reinterpret_cast<char*>(workspace) + w.part_top) : nullptr;
  a.top = top;
  a.logprobs = logprobs;
  a.entropy = entropy;
  a.top_logprobs = top_logprobs;
  a.top_tokens = top_tokens;
  a.stats = stats;
  const bool ent = entropy != nullptr;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  const bool bf16 = logits->dtype == TTAMD_BF16;
#define TT_FWD(E, K)                  \
  if (bf16)                           \
    launch_fwd<BF16, E, K>(a, st);    \
  else                                \
    launch_fwd<F32, E, K>(a, st);
  if (ent && top) {
    TT_FWD(true, true)
  } else if (ent) {
    TT_FWD(true, false)
  } else if (top) {
    TT_FWD(false, true)
  } else {
    TT_FWD(false, false)
  }
#undef TT_FWD
  return check_launch("token_logprobs_fwd");
}

extern "C" int ttamd_token_logprobs_bwd(const ttamd_logits* logits, const int64_t* tokens, int64_t n_tokens, int64_t ignore_index,
                                        float temperature, const float* stats, const float* g_logprobs, const float* g_entropy, void* grad,
                                        void* stream) {
  GradArgs a;
  if (int rc = prepare("token_logprobs_bwd", a.f, logits, tokens, n_tokens, ignore_index, temperature)) return rc;
  TT_REQUIRE(stats && grad && (g_logprobs || g_entropy), "token_logprobs_bwd: null pointer argument");
  a.f.stats = const_cast<float*>(stats);
  a.g_logprobs = n_tokens ? g_logprobs : nullptr;
  a.g_entropy = g_entropy;
  a.grad = grad;
  const int64_t piece = kBwdThreads * kBwdPieces * 8, per_row = (logits->V + piece - 1) / piece;
  TT_REQUIRE(logits->rows * per_row < (int64_t(1) << 31), "token_logprobs_bwd: too many logits for one launch");
  a.per_row = (uint32_t)per_row;
  const dim3 grid((unsigned)(logits->rows * per_row)), block(kBwdThreads);
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (logits->dtype == TTAMD_BF16) {
    if (g_entropy)
      token_logprobs_bwd_kernel<BF16, true><<<grid, block, 0, st>>>(a);
    else
      token_logprobs_bwd_kernel<BF16, false><<<grid, block, 0, st>>>(a);
  } else if (g_entropy) {
    token_logprobs_bwd_kernel<F32, true><<<grid, block, 0, st>>>(a);
  } else {
    token_logprobs_bwd_kernel<F32, false><<<grid, block, 0, st>>>(a);
  }
  return check_launch("token_logprobs_bwd");
}
