// Sums over the rows of a bf16 matrix, out[N] = bf16(sum_m x[m, N]) with fp32 sums: the gradient of a linear's bias.
//
// A workgroup adds up a stretch of rows of 128 columns: 16 lanes lie side by side along a row, 16 bytes each (rows of an odd
// length start anywhere; those bytes are loaded unaligned), a thread takes every 16th row, four of them in flight, and the threads
// of a column meet in LDS.  With more than one stretch a second launch adds the stretches' fp32 sums.  Both orders are fixed, no
// memory has to be cleared and nothing is counted, so a recorded launch gives on every replay what a call gives.  Bound: HBM, one
// pass over x: 8192 x 14336 44.8 us (5.2 TB/s), 8192 x 4096 15.7 us, 2000 x 10001 17.1 us, 350 x 2048 5.8 us (the two launches).
#include <algorithm>

#include "common.h"

namespace ttamd {
namespace {

typedef __bf16 bf16_t;
struct __attribute__((packed, aligned(2))) Eight {
  uint32_t d[4];
};

constexpr int kLanes = 16, kRows = 16, kCols = 8 * kLanes, kInFlight = 4;

__global__ __launch_bounds__(kLanes * kRows) void column_sum_kernel(const uint16_t* __restrict__ x, int64_t M, int64_t N, int64_t rows_per_stretch,
                                                                    float* __restrict__ part, uint16_t* __restrict__ out) {
  __shared__ float sums[kRows][kCols];
  const int lane = threadIdx.x % kLanes, r = threadIdx.x / kLanes;
  const int64_t c0 = (int64_t)blockIdx.x * kCols, col = c0 + 8 * lane;
  const int64_t m_begin = (int64_t)blockIdx.y * rows_per_stretch, m_end = m_begin + rows_per_stretch < M ? m_begin + rows_per_stretch : M;
  const int here = N - col < 8 ? (int)(N - col) : 8;  // columns of this thread
  float acc[kInFlight][8];
#pragma unroll
  for (int u = 0; u < kInFlight; ++u)
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[u][e] = 0.f;
  if (here == 8) {
    for (int64_t m = m_begin + r; m < m_end; m += kInFlight * kRows) {
      Eight v[kInFlight];
#pragma unroll
      for (int u = 0; u < kInFlight; ++u) {
        v[u] = Eight{{0, 0, 0, 0}};
        if (m + u * kRows < m_end) v[u] = *reinterpret_cast<const Eight*>(x + (m + u * kRows) * N + col);
      }
#pragma unroll
      for (int u = 0; u < kInFlight; ++u)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          acc[u][2 * e] += __builtin_bit_cast(float, v[u].d[e] << 16);
          acc[u][2 * e + 1] += __builtin_bit_cast(float, v[u].d[e] & 0xffff0000u);
        }
    }
  } else {  // the end of the rows
    for (int64_t m = m_begin + r; m < m_end; m += kRows)
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (e < here) acc[0][e] += __builtin_bit_cast(float, (uint32_t)x[m * N + col + e] << 16);
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) sums[r][8 * lane + e] = (acc[0][e] + acc[1][e]) + (acc[2][e] + acc[3][e]);
  __syncthreads();
  if (threadIdx.x >= kCols || c0 + threadIdx.x >= N) return;
  float s = 0.f;
#pragma unroll
  for (int q = 0; q < kRows; ++q) s += sums[q][threadIdx.x];
  if (part)
    part[(int64_t)blockIdx.y * N + c0 + threadIdx.x] = s;
  else
    out[c0 + threadIdx.x] = __builtin_bit_cast(uint16_t, (bf16_t)s);
}

// out[n] = bf16(sum of the stretches' sums): sixteen waves take every sixteenth stretch of 64 columns
constexpr int kSumWaves = 16;
__global__ __launch_bounds__(64 * kSumWaves) void column_sum_stretches_kernel(const float* __restrict__ part, int stretches, int64_t N, uint16_t* __restrict__ out) {
  __shared__ float sums[kSumWaves][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t n = (int64_t)blockIdx.x * 64 + lane;
  float s = 0.f;
  if (n < N)
#pragma unroll 4
    for (int q = wave; q < stretches; q += kSumWaves) s += part[(int64_t)q * N + n];
  sums[wave][lane] = s;
  __syncthreads();
  if (wave > 0 || n >= N) return;
  s = 0.f;
#pragma unroll
  for (int w = 0; w < kSumWaves; ++w) s += sums[w][lane];
  out[n] = __builtin_bit_cast(uint16_t, (bf16_t)s);
}

struct ColumnPlan {
  int64_t tiles, rows;  // of columns; of a stretch
  int stretches;
};
// Workgroups for four to a CU, but no stretch below 64 rows (a single launch takes 3.3 us, two 5.8) and at most 512
ColumnPlan plan_columns(int64_t M, int64_t N) {
  ColumnPlan p;
  p.tiles = (N + kCols - 1) / kCols;
  const int64_t most = std::min<int64_t>(512, std::max<int64_t>(1, 1024 / p.tiles));
  const int64_t n = std::max<int64_t>(1, std::min(most, M / 64));
  p.rows = std::max<int64_t>(1, (M + n - 1) / n);
  p.stretches = (int)std::max<int64_t>(1, (M + p.rows - 1) / p.rows);
  return p;
}

}  // namespace
}  // namespace ttamd

using namespace ttamd;

extern "C" size_t ttamd_column_sum_workspace_bytes(int64_t M, int64_t N) {
  if (M <= 0 || N <= 0) return 0;
  const ColumnPlan p = plan_columns(M, N);
  return p.stretches > 1 ? (size_t)p.stretches * N * sizeof(float) : 0;
}

extern "C" int ttamd_column_sum_bf16(const void* x, void* out, int64_t M, int64_t N, void* workspace, size_t workspace_bytes, void* stream) {
  TT_REQUIRE(M >= 0 && N >= 0, "column_sum: bad shape M=%lld N=%lld", (long long)M, (long long)N);
  if (N == 0) return TTAMD_OK;
  if (N >= (int64_t(1) << 29)) return fail(TTAMD_EUNSUPPORTED, "column_sum: N=%lld is too large", (long long)N);
  TT_REQUIRE((x || M == 0) && out && aligned16(x) && (reinterpret_cast<uintptr_t>(out) & 1u) == 0, "column_sum: pointers must be non-null, x 16-byte aligned");
  const size_t need = ttamd_column_sum_workspace_bytes(M, N);
  if (need > 0 && (!workspace || !aligned16(workspace) || workspace_bytes < need))
    return fail(TTAMD_EWORKSPACE, "column_sum: needs %zu bytes of 16-byte aligned workspace, got %zu", need, workspace_bytes);
  const ColumnPlan p = plan_columns(M, N);
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const uint16_t* in = reinterpret_cast<const uint16_t*>(x);
  uint16_t* o = reinterpret_cast<uint16_t*>(out);
  float* part = p.stretches > 1 ? reinterpret_cast<float*>(workspace) : nullptr;
  const dim3 grid((unsigned)p.tiles, (unsigned)p.stretches);
  column_sum_kernel<<<grid, dim3(kLanes * kRows), 0, s>>>(in, M, N, p.rows, part, o);
  if (int rc = check_launch("column_sum")) return rc;
  if (!part) return TTAMD_OK;
  column_sum_stretches_kernel<<<dim3((unsigned)((N + 63) / 64)), dim3(64 * kSumWaves), 0, s>>>(part, p.stretches, N, o);
  return check_launch("column_sum");
}
