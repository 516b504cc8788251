// One training step's two directions of frozen mxfp4 linears with low-rank adapters that read the same input
// (torchtune/modules/peft/lora.py:128-147 over a microscaled base weight):
//
//   forward   x^ = mxfp8(x);  h_i = bf16(x^ . A_i^T);  y_i = x^ . W_i^T (+ bias_i) + s_i . h_i . B_i^T
//   backward  gh_i = bf16(s_i . gy_i . B_i);  gA_i = gh_i^T . x^;  gB_i = s_i . gy_i^T . h_i;  gx = sum gy_i . W_i + gh_i . A_i
//
// The 8-bit input that the products read is also what the backward pass reads: 1 + 1 / 32 bytes per element are kept
// instead of 2, once for all members, and the adapter gradients are those of the products that ran.
#include "group.h"
#include "mx_math.h"

namespace ttamd {
namespace {

constexpr int64_t kMaxGradN = int64_t(1) << 22;  // 256 rows of the output's gradient, 512 N bytes, are counted in 32 bits

struct Members {
  GroupSkinny sk;
  GroupDx dx;
  const uint8_t *codes[kGroupMax], *scales[kGroupMax];
};

int decode(const char* who, const ttamd_mx_lora_member* m, int n, int64_t M, int64_t K, bool backward, Members& d) {
  d = Members{};
  TT_REQUIRE(m && n >= 1 && n <= kGroupMax, "%s: 1 to %d members (got %d)", who, kGroupMax, n);
  TT_REQUIRE(M > 0 && K > 0 && K % 64 == 0, "%s: K (%lld) must be a positive multiple of 64 (M %lld)", who, (long long)K, (long long)M);
  d.sk.n = d.dx.n = n;
  d.sk.M = d.dx.M = M;
  d.sk.K = d.dx.K = K;
  int r = 0;
  bool adapters = false;  // none of their gradients wanted: all of the pointers are null
  for (int i = 0; i < n; ++i) adapters = adapters || m[i].grad_lora_a || m[i].grad_lora_b;
  for (int i = 0; i < n; ++i) {
    TT_REQUIRE(m[i].N > 0 && m[i].N % 64 == 0, "%s: member %d: N (%lld) must be a positive multiple of 64", who, i, (long long)m[i].N);
    TT_REQUIRE(m[i].rank > 0 && m[i].rank % 8 == 0, "%s: member %d: the rank (%d) must be a positive multiple of 8", who, i, m[i].rank);
    if (int rc = check_mx_product(who, M, m[i].N, K)) return rc;
    if (m[i].N >= kMaxGradN) return fail(TTAMD_EUNSUPPORTED, "%s: member %d: N (%lld) is too large", who, i, (long long)m[i].N);
    TT_REQUIRE(m[i].codes && m[i].scales && m[i].lora_a && m[i].lora_b && m[i].y && aligned16(m[i].codes) && aligned16(m[i].scales) &&
                   aligned16(m[i].lora_a) && aligned16(m[i].lora_b) && aligned16(m[i].y) && (reinterpret_cast<uintptr_t>(m[i].bias) & 1u) == 0,
               "%s: member %d: pointers must be non-null and 16-byte aligned", who, i);
    TT_REQUIRE(!backward || !adapters || (m[i].grad_lora_a && m[i].grad_lora_b && aligned16(m[i].grad_lora_a) && aligned16(m[i].grad_lora_b)),
               "%s: member %d: the adapter gradients must be non-null (or null for all members) and 16-byte aligned", who, i);
    d.codes[i] = m[i].codes;
    d.scales[i] = m[i].scales;
    d.sk.N[i] = d.dx.N[i] = m[i].N;
    d.sk.rank[i] = d.dx.rank[i] = m[i].rank;
    d.sk.r_off[i] = d.dx.r_off[i] = r;
    d.sk.scale[i] = m[i].scale;
    d.sk.lora_a[i] = d.dx.lora_a[i] = reinterpret_cast<const uint16_t*>(m[i].lora_a);
    d.sk.lora_b[i] = reinterpret_cast<const uint16_t*>(m[i].lora_b);
    d.sk.gy[i] = d.dx.gy[i] = reinterpret_cast<const uint16_t*>(m[i].y);
    d.sk.ga[i] = reinterpret_cast<uint16_t*>(m[i].grad_lora_a);
    d.sk.gb[i] = reinterpret_cast<uint16_t*>(m[i].grad_lora_b);
    r += m[i].rank;
  }
  TT_REQUIRE(r <= 64, "%s: the members' ranks add up to %d, at most 64 are supported", who, r);
  int64_t n_total = 0;
  for (int i = 0; i < n; ++i) n_total += m[i].N;
  if (n_total >= 2 * kMaxGradN) return fail(TTAMD_EUNSUPPORTED, "%s: the members' outputs (%lld) are too many for one grad-input", who, (long long)n_total);
  d.sk.r_off[n] = d.dx.r_off[n] = r;
  return TTAMD_OK;
}

size_t align256(size_t v) { return (v + 255) & ~size_t(255); }

struct Cut {  // consecutive stretches of a workspace
  char* p;
  size_t used = 0;
  template <typename T>
  T* take(size_t bytes) {
    T* q = reinterpret_cast<T*>(p ? p + used : nullptr);
    used += align256(bytes);
    return q;
  }
};

struct FwdSpace {
  uint8_t* pieces[kGroupMax];
  float* part;
  size_t bytes;
};
FwdSpace fwd_space(const Members& d, void* workspace) {
  Cut c{reinterpret_cast<char*>(workspace)};
  FwdSpace f = {};
  const GroupSkinny& g = d.sk;
  size_t part = mx_hidden_part_bytes(g.M, g.K, g.r_off[g.n]);
  for (int i = 0; i < g.n; ++i) {
    f.pieces[i] = c.take<uint8_t>(mx_piece_bytes(g.N[i], g.K));
    const size_t p = mx_gemm_part_bytes(g.M, g.N[i], g.K, TTAMD_MXFP8);
    part = p > part ? p : part;
  }
  f.part = c.take<float>(part);
  f.bytes = c.used;
  return f;
}

struct BwdSpace {
  float *skinny, *part;
  char* tiles;
  size_t bytes;
};
int64_t sum_n(const GroupDx& d) {
  int64_t n = 0;
  for (int i = 0; i < d.n; ++i) n += d.N[i];
  return n;
}
// gx: on the codes where the fused kernel serves the shape, else on the weights expanded to bf16 tiles
int run_dx(const GroupDx& d, const uint8_t* const* codes, const uint8_t* const* scales, const void* gh, void* gx, float* part, char* tiles, hipStream_t s) {
  if (mx_dx_fused(d.M, sum_n(d), d.K)) return run_mx_dx(d, codes, scales, gh, gx, part, s);
  int64_t n = 0;
  for (int i = 0; i < d.n; ++i) {
    if (int rc = run_mx_expand_tiles(codes[i], scales[i], d.N[i], d.K, tiles + 2 * n * d.K, s)) return rc;
    n += d.N[i];
  }
  // the dense launch addresses a gradient with 32 bits: longer batches go in stretches of rows
  int64_t widest = 0;
  for (int i = 0; i < d.n; ++i) widest = d.N[i] > widest ? d.N[i] : widest;
  const int64_t rows = ((int64_t(1) << 32) - 1) / (2 * widest) / 256 * 256;
  for (int64_t r = 0; r < d.M; r += rows) {
    GroupDx part = d;
    part.M = d.M - r < rows ? d.M - r : rows;
    for (int i = 0; i < d.n; ++i) part.gy[i] = d.gy[i] + r * d.N[i];
    if (int rc = run_dense_dx_on_tiles(part, reinterpret_cast<const uint16_t*>(gh) + r * d.r_off[d.n], reinterpret_cast<uint16_t*>(gx) + r * d.K, tiles, s)) return rc;
  }
  return TTAMD_OK;
}
BwdSpace bwd_space(const Members& d, void* workspace) {
  Cut c{reinterpret_cast<char*>(workspace)};
  BwdSpace b = {};
  const GroupSkinny& g = d.sk;
  b.skinny = c.take<float>(group_lora_bwd_ws_bytes(g));
  const int64_t n = sum_n(d.dx);
  const bool fused = mx_dx_fused(g.M, n, g.K);
  b.part = c.take<float>(fused ? mx_dx_fused_bytes(g.M, n, g.K) : 0);
  b.tiles = c.take<char>(fused ? 0 : 2 * n * g.K);
  b.bytes = c.used;
  return b;
}

}  // namespace
}  // namespace ttamd

using namespace ttamd;

extern "C" size_t ttamd_mx_kept_codes_bytes(int64_t M, int64_t K) { return M > 0 && K > 0 ? (size_t)M * mx_padded_k(K) : 0; }
extern "C" size_t ttamd_mx_kept_scales_bytes(int64_t M, int64_t K) { return M > 0 && K > 0 ? (size_t)mx_piece_bytes(M, K) : 0; }

extern "C" size_t ttamd_mx_lora_fwd_workspace_bytes(const ttamd_mx_lora_member* members, int n_members, int64_t M, int64_t K) {
  Members d;
  return decode("mx_lora_fwd", members, n_members, M, K, false, d) ? 0 : fwd_space(d, nullptr).bytes;
}

extern "C" int ttamd_mx_lora_fwd_bf16(const void* x, const ttamd_mx_lora_member* members, int n_members, uint8_t* kept_codes,
                                      uint8_t* kept_scales, void* h_cat, int64_t M, int64_t K, void* workspace, size_t workspace_bytes,
                                      void* stream) {
  Members d;
  if (int rc = decode("mx_lora_fwd", members, n_members, M, K, false, d)) return rc;
  TT_REQUIRE(x && kept_codes && kept_scales && h_cat && aligned16(x) && aligned16(kept_codes) && aligned16(kept_scales) && aligned16(h_cat),
             "mx_lora_fwd: pointers must be non-null and 16-byte aligned");
  const FwdSpace f = fwd_space(d, workspace);
  if (!workspace || !aligned16(workspace) || workspace_bytes < f.bytes)
    return fail(TTAMD_EWORKSPACE, "mx_lora_fwd: needs %zu bytes of 16-byte aligned workspace, got %zu", f.bytes, workspace_bytes);
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  uint16_t* h = reinterpret_cast<uint16_t*>(h_cat);
  if (int rc = run_mx_quantize_hidden(x, M, K, kept_codes, kept_scales, d.sk.lora_a, d.sk.r_off, n_members, h, f.part, d.scales, d.sk.N, f.pieces, s)) return rc;
  MxProduct q[kGroupMax] = {};
  for (int i = 0; i < n_members; ++i) {
    q[i].x_codes = kept_codes; q[i].x_pieces = kept_scales;
    q[i].w_codes = d.codes[i]; q[i].w_pieces = f.pieces[i];
    q[i].h = h + d.sk.r_off[i]; q[i].ldh = d.sk.r_off[n_members]; q[i].rank = d.sk.rank[i]; q[i].lora_b = d.sk.lora_b[i]; q[i].lscale = d.sk.scale[i];
    q[i].bias = reinterpret_cast<const uint16_t*>(members[i].bias);
    q[i].y = reinterpret_cast<uint16_t*>(members[i].y);
  }
  return run_mx_gemm_group(q, n_members, M, d.sk.N, K, f.part, s);
}

extern "C" size_t ttamd_mx_lora_bwd_workspace_bytes(const ttamd_mx_lora_member* members, int n_members, int64_t M, int64_t K) {
  Members d;
  return decode("mx_lora_bwd", members, n_members, M, K, false, d) ? 0 : bwd_space(d, nullptr).bytes;
}

extern "C" int ttamd_mx_lora_bwd_bf16(const uint8_t* kept_codes, const uint8_t* kept_scales, const void* h_cat,
                                      const ttamd_mx_lora_member* members, int n_members, void* gh_cat, void* gx, int64_t M, int64_t K,
                                      void* workspace, size_t workspace_bytes, void* stream) {
  Members d;
  if (int rc = decode("mx_lora_bwd", members, n_members, M, K, true, d)) return rc;
  TT_REQUIRE(kept_codes && kept_scales && h_cat && gh_cat && aligned16(kept_codes) && aligned16(kept_scales) && aligned16(h_cat) &&
                 aligned16(gh_cat) && aligned16(gx),
             "mx_lora_bwd: pointers must be non-null and 16-byte aligned (gx may be NULL)");
  const BwdSpace b = bwd_space(d, workspace);
  if (!workspace || !aligned16(workspace) || workspace_bytes < b.bytes)
    return fail(TTAMD_EWORKSPACE, "mx_lora_bwd: needs %zu bytes of 16-byte aligned workspace, got %zu", b.bytes, workspace_bytes);
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  uint16_t* gh = reinterpret_cast<uint16_t*>(gh_cat);
  d.sk.kept = KeptInput{kept_codes, kept_scales, mx_padded_k(K)};
  if (int rc = run_group_lora_bwd(nullptr, reinterpret_cast<const uint16_t*>(h_cat), d.sk, gh, b.skinny, s, nullptr)) return rc;
  return gx ? run_dx(d.dx, d.codes, d.scales, gh, gx, b.part, b.tiles, s) : TTAMD_OK;
}

// the grad-input of a product without adapters: gx = gy . W
extern "C" size_t ttamd_mx_linear_dx_workspace_bytes(int64_t M, int64_t N, int64_t K) {
  if (!(M > 0 && N > 0 && K > 0 && N % 64 == 0 && K % 64 == 0)) return 0;
  return mx_dx_fused(M, N, K) ? mx_dx_fused_bytes(M, N, K) : align256(2 * (size_t)N * K);
}
extern "C" int ttamd_mx_linear_dx_bf16(const void* gy, const uint8_t* w_codes, const uint8_t* w_scales, void* gx, int64_t M, int64_t N,
                                       int64_t K, void* workspace, size_t workspace_bytes, void* stream) {
  if (int rc = check_mx_product("mx_linear_dx", M, N, K)) return rc;
  if (N >= kMaxGradN) return fail(TTAMD_EUNSUPPORTED, "mx_linear_dx: N (%lld) is too large", (long long)N);
  TT_REQUIRE(N % 64 == 0 && K % 64 == 0, "mx_linear_dx: N (%lld) and K (%lld) must be multiples of 64", (long long)N, (long long)K);
  TT_REQUIRE(gy && w_codes && w_scales && gx && aligned16(gy) && aligned16(w_codes) && aligned16(w_scales) && aligned16(gx),
             "mx_linear_dx: pointers must be non-null and 16-byte aligned");
  const size_t need = ttamd_mx_linear_dx_workspace_bytes(M, N, K);
  if (need > 0 && (!workspace || !aligned16(workspace) || workspace_bytes < need))
    return fail(TTAMD_EWORKSPACE, "mx_linear_dx: needs %zu bytes of 16-byte aligned workspace, got %zu", need, workspace_bytes);
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  GroupDx d = {};
  d.n = 1;
  d.M = M; d.K = K;
  d.N[0] = N;
  d.gy[0] = reinterpret_cast<const uint16_t*>(gy);
  return run_dx(d, &w_codes, &w_scales, nullptr, gx, reinterpret_cast<float*>(workspace), reinterpret_cast<char*>(workspace), s);
}
