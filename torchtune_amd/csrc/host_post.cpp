// Host path of what surrounds the linears of a post-training step: the norm and rotation of queries and keys, the log
// probabilities of tokens, and the optimizer's step.  Argument checks, allocations, autograd nodes and the library calls in
// native code: at one token the kernels take a few microseconds, and the optimizer walks over hundreds of tensors in each step.
// Checks of shapes and types come before those of the device, so that they hold without one.
#include "host_common.h"

#include <ATen/MemoryOverlap.h>
#include <c10/hip/HIPCachingAllocator.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/variable.h>

#include <mutex>

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using namespace ttamd_host;
typedef std::optional<Tensor> Maybe;

int type_code(const Tensor& t, const char* what) {
  TORCH_CHECK_TYPE(t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kFloat, what, ": dtype ", t.scalar_type(),
                   " is not supported (bfloat16 and float32 are)");
  return t.scalar_type() == at::kBFloat16 ? TTAMD_BF16 : TTAMD_F32;
}

void same_device(const Tensor& t, const Tensor& as, const char* what, const char* name) {
  TORCH_CHECK(t.device() == as.device(), what, ": ", name, " is on ", t.device().str(), ", expected ", as.device().str());
}

// The backward passes are kernels that autograd does not see into.
void first_order(const char* what) {
  TORCH_CHECK(!at::GradMode::is_enabled(), what, ": the backward pass cannot be differentiated (create_graph=True)");
}

// ---------------------------------------------------------------------------------------------------
// norm and rotation of queries and keys
// ---------------------------------------------------------------------------------------------------
constexpr const char* kRope = "qk_norm_rope";

Tensor dense(const Tensor& t) { return t.defined() ? t.contiguous() : t; }

// rows whose elements lie together; a copy only of what does not
Tensor rows(const Tensor& t) { return t.stride(-1) == 1 || t.size(-1) == 1 ? t : t.contiguous(); }

ttamd_rope_heads part_of(const Tensor& x, const Tensor& scale, const Tensor& gy) {
  ttamd_rope_heads p = {};
  const Tensor& shape = x.defined() ? x : gy;
  p.heads = shape.size(2);
  for (int d = 0; d < 3; ++d) {
    if (x.defined()) p.x_stride[d] = x.stride(d);
    if (gy.defined()) p.gy_stride[d] = gy.stride(d);
  }
  p.x = x.defined() ? x.data_ptr() : nullptr;
  p.scale = scale.defined() ? scale.data_ptr() : nullptr;
  p.gy = gy.defined() ? gy.data_ptr() : nullptr;
  return p;
}

struct Places {
  Tensor cache, positions;
  ttamd_rope_positions at = {};
  Places(const Tensor& cache_, const Tensor& positions_, const std::vector<int64_t>& sections, bool interleaved) {
    cache = cache_.contiguous();
    if (reinterpret_cast<uintptr_t>(cache.data_ptr()) & 7u) cache = cache.clone();
    at.cache = cache.data_ptr<float>();
    at.cache_rows = cache.size(0);
    at.n_axes = sections.empty() ? 1 : (int)sections.size();
    at.interleaved = interleaved;
    for (size_t i = 0; i < sections.size(); ++i) at.section[i] = (int)sections[i];
    if (!positions_.defined()) return;
    positions = positions_;
    at.positions = positions.data_ptr<int64_t>();
    const int first = positions.dim() == 3;
    at.stride[0] = first ? positions.stride(0) : 0;
    at.stride[1] = positions.stride(first);
    at.stride[2] = positions.stride(first + 1);
  }
};

std::pair<Tensor, Tensor> rope_forward(const Tensor& q_, const Tensor& k_, const Tensor& cache, const Tensor& qw, const Tensor& kw, double eps,
                                       const Tensor& positions, const std::vector<int64_t>& sections, bool interleaved) {
  const c10::DeviceGuard guard(q_.device());
  const Tensor q = rows(q_), k = rows(k_);
  Tensor qo = at::empty(q.sizes(), q.options()), ko = at::empty(k.sizes(), k.options());
  if (q.numel() + k.numel() == 0) return {qo, ko};
  const Places places(cache, positions, sections, interleaved);
  ttamd_rope_heads parts[2] = {part_of(q, qw, Tensor()), part_of(k, kw, Tensor())};
  parts[0].out = qo.data_ptr();
  parts[1].out = ko.data_ptr();
  check(ttamd_qk_norm_rope_fwd(parts, &places.at, type_code(q, kRope), (float)eps, q.size(0), q.size(1), q.size(3), stream_of(q)), kRope);
  return {qo, ko};
}

struct QKNormRopeFn : torch::autograd::Function<QKNormRopeFn> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& cache, const Maybe& qw, const Maybe& kw,
                               double eps, const Maybe& positions, const std::vector<int64_t>& sections, bool interleaved) {
    const Tensor w1 = qw ? *qw : Tensor(), w2 = kw ? *kw : Tensor(), pos = positions ? *positions : Tensor();
    auto [qo, ko] = rope_forward(q, k, cache, dense(w1), dense(w2), eps, pos, sections, interleaved);
    // a rotation needs nothing of what it turned
    ctx->save_for_backward({w1.defined() ? q : Tensor(), w1.defined() ? k : Tensor(), cache, w1, w2, pos});
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["sections"] = sections;
    ctx->saved_data["interleaved"] = interleaved;
    ctx->saved_data["norm"] = w1.defined();
    ctx->set_materialize_grads(false);
    return {qo, ko};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    first_order(kRope);
    const bool norm = ctx->saved_data["norm"].toBool();
    // the edges of the call: q, k, cache, then the scales where there are any, then the positions where they are given
    const bool want_x[2] = {ctx->needs_input_grad(0), ctx->needs_input_grad(1)};
    const bool want_w[2] = {norm && ctx->needs_input_grad(3), norm && ctx->needs_input_grad(4)};
    variable_list out(9);
    if (!g[0].defined() && !g[1].defined()) return out;
    const auto saved = ctx->get_saved_variables();
    const double eps = ctx->saved_data["eps"].toDouble();
    const std::vector<int64_t> sections = ctx->saved_data["sections"].toIntVector();
    const Tensor& like = g[0].defined() ? g[0] : g[1];
    const c10::DeviceGuard guard(like.device());
    const Places places(saved[2], saved[5], sections, ctx->saved_data["interleaved"].toBool());
    ttamd_rope_heads parts[2] = {{}, {}};
    Tensor kept[2], gy[2], gx[2], gw[2], w[2];
    bool sums = false, any = false;
    for (int i = 0; i < 2; ++i) {
      if (norm) w[i] = saved[3 + i].contiguous();
      if (!g[i].defined() || !(want_x[i] || want_w[i])) continue;
      gy[i] = rows(g[i]);
      if (norm) kept[i] = rows(saved[i]);
      if (want_x[i]) gx[i] = at::empty(gy[i].sizes(), gy[i].options());
      if (want_w[i]) gw[i] = gy[i].numel() ? at::empty_like(w[i]) : at::zeros_like(w[i]);
      if (gy[i].numel() == 0) continue;
      parts[i] = part_of(kept[i], w[i], gy[i]);
      parts[i].out = gx[i].defined() ? gx[i].data_ptr() : nullptr;
      parts[i].gscale = gw[i].defined() ? gw[i].data_ptr() : nullptr;
      sums = sums || gw[i].defined();
      any = true;
    }
    if (any) {
      const int64_t D = like.size(3);
      const size_t bytes = sums ? ttamd_qk_norm_rope_bwd_workspace_bytes(D) : 0;
      const Tensor ws = bytes ? scratch(bytes, like) : Tensor();
      check(ttamd_qk_norm_rope_bwd(parts, &places.at, type_code(like, kRope), (float)eps, like.size(0), like.size(1), D,
                                   bytes ? ws.data_ptr() : nullptr, bytes, stream_of(like)),
            kRope);
    }
    out[0] = gx[0];
    out[1] = gx[1];
    out[3] = gw[0];
    out[4] = gw[1];
    return out;
  }
};

std::pair<Tensor, Tensor> qk_norm_rope(const Tensor& q, const Tensor& k, const Tensor& cache, const Maybe& q_scale, const Maybe& k_scale, double eps,
                                       const Maybe& positions_, const std::vector<int64_t>& sections, bool interleaved) {
  type_code(q, kRope);
  TORCH_CHECK_TYPE(k.scalar_type() == q.scalar_type(), kRope, ": q is ", q.scalar_type(), ", k ", k.scalar_type());
  TORCH_CHECK_VALUE(q.dim() == 4 && k.dim() == 4 && q.size(0) == k.size(0) && q.size(1) == k.size(1) && q.size(3) == k.size(3), kRope,
                    ": expected [b, s, n_h, h_d] and [b, s, n_kv, h_d], got ", q.sizes(), " and ", k.sizes());
  const int64_t B = q.size(0), S = q.size(1), D = q.size(3);
  TORCH_CHECK_VALUE(D >= 16 && D <= 512 && D % 16 == 0, kRope, ": the head dimension must be a multiple of 16, at most 512, got ", D);
  TORCH_CHECK_TYPE(cache.scalar_type() == at::kFloat, kRope, ": cache must be float32, got ", cache.scalar_type());
  TORCH_CHECK_VALUE(cache.dim() == 3 && cache.size(0) > 0 && cache.size(1) == D / 2 && cache.size(2) == 2, kRope, ": cache must be [positions, ", D / 2,
                    ", 2], got ", cache.sizes());
  TORCH_CHECK_VALUE(q_scale.has_value() == k_scale.has_value(), kRope, ": scales for the queries and for the keys, or for neither");
  for (const Maybe* w : {&q_scale, &k_scale}) {
    if (!*w) continue;
    TORCH_CHECK_TYPE((*w)->scalar_type() == q.scalar_type(), kRope, ": a scale is ", (*w)->scalar_type(), ", q ", q.scalar_type());
    TORCH_CHECK_VALUE((*w)->dim() == 1 && (*w)->size(0) == D, kRope, ": a scale must be [", D, "], got ", (*w)->sizes());
    same_device(**w, q, kRope, "a scale");
  }
  Maybe positions = positions_;
  if (!sections.empty()) {
    int64_t sum = 0;
    for (int64_t n : sections) {
      TORCH_CHECK_VALUE(n >= 0 && n <= D / 2, kRope, ": a section of ", n, " frequencies");
      sum += n;
    }
    TORCH_CHECK_VALUE(sections.size() >= 2 && sections.size() <= 4 && sum == D / 2, kRope, ": sections are two to four numbers that add up to ", D / 2);
    TORCH_CHECK_VALUE(positions && positions->dim() == 3 && positions->size(0) == (int64_t)sections.size(), kRope, ": ", sections.size(),
                      " sections need positions [", sections.size(), ", b, s]");
  }
  if (positions) {
    TORCH_CHECK_TYPE(positions->scalar_type() == at::kLong || positions->scalar_type() == at::kInt, kRope, ": positions must be int64 or int32, got ",
                     positions->scalar_type());
    std::vector<int64_t> want = {B, S};
    if (!sections.empty()) want.insert(want.begin(), (int64_t)sections.size());
    TORCH_CHECK_VALUE(positions->dim() <= (int64_t)want.size(), kRope, ": positions ", positions->sizes(), " do not fit ", want);
    bool fits = true;
    for (int64_t d = 1; d <= positions->dim(); ++d) {
      const int64_t n = positions->size(-d);
      fits = fits && (n == want[want.size() - d] || n == 1);
    }
    TORCH_CHECK_VALUE(fits, kRope, ": positions ", positions->sizes(), " do not fit ", want);
    same_device(*positions, q, kRope, "positions");
    positions = positions->to(at::kLong).expand(want);
  } else {
    TORCH_CHECK_VALUE(cache.size(0) >= S, kRope, ": the cache has ", cache.size(0), " positions, the sequence ", S);
  }
  same_device(k, q, kRope, "k");
  same_device(cache, q, kRope, "the cache");
  TORCH_CHECK(!(at::GradMode::is_enabled() && cache.requires_grad()), kRope, ": there is no gradient with respect to the cache");
  need_gpu(q, kRope);
  const Tensor w1 = q_scale ? *q_scale : Tensor(), w2 = k_scale ? *k_scale : Tensor();
  if (wants_grad({&q, &k, &w1, &w2})) {
    variable_list o = QKNormRopeFn::apply(q, k, cache, q_scale, k_scale, eps, positions, sections, interleaved);
    return {o[0], o[1]};
  }
  return rope_forward(q, k, cache, dense(w1), dense(w2), eps, positions ? *positions : Tensor(), sections, interleaved);
}

// ---------------------------------------------------------------------------------------------------
// log probabilities of tokens
// ---------------------------------------------------------------------------------------------------
constexpr const char* kLogprobs = "token_logprobs";

// The rows of a tensor [.., V] as two nested strides; false where there are more.
bool as_rows(const Tensor& t, ttamd_logits& l) {
  l.dtype = type_code(t, kLogprobs);
  l.data = t.data_ptr();
  l.V = t.size(-1);
  l.rows = t.numel() / l.V;
  if (l.V > 1 && t.stride(-1) != 1) return false;
  std::vector<std::pair<int64_t, int64_t>> dims;  // (size, stride), outermost first, neighbours joined where they make one
  for (int64_t d = 0; d + 1 < t.dim(); ++d) {
    if (t.size(d) == 1) continue;
    if (!dims.empty() && dims.back().second == t.size(d) * t.stride(d)) {
      dims.back() = {dims.back().first * t.size(d), t.stride(d)};
    } else {
      dims.push_back({t.size(d), t.stride(d)});
    }
  }
  if (dims.size() > 2) return false;
  l.n_inner = dims.empty() ? 1 : dims.back().first;
  l.stride_inner = dims.empty() ? 0 : dims.back().second;
  l.stride_outer = dims.size() == 2 ? dims[0].second : 0;
  return true;
}

struct Logprobs {
  Tensor logprobs, entropy, top_logprobs, top_tokens, stats;
};

Logprobs logprobs_forward(const Tensor& logits_, const Tensor& tokens_, double temperature, bool entropy, int64_t top, int64_t ignore_index,
                          bool keep) {
  const c10::DeviceGuard guard(logits_.device());
  const Tensor tokens = tokens_.contiguous();
  Tensor logits = logits_;
  const std::vector<int64_t> lead(logits.sizes().begin(), logits.sizes().end() - 1);
  const int64_t n_rows = c10::multiply_integers(lead);
  const auto f32 = logits.options().dtype(at::kFloat);
  std::vector<int64_t> top_shape = lead;
  top_shape.push_back(top);
  Logprobs o;
  o.logprobs = at::empty(tokens.sizes(), f32);
  o.entropy = at::empty(entropy ? at::IntArrayRef(lead) : at::IntArrayRef({0}), f32);
  o.top_logprobs = at::empty(top_shape, f32);
  o.top_tokens = at::empty(top_shape, f32.dtype(at::kLong));
  o.stats = at::empty({keep ? n_rows : 0, 4}, f32);
  if (n_rows == 0) return o;
  ttamd_logits l = {};
  if (!as_rows(logits, l)) {
    logits = logits.contiguous();
    as_rows(logits, l);
  }
  const size_t bytes = ttamd_token_logprobs_workspace_bytes(l.rows, l.V, (int)top);
  const Tensor ws = bytes ? scratch(bytes, logits) : Tensor();
  check(ttamd_token_logprobs_fwd(&l, tokens.data_ptr<int64_t>(), tokens.numel() / n_rows, ignore_index, (float)temperature, o.logprobs.data_ptr<float>(),
                                 entropy ? o.entropy.data_ptr<float>() : nullptr, (int)top, top ? o.top_logprobs.data_ptr<float>() : nullptr,
                                 top ? o.top_tokens.data_ptr<int64_t>() : nullptr, keep ? o.stats.data_ptr<float>() : nullptr,
                                 bytes ? ws.data_ptr() : nullptr, bytes, stream_of(logits)),
        kLogprobs);
  return o;
}

struct TokenLogprobsFn : torch::autograd::Function<TokenLogprobsFn> {
  static variable_list forward(AutogradContext* ctx, const Tensor& logits, const Tensor& tokens, double temperature, bool entropy, int64_t top,
                               int64_t ignore_index) {
    Logprobs o = logprobs_forward(logits, tokens, temperature, entropy, top, ignore_index, true);
    ctx->save_for_backward({logits, tokens, o.stats});
    ctx->saved_data["temperature"] = temperature;
    ctx->saved_data["ignore_index"] = ignore_index;
    ctx->saved_data["entropy"] = entropy;
    variable_list plain = {o.top_logprobs, o.top_tokens};
    if (!entropy) plain.push_back(o.entropy);
    ctx->mark_non_differentiable(plain);
    ctx->set_materialize_grads(false);
    return {o.logprobs, o.entropy, o.top_logprobs, o.top_tokens};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    first_order(kLogprobs);
    variable_list out(6);
    const bool entropy = ctx->saved_data["entropy"].toBool() && g[1].defined();
    if (!g[0].defined() && !entropy) return out;
    const auto saved = ctx->get_saved_variables();
    Tensor logits = saved[0];
    const Tensor tokens = saved[1].contiguous(), stats = saved[2];
    const c10::DeviceGuard guard(logits.device());
    out[0] = at::empty(logits.sizes(), logits.options());
    if (logits.numel() == 0) return out;
    ttamd_logits l = {};
    if (!as_rows(logits, l)) {
      logits = logits.contiguous();
      as_rows(logits, l);
    }
    const Tensor gl = g[0].defined() ? g[0].to(at::kFloat).contiguous() : Tensor(), gh = entropy ? g[1].to(at::kFloat).contiguous() : Tensor();
    check(ttamd_token_logprobs_bwd(&l, tokens.data_ptr<int64_t>(), tokens.numel() / l.rows, ctx->saved_data["ignore_index"].toInt(),
                                   (float)ctx->saved_data["temperature"].toDouble(), stats.data_ptr<float>(),
                                   gl.defined() && gl.numel() ? gl.data_ptr<float>() : nullptr, gh.defined() ? gh.data_ptr<float>() : nullptr,
                                   out[0].data_ptr(), stream_of(logits)),
          kLogprobs);
    return out;
  }
};

// (logprobs, entropy, top_logprobs, top_tokens); the second without elements where it is not wanted
std::tuple<Tensor, Tensor, Tensor, Tensor> token_logprobs(const Tensor& logits, const Tensor& tokens, double temperature, bool entropy, int64_t top,
                                                          int64_t ignore_index) {
  type_code(logits, kLogprobs);
  TORCH_CHECK_VALUE(logits.dim() >= 1 && logits.size(-1) > 0, kLogprobs, ": expected logits [.., vocabulary], got ", logits.sizes());
  TORCH_CHECK_TYPE(tokens.scalar_type() == at::kLong, kLogprobs, ": tokens must be int64, got ", tokens.scalar_type());
  bool fits = tokens.dim() == logits.dim() - 1 || tokens.dim() == logits.dim();
  for (int64_t d = 0; fits && d + 1 < logits.dim(); ++d) fits = tokens.size(d) == logits.size(d);
  TORCH_CHECK_VALUE(fits && !(tokens.dim() == logits.dim() && tokens.size(-1) == 0), kLogprobs, ": tokens ", tokens.sizes(), " do not fit logits ", logits.sizes(),
                    " (one token a row, or [.., tokens])");
  TORCH_CHECK_VALUE(temperature > 1e-6 && temperature < 1e6, kLogprobs, ": the temperature must be positive (1e-6 to 1e6), got ", temperature);
  TORCH_CHECK_VALUE(top >= 0 && top <= 64 && top <= logits.size(-1), kLogprobs, ": top must be 0 to 64 and at most the vocabulary, got ", top);
  same_device(tokens, logits, kLogprobs, "tokens");
  need_gpu(logits, kLogprobs);
  if (wants_grad({&logits})) {
    variable_list o = TokenLogprobsFn::apply(logits, tokens, temperature, entropy, top, ignore_index);
    return {o[0], o[1], o[2], o[3]};
  }
  Logprobs o = logprobs_forward(logits, tokens, temperature, entropy, top, ignore_index, false);
  return {o.logprobs, o.entropy, o.top_logprobs, o.top_tokens};
}

// ---------------------------------------------------------------------------------------------------
// AdamW
// ---------------------------------------------------------------------------------------------------
constexpr const char* kAdamW = "AdamW";

// From the first byte of a tensor's elements to behind the last (of one that has any).
int64_t span_bytes(const Tensor& t) {
  int64_t last = 0;
  for (int64_t d = 0; d < t.dim(); ++d) last += (t.size(d) - 1) * t.stride(d);
  return (last + 1) * (int64_t)t.itemsize();
}

// A tensor's memory may have been given up under it (sharding and offloading resize storages).
void check_memory(const Tensor& t, const char* name) {
  const int64_t there = (int64_t)t.storage().nbytes(), size = (int64_t)t.itemsize(), from = t.storage_offset() * size;
  TORCH_CHECK(t.numel() == 0 || there >= from + (t.is_non_overlapping_and_dense() ? t.numel() * size : span_bytes(t)), kAdamW, ": the memory of ", name,
              " ", t.sizes(), " is not there, its storage has ", there, " bytes");
}

void check_param(const Tensor& p) {
  TORCH_CHECK(!p.key_set().has(c10::DispatchKey::Python) && p.layout() == at::kStrided, kAdamW, ": parameters must be plain dense tensors");
  type_code(p, kAdamW);
  check_memory(p, "a parameter");
  need_gpu(p, kAdamW);
  if (!p.is_non_overlapping_and_dense()) at::assert_no_internal_overlap(p);
}

void check_gradient(const Tensor& g) {
  TORCH_CHECK(g.layout() == at::kStrided && !g.key_set().has(c10::DispatchKey::Python), kAdamW, ": gradients must be plain dense tensors");
  check_memory(g, "a gradient");
}

// Whether two tensors are seen to share no byte: their elements' places modulo the pitch of one of their dimensions lie in
// intervals that do not meet, as those of columns of one matrix.
bool apart(const Tensor& a, const Tensor& b) {
  const auto place = [](const Tensor& t) { return (uint64_t)reinterpret_cast<uintptr_t>(t.data_ptr()); };
  const auto width = [](const Tensor& t, int64_t pitch) {  // of the interval
    int64_t w = (int64_t)t.itemsize();
    for (int64_t d = 0; d < t.dim(); ++d)
      if (t.size(d) > 1 && t.stride(d) * (int64_t)t.itemsize() % pitch) w += (t.size(d) - 1) * t.stride(d) * (int64_t)t.itemsize();
    return w;
  };
  for (const Tensor* t : {&a, &b}) {
    for (int64_t d = 0; d < t->dim(); ++d) {
      const int64_t pitch = t->stride(d) * (int64_t)t->itemsize();
      if (t->size(d) < 2 || pitch <= 0) continue;
      const int64_t shift = (int64_t)((place(b) % pitch + pitch - place(a) % pitch) % pitch);
      if (width(a, pitch) <= shift && shift + width(b, pitch) <= pitch) return true;
    }
  }
  return false;
}

// Two of these tensors that share memory or cannot be seen not to.  Those that lie densely, one after another, cost a sort.
std::optional<std::pair<int64_t, int64_t>> overlapping(const std::vector<Tensor>& tensors) {
  struct Span {
    uintptr_t begin, end;
    int64_t of;
  };
  std::vector<Span> spans, open;
  for (size_t i = 0; i < tensors.size(); ++i) {
    const Tensor& t = tensors[i];
    if (!t.defined() || t.numel() == 0) continue;
    const uintptr_t begin = reinterpret_cast<uintptr_t>(t.data_ptr());
    spans.push_back({begin, begin + (uintptr_t)span_bytes(t), (int64_t)i});
  }
  std::sort(spans.begin(), spans.end(), [](const Span& a, const Span& b) { return a.begin < b.begin; });
  for (const Span& s : spans) {
    open.erase(std::remove_if(open.begin(), open.end(), [&](const Span& o) { return o.end <= s.begin; }), open.end());
    for (const Span& o : open)
      if (!apart(tensors[o.of], tensors[s.of])) return std::make_pair(std::min(o.of, s.of), std::max(o.of, s.of));
    open.push_back(s);
  }
  return std::nullopt;
}

// The order of a dense tensor's elements in its states, as it lies in memory.  (One with gaps: row by row.)  Strides of single
// elements say nothing.
std::vector<int64_t> order_of(const Tensor& p) {
  std::vector<int64_t> s = p.strides().vec();
  for (int64_t d = 0; d < p.dim(); ++d)
    if (p.size(d) <= 1) s[d] = 0;
  return s;
}

// Parameters of one type on one device with the buffers that hold their moments.
struct Block {
  std::vector<Tensor> params;
  std::vector<int64_t> numbers;
  std::vector<std::vector<int64_t>> order;  // empty: row by row
  std::vector<Tensor> shadow;  // of parameters that do not lie densely
  std::vector<void*> address;  // that the table holds
  struct Place {
    int64_t offset, numel, block;
  };
  std::vector<Place> places;
  std::vector<uint32_t> chunks;  // first chunk of each tensor, and the end
  bool shared = false;          // some of the addresses may be in several parameters
  Tensor table, exp_avg, exp_avg_sq, exp_avg_exponent, exp_avg_sq_exponent, steps;
  int bits;
  at::ScalarType type;         // of the parameters
  c10::hip::HIPStream stream;  // that the buffers were made on

  Block(std::vector<Tensor> ps, std::vector<int64_t> numbers_, int bits_)
      : params(std::move(ps)), numbers(std::move(numbers_)), bits(bits_), type(params[0].scalar_type()), stream(c10::hip::getCurrentHIPStream(params[0].get_device())) {
    const c10::DeviceGuard guard(params[0].device());
    int64_t n = 0, blocks = 0;
    uint64_t chunk = 0;
    for (size_t i = 0; i < params.size(); ++i) {
      const int64_t m = params[i].numel();
      places.push_back({n, m, blocks});
      chunks.push_back((uint32_t)chunk);
      order.push_back(params[i].is_contiguous() || !params[i].is_non_overlapping_and_dense() ? std::vector<int64_t>() : order_of(params[i]));
      n += m;
      blocks += (m + TTAMD_ADAMW_BLOCK - 1) / TTAMD_ADAMW_BLOCK;
      chunk += (m + TTAMD_ADAMW_CHUNK - 1) / TTAMD_ADAMW_CHUNK;
    }
    TORCH_CHECK(chunk < (uint64_t(1) << 31), kAdamW, ": too many parameters in one group");
    chunks.push_back((uint32_t)chunk);
    const auto dev = params[0].options();
    exp_avg = at::zeros({n}, dev.dtype(bits == 8 ? at::kByte : at::kFloat));
    exp_avg_sq = at::zeros_like(exp_avg);
    if (bits == 8) {
      exp_avg_exponent = at::full({blocks}, 16, dev.dtype(at::kByte));
      exp_avg_sq_exponent = at::full_like(exp_avg_exponent, 16);
    }
    steps = at::zeros({(int64_t)params.size()}, at::kLong);
    shadow.resize(params.size());
    address.resize(params.size());
  }

  // Where the kernel finds tensor i: the parameter, or a copy of one with gaps, which lives as long as the states.
  void* find(size_t i) {
    if (params[i].is_non_overlapping_and_dense()) return params[i].data_ptr();
    if (!shadow[i].defined() || shadow[i].sizes() != params[i].sizes()) shadow[i] = at::empty(params[i].sizes(), params[i].options());
    return shadow[i].data_ptr();
  }

  // The table of chunks, made again when a parameter's memory has moved.
  void point() {
    bool same = table.defined();
    for (size_t i = 0; i < params.size(); ++i) {
      void* now = find(i);
      same = same && now == address[i];
      address[i] = now;
    }
    if (same) return;
    shared = overlapping(params).has_value();
    const Tensor host = at::empty({(int64_t)(std::max<uint32_t>(chunks.back(), 1) * sizeof(ttamd_adamw_chunk))}, at::kByte);
    ttamd_adamw_chunk* to = (ttamd_adamw_chunk*)host.data_ptr();
    for (size_t i = 0; i < params.size(); ++i)
      for (uint32_t j = chunks[i]; j < chunks[i + 1]; ++j)
        to[j] = {address[i], (int64_t)(j - chunks[i]) * TTAMD_ADAMW_CHUNK, places[i].numel, places[i].offset, places[i].block, (uint32_t)i, (uint32_t)numbers[i]};
    table = host.to(exp_avg.device());
  }

  ttamd_adamw_states states() const {
    ttamd_adamw_states s = {};
    s.chunks = (const ttamd_adamw_chunk*)table.data_ptr();
    s.exp_avg = exp_avg.data_ptr();
    s.exp_avg_sq = exp_avg_sq.data_ptr();
    if (bits == 8) {
      s.exp_avg_exponent = exp_avg_exponent.data_ptr<uint8_t>();
      s.exp_avg_sq_exponent = exp_avg_sq_exponent.data_ptr<uint8_t>();
    }
    s.state_bits = bits;
    return s;
  }

  // The buffers outlive what another stream does with them (the later ones were made on whatever stream was current).
  void used_on(const c10::hip::HIPStream& now) const {
    auto record = [&](const Tensor& t) {
      if (t.defined()) c10::hip::HIPCachingAllocator::recordStream(t.storage().data_ptr(), now);
    };
    record(table);
    for (const Tensor& t : shadow) record(t);
    if (now == stream) return;
    for (const Tensor* t : {&exp_avg, &exp_avg_sq, &exp_avg_exponent, &exp_avg_sq_exponent}) record(*t);
  }

  // a flat buffer's part of tensor i, laid out as the parameter is
  Tensor like(const Tensor& flat, size_t i) const {
    const Tensor& p = params[i];
    const Tensor part = flat.narrow(0, places[i].offset, places[i].numel);
    return p.is_non_overlapping_and_dense() ? part.as_strided(p.sizes(), p.strides(), part.storage_offset()) : part.view(p.sizes());
  }
  Tensor exponents(const Tensor& flat, size_t i) const {
    return flat.narrow(0, places[i].block, (places[i].numel + TTAMD_ADAMW_BLOCK - 1) / TTAMD_ADAMW_BLOCK);
  }

  std::pair<Tensor, Tensor> moments() {
    if (bits == 32) return {exp_avg, exp_avg_sq};
    const c10::DeviceGuard guard(exp_avg.device());
    Tensor m = at::empty(exp_avg.sizes(), exp_avg.options().dtype(at::kBFloat16)), v = at::empty_like(m);
    if (chunks.back() == 0) return {m, v};
    point();
    used_on(c10::hip::getCurrentHIPStream(exp_avg.get_device()));
    const ttamd_adamw_states s = states();
    check(ttamd_adamw_moments_bf16(&s, chunks.back(), m.data_ptr(), v.data_ptr(), stream_of(m)), kAdamW);
    return {m, v};
  }

  // The gradients (undefined: none) of a step that can be taken; nothing is changed here.
  std::vector<Tensor> gradients() const {
    const c10::DeviceGuard guard(params[0].device());
    TORCH_CHECK(c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None, kAdamW,
                ": a step cannot be recorded into a graph (its count, and with it the bias corrections, would stand still)");
    const size_t n = params.size();
    std::vector<Tensor> grads(n);
    for (size_t i = 0; i < n; ++i) {
      const Tensor& p = params[i];
      const Tensor& g = grads[i] = p.grad();
      if (!g.defined()) continue;
      check_gradient(g);
      check_param(p);
      TORCH_CHECK_TYPE(g.scalar_type() == p.scalar_type(), kAdamW, ": a gradient is ", g.scalar_type(), ", its parameter ", p.scalar_type());
      TORCH_CHECK(g.device() == p.device() && p.device() == exp_avg.device(), kAdamW, ": a parameter or its gradient has left ", exp_avg.device().str());
      TORCH_CHECK(p.numel() == places[i].numel && g.sizes() == p.sizes() && p.scalar_type() == type, kAdamW,
                  ": a parameter's size or type has changed");
      TORCH_CHECK(order[i].empty() ? p.is_contiguous() || !p.is_non_overlapping_and_dense() : order_of(p) == order[i], kAdamW,
                  ": the order of a parameter's elements in memory has changed");
    }
    return grads;
  }

  // One launch steps many parameters at a time, so that none may be part of another.
  void check_apart(const std::vector<Tensor>& grads) const {
    if (!shared) return;
    std::vector<Tensor> stepped(params.size());
    for (size_t i = 0; i < params.size(); ++i)
      if (grads[i].defined()) stepped[i] = params[i];
    const auto two = overlapping(stepped);
    TORCH_CHECK(!two, kAdamW, ": parameters ", numbers[two->first], " and ", numbers[two->second], ", ", stepped[two->first].sizes(), " and ",
                stepped[two->second].sizes(), ", share memory");
  }

  // grads: what gradients() gave, and point() has been called since
  void step(const std::vector<Tensor>& grads, const ttamd_adamw_scalars& scalars) {
    const c10::DeviceGuard guard(params[0].device());
    const auto now = c10::hip::getCurrentHIPStream(params[0].get_device());
    const size_t n = params.size();
    used_on(now);
    const ttamd_adamw_states s = states();
    const int dtype = type == at::kBFloat16 ? TTAMD_BF16 : TTAMD_F32;
    int64_t* count = steps.data_ptr<int64_t>();
    const void* g[TTAMD_ADAMW_TENSORS];
    for (size_t first = 0; first < n;) {
      if (!grads[first].defined()) {
        ++first;
        continue;
      }
      // neighbours that have taken as many steps
      std::vector<Tensor> hold;
      std::vector<size_t> back;
      size_t end = first;
      for (; end < n && end - first < TTAMD_ADAMW_TENSORS && grads[end].defined() && count[end] == count[first]; ++end) {
        const Tensor &t = params[end], &grad = grads[end];
        const bool dense = t.is_non_overlapping_and_dense();
        if (!dense) {
          shadow[end].copy_(t);
          back.push_back(end);
        }
        if (dense && grad.strides() == t.strides()) {
          g[end - first] = grad.data_ptr();
        } else {
          // as the parameter lies in memory
          hold.push_back(!dense || t.is_contiguous() ? grad.contiguous() : at::empty_strided(t.sizes(), t.strides(), grad.options()).copy_(grad));
          g[end - first] = hold.back().data_ptr();
        }
        // an empty tensor has no address; nothing reads it
        if (t.numel() == 0) g[end - first] = table.data_ptr();
      }
      ttamd_adamw_scalars c = scalars;
      c.step = count[first] + 1;
      if (chunks[end] > chunks[first])
        check(ttamd_adamw_step(g, (int)(end - first), dtype, &s, (uint32_t)first, chunks[first], chunks[end] - chunks[first], &c, now.stream()), kAdamW);
      for (size_t i : back) params[i].detach().copy_(shadow[i]);
      for (size_t i = first; i < end; ++i) {
        ++count[i];
        if (!params[i].is_inference()) params[i].unsafeGetTensorImpl()->bump_version();
      }
      first = end;
    }
  }
};

// A parameter group: blocks are made for parameters when they first have a gradient, or when their states are given.
struct AdamWGroup {
  std::vector<Tensor> params;
  std::vector<std::pair<int, int>> where;  // block and place in it, or -1
  std::vector<std::unique_ptr<Block>> blocks;
  int64_t number;
  int bits;
  std::mutex mutex;  // calls run without the interpreter's lock

  AdamWGroup(std::vector<Tensor> ps, int64_t first_number, int64_t bits_)
      : params(std::move(ps)), where(params.size(), {-1, -1}), number(first_number), bits((int)bits_) {}

  // whether a list still holds these parameters (the tensors themselves: an element may have been replaced)
  bool holds(const py::handle& list) const {
    const py::object items = py::reinterpret_steal<py::object>(PySequence_Fast(list.ptr(), "expected a list of parameters"));
    if (!items) throw py::error_already_set();
    if (PySequence_Fast_GET_SIZE(items.ptr()) != (Py_ssize_t)params.size()) return false;
    for (size_t i = 0; i < params.size(); ++i) {
      PyObject* p = PySequence_Fast_GET_ITEM(items.ptr(), (Py_ssize_t)i);
      if (!THPVariable_Check(p) || THPVariable_Unpack(p).unsafeGetTensorImpl() != params[i].unsafeGetTensorImpl()) return false;
    }
    return true;
  }

  // states for these parameters, a block for each device and type; what has them already keeps them
  void make(const std::vector<int64_t>& of) {
    const std::lock_guard<std::mutex> lock(mutex);
    const at::NoGradGuard no_grad;
    std::vector<int64_t> left;
    for (int64_t i : of)
      if (where.at(i).first < 0) left.push_back(i);
    for (int64_t i : left) check_param(params[i]);
    while (!left.empty()) {
      const Tensor& like = params[left[0]];
      std::vector<Tensor> ps;
      std::vector<int64_t> numbers, other;
      for (int64_t i : left) {
        if (params[i].device() != like.device() || params[i].scalar_type() != like.scalar_type()) {
          other.push_back(i);
          continue;
        }
        ps.push_back(params[i]);
        numbers.push_back(number + i);
      }
      const int block = (int)blocks.size();
      blocks.push_back(std::make_unique<Block>(std::move(ps), numbers, bits));
      for (size_t k = 0; k < numbers.size(); ++k) where[numbers[k] - number] = {block, (int)k};
      left = std::move(other);
    }
  }

  // (step, exp_avg, exp_avg_sq[, exponents of both]) of a parameter
  std::vector<Tensor> state(int64_t i) {
    const std::lock_guard<std::mutex> lock(mutex);
    const Block& b = *blocks.at(where.at(i).first);
    const size_t at = where[i].second;
    std::vector<Tensor> s = {b.steps.select(0, at), b.like(b.exp_avg, at), b.like(b.exp_avg_sq, at)};
    if (bits == 8) {
      s.push_back(b.exponents(b.exp_avg_exponent, at));
      s.push_back(b.exponents(b.exp_avg_sq_exponent, at));
    }
    return s;
  }

  // the places of parameters that have a gradient and no states yet; none if the list holds other parameters than these
  std::optional<std::vector<int64_t>> fresh(const py::handle& list) {
    if (!holds(list)) return std::nullopt;
    const py::gil_scoped_release unlocked;
    const std::lock_guard<std::mutex> lock(mutex);
    std::vector<int64_t> found;
    for (size_t i = 0; i < params.size(); ++i) {
      if (where[i].first >= 0 || !params[i].grad().defined()) continue;
      const Tensor g = params[i].grad();
      check_gradient(g);
      check_param(params[i]);
      TORCH_CHECK(c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None, kAdamW, ": a step cannot be recorded into a graph");
      found.push_back((int64_t)i);
    }
    return found;
  }

  // the flat moments, where one block holds all parameters in their order
  std::optional<std::pair<Tensor, Tensor>> whole() {
    const std::lock_guard<std::mutex> lock(mutex);
    if (blocks.size() != 1 || blocks[0]->params.size() != params.size()) return std::nullopt;
    return blocks[0]->moments();
  }
  // else those of each parameter that has them, in their order
  std::vector<std::pair<Tensor, Tensor>> moments() {
    const std::lock_guard<std::mutex> lock(mutex);
    std::vector<std::pair<Tensor, Tensor>> all, out;
    for (const auto& b : blocks) all.push_back(b->moments());
    for (const auto& [b, at] : where) {
      if (b < 0) continue;
      const Block::Place& p = blocks[b]->places[at];
      out.push_back({all[b].first.narrow(0, p.offset, p.numel), all[b].second.narrow(0, p.offset, p.numel)});
    }
    return out;
  }
};

// group, lr, beta1, beta2, eps, weight_decay, seed, stochastic
typedef std::tuple<AdamWGroup*, double, double, double, double, double, int64_t, bool> GroupStep;

// One step of several groups: everything is checked, in all of them, before anything is changed.
void adamw_step(const std::vector<GroupStep>& groups) {
  const at::NoGradGuard no_grad;
  std::vector<std::unique_lock<std::mutex>> locks;
  struct Ready {
    Block* block;
    std::vector<Tensor> grads;
    ttamd_adamw_scalars scalars;
  };
  std::vector<Ready> ready;
  for (const auto& [group, lr, beta1, beta2, eps, weight_decay, seed, stochastic] : groups) {
    locks.emplace_back(group->mutex);
    ttamd_adamw_scalars c = {};
    c.lr = lr;
    c.beta1 = beta1;
    c.beta2 = beta2;
    c.eps = eps;
    c.weight_decay = weight_decay;
    c.seed = seed;
    for (auto& b : group->blocks) {
      c.stochastic = stochastic && b->type == at::kBFloat16;
      std::vector<Tensor> grads = b->gradients();
      if (std::none_of(grads.begin(), grads.end(), [](const Tensor& g) { return g.defined(); })) continue;
      TORCH_CHECK_VALUE(beta1 >= 0 && beta1 < 1 && beta2 >= 0 && beta2 < 1 && eps >= 0, kAdamW, ": betas ", beta1, ", ", beta2, " and eps ", eps);
      ready.push_back({b.get(), std::move(grads), c});
    }
  }
  for (Ready& r : ready) {
    const c10::DeviceGuard guard(r.block->params[0].device());
    r.block->point();
    r.block->check_apart(r.grads);
  }
  for (Ready& r : ready) r.block->step(r.grads, r.scalars);
}

}  // namespace

void bind_post(py::module_& m) {
  const py::call_guard<py::gil_scoped_release> unlocked;
  m.def("qk_norm_rope", &qk_norm_rope, unlocked);
  m.def("token_logprobs", &token_logprobs, unlocked);
  py::class_<AdamWGroup>(m, "AdamWGroup")
      .def(py::init<std::vector<Tensor>, int64_t, int64_t>())
      .def("holds", &AdamWGroup::holds)
      .def("make", &AdamWGroup::make, unlocked)
      .def("state", &AdamWGroup::state, unlocked)
      .def("fresh", &AdamWGroup::fresh)
      .def("whole", &AdamWGroup::whole, unlocked)
      .def("moments", &AdamWGroup::moments, unlocked);
  // one group, as most optimizers have, without the list: half a microsecond
  m.def("adamw_step",
        [](AdamWGroup& group, double lr, double beta1, double beta2, double eps, double weight_decay, int64_t seed, bool stochastic) {
          adamw_step({GroupStep(&group, lr, beta1, beta2, eps, weight_decay, seed, stochastic)});
        },
        unlocked);
  m.def("adamw_step", &adamw_step, unlocked);
  m.def("overlapping", &overlapping);
}
