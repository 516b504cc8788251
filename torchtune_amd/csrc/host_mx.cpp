// Host path of the microscaled tensors: argument checks, output and workspace allocation, autograd nodes and the library calls
// of to_mx, linear_mx and lora_linear_mx in native code.  The kernels of a small call take 4 - 12 us; through Python wrappers
// and a torch.autograd.Function the host took 11 (codec), 20 (linear) and 200 us (adapter layers, both directions).
// Checks of shapes and types come before those of the device, so that they hold without one.
#include "host_common.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using namespace ttamd_host;

int64_t per_block(int64_t format) { return format == TTAMD_MXFP4 ? 16 : 32; }  // bytes of codes

// Contiguous and 16-byte aligned, a copy only where it is not.
Tensor dense(const Tensor& t) {
  const Tensor c = t.contiguous();
  return (reinterpret_cast<uintptr_t>(c.data_ptr()) & 15u) == 0 ? c : c.clone();
}

int codec_dtype(at::ScalarType t, const char* what) {
  TORCH_CHECK_TYPE(t == at::kBFloat16 || t == at::kFloat, what, ": dtype ", t, " is not supported (bfloat16 and float32 are)");
  return t == at::kBFloat16 ? TTAMD_BF16 : TTAMD_F32;
}

std::vector<int64_t> resized(const Tensor& t, int64_t last) {
  std::vector<int64_t> s = t.sizes().vec();
  s.back() = last;
  return s;
}

std::tuple<Tensor, Tensor> mx_quantize(const Tensor& x_, int64_t format) {
  const int dtype = codec_dtype(x_.scalar_type(), "to_mx");
  TORCH_CHECK_VALUE(x_.dim() > 0 && x_.size(-1) > 0 && x_.size(-1) % 32 == 0, "to_mx: the last dimension must be a positive multiple of 32, got ",
                    x_.sizes());
  need_gpu(x_, "to_mx");
  const c10::DeviceGuard guard(x_.device());
  const Tensor x = dense(x_.detach());
  const int64_t K = x.size(-1);
  const auto u8 = x.options().dtype(at::kByte);
  Tensor codes = at::empty(resized(x, K / 32 * per_block(format)), u8), scales = at::empty(resized(x, K / 32), u8);
  check(ttamd_mx_quantize(x.data_ptr(), dtype, x.numel() / K, K, (int)format, (uint8_t*)codes.data_ptr(), (uint8_t*)scales.data_ptr(), stream_of(x)),
        "to_mx");
  return {codes, scales};
}

void check_parts(const Tensor& codes, const Tensor& scales, int64_t format, const char* what) {
  TORCH_CHECK_TYPE(codes.scalar_type() == at::kByte && scales.scalar_type() == at::kByte, what, ": codes and scales must be uint8, got ",
                   codes.scalar_type(), " and ", scales.scalar_type());
  bool fits = codes.dim() > 0 && codes.dim() == scales.dim() && codes.size(-1) == per_block(format) * scales.size(-1);
  for (int64_t d = 0; fits && d + 1 < codes.dim(); ++d) fits = codes.size(d) == scales.size(d);
  TORCH_CHECK_VALUE(fits, what, ": codes ", codes.sizes(), " and scales ", scales.sizes(), " do not fit each other");
  TORCH_CHECK_VALUE(codes.device() == scales.device(), what, ": codes on ", codes.device().str(), ", scales on ", scales.device().str());
}

Tensor mx_dequantize(const Tensor& codes_, const Tensor& scales_, int64_t format, at::ScalarType type) {
  const int dtype = codec_dtype(type, "MXTensor.to");
  check_parts(codes_, scales_, format, "MXTensor.to");
  need_gpu(codes_, "MXTensor.to");
  const c10::DeviceGuard guard(codes_.device());
  const Tensor codes = dense(codes_), scales = scales_.contiguous();
  const int64_t K = 32 * scales.size(-1);
  Tensor out = at::empty(resized(codes, K), codes.options().dtype(type));
  if (K == 0) return out;
  check(ttamd_mx_dequantize((const uint8_t*)codes.data_ptr(), (const uint8_t*)scales.data_ptr(), (int)format, scales.numel() / scales.size(-1), K,
                            dtype, out.data_ptr(), stream_of(codes)),
        "MXTensor.to");
  return out;
}

// The backward passes are kernels that autograd does not see into.
void first_order(const char* what) {
  TORCH_CHECK(!at::GradMode::is_enabled(), what, ": the backward pass cannot be differentiated (create_graph=True)");
}

// the weight of a product: 2-D mxfp4
void check_weight(const Tensor& codes, const Tensor& scales, const Tensor& x, const char* what) {
  check_parts(codes, scales, TTAMD_MXFP4, what);
  TORCH_CHECK_VALUE(codes.dim() == 2 && codes.size(1) > 0, what, ": the weight must have two dimensions and inputs, got codes ", codes.sizes());
  TORCH_CHECK_TYPE(x.scalar_type() == at::kBFloat16, what, ": expected a bfloat16 input, got ", x.scalar_type());
  TORCH_CHECK(x.dim() > 0 && x.size(-1) == 2 * codes.size(1), what, ": mat1 and mat2 shapes cannot be multiplied (", x.sizes(), " and ",
              2 * codes.size(1), "x", codes.size(0), ")");
  TORCH_CHECK(x.device() == codes.device(), what, ": the input is on ", x.device().str(), ", the weight on ", codes.device().str());
}

void check_bias(const Tensor& bias, int64_t N, const Tensor& x, const char* what) {
  if (!bias.defined()) return;
  TORCH_CHECK_TYPE(bias.scalar_type() == at::kBFloat16, what, ": the bias must be bfloat16, got ", bias.scalar_type());
  TORCH_CHECK_VALUE(bias.dim() == 1 && bias.size(0) == N, what, ": bias ", bias.sizes(), " does not fit ", N, " outputs");
  TORCH_CHECK(bias.device() == x.device(), what, ": the input is on ", x.device().str(), ", the bias on ", bias.device().str());
}

void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

Tensor linear_forward(const Tensor& x_, const Tensor& codes_, const Tensor& scales_, const Tensor& bias_, int64_t activation) {
  need_gpu(x_, "linear_mx");
  const c10::DeviceGuard guard(x_.device());
  const Tensor x = dense(x_), codes = dense(codes_), scales = dense(scales_), bias = bias_.defined() ? bias_.contiguous() : bias_;
  const int64_t K = x.size(-1), N = codes.size(0), M = x.numel() / K;
  Tensor y = at::empty(resized(x, N), x.options());
  if (y.numel() == 0) return y;
  const size_t bytes = ttamd_mx_linear_workspace_bytes(M, N, K, (int)activation);
  const Tensor ws = bytes ? scratch(bytes, x) : Tensor();
  check(ttamd_mx_linear_bf16(x.data_ptr(), (int)activation, (const uint8_t*)codes.data_ptr(), (const uint8_t*)scales.data_ptr(), ptr(bias), y.data_ptr(),
                             M, N, K, ptr(ws), bytes, stream_of(x)),
        "linear_mx");
  return y;
}

struct LinearMXFn : torch::autograd::Function<LinearMXFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& codes, const Tensor& scales, const std::optional<Tensor>& bias,
                        int64_t activation) {
    ctx->save_for_backward({codes, scales});
    ctx->saved_data["shape"] = x.sizes().vec();
    ctx->saved_data["bias"] = bias.has_value();  // an absent one has no edge to ask about
    return linear_forward(x, codes, scales, bias ? *bias : Tensor(), activation);
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    first_order("linear_mx");
    const auto saved = ctx->get_saved_variables();
    const Tensor codes = dense(saved[0]), scales = dense(saved[1]);
    const int64_t N = codes.size(0), K = 2 * codes.size(1);
    const c10::DeviceGuard guard(codes.device());
    Tensor gx, gbias;
    const std::vector<int64_t> shape = ctx->saved_data["shape"].toIntVector();
    const int64_t M = c10::multiply_integers(shape) / K;
    const Tensor gy = dense(g[0]).reshape({M, N});
    if (ctx->needs_input_grad(0)) {
      gx = gy.numel() ? at::empty(shape, gy.options()) : at::zeros(shape, gy.options());
      if (gy.numel()) {
        const Tensor ws = scratch(ttamd_mx_linear_dx_workspace_bytes(M, N, K), gy);
        check(ttamd_mx_linear_dx_bf16(gy.data_ptr(), (const uint8_t*)codes.data_ptr(), (const uint8_t*)scales.data_ptr(), gx.data_ptr(), M, N, K,
                                      ws.data_ptr(), ws.numel(), stream_of(gy)),
              "linear_mx");
      }
    }
    if (ctx->saved_data["bias"].toBool() && ctx->needs_input_grad(3)) gbias = column_sum(gy);
    return {gx, Tensor(), Tensor(), gbias, Tensor()};
  }
};

Tensor mx_linear(const Tensor& x, const Tensor& codes, const Tensor& scales, const std::optional<Tensor>& bias, int64_t activation) {
  check_weight(codes, scales, x, "linear_mx");
  const Tensor b = bias ? *bias : Tensor();
  check_bias(b, codes.size(0), x, "linear_mx");
  if (!wants_grad({&x, &b})) return linear_forward(x, codes, scales, b, activation);
  const int64_t N = codes.size(0), K = 2 * codes.size(1);
  TORCH_CHECK_VALUE(!x.requires_grad() || (N % 64 == 0 && K % 64 == 0), "linear_mx: the gradient of the input needs a weight whose sides are multiples of 64, got ", N,
                    " x ", K);
  return LinearMXFn::apply(x, codes, scales, bias, activation);
}

// ---------------------------------------------------------------------------------------------------
// adapter linears over the same input
// ---------------------------------------------------------------------------------------------------
struct MxMember {
  Tensor codes, scales, a, b, bias;
  double scale = 0;
};

void fill(ttamd_mx_lora_member& e, const MxMember& m, const Tensor& y) {
  e = {};
  e.codes = (const uint8_t*)m.codes.data_ptr();
  e.scales = (const uint8_t*)m.scales.data_ptr();
  e.lora_a = m.a.data_ptr();
  e.lora_b = m.b.data_ptr();
  e.bias = ptr(m.bias);
  e.y = y.data_ptr();
  e.N = m.codes.size(0);
  e.rank = (int)m.a.size(0);
  e.scale = (float)m.scale;
}

// What the backward pass reads, in one piece of memory: the input's codes and scales, and h [M, ranks].
struct Kept {
  size_t scales, h, bytes;  // offsets
  Kept(int64_t M, int64_t K, int64_t ranks)
      : scales(align256(ttamd_mx_kept_codes_bytes(M, K))), h(scales + align256(ttamd_mx_kept_scales_bytes(M, K))), bytes(h + 2 * M * ranks) {}
};

struct LoraOut {
  std::vector<Tensor> ys;
  Tensor kept;
};

LoraOut lora_forward(const Tensor& x_, const std::vector<MxMember>& given) {
  need_gpu(x_, "lora_linear_mx");
  const c10::DeviceGuard guard(x_.device());
  const Tensor x = dense(x_);
  const int64_t K = x.size(-1), M = x.numel() / K;
  const int n = (int)given.size();
  LoraOut o;
  std::vector<MxMember> ms = given;
  ttamd_mx_lora_member arr[TTAMD_GROUP_MAX];
  int64_t ranks = 0;
  for (int i = 0; i < n; ++i) {
    MxMember& m = ms[i];
    for (Tensor* t : {&m.codes, &m.scales, &m.a, &m.b}) *t = dense(*t);
    if (m.bias.defined()) m.bias = m.bias.contiguous();
    o.ys.push_back(at::empty(resized(x, m.codes.size(0)), x.options()));
    fill(arr[i], m, o.ys[i]);
    ranks += m.a.size(0);
  }
  const Kept at(M, K, ranks);
  o.kept = at::empty({(int64_t)at.bytes}, x.options().dtype(at::kByte));
  if (M == 0) return o;
  uint8_t* kept = (uint8_t*)o.kept.data_ptr();
  const Tensor ws = scratch(ttamd_mx_lora_fwd_workspace_bytes(arr, n, M, K), x);
  check(ttamd_mx_lora_fwd_bf16(x.data_ptr(), arr, n, kept, kept + at.scales, kept + at.h, M, K, ws.data_ptr(),
                               ws.numel(), stream_of(x)),
        "lora_linear_mx");
  return o;
}

// Differentiable inputs: x, then per member lora_a, lora_b and, where there is one, the bias.
struct LoraMXFn : torch::autograd::Function<LoraMXFn> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, at::TensorList /*inputs*/, const std::vector<MxMember>& ms) {
    LoraOut o = lora_forward(x, ms);
    variable_list save = {o.kept};
    std::vector<double> factors;
    std::vector<int64_t> bias;
    for (const MxMember& m : ms) {
      for (const Tensor& t : {m.codes, m.scales, m.a, m.b}) save.push_back(t);
      factors.push_back(m.scale);
      bias.push_back(m.bias.defined() ? 1 : 0);
    }
    ctx->save_for_backward(std::move(save));
    ctx->saved_data["factors"] = factors;
    ctx->saved_data["bias"] = bias;
    ctx->saved_data["shape"] = x.sizes().vec();
    return o.ys;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    first_order("lora_linear_mx");
    const auto saved = ctx->get_saved_variables();
    const Tensor& kept = saved[0];
    const std::vector<double> factors = ctx->saved_data["factors"].toDoubleVector();
    const std::vector<int64_t> bias = ctx->saved_data["bias"].toIntVector(), shape = ctx->saved_data["shape"].toIntVector();
    const int n = (int)factors.size();
    const c10::DeviceGuard guard(kept.device());
    const int64_t K = shape.back(), M = c10::multiply_integers(shape) / K;
    int64_t ranks = 0;
    std::vector<Tensor> gys(n), ga(n), gb(n);
    std::vector<MxMember> ms(n);
    ttamd_mx_lora_member arr[TTAMD_GROUP_MAX];
    // what is wanted: x's gradient, any adapter's, and which of the biases'
    const bool need_x = ctx->needs_input_grad(0);
    bool need_ab = false, need_bias[TTAMD_GROUP_MAX] = {};
    size_t edge = 1;
    for (int i = 0; i < n; ++i) {
      need_ab = need_ab || ctx->needs_input_grad(edge) || ctx->needs_input_grad(edge + 1);
      edge += 2;
      if (bias[i]) need_bias[i] = ctx->needs_input_grad(edge++);
    }
    for (int i = 0; i < n; ++i) {
      MxMember& m = ms[i];
      m.codes = dense(saved[1 + 4 * i]);
      m.scales = dense(saved[2 + 4 * i]);
      m.a = dense(saved[3 + 4 * i]);
      m.b = dense(saved[4 + 4 * i]);
      m.scale = factors[i];
      ranks += m.a.size(0);
      gys[i] = dense(g[i]).reshape({M, m.codes.size(0)});
      fill(arr[i], m, gys[i]);
      if (!need_ab) continue;
      ga[i] = M ? at::empty_like(m.a) : at::zeros_like(m.a);
      gb[i] = M ? at::empty_like(m.b) : at::zeros_like(m.b);
      arr[i].grad_lora_a = ga[i].data_ptr();
      arr[i].grad_lora_b = gb[i].data_ptr();
    }
    Tensor gx;
    if (need_x) gx = at::empty(shape, gys[0].options());
    if (M && (need_x || need_ab)) {
      const Kept at(M, K, ranks);
      const uint8_t* k = (const uint8_t*)kept.data_ptr();
      const size_t bytes = ttamd_mx_lora_bwd_workspace_bytes(arr, n, M, K), gh = align256(bytes);  // the gradient of h behind the workspace
      const Tensor ws = scratch(gh + 2 * M * ranks, kept);
      check(ttamd_mx_lora_bwd_bf16(k, k + at.scales, k + at.h, arr, n, (uint8_t*)ws.data_ptr() + gh, ptr(gx), M, K, ws.data_ptr(), bytes, stream_of(kept)),
            "lora_linear_mx");
    }
    variable_list out = {gx};
    for (int i = 0; i < n; ++i) {
      out.push_back(ga[i]);
      out.push_back(gb[i]);
      if (bias[i]) out.push_back(need_bias[i] ? column_sum(gys[i]) : Tensor());
    }
    out.push_back(Tensor());
    return out;
  }
};

// flat: codes, scales, lora_a, lora_b and bias (or None) of each member in turn
std::vector<Tensor> mx_lora(const Tensor& x, const std::vector<double>& factors, const py::args& flat) {
  const int n = (int)factors.size();
  TORCH_CHECK_VALUE(n >= 1 && n <= TTAMD_GROUP_MAX && (int)flat.size() == 5 * n, "lora_linear_mx: takes 1 to ", TTAMD_GROUP_MAX,
                    " weights and as many adapters, scales and biases, got ", n);
  std::vector<MxMember> ms(n);
  for (int i = 0; i < n; ++i) {
    MxMember& m = ms[i];
    Tensor* to[5] = {&m.codes, &m.scales, &m.a, &m.b, &m.bias};
    for (int k = 0; k < 5; ++k)
      if (!flat[5 * i + k].is_none()) *to[k] = flat[5 * i + k].cast<Tensor>();
    m.scale = factors[i];
  }
  const py::gil_scoped_release unlocked;
  int64_t ranks = 0;
  variable_list inputs;
  bool grad = wants_grad({&x});
  for (const MxMember& m : ms) {
    const char* what = "lora_linear_mx";
    TORCH_CHECK_VALUE(m.codes.defined() && m.scales.defined() && m.a.defined() && m.b.defined(), what, ": a weight or an adapter is missing");
    check_weight(m.codes, m.scales, x, what);
    const int64_t N = m.codes.size(0), K = 2 * m.codes.size(1), r = m.a.dim() == 2 ? m.a.size(0) : 0;
    TORCH_CHECK_VALUE(r > 0 && r % 8 == 0 && m.a.size(1) == K && m.b.dim() == 2 && m.b.size(0) == N && m.b.size(1) == r, what, ": lora_a ", m.a.sizes(),
                      " and lora_b ", m.b.sizes(), " do not fit a weight of ", N, " x ", K, " with a rank that is a multiple of 8");
    TORCH_CHECK_VALUE(N > 0 && K > 0 && N % 64 == 0 && K % 64 == 0, what, ": the weight's sides must be multiples of 64, got ", N, " x ", K);
    check_bias(m.bias, N, x, what);
    for (const Tensor* t : {&m.a, &m.b}) {
      TORCH_CHECK_TYPE(t->scalar_type() == at::kBFloat16, what, ": adapters must be bfloat16, got ", t->scalar_type());
      TORCH_CHECK(t->device() == x.device(), what, ": the input is on ", x.device().str(), ", an adapter on ", t->device().str());
    }
    ranks += r;
    inputs.push_back(m.a);
    inputs.push_back(m.b);
    if (m.bias.defined()) inputs.push_back(m.bias);
    grad = grad || wants_grad({&m.a, &m.b, &m.bias});
  }
  TORCH_CHECK_VALUE(ranks <= 64, "lora_linear_mx: the members' ranks add up to ", ranks, ", at most 64 are supported");
  need_gpu(x, "lora_linear_mx");
  return grad ? LoraMXFn::apply(x, at::TensorList(inputs), ms) : lora_forward(x, ms).ys;
}

}  // namespace

void bind_mx(py::module_& m) {
  const py::call_guard<py::gil_scoped_release> unlocked;
  m.def("mx_quantize", &mx_quantize, unlocked);
  m.def("mx_dequantize", &mx_dequantize, unlocked);
  m.def("mx_linear", &mx_linear, unlocked);
  m.def("mx_lora", [](const Tensor& x, const std::vector<double>& factors, const py::args& flat) {
    const std::vector<Tensor> ys = mx_lora(x, factors, flat);
    return py::tuple(py::cast(ys));
  });
}
