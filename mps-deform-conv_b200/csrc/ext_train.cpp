// ext_train.cpp -- the training-block operators of the Python module
// `mps_deform_conv._C`: tensors to pointers and shapes over the C ABI.
#include <exception>
#include <optional>
#include <tuple>
#include <vector>

#include "ext_common.h"

namespace {

using Tensors = std::vector<at::Tensor>;

// The two tensors' elements lie in the same order in memory.
bool same_order(const at::Tensor& a, const at::Tensor& b) {
  return (a.is_contiguous() && b.is_contiguous()) || a.strides() == b.strides();
}

// A kernel wrote the tensor: autograd and the weight image cache go by its version.
void written(const at::Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

void check_count(const Tensors& t, size_t n, const char* name) {
  TORCH_CHECK(t.size() == n, name, " has ", t.size(), " tensors, params has ", n);
}

void check_on(const at::Tensor& t, const char* name, size_t i, const at::Device& dev) {
  TORCH_CHECK(t.is_cuda(), name, "[", i, "] must be a CUDA tensor");
  TORCH_CHECK(t.device() == dev, name, "[", i, "] must be on ", dev, " as the first tensor, got ", t.device());
}

// A state, scale or master tensor of params[i].
void check_state(const at::Tensor& t, const char* name, size_t i, const at::Tensor& p, at::ScalarType type) {
  check_on(t, name, i, p.device());
  TORCH_CHECK(t.scalar_type() == type, name, "[", i, "] must be ", type, ", got ", t.scalar_type());
  TORCH_CHECK(t.sizes() == p.sizes() && same_order(t, p), name, "[", i,
              "] must have the shape and memory format of params[", i, "] ", p.sizes(), ", got ", t.sizes());
}

const float* scalar_ptr(const std::optional<at::Tensor>& t, const char* name, const at::Device& dev) {
  if (!t.has_value() || !t->defined()) return nullptr;
  TORCH_CHECK(t->is_cuda() && t->device() == dev && t->scalar_type() == at::kFloat && t->numel() == 1, name,
              " must be one float32 element on ", dev);
  return t->const_data_ptr<float>();
}

}  // namespace

// ---------------------------------------------------------------- gated feed-forward block
namespace {

// A dense copy-free view where the tensor allows it, else a dense copy; 16-byte aligned.
at::Tensor dense16(const at::Tensor& t) {
  at::Tensor r = t.contiguous();
  if ((reinterpret_cast<uintptr_t>(r.data_ptr()) & 15) != 0) r = r.clone(at::MemoryFormat::Contiguous);
  return r;
}

using OptTensor = std::optional<at::Tensor>;

struct FfnArgs {
  dcn_ffn_desc d;
  at::Tensor x, w_gate, w_up, w_down, b_gate, b_up, b_down;  // dense; biases may be undefined
  dcn_ffn_tensors t;
  FfnArgs(const at::Tensor& input, const at::Tensor& wg, const at::Tensor& wu, const at::Tensor& wd,
          const OptTensor& bg, const OptTensor& bu, const OptTensor& bd, int64_t activation) {
    TORCH_CHECK_VALUE(input.is_cuda(), "Input must be on CUDA device, got ", input.device());
    TORCH_CHECK_VALUE(input.dim() >= 1, "input must have a channel dimension");
    const int64_t c = input.size(-1);
    auto placed = [&](const at::Tensor& t, const char* name) {
      TORCH_CHECK_VALUE(t.device() == input.device(), name, " must be on same device as input (", input.device(),
                        "), got ", t.device());
      check_cuda(t, name, input);
    };
    placed(wg, "w_gate");
    placed(wu, "w_up");
    placed(wd, "w_down");
    TORCH_CHECK_VALUE(wg.dim() == 2 && wg.size(1) == c, "w_gate must have shape (hidden, ", c, "), got ", wg.sizes());
    const int64_t f = wg.size(0);
    TORCH_CHECK_VALUE(wu.sizes() == wg.sizes(), "w_up must have shape ", wg.sizes(), " as w_gate, got ", wu.sizes());
    TORCH_CHECK_VALUE(wd.dim() == 2 && wd.size(0) == c && wd.size(1) == f, "w_down must have shape (", c, ", ", f,
                      "), got ", wd.sizes());
    TORCH_CHECK_VALUE(c > 0 && f > 0, "channels and hidden must be positive, got ", c, " and ", f);
    TORCH_CHECK_VALUE(bg.has_value() == bu.has_value(), "b_gate and b_up go together");
    d.dtype = dtype_code(input, "gated_feed_forward");
    d.activation = (int32_t)activation;
    d.channels = c;
    d.hidden = f;
    d.tokens = c > 0 ? input.numel() / c : 0;
    check_status(dcn_ffn_validate(&d));
    x = dense16(input);
    w_gate = dense16(wg);
    w_up = dense16(wu);
    w_down = dense16(wd);
    auto bias = [&](const OptTensor& b, const char* name, int64_t n) {
      if (!b.has_value()) return at::Tensor();
      placed(*b, name);
      TORCH_CHECK_VALUE(b->dim() == 1 && b->size(0) == n, name, " must have shape (", n, ",), got ", b->sizes());
      return b->contiguous();
    };
    b_gate = bias(bg, "b_gate", f);
    b_up = bias(bu, "b_up", f);
    b_down = bias(bd, "b_down", c);
    auto p = [](const at::Tensor& v) -> const void* { return v.defined() ? v.data_ptr() : nullptr; };
    t = {p(x), p(w_gate), p(w_up), p(w_down), p(b_gate), p(b_up), p(b_down)};
  }
};

}  // namespace

// (output, saved state); the state is empty unless keep_saved, the output when !want_output.
std::tuple<at::Tensor, at::Tensor> gated_feed_forward_forward(const at::Tensor& input, const at::Tensor& w_gate,
                                                              const at::Tensor& w_up, const at::Tensor& w_down,
                                                              const OptTensor& b_gate, const OptTensor& b_up,
                                                              const OptTensor& b_down, int64_t activation,
                                                              bool keep_saved, bool want_output) {
  TORCH_CHECK(input.is_cuda(), "input must be a CUDA tensor");
  c10::cuda::CUDAGuard guard(input.device());
  const FfnArgs a(input, w_gate, w_up, w_down, b_gate, b_up, b_down, activation);
  at::Tensor out = want_output ? at::empty_like(a.x) : at::empty({0}, input.options());
  const size_t sbytes = keep_saved ? dcn_ffn_saved_bytes(&a.d) : 0;
  auto saved = at::empty({(int64_t)sbytes}, input.options().dtype(at::kByte));
  auto ws = workspace(dcn_ffn_forward_workspace_size(&a.d, sbytes != 0), input);
  check_status(dcn_ffn_forward(&a.d, &a.t, want_output ? out.data_ptr() : nullptr, sbytes ? saved.data_ptr() : nullptr,
                               sbytes, ws.data_ptr(), (size_t)ws.numel(), stream_of(input)));
  return {out, saved};
}

// Gradients of (input, w_gate, w_up, w_down, b_gate, b_up, b_down) by output_mask;
// the others are undefined.  params_ready(grad_weight, grad_bias), when given, is
// called for each of the three weights once they are enqueued.
std::vector<at::Tensor> gated_feed_forward_backward(const at::Tensor& grad_output, const at::Tensor& input,
                                                    const at::Tensor& w_gate, const at::Tensor& w_up,
                                                    const at::Tensor& w_down, const OptTensor& b_gate,
                                                    const OptTensor& b_up, const OptTensor& b_down, int64_t activation,
                                                    const at::Tensor& saved, std::vector<bool> output_mask,
                                                    const std::optional<py::function>& params_ready) {
  TORCH_CHECK(input.is_cuda(), "input must be a CUDA tensor");
  c10::cuda::CUDAGuard guard(input.device());
  check_cuda(grad_output, "grad_output", input);
  TORCH_CHECK(grad_output.sizes() == input.sizes(), "grad_output must have shape ", input.sizes(), ", got ",
              grad_output.sizes());
  TORCH_CHECK(output_mask.size() == 7, "output_mask must have 7 entries");
  const FfnArgs a(input, w_gate, w_up, w_down, b_gate, b_up, b_down, activation);
  if (a.d.tokens > 0)
    TORCH_CHECK(saved.is_cuda() && saved.device() == input.device() && saved.scalar_type() == at::kByte &&
                    saved.is_contiguous(),
                "saved state must be a contiguous uint8 tensor on the input's device");
  const at::Tensor dy = dense16(grad_output);
  const at::Tensor like[7] = {a.x, a.w_gate, a.w_up, a.w_down, a.b_gate, a.b_up, a.b_down};
  std::vector<at::Tensor> g(7);
  void* ptr[7];
  for (int i = 0; i < 7; ++i) {
    if (output_mask[i] && like[i].defined()) g[i] = at::empty_like(like[i], at::MemoryFormat::Contiguous);
    ptr[i] = g[i].defined() ? g[i].data_ptr() : nullptr;
  }
  const dcn_ffn_grads grads{ptr[0], ptr[1], ptr[2], ptr[3], ptr[4], ptr[5], ptr[6]};
  auto ws = workspace(dcn_ffn_backward_workspace_size(&a.d), input);
  // a Python exception of the hook is held and re-raised after the call, never thrown through the C ABI
  struct Ready {
    const py::function* fn;
    const std::vector<at::Tensor>* g;
    std::exception_ptr err;
  } ready{nullptr, &g, nullptr};
  const bool hook = params_ready.has_value() && !params_ready->is_none();
  if (hook) ready.fn = &*params_ready;
  auto tramp = [](void* u) {
    auto* r = static_cast<Ready*>(u);
    try {
      auto cast = [](const at::Tensor& t) -> py::object { return t.defined() ? py::cast(t) : py::none(); };
      for (int i = 1; i <= 3; ++i) {
        const at::Tensor &w = (*r->g)[i], &b = (*r->g)[i + 3];
        if (w.defined() || b.defined()) (*r->fn)(cast(w), cast(b));
      }
    } catch (...) {
      r->err = std::current_exception();
    }
  };
  const int rc = dcn_ffn_backward(&a.d, &a.t, dy.data_ptr(), a.d.tokens ? saved.data_ptr() : nullptr,
                                  (size_t)saved.numel(), &grads, ws.data_ptr(), (size_t)ws.numel(), stream_of(input),
                                  hook ? +tramp : nullptr, hook ? &ready : nullptr);
  if (ready.err) std::rethrow_exception(ready.err);
  check_status(rc);
  return g;
}

void adamw_step(const Tensors& params, const Tensors& grads, const Tensors& exp_avgs, const Tensors& exp_avg_sqs,
                const Tensors& steps, const std::optional<Tensors>& masters,
                const std::optional<Tensors>& exp_avg_scales, const std::optional<Tensors>& exp_avg_sq_scales,
                double lr, const std::optional<at::Tensor>& lr_tensor, double beta1, double beta2, double eps,
                double weight_decay, const std::optional<at::Tensor>& grad_scale, int64_t seed) {
  const size_t n = params.size();
  check_count(grads, n, "grads");
  check_count(exp_avgs, n, "exp_avgs");
  check_count(exp_avg_sqs, n, "exp_avg_sqs");
  check_count(steps, n, "steps");
  if (masters) check_count(*masters, n, "masters");
  TORCH_CHECK(exp_avg_scales.has_value() == exp_avg_sq_scales.has_value(),
              "exp_avg_scales and exp_avg_sq_scales go together");
  const bool bits8 = exp_avg_scales.has_value();
  if (bits8) {
    check_count(*exp_avg_scales, n, "exp_avg_scales");
    check_count(*exp_avg_sq_scales, n, "exp_avg_sq_scales");
  }
  if (n == 0) return;
  const at::Device dev = params[0].device();
  TORCH_CHECK(dev.is_cuda(), "params[0] must be a CUDA tensor");
  c10::cuda::CUDAGuard guard(dev);
  dcn_adamw_options o{};
  o.lr = lr; o.beta1 = beta1; o.beta2 = beta2; o.eps = eps; o.weight_decay = weight_decay;
  o.lr_device = scalar_ptr(lr_tensor, "lr", dev);
  o.grad_scale = scalar_ptr(grad_scale, "grad_scale", dev);
  o.state_bits = bits8 ? 8 : 32;
  o.seed = (uint32_t)seed;
  const at::ScalarType state = bits8 ? at::kFloat8_e4m3fn : at::kFloat;
  std::vector<dcn_adamw_tensor> e(n);
  Tensors relaid;  // gradients whose memory format differs from their parameter's
  for (size_t i = 0; i < n; ++i) {
    const at::Tensor& p = params[i];
    at::Tensor g = grads[i];
    check_on(p, "params", i, dev);
    TORCH_CHECK(p.is_non_overlapping_and_dense(), "params[", i, "] must be dense in memory (no gaps, no overlaps)");
    check_on(g, "grads", i, dev);
    TORCH_CHECK(g.layout() == at::kStrided && g.scalar_type() == p.scalar_type() && g.sizes() == p.sizes(), "grads[", i,
                "] must be a strided ", p.scalar_type(), " tensor of shape ", p.sizes(), " as its parameter, got ",
                g.scalar_type(), " ", g.sizes());
    check_state(exp_avgs[i], "exp_avgs", i, p, state);
    check_state(exp_avg_sqs[i], "exp_avg_sqs", i, p, state);
    const at::Tensor& s = steps[i];
    check_on(s, "steps", i, dev);
    TORCH_CHECK(s.scalar_type() == at::kInt && s.numel() == 2 && s.is_contiguous(), "steps[", i,
                "] must hold two int32: the steps taken and a ticket (0)");
    if (!same_order(g, p)) {
      relaid.push_back(at::empty_strided(p.sizes(), p.strides(), p.options()).copy_(g));
      g = relaid.back();
    }
    dcn_adamw_tensor& t = e[i];
    t.param = p.data_ptr();
    t.grad = g.data_ptr();
    t.exp_avg = exp_avgs[i].data_ptr();
    t.exp_avg_sq = exp_avg_sqs[i].data_ptr();
    t.exp_avg_scale = t.exp_avg_sq_scale = nullptr;
    if (bits8) {
      const int64_t blocks = (p.numel() + 255) / 256;
      for (const Tensors* l : {&*exp_avg_scales, &*exp_avg_sq_scales}) {
        const at::Tensor& c = (*l)[i];
        check_on(c, "scales", i, dev);
        TORCH_CHECK(c.scalar_type() == at::kFloat && c.numel() == blocks && c.is_contiguous(), "scales[", i,
                    "] must hold one float32 per 256 elements (", blocks, "), got ", c.numel());
      }
      t.exp_avg_scale = (*exp_avg_scales)[i].data_ptr<float>();
      t.exp_avg_sq_scale = (*exp_avg_sq_scales)[i].data_ptr<float>();
    }
    t.master = nullptr;
    if (masters) {
      check_state((*masters)[i], "masters", i, p, at::kFloat);
      t.master = (*masters)[i].data_ptr<float>();
    }
    t.step = s.data_ptr<int32_t>();
    t.numel = p.numel();
    t.dtype = dtype_code(p, "adamw_step");
    t.reserved = 0;
  }
  check_status(dcn_adamw_step(&o, e.data(), (int64_t)n, stream_of(params[0])));
  for (size_t i = 0; i < n; ++i) {
    written(params[i]);
    written(exp_avgs[i]);
    written(exp_avg_sqs[i]);
    written(steps[i]);
    if (masters) written((*masters)[i]);
    if (bits8) {
      written((*exp_avg_scales)[i]);
      written((*exp_avg_sq_scales)[i]);
    }
  }
}

// (norm, factor), two 0-d float32 tensors; max_norm < 0 clips nothing.
std::tuple<at::Tensor, at::Tensor> grad_norm(const Tensors& grads, double max_norm, double loss_scale) {
  TORCH_CHECK(!grads.empty(), "grads is empty");
  const at::Device dev = grads[0].device();
  TORCH_CHECK(dev.is_cuda(), "grads[0] must be a CUDA tensor");
  c10::cuda::CUDAGuard guard(dev);
  std::vector<dcn_tensor_ref> refs(grads.size());
  Tensors dense;  // copies of gradients with gaps or overlaps
  for (size_t i = 0; i < grads.size(); ++i) {
    at::Tensor g = grads[i];
    check_on(g, "grads", i, dev);
    TORCH_CHECK(g.layout() == at::kStrided, "grads[", i, "] must be a strided tensor");
    if (!g.is_non_overlapping_and_dense()) {
      dense.push_back(g.contiguous());
      g = dense.back();
    }
    refs[i] = {g.data_ptr(), g.numel(), dtype_code(g, "grad_norm"), 0};
  }
  auto opt = grads[0].options().dtype(at::kFloat);
  auto out = at::empty({2}, opt);
  auto ws = workspace(dcn_grad_norm_workspace_size(refs.data(), (int64_t)refs.size()), grads[0]);
  check_status(dcn_grad_norm(refs.data(), (int64_t)refs.size(), max_norm, loss_scale, out.data_ptr<float>(),
                             out.data_ptr<float>() + 1, ws.data_ptr(), (size_t)ws.numel(), stream_of(grads[0])));
  return {out[0], out[1]};
}

void bind_train(py::module_& m) {
  m.def("gated_feed_forward_forward", &gated_feed_forward_forward, "Gated feed-forward block: (output, saved)",
        py::arg("input"), py::arg("w_gate"), py::arg("w_up"), py::arg("w_down"), py::arg("b_gate"), py::arg("b_up"),
        py::arg("b_down"), py::arg("activation"), py::arg("keep_saved") = false, py::arg("want_output") = true);
  m.def("gated_feed_forward_backward", &gated_feed_forward_backward,
        "Gradients of (input, w_gate, w_up, w_down, b_gate, b_up, b_down)", py::arg("grad_output"), py::arg("input"),
        py::arg("w_gate"), py::arg("w_up"), py::arg("w_down"), py::arg("b_gate"), py::arg("b_up"), py::arg("b_down"),
        py::arg("activation"), py::arg("saved"), py::arg("output_mask"), py::arg("params_ready") = py::none());
  m.def("adamw_step", &adamw_step, "AdamW step over many tensors, in place", py::arg("params"), py::arg("grads"),
        py::arg("exp_avgs"), py::arg("exp_avg_sqs"), py::arg("steps"), py::arg("masters"), py::arg("exp_avg_scales"),
        py::arg("exp_avg_sq_scales"), py::arg("lr"), py::arg("lr_tensor"), py::arg("beta1"), py::arg("beta2"),
        py::arg("eps"), py::arg("weight_decay"), py::arg("grad_scale"), py::arg("seed"));
  m.def("grad_norm", &grad_norm, "Global gradient norm and clipping factor: (norm, factor)", py::arg("grads"),
        py::arg("max_norm"), py::arg("loss_scale"));
}
