// ext_train.cpp -- the training-block operators of the Python module
// `mps_deform_conv._C`: tensors to pointers and shapes over the C ABI.
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
    t.dtype = dtype_code(p);
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
    refs[i] = {g.data_ptr(), g.numel(), dtype_code(g), 0};
  }
  auto opt = grads[0].options().dtype(at::kFloat);
  auto out = at::empty({2}, opt);
  auto ws = workspace(dcn_grad_norm_workspace_size(refs.data(), (int64_t)refs.size()), grads[0]);
  check_status(dcn_grad_norm(refs.data(), (int64_t)refs.size(), max_norm, loss_scale, out.data_ptr<float>(),
                             out.data_ptr<float>() + 1, ws.data_ptr(), (size_t)ws.numel(), stream_of(grads[0])));
  return {out[0], out[1]};
}

void bind_train(py::module_& m) {
  m.def("adamw_step", &adamw_step, "AdamW step over many tensors, in place", py::arg("params"), py::arg("grads"),
        py::arg("exp_avgs"), py::arg("exp_avg_sqs"), py::arg("steps"), py::arg("masters"), py::arg("exp_avg_scales"),
        py::arg("exp_avg_sq_scales"), py::arg("lr"), py::arg("lr_tensor"), py::arg("beta1"), py::arg("beta2"),
        py::arg("eps"), py::arg("weight_decay"), py::arg("grad_scale"), py::arg("seed"));
  m.def("grad_norm", &grad_norm, "Global gradient norm and clipping factor: (norm, factor)", py::arg("grads"),
        py::arg("max_norm"), py::arg("loss_scale"));
}
