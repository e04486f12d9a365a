// dcn_abi_train.cu -- the extern "C" entry points of the training-block
// operators of include/dcn_b200.h: argument checks and dispatch.
#include <float.h>
#include <math.h>

#include <algorithm>
#include <new>
#include <utility>
#include <vector>

#include "dcn_ffn.h"
#include "dcn_optim.h"

namespace dcn {

static bool dtype_ok(int32_t d) { return d == DCN_FLOAT32 || d == DCN_FLOAT16 || d == DCN_BFLOAT16; }
static int64_t elem_bytes(int32_t d) { return d == DCN_FLOAT32 ? 4 : 2; }

// No C++ exception leaves a C entry: the host-side tables are std::vectors.
template <typename F>
static int guarded(F&& f) {
  try {
    return f();
  } catch (const std::bad_alloc&) {
    return fail(DCN_ERR_CUDA, "out of host memory");
  } catch (...) {
    return fail(DCN_ERR_CUDA, "unexpected host error");
  }
}

// A kernel reads and writes whole elements: elsewhere it would fault.
static bool on(const void* p, int64_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (uintptr_t)(bytes - 1)) == 0; }

constexpr int64_t kMaxNumel = int64_t(1) << 40;  // keeps every chunk count and byte offset in range

static int check_adamw(const dcn_adamw_options* o, const dcn_adamw_tensor* t, int64_t n) {
  if (!o) return fail(DCN_ERR_INVALID_ARGUMENT, "options are NULL");
  if (n < 0 || (n > 0 && !t)) return fail(DCN_ERR_INVALID_ARGUMENT, "tensor list is NULL or its length negative");
  if (o->state_bits != 32 && o->state_bits != 8)
    return fail(DCN_ERR_UNSUPPORTED, "state_bits must be 32 or 8, got %d", o->state_bits);
  if (!o->lr_device && !(o->lr >= 0.0 && isfinite(o->lr)))
    return fail(DCN_ERR_INVALID_ARGUMENT, "lr must be non-negative and finite, got %g", o->lr);
  if (!(o->beta1 >= 0.0 && o->beta1 < 1.0) || !(o->beta2 >= 0.0 && o->beta2 < 1.0))
    return fail(DCN_ERR_INVALID_ARGUMENT, "betas must be in [0, 1), got (%g, %g)", o->beta1, o->beta2);
  if (!(o->eps >= 0.0 && isfinite(o->eps)))
    return fail(DCN_ERR_INVALID_ARGUMENT, "eps must be non-negative and finite, got %g", o->eps);
  // the kernel's reciprocal takes a subnormal for 0: 0 / eps would be NaN
  if (o->eps > 0.0 && !((float)o->eps >= FLT_MIN))
    return fail(DCN_ERR_INVALID_ARGUMENT, "eps must be 0 or at least 2^-126, got %g", o->eps);
  if (!(o->weight_decay >= 0.0 && isfinite(o->weight_decay)))
    return fail(DCN_ERR_INVALID_ARGUMENT, "weight_decay must be non-negative and finite, got %g", o->weight_decay);
  std::vector<std::pair<uintptr_t, uintptr_t>> written;
  written.reserve((size_t)n * 4);
  for (int64_t i = 0; i < n; ++i) {
    const dcn_adamw_tensor& e = t[i];
    if (!dtype_ok(e.dtype))
      return fail(DCN_ERR_UNSUPPORTED, "tensor %lld: dtype %d is not one of float32, float16, bfloat16", (long long)i,
                  e.dtype);
    if (e.numel < 0 || e.numel > kMaxNumel)
      return fail(DCN_ERR_UNSUPPORTED, "tensor %lld: %lld elements", (long long)i, (long long)e.numel);
    if (!e.step) return fail(DCN_ERR_INVALID_ARGUMENT, "tensor %lld: step counter is NULL", (long long)i);
    if (e.numel == 0) continue;
    if (!e.param || !e.grad || !e.exp_avg || !e.exp_avg_sq)
      return fail(DCN_ERR_INVALID_ARGUMENT, "tensor %lld: NULL pointer (param, grad, exp_avg, exp_avg_sq)", (long long)i);
    if (o->state_bits == 8 && (!e.exp_avg_scale || !e.exp_avg_sq_scale))
      return fail(DCN_ERR_INVALID_ARGUMENT, "tensor %lld: 8-bit states need exp_avg_scale and exp_avg_sq_scale",
                  (long long)i);
    const int64_t state = o->state_bits == 8 ? 1 : 4;
    auto add = [&](const void* p, int64_t bytes) {
      if (p) written.emplace_back((uintptr_t)p, (uintptr_t)p + (uintptr_t)bytes);
    };
    add(e.param, e.numel * elem_bytes(e.dtype));
    add(e.master, e.numel * 4);
    add(e.exp_avg, e.numel * state);
    add(e.exp_avg_sq, e.numel * state);
    if (o->state_bits == 8) {
      add(e.exp_avg_scale, (e.numel + 255) / 256 * 4);
      add(e.exp_avg_sq_scale, (e.numel + 255) / 256 * 4);
    }
  }
  // two CTAs must not update the same memory, nor one read what another updates
  std::sort(written.begin(), written.end());
  for (size_t i = 1; i < written.size(); ++i)
    if (written[i].first < written[i - 1].second)
      return fail(DCN_ERR_INVALID_ARGUMENT,
                  "parameters, master copies and states must not overlap one another (the same tensor twice?)");
  auto meets = [&](const void* p, int64_t bytes) {
    const uintptr_t a = (uintptr_t)p;
    // the first range that starts at or past the end; the one before it reaches furthest
    auto it = std::lower_bound(written.begin(), written.end(), std::make_pair(a + (uintptr_t)bytes, uintptr_t(0)));
    return p && it != written.begin() && (it - 1)->second > a;
  };
  std::vector<uintptr_t> counters;
  counters.reserve((size_t)n);
  for (int64_t i = 0; i < n; ++i) {
    const char* what = t[i].numel && meets(t[i].grad, t[i].numel * elem_bytes(t[i].dtype)) ? "grad"
                       : meets(t[i].step, 8)                                               ? "step"
                                                                                           : nullptr;
    if (what)
      return fail(DCN_ERR_INVALID_ARGUMENT, "tensor %lld: %s must not overlap a parameter, master copy or state",
                  (long long)i, what);
    counters.push_back((uintptr_t)t[i].step);
  }
  std::sort(counters.begin(), counters.end());
  counters.erase(std::unique(counters.begin(), counters.end()), counters.end());
  for (size_t i = 1; i < counters.size(); ++i)
    if (counters[i] - counters[i - 1] < 8)
      return fail(DCN_ERR_INVALID_ARGUMENT, "step counters must be the same or not overlap");
  auto meets_any = [&](const float* p) {
    const uintptr_t a = (uintptr_t)p;
    auto it = std::lower_bound(counters.begin(), counters.end(), a + 4);
    return p && (meets(p, 4) || (it != counters.begin() && *(it - 1) + 8 > a));
  };
  const char* scalar = meets_any(o->grad_scale) ? "grad_scale" : meets_any(o->lr_device) ? "lr_device" : nullptr;
  if (scalar)
    return fail(DCN_ERR_INVALID_ARGUMENT, "%s must not overlap a parameter, master copy, state or step counter", scalar);
  for (int64_t i = 0; i < n; ++i) {
    const dcn_adamw_tensor& e = t[i];
    const int64_t es = elem_bytes(e.dtype), state = o->state_bits == 8 ? 1 : 4;
    const bool scales = o->state_bits != 8 || (on(e.exp_avg_scale, 4) && on(e.exp_avg_sq_scale, 4));
    if (!on(e.step, 4) || (e.numel && !(on(e.param, es) && on(e.grad, es) && on(e.exp_avg, state) &&
                                        on(e.exp_avg_sq, state) && on(e.master, 4) && scales)))
      return fail(DCN_ERR_INVALID_ARGUMENT, "tensor %lld: a pointer is not aligned to its elements", (long long)i);
  }
  if (!on(o->grad_scale, 4) || !on(o->lr_device, 4))
    return fail(DCN_ERR_INVALID_ARGUMENT, "grad_scale or lr_device is not aligned to 4 bytes");
  return DCN_OK;
}

static int check_refs(const dcn_tensor_ref* t, int64_t n) {
  if (n < 0 || (n > 0 && !t)) return fail(DCN_ERR_INVALID_ARGUMENT, "tensor list is NULL or its length negative");
  for (int64_t i = 0; i < n; ++i) {
    if (!dtype_ok(t[i].dtype))
      return fail(DCN_ERR_UNSUPPORTED, "tensor %lld: dtype %d is not one of float32, float16, bfloat16", (long long)i,
                  t[i].dtype);
    if (t[i].numel < 0 || t[i].numel > kMaxNumel)
      return fail(DCN_ERR_UNSUPPORTED, "tensor %lld: %lld elements", (long long)i, (long long)t[i].numel);
  }
  return DCN_OK;
}

static int check_ffn(const dcn_ffn_desc* d) {
  if (!d) return fail(DCN_ERR_INVALID_ARGUMENT, "descriptor is NULL");
  if (!dtype_ok(d->dtype))
    return fail(DCN_ERR_UNSUPPORTED, "dtype %d is not one of float32, float16, bfloat16", d->dtype);
  if (d->activation < DCN_ACT_SILU || d->activation > DCN_ACT_SIGMOID)
    return fail(DCN_ERR_INVALID_ARGUMENT, "unknown activation %d", d->activation);
  if (d->tokens < 0 || d->channels <= 0 || d->hidden <= 0)
    return fail(DCN_ERR_INVALID_ARGUMENT,
                "sizes must be positive (tokens may be 0): tokens=%lld channels=%lld hidden=%lld", (long long)d->tokens,
                (long long)d->channels, (long long)d->hidden);
  // tensor-map extents, tile indices and byte strides stay in range
  const int64_t lim = int64_t(1) << 20;
  if (d->channels > lim || d->hidden > lim)
    return fail(DCN_ERR_UNSUPPORTED, "channels (%lld) and hidden (%lld) may be at most %lld", (long long)d->channels,
                (long long)d->hidden, (long long)lim);
  const int64_t wide = d->channels > d->hidden ? d->channels : d->hidden;
  if (d->tokens > (int64_t(1) << 30) || d->tokens > (int64_t(1) << 38) / wide)
    return fail(DCN_ERR_UNSUPPORTED, "tokens (%lld) x %lld exceeds the size limit", (long long)d->tokens, (long long)wide);
  return DCN_OK;
}

static FfnProblem problem(const dcn_ffn_desc* d) {
  return {d->dtype, d->activation, d->tokens, d->channels, d->hidden};
}

static bool on16(const void* p) { return on(p, 16); }

static int check_ffn_tensors(const dcn_ffn_tensors* t, int64_t es) {
  if (!t || !t->x || !t->w_gate || !t->w_up || !t->w_down)
    return fail(DCN_ERR_INVALID_ARGUMENT, "NULL tensor pointer (x, w_gate, w_up, w_down)");
  if ((t->b_gate != nullptr) != (t->b_up != nullptr))
    return fail(DCN_ERR_INVALID_ARGUMENT, "b_gate and b_up go together");
  if (!on16(t->x) || !on16(t->w_gate) || !on16(t->w_up) || !on16(t->w_down))
    return fail(DCN_ERR_INVALID_ARGUMENT, "x and the weights must be 16-byte aligned");
  if (!on(t->b_gate, es) || !on(t->b_up, es) || !on(t->b_down, es))
    return fail(DCN_ERR_INVALID_ARGUMENT, "a bias is not aligned to its elements");
  return DCN_OK;
}

static int check_buffer(const void* p, size_t have, size_t need, const char* what) {
  if (need == 0) return DCN_OK;
  if (!p || have < need) return fail(DCN_ERR_WORKSPACE, "%s too small: need %zu bytes, got %zu", what, need, p ? have : 0);
  if (reinterpret_cast<uintptr_t>(p) & 255) return fail(DCN_ERR_INVALID_ARGUMENT, "%s must be 256-byte aligned", what);
  return DCN_OK;
}

}  // namespace dcn

using namespace dcn;

extern "C" {

int dcn_adamw_step(const dcn_adamw_options* opt, const dcn_adamw_tensor* tensors, int64_t n, void* stream) {
  return guarded([&] {
    const int r = check_adamw(opt, tensors, n);
    if (r != DCN_OK) return r;
    const cudaError_t e = adamw_step(*opt, tensors, n, (cudaStream_t)stream);
    return e == cudaSuccess ? ok() : cuda_fail(e, "adamw_step");
  });
}

size_t dcn_grad_norm_workspace_size(const dcn_tensor_ref* grads, int64_t n) {
  size_t bytes = 0;
  guarded([&] {
    const int r = check_refs(grads, n);
    if (r == DCN_OK) bytes = grad_norm_workspace(grads, n);
    return r;
  });
  return bytes;
}

int dcn_grad_norm(const dcn_tensor_ref* grads, int64_t n, double max_norm, double loss_scale, float* norm,
                  float* factor, void* workspace, size_t workspace_bytes, void* stream) {
  return guarded([&] {
    int r = check_refs(grads, n);
    if (r != DCN_OK) return r;
    if (!(loss_scale > 0.0 && isfinite(loss_scale)))
      return fail(DCN_ERR_INVALID_ARGUMENT, "loss_scale must be positive and finite, got %g", loss_scale);
    if (isnan(max_norm)) return fail(DCN_ERR_INVALID_ARGUMENT, "max_norm is NaN");
    if (!norm || !factor) return fail(DCN_ERR_INVALID_ARGUMENT, "NULL output (norm, factor)");
    if (!on(norm, 4) || !on(factor, 4)) return fail(DCN_ERR_INVALID_ARGUMENT, "norm or factor is not aligned to 4 bytes");
    for (int64_t i = 0; i < n; ++i) {
      if (grads[i].numel && !grads[i].data)
        return fail(DCN_ERR_INVALID_ARGUMENT, "tensor %lld: NULL pointer", (long long)i);
      if (grads[i].numel && !on(grads[i].data, elem_bytes(grads[i].dtype)))
        return fail(DCN_ERR_INVALID_ARGUMENT, "tensor %lld: the pointer is not aligned to its elements", (long long)i);
    }
    if ((r = check_buffer(workspace, workspace_bytes, grad_norm_workspace(grads, n), "grad_norm workspace")) != DCN_OK) return r;
    const cudaError_t e = grad_norm(grads, n, max_norm, loss_scale, norm, factor, workspace, (cudaStream_t)stream);
    return e == cudaSuccess ? ok() : cuda_fail(e, "grad_norm");
  });
}

int dcn_ffn_validate(const dcn_ffn_desc* desc) {
  const int r = check_ffn(desc);
  return r == DCN_OK ? ok() : r;
}

size_t dcn_ffn_saved_bytes(const dcn_ffn_desc* desc) {
  return check_ffn(desc) == DCN_OK && desc->tokens ? ffn_saved_bytes(problem(desc)) : 0;
}

size_t dcn_ffn_forward_workspace_size(const dcn_ffn_desc* desc, int save) {
  return check_ffn(desc) == DCN_OK && desc->tokens ? ffn_forward_workspace(problem(desc), save != 0) : 0;
}

size_t dcn_ffn_backward_workspace_size(const dcn_ffn_desc* desc) {
  return check_ffn(desc) == DCN_OK && desc->tokens ? ffn_backward_workspace(problem(desc)) : 0;
}

int dcn_ffn_forward(const dcn_ffn_desc* desc, const dcn_ffn_tensors* t, void* y, void* saved, size_t saved_bytes,
                    void* workspace, size_t workspace_bytes, void* stream) {
  return guarded([&] {
    int r = check_ffn(desc);
    if (r != DCN_OK) return r;
    if (desc->tokens == 0) return ok();
    if ((r = check_ffn_tensors(t, elem_bytes(desc->dtype))) != DCN_OK) return r;
    if (!y && !saved) return fail(DCN_ERR_INVALID_ARGUMENT, "y and saved are both NULL");
    if (y && !on16(y)) return fail(DCN_ERR_INVALID_ARGUMENT, "y must be 16-byte aligned");
    const FfnProblem p = problem(desc);
    if (saved && (r = check_buffer(saved, saved_bytes, ffn_saved_bytes(p), "saved state")) != DCN_OK) return r;
    if ((r = check_buffer(workspace, workspace_bytes, ffn_forward_workspace(p, saved != nullptr), "forward workspace")) != DCN_OK)
      return r;
    const FfnTensors in{t->x, t->w_gate, t->w_up, t->w_down, t->b_gate, t->b_up, t->b_down};
    const cudaError_t e = ffn_forward(p, in, y, saved, workspace, (cudaStream_t)stream);
    return e == cudaSuccess ? ok() : cuda_fail(e, "ffn_forward");
  });
}

int dcn_ffn_backward(const dcn_ffn_desc* desc, const dcn_ffn_tensors* t, const void* grad_y, const void* saved,
                     size_t saved_bytes, const dcn_ffn_grads* grads, void* workspace, size_t workspace_bytes,
                     void* stream, void (*params_ready)(void* user_data), void* user_data) {
  return guarded([&] {
    int r = check_ffn(desc);
    if (r != DCN_OK) return r;
    if (!grads) return fail(DCN_ERR_INVALID_ARGUMENT, "grads is NULL");
    const FfnGrads g{grads->x, grads->w_gate, grads->w_up, grads->w_down, grads->b_gate, grads->b_up, grads->b_down};
    if (!on16(g.x) || !on16(g.w_gate) || !on16(g.w_up) || !on16(g.w_down))
      return fail(DCN_ERR_INVALID_ARGUMENT, "gradients of x and of the weights must be 16-byte aligned");
    const int64_t size = elem_bytes(desc->dtype);
    if (!on(g.b_gate, size) || !on(g.b_up, size) || !on(g.b_down, size))
      return fail(DCN_ERR_INVALID_ARGUMENT, "a bias gradient is not aligned to its elements");
    cudaStream_t st = (cudaStream_t)stream;
    if (desc->tokens == 0) {  // sums over no rows
      const size_t es = (size_t)size, c = (size_t)desc->channels, f = (size_t)desc->hidden;
      const std::pair<void*, size_t> zero[6] = {{g.w_gate, c * f}, {g.w_up, c * f}, {g.w_down, c * f},
                                                {g.b_gate, f},     {g.b_up, f},     {g.b_down, c}};
      for (auto& z : zero)
        if (z.first) {
          const cudaError_t e = cudaMemsetAsync(z.first, 0, z.second * es, st);
          if (e != cudaSuccess) return cuda_fail(e, "ffn_backward");
        }
      if (params_ready) params_ready(user_data);
      return ok();
    }
    if ((r = check_ffn_tensors(t, elem_bytes(desc->dtype))) != DCN_OK) return r;
    if (!grad_y || !on16(grad_y))
      return fail(DCN_ERR_INVALID_ARGUMENT, "grad_y is NULL or not 16-byte aligned");
    const FfnProblem p = problem(desc);
    if ((r = check_buffer(saved, saved_bytes, ffn_saved_bytes(p), "saved state")) != DCN_OK) return r;
    if ((r = check_buffer(workspace, workspace_bytes, ffn_backward_workspace(p), "backward workspace")) != DCN_OK) return r;
    const FfnTensors in{t->x, t->w_gate, t->w_up, t->w_down, t->b_gate, t->b_up, t->b_down};
    const cudaError_t e = ffn_backward(p, in, grad_y, saved, g, workspace, st, params_ready, user_data);
    return e == cudaSuccess ? ok() : cuda_fail(e, "ffn_backward");
  });
}

}  // extern "C"
