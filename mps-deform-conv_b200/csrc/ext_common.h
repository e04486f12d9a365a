// ext_common.h -- what the files of the Python module `mps_deform_conv._C` share.
#pragma once

#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include <algorithm>

#include "dcn_b200.h"

inline int32_t dtype_code(const at::Tensor& t, const char* op) {
  switch (t.scalar_type()) {
    case at::kFloat: return DCN_FLOAT32;
    case at::kHalf: return DCN_FLOAT16;
    case at::kBFloat16: return DCN_BFLOAT16;
    default:
      TORCH_CHECK(false, op, ": unsupported dtype ", t.scalar_type(),
                  " (expected float32, float16 or bfloat16)");
  }
  return 0;
}

inline void check_cuda(const at::Tensor& t, const char* name, const at::Tensor& ref) {
  TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor");
  TORCH_CHECK(t.device() == ref.device(), name, " must be on the same device as input (",
              ref.device(), "), got ", t.device());
  TORCH_CHECK(t.scalar_type() == ref.scalar_type(), name, " must have the same dtype as input (",
              ref.scalar_type(), "), got ", t.scalar_type());
}

inline void check_status(int rc) {
  TORCH_CHECK(rc == DCN_OK, dcn_last_error());
}

inline at::Tensor workspace(size_t bytes, const at::Tensor& like) {
  return at::empty({(int64_t)std::max<size_t>(bytes, 1)}, like.options().dtype(at::kByte));
}

inline void* stream_of(const at::Tensor& t) {
  return (void*)at::cuda::getCurrentCUDAStream(t.device().index()).stream();
}

// Adds the training-block operators (ext_train.cpp) to the module.
void bind_train(py::module_& m);
