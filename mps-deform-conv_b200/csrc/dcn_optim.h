// dcn_optim.h -- launchers of the optimizer step and the gradient norm (dcn_optim.cu).
#pragma once

#include "dcn_internal.h"

namespace dcn {

// Arguments checked by the C ABI layer (dcn_abi_train.cu).
cudaError_t adamw_step(const dcn_adamw_options& o, const dcn_adamw_tensor* tensors, int64_t n, cudaStream_t st);
size_t grad_norm_workspace(const dcn_tensor_ref* tensors, int64_t n);
cudaError_t grad_norm(const dcn_tensor_ref* tensors, int64_t n, double max_norm, double loss_scale, float* norm,
                      float* factor, void* workspace, cudaStream_t st);

}  // namespace dcn
