// dcn_ffn.cu -- entry of the gated feed-forward block: buffer sizes, and the
// pass of the data type at hand (dcn_ffn_impl.cuh).
#include "dcn_ffn_layout.h"

namespace dcn {

#define DCN_FFN_DECLARE(name)                                                                                 \
  cudaError_t ffn_forward_##name(const FfnProblem&, const FfnTensors&, void*, void*, void*, cudaStream_t);    \
  cudaError_t ffn_backward_##name(const FfnProblem&, const FfnTensors&, const void*, const void*,             \
                                  const FfnGrads&, void*, cudaStream_t, dcn_params_ready_fn, void*);
DCN_FFN_DECLARE(bf16)
DCN_FFN_DECLARE(fp16)
DCN_FFN_DECLARE(fp32)

size_t ffn_forward_workspace(const FfnProblem& p, bool save) {
  // any non-null pointer stands for hidden values that live in the saved state
  int there = 0;
  return ffn::ForwardWs(p, FfnTensors{}, nullptr, save ? &there : nullptr).total;
}
size_t ffn_saved_bytes(const FfnProblem& p) {
  const ffn::Shape s(p);
  return s.blocks_bytes() + s.panels_bytes();
}
size_t ffn_backward_workspace(const FfnProblem& p) {
  return ffn::BackwardWs(p, FfnTensors{}, nullptr, nullptr).total;
}

cudaError_t ffn_forward(const FfnProblem& p, const FfnTensors& t, void* y, void* saved, void* workspace,
                        cudaStream_t st) {
  if (p.dtype == DCN_FLOAT32) return ffn_forward_fp32(p, t, y, saved, workspace, st);
  if (p.dtype == DCN_FLOAT16) return ffn_forward_fp16(p, t, y, saved, workspace, st);
  return ffn_forward_bf16(p, t, y, saved, workspace, st);
}

cudaError_t ffn_backward(const FfnProblem& p, const FfnTensors& t, const void* dy, const void* saved,
                         const FfnGrads& g, void* workspace, cudaStream_t st, dcn_params_ready_fn ready, void* user) {
  if (p.dtype == DCN_FLOAT32) return ffn_backward_fp32(p, t, dy, saved, g, workspace, st, ready, user);
  if (p.dtype == DCN_FLOAT16) return ffn_backward_fp16(p, t, dy, saved, g, workspace, st, ready, user);
  return ffn_backward_bf16(p, t, dy, saved, g, workspace, st, ready, user);
}

}  // namespace dcn
