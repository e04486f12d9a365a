// dcn_ffn.h -- the gated feed-forward block: problem, workspace layouts and
// launchers (dcn_ffn.cu).
#pragma once

#include "dcn_internal.h"

namespace dcn {

struct FfnProblem {
  int dtype, act;
  int64_t M, C, F;  // rows, channels, hidden width
};

struct FfnTensors {
  const void *x, *w_gate, *w_up, *w_down, *b_gate, *b_up, *b_down;
};
struct FfnGrads {
  void *x, *w_gate, *w_up, *w_down, *b_gate, *b_up, *b_down;
};

size_t ffn_forward_workspace(const FfnProblem& p, bool save);
size_t ffn_saved_bytes(const FfnProblem& p);
size_t ffn_backward_workspace(const FfnProblem& p);
// saved: null for a forward that keeps nothing.
cudaError_t ffn_forward(const FfnProblem& p, const FfnTensors& t, void* y, void* saved, void* workspace,
                        cudaStream_t st);
// Gradient pointers may be null.  ready(user), when given, is called once the
// parameter gradients are enqueued.
cudaError_t ffn_backward(const FfnProblem& p, const FfnTensors& t, const void* dy, const void* saved,
                         const FfnGrads& g, void* workspace, cudaStream_t st, dcn_params_ready_fn ready, void* user);

}  // namespace dcn
