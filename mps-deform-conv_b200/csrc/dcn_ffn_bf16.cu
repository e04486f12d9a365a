// dcn_ffn_bf16.cu -- the gated feed-forward block on bf16 data.
#include "dcn_ffn_impl.cuh"

namespace dcn {
DCN_FFN_INSTANTIATE(__nv_bfloat16, bf16)
}  // namespace dcn
