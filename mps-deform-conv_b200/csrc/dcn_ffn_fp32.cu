// dcn_ffn_fp32.cu -- the gated feed-forward block on fp32 data.
#include "dcn_ffn_impl.cuh"

namespace dcn {
DCN_FFN_INSTANTIATE(float, fp32)
}  // namespace dcn
