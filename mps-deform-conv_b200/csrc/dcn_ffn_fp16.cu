// dcn_ffn_fp16.cu -- the gated feed-forward block on fp16 data.
#include "dcn_ffn_impl.cuh"

namespace dcn {
DCN_FFN_INSTANTIATE(__half, fp16)
}  // namespace dcn
