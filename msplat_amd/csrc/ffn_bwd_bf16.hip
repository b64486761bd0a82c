// ffn_bwd_bf16.hip — the gated feed-forward block's backward kernels for __bf16.
#include "ffn.hpp"

namespace msp {

template <>
void ffn_backward<__bf16>(hipStream_t s, const FfnArgs& a) {
    ffn::backward<__bf16>(s, a);
}

}  // namespace msp
