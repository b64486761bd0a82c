// ffn_fwd_bf16.hip — the gated feed-forward block's forward kernels for __bf16.
#include "ffn.hpp"

namespace msp {

template <>
void ffn_forward<__bf16>(hipStream_t s, const FfnArgs& a) {
    ffn::forward<__bf16>(s, a);
}

}  // namespace msp
