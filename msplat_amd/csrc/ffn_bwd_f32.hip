// ffn_bwd_f32.hip — the gated feed-forward block's backward kernels for float.
#include "ffn.hpp"

namespace msp {

template <>
void ffn_backward<float>(hipStream_t s, const FfnArgs& a) {
    ffn::backward<float>(s, a);
}

}  // namespace msp
