// ffn_fwd_f32.hip — the gated feed-forward block's forward kernels for float.
#include "ffn.hpp"

namespace msp {

template <>
void ffn_forward<float>(hipStream_t s, const FfnArgs& a) {
    ffn::forward<float>(s, a);
}

}  // namespace msp
