// ffn_bwd_f16.hip — the gated feed-forward block's backward kernels for _Float16.
#include "ffn.hpp"

namespace msp {

template <>
void ffn_backward<_Float16>(hipStream_t s, const FfnArgs& a) {
    ffn::backward<_Float16>(s, a);
}

}  // namespace msp
