// ffn_fwd_f16.hip — the gated feed-forward block's forward kernels for _Float16.
#include "ffn.hpp"

namespace msp {

template <>
void ffn_forward<_Float16>(hipStream_t s, const FfnArgs& a) {
    ffn::forward<_Float16>(s, a);
}

}  // namespace msp
