// linear_fwd_bf16_f32.hip — the linear layer's forward kernels for __bf16, the result in float.
#include "linear.hpp"

namespace msp {

template <>
void linear_forward<__bf16, float, false>(hipStream_t s, const LinearArgs& a) {
    linear::product<__bf16, float, false, false>(s, a);
}

}  // namespace msp
