// linear_fwd_mx8_f32.hip — the linear layer's forward kernels for 8-bit operands, the result in float.
#include "linear.hpp"

namespace msp {

template <>
void linear_forward<__bf16, float, true>(hipStream_t s, const LinearArgs& a) {
    linear::product<__bf16, float, true, false>(s, a);
}

}  // namespace msp
