// linear_fwd_mx8_bf16.hip — the linear layer's forward kernels for 8-bit operands, the result in __bf16.
#include "linear.hpp"

namespace msp {

template <>
void linear_forward<__bf16, __bf16, true>(hipStream_t s, const LinearArgs& a) {
    linear::product<__bf16, __bf16, true, false>(s, a);
}

}  // namespace msp
