// linear_fwd_mx8_f16.hip — the linear layer's forward kernels for 8-bit operands, the result in _Float16.
#include "linear.hpp"

namespace msp {

template <>
void linear_forward<__bf16, _Float16, true>(hipStream_t s, const LinearArgs& a) {
    linear::product<__bf16, _Float16, true, false>(s, a);
}

}  // namespace msp
