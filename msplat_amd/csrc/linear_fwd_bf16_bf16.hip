// linear_fwd_bf16_bf16.hip — the linear layer's forward kernels for __bf16, the result in __bf16.
#include "linear.hpp"

namespace msp {

template <>
void linear_forward<__bf16, __bf16, false>(hipStream_t s, const LinearArgs& a) {
    linear::product<__bf16, __bf16, false, false>(s, a);
}

}  // namespace msp
