// linear_fwd_f32_bf16.hip — the linear layer's forward kernels for float, the result in __bf16.
#include "linear.hpp"

namespace msp {

template <>
void linear_forward<float, __bf16, false>(hipStream_t s, const LinearArgs& a) {
    linear::product<float, __bf16, false, false>(s, a);
}

}  // namespace msp
