// linear_fwd_f16_bf16.hip — the linear layer's forward kernels for _Float16, the result in __bf16.
#include "linear.hpp"

namespace msp {

template <>
void linear_forward<_Float16, __bf16, false>(hipStream_t s, const LinearArgs& a) {
    linear::product<_Float16, __bf16, false, false>(s, a);
}

}  // namespace msp
