// linear_fwd_bf16_f16.hip — the linear layer's forward kernels for __bf16, the result in _Float16.
#include "linear.hpp"

namespace msp {

template <>
void linear_forward<__bf16, _Float16, false>(hipStream_t s, const LinearArgs& a) {
    linear::product<__bf16, _Float16, false, false>(s, a);
}

}  // namespace msp
