// linear_fwd_f16_f16.hip — the linear layer's forward kernels for _Float16, the result in _Float16.
#include "linear.hpp"

namespace msp {

template <>
void linear_forward<_Float16, _Float16, false>(hipStream_t s, const LinearArgs& a) {
    linear::product<_Float16, _Float16, false, false>(s, a);
}

}  // namespace msp
