// linear_fwd_f16_f32.hip — the linear layer's forward kernels for _Float16, the result in float.
#include "linear.hpp"

namespace msp {

template <>
void linear_forward<_Float16, float, false>(hipStream_t s, const LinearArgs& a) {
    linear::product<_Float16, float, false, false>(s, a);
}

}  // namespace msp
