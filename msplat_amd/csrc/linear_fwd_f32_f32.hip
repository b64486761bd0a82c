// linear_fwd_f32_f32.hip — the linear layer's forward kernels for float, the result in float.
#include "linear.hpp"

namespace msp {

template <>
void linear_forward<float, float, false>(hipStream_t s, const LinearArgs& a) {
    linear::product<float, float, false, false>(s, a);
}

}  // namespace msp
