// linear_fwd_f32_f16.hip — the linear layer's forward kernels for float, the result in _Float16.
#include "linear.hpp"

namespace msp {

template <>
void linear_forward<float, _Float16, false>(hipStream_t s, const LinearArgs& a) {
    linear::product<float, _Float16, false, false>(s, a);
}

}  // namespace msp
