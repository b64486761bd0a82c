// linear_bwd_f32.hip — the linear layer's backward kernels for float.
#include "linear.hpp"

namespace msp {

template <>
void linear_backward<float>(hipStream_t s, const LinearGradArgs& a) {
    linear::backward<float>(s, a);
}

}  // namespace msp
