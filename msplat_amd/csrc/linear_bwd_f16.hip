// linear_bwd_f16.hip — the linear layer's backward kernels for _Float16.
#include "linear.hpp"

namespace msp {

template <>
void linear_backward<_Float16>(hipStream_t s, const LinearGradArgs& a) {
    linear::backward<_Float16>(s, a);
}

}  // namespace msp
