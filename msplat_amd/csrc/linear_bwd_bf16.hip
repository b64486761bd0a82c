// linear_bwd_bf16.hip — the linear layer's backward kernels for __bf16.
#include "linear.hpp"

namespace msp {

template <>
void linear_backward<__bf16>(hipStream_t s, const LinearGradArgs& a) {
    linear::backward<__bf16>(s, a);
}

}  // namespace msp
