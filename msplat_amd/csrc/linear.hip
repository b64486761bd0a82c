// linear.hip — the linear layer's launches by operand type.
#include "linear.hpp"

namespace msp {

template <>
void linear_forward<float, float, false>(hipStream_t, const LinearArgs&);
template <>
void linear_forward<float, _Float16, false>(hipStream_t, const LinearArgs&);
template <>
void linear_forward<float, __bf16, false>(hipStream_t, const LinearArgs&);
template <>
void linear_forward<_Float16, float, false>(hipStream_t, const LinearArgs&);
template <>
void linear_forward<_Float16, _Float16, false>(hipStream_t, const LinearArgs&);
template <>
void linear_forward<_Float16, __bf16, false>(hipStream_t, const LinearArgs&);
template <>
void linear_forward<__bf16, float, false>(hipStream_t, const LinearArgs&);
template <>
void linear_forward<__bf16, _Float16, false>(hipStream_t, const LinearArgs&);
template <>
void linear_forward<__bf16, __bf16, false>(hipStream_t, const LinearArgs&);
template <>
void linear_forward<__bf16, float, true>(hipStream_t, const LinearArgs&);
template <>
void linear_forward<__bf16, _Float16, true>(hipStream_t, const LinearArgs&);
template <>
void linear_forward<__bf16, __bf16, true>(hipStream_t, const LinearArgs&);
template <>
void linear_backward<float>(hipStream_t, const LinearGradArgs&);
template <>
void linear_backward<_Float16>(hipStream_t, const LinearGradArgs&);
template <>
void linear_backward<__bf16>(hipStream_t, const LinearGradArgs&);

void launch_linear_fwd(hipStream_t s, int dtype, const LinearArgs& a) {
    with_type(a.y_dtype, [&](auto y) {
        if (a.x_scales) return linear_forward<__bf16, decltype(y), true>(s, a);
        with_type(dtype, [&](auto t) { linear_forward<decltype(t), decltype(y), false>(s, a); });
    });
}

size_t linear_workspace(int dtype, int64_t rows, int inner, int outer) {
    size_t n = 0;
    with_type(dtype, [&](auto t) { n = (size_t)linear::product_workspace<decltype(t)>(rows, inner, outer); });
    return n;
}

size_t linear_grad_workspace(int dtype, int y_dtype, int64_t rows, int inner, int outer, int act) {
    size_t n = 0;
    with_type(dtype, [&](auto t) {
        n = (size_t)linear::plan<decltype(t)>(rows, inner, outer, act, y_dtype == dtype).bytes();
    });
    return n;
}

void launch_linear_bwd(hipStream_t s, const LinearGradArgs& a) {
    with_type(a.dtype, [&](auto t) { linear_backward<decltype(t)>(s, a); });
}

}  // namespace msp
