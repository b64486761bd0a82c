// ffn.hip — the gated feed-forward block's launches by element type.
#include "ffn.hpp"

namespace msp {

template <>
void ffn_forward<float>(hipStream_t, const FfnArgs&);
template <>
void ffn_forward<_Float16>(hipStream_t, const FfnArgs&);
template <>
void ffn_forward<__bf16>(hipStream_t, const FfnArgs&);
template <>
void ffn_backward<float>(hipStream_t, const FfnArgs&);
template <>
void ffn_backward<_Float16>(hipStream_t, const FfnArgs&);
template <>
void ffn_backward<__bf16>(hipStream_t, const FfnArgs&);

size_t ffn_workspace(int dtype, int64_t rows, int dim, int hidden, bool backward) {
    size_t n = 0;
    with_type(dtype, [&](auto t) { n = ffn::workspace<decltype(t)>(rows, dim, hidden, backward); });
    return n;
}

void launch_ffn_fwd(hipStream_t s, int dtype, const FfnArgs& a) {
    with_type(dtype, [&](auto t) { ffn_forward<decltype(t)>(s, a); });
}

void launch_ffn_bwd(hipStream_t s, int dtype, const FfnArgs& a) {
    with_type(dtype, [&](auto t) { ffn_backward<decltype(t)>(s, a); });
}

}  // namespace msp
