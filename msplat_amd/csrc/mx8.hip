// mx8.hip — rows packed into 8 bits and back (mx8.hpp has the format).
//
// Bound by HBM: a thread has a 16-byte piece of a row, 4 (16-bit types) or 8
// lanes a block, whose largest magnitude goes round them by lane swaps.
//   1.09M rows of 64 bf16: packed in 43 us, 4.9 TB/s, unpacked in 32, 6.6 TB/s
//   120k rows of 45 f32 (180 bytes, off the 16-byte grid): 11.4 and 9.5 us
#include "mx8.hpp"

#include <algorithm>

namespace msp {
namespace {

constexpr int THREADS = 256;

// tx threads along a row (a power of two, at least a block's), 256 / tx rows a
// workgroup at once.
template <class T>
__global__ __launch_bounds__(THREADS) void k_mx8_pack(Mx8Args a, int tx) {
    const int lane = threadIdx.x & (tx - 1), sub = threadIdx.x / tx, rb = THREADS / tx;
    const int64_t ds = mx8::data_stride(a.dim), ss = mx8::scale_stride(a.dim);
    for (int64_t row = (int64_t)blockIdx.x * rb + sub; row < a.rows; row += (int64_t)gridDim.x * rb)
        for (int64_t k = lane * E<T>; k < ds; k += tx * E<T>) {
            const piece_t<T> p = k < a.dim ? load_piece(static_cast<const T*>(a.x) + row * a.x_stride, (int)k, a.dim)
                                           : piece_t<T>{};
            float v[E<T>];
#pragma unroll
            for (int j = 0; j < E<T>; ++j) v[j] = (float)p[j];
            uint32_t bytes[E<T> / 4];
            const int code = mx8::pack_block<T>(v, bytes);
            mx8::store<T>(a.data + row * ds, a.scales + row * ss, (int)k, a.dim, bytes, code);
        }
}

template <class T>
__global__ __launch_bounds__(THREADS) void k_mx8_unpack(Mx8Args a, int tx) {
    const int lane = threadIdx.x & (tx - 1), sub = threadIdx.x / tx, rb = THREADS / tx;
    const int64_t ds = mx8::data_stride(a.dim), ss = mx8::scale_stride(a.dim);
    for (int64_t row = (int64_t)blockIdx.x * rb + sub; row < a.rows; row += (int64_t)gridDim.x * rb)
        for (int64_t k = lane * E<T>; k < a.dim; k += tx * E<T>) {
            float v[E<T>];
            mx8::load<T>(a.data + row * ds, a.scales + row * ss, (int)k, v);
            piece_t<T> o;
#pragma unroll
            for (int j = 0; j < E<T>; ++j) o[j] = (T)v[j];
            store_piece(static_cast<T*>(a.y) + row * a.y_stride, (int)k, a.dim, o);
        }
}

// Threads along a row, and workgroups.
template <class T>
int along(int dim) {
    const int64_t pieces = mx8::data_stride(dim) / E<T>;
    int tx = mx8::LANES<T>;
    while (tx < pieces && tx < THREADS) tx *= 2;
    return tx;
}
int groups(int64_t rows, int tx) { return (int)std::min<int64_t>((rows + THREADS / tx - 1) / (THREADS / tx), 8192); }

}  // namespace

void launch_mx8_pack(hipStream_t s, int dtype, const Mx8Args& a) {
    with_type(dtype, [&](auto t) {
        const int tx = along<decltype(t)>(a.dim);
        k_mx8_pack<decltype(t)><<<groups(a.rows, tx), THREADS, 0, s>>>(a, tx);
    });
}

void launch_mx8_unpack(hipStream_t s, int dtype, const Mx8Args& a) {
    with_type(dtype, [&](auto t) {
        const int tx = along<decltype(t)>(a.dim);
        k_mx8_unpack<decltype(t)><<<groups(a.rows, tx), THREADS, 0, s>>>(a, tx);
    });
}

}  // namespace msp
