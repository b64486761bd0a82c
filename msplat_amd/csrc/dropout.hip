// dropout.hip — dropout added to a residual, with a mask that is never stored.
//
//   y = residual + (keep ? x / (1 - p) : 0)
//
// The mask is a function of (seed, offset, row, column): a word of Philox 4x32
// with seven rounds (Salmon, Moraes, Dror and Shaw, "Parallel random numbers:
// as easy as 1, 2, 3", SC 2011; seven is the smallest count that passes their
// test batteries), key = seed, counter = (column / 4, row, offset), word
// column % 4, kept where it is at least p 2^32.  The backward makes the same
// words again.  A dropped element counts as zero whatever it holds.
//
// Bound by HBM: 14 32x32-bit products make four words, which fits behind the 24
// bytes (16-bit types: 1.09M rows of 64 f16 with a residual 74 us, 5.6 TB/s; a
// large copy 5.1); ten rounds cost 2.5% more, 80.1 against 78.1 us a call.  A thread
// has a 16-byte piece of a row.
#include "nn.hpp"

#include <algorithm>

namespace msp {
namespace {

constexpr int THREADS = 256;

struct Words {
    uint32_t w[4];
};

__device__ __forceinline__ Words philox(uint32_t c0, uint32_t c1, uint32_t c2, uint32_t c3, uint32_t k0, uint32_t k1) {
#pragma unroll
    for (int r = 0; r < 7; ++r) {
        const uint64_t a = (uint64_t)c0 * 0xD2511F53u, b = (uint64_t)c2 * 0xCD9E8D57u;
        c0 = (uint32_t)(b >> 32) ^ c1 ^ k0;
        c2 = (uint32_t)(a >> 32) ^ c3 ^ k1;
        c1 = (uint32_t)b;
        c3 = (uint32_t)a;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return {{c0, c1, c2, c3}};
}

// tx threads along a row (a power of two), 256 / tx rows a workgroup at once.
template <class T, bool RES>
__global__ __launch_bounds__(THREADS) void k_dropout(DropArgs a, int tx) {
    const int lane = threadIdx.x & (tx - 1), sub = threadIdx.x / tx, rb = THREADS / tx;
    const T* x = static_cast<const T*>(a.x);
    const T* res = static_cast<const T*>(a.residual);
    T* out = static_cast<T*>(a.out);
    const uint64_t offset = a.offset_at ? *a.offset_at : a.offset;
    for (int64_t row = (int64_t)blockIdx.x * rb + sub; row < a.rows; row += (int64_t)gridDim.x * rb)
        // at runs to dim + THREADS * E - 1, which passes 2^31 at the largest widths
        for (uint32_t at = lane * E<T>; at < (uint32_t)a.dim; at += tx * E<T>) {
            const int k = (int)at;
            const piece_t<T> v = load_piece(x + row * a.x_stride, k, a.dim);
            piece_t<T> r = {};
            if (RES) r = load_piece(res + row * a.residual_stride, k, a.dim);
            piece_t<T> o;
#pragma unroll
            for (int q = 0; q < E<T> / 4; ++q) {
                const Words w = philox((uint32_t)(k / 4 + q), (uint32_t)row, (uint32_t)offset, (uint32_t)(offset >> 32),
                                       (uint32_t)a.seed, (uint32_t)(a.seed >> 32));
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float t = w.w[j] >= a.threshold ? (float)v[4 * q + j] * a.scale : 0.f;
                    o[4 * q + j] = (T)(RES ? (float)r[4 * q + j] + t : t);
                }
            }
            store_piece(out + row * a.out_stride, k, a.dim, o);
        }
}

}  // namespace

void launch_dropout(hipStream_t s, int dtype, const DropArgs& a) {
    with_type(dtype, [&](auto t) {
        using T = decltype(t);
        const int pieces = (a.dim + E<T> - 1) / E<T>;
        int tx = 1;
        while (tx < pieces && tx < THREADS) tx *= 2;
        const int64_t rb = THREADS / tx;
        const int grid = (int)std::min<int64_t>((a.rows + rb - 1) / rb, 8192);
        if (a.residual) k_dropout<T, true><<<grid, THREADS, 0, s>>>(a, tx);
        else k_dropout<T, false><<<grid, THREADS, 0, s>>>(a, tx);
    });
}

}  // namespace msp
