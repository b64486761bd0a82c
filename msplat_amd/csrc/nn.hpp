// nn.hpp — what the learned-head kernels (norm, dropout, gated feed-forward)
// share: element types, 16-byte pieces of a row, reductions over lanes.
//
// A call's tensors hold one type T (float, _Float16 or __bf16).  Kernels
// read and write rows in pieces of 16 bytes, E<T> elements; all arithmetic is
// in 32-bit floats, and a result is rounded to T once, when it is stored.
// Rows may start at any element: gfx950 reads and writes 16 bytes at any
// address, so there is one path for every alignment and stride.
#pragma once

#include "common.hpp"
#include "kernels.hpp"

namespace msp {

typedef float f32x4 __attribute__((ext_vector_type(4)));

template <class T>
constexpr int E = 16 / (int)sizeof(T);   // elements of a piece

template <class T>
struct Piece {
    typedef T type __attribute__((ext_vector_type(16 / sizeof(T))));
};
template <class T>
using piece_t = typename Piece<T>::type;

// v's elements moved down by n (0 .. E - 1, the same in every lane), zeros
// behind them.
template <class T>
__device__ __forceinline__ piece_t<T> moved_down(piece_t<T> v, int n) {
    typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
    u32x4 w;
    __builtin_memcpy(&w, &v, 16);
    const int bytes = n * (int)sizeof(T);
    if (bytes & 8) w = u32x4{w[2], w[3], 0, 0};
    if (bytes & 4) w = u32x4{w[1], w[2], w[3], 0};
    if (bytes & 2) w = u32x4{w[0] >> 16 | w[1] << 16, w[1] >> 16 | w[2] << 16, w[2] >> 16 | w[3] << 16, w[3] >> 16};
    __builtin_memcpy(&v, &w, 16);
    return v;
}

// Elements k .. k + E - 1 of a row of n >= E (k a multiple of E), zero from n
// on, in two steps so that a read may be under way while something else runs.
// The last piece of a row that E does not divide is read so that it ends with
// the row, and moved down: one read for every piece.
template <class T>
__device__ __forceinline__ piece_t<T> read_piece(const T* row, int k, int n) {
    piece_t<T> v;
    __builtin_memcpy(&v, row + min(k, n - E<T>), 16);
    return v;
}
template <class T>
__device__ __forceinline__ piece_t<T> settle_piece(piece_t<T> v, int k, int n, bool live) {
    if (n % E<T> != 0 && k > n - E<T>) v = moved_down<T>(v, E<T> - n % E<T>);
    if (k >= n || !live) v = piece_t<T>{};
    return v;
}

// The same in one step, for rows of any length.
template <class T>
__device__ __forceinline__ piece_t<T> load_piece(const T* row, int k, int n) {
    if (n >= E<T>) return settle_piece<T>(read_piece(row, k, n), k, n, true);
    piece_t<T> v = {};
#pragma unroll
    for (int j = 0; j < E<T>; ++j)
        if (k + j < n) v[j] = row[k + j];
    return v;
}

template <class T>
__device__ __forceinline__ void store_piece(T* row, int k, int n, piece_t<T> v) {
    if (k + E<T> <= n) {
        __builtin_memcpy(row + k, &v, 16);
    } else {
#pragma unroll
        for (int j = 0; j < E<T>; ++j)
            if (k + j < n) row[k + j] = v[j];
    }
}

// Sum over groups of L consecutive lanes (a power of two up to 64); every
// lane of a group gets the same bits.  All 64 lanes must be active.  After a
// step the lanes that it joined agree, so the mirrors of the steps 4 and 8
// pair the same groups as an exclusive or would.
template <int L>
__device__ __forceinline__ float group_sum(float v) {
    if (L >= 2) v += dpp<0xB1>(v);     // quad_perm [1,0,3,2]
    if (L >= 4) v += dpp<0x4E>(v);     // quad_perm [2,3,0,1]
    if (L >= 8) v += dpp<0x141>(v);    // row_half_mirror
    if (L >= 16) v += dpp<0x140>(v);   // row_mirror
    if (L >= 32) {
        const auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = __uint_as_float(s[0]) + __uint_as_float(s[1]);
    }
    if (L >= 64) {
        const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = __uint_as_float(s[0]) + __uint_as_float(s[1]);
    }
    return v;
}

// Calls f with a value of the element type that dtype (MSPLAT_F32 = 0,
// MSPLAT_F16 = 1, MSPLAT_BF16 = 2) names.
template <class F>
inline void with_type(int dtype, F&& f) {
    if (dtype == 0) f(float{});
    else if (dtype == 1) f(_Float16{});
    else f(__bf16{});
}

}  // namespace msp
