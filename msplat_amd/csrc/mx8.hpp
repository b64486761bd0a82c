// mx8.hpp — rows of numbers in 8 bits: the OCP microscaling format MXFP8 with
// e4m3 elements.  32 adjacent columns of a row are a block with one scale, a
// power of two 2^(code - 127).  A row of dim columns takes
//
//   32 ceil(dim / 32) bytes of data, zeros from dim on, and
//   4 ceil(dim / 128) bytes of scales, one a block, zeros behind the last,
//
// row after row; both start on a 16-byte boundary.  gfx950's scaled matrix
// instructions take 32 such bytes a lane with the block's scale, and a dword of
// scales is what a row has in the 128 columns of one instruction.
//
// Packing takes the least scale with which the block's largest magnitude is at
// most 448 (so that nothing saturates), not below 2^-126, and rounds to the
// nearest element, ties to even.  Infinities and NaN become NaN.  An element
// in [1.75, 2) 2^Emax of its type would round to 2^(Emax + 1), beyond the type:
// magnitudes over 1.875 2^Emax count as that.
#pragma once

#include "nn.hpp"

#include <type_traits>

namespace msp {
namespace mx8 {

constexpr int BLOCK = 32;
template <class T>
constexpr int LANES = BLOCK / E<T>;   // lanes that hold a block, a piece each

__host__ __device__ inline int64_t data_stride(int dim) { return ((int64_t)dim + 31) / 32 * 32; }
__host__ __device__ inline int64_t scale_stride(int dim) { return ((int64_t)dim + 127) / 128 * 4; }

// 1.875 2^Emax of a type, as a float's bits.
template <class T>
constexpr uint32_t LARGEST = std::is_same<T, _Float16>::value ? 0x47700000u : 0x7F700000u;   // 61440, 1.875 2^127

// Maximum over groups of L lanes (4 or 8); all lanes of a group must be active.
template <int L>
__device__ __forceinline__ uint32_t group_max(uint32_t v) {
    auto other = [](uint32_t u, auto ctrl) {
        return (uint32_t)__builtin_amdgcn_mov_dpp((int)u, decltype(ctrl)::value, 0xF, 0xF, true);
    };
    v = max(v, other(v, std::integral_constant<int, 0xB1>{}));          // quad_perm [1,0,3,2]
    v = max(v, other(v, std::integral_constant<int, 0x4E>{}));          // quad_perm [2,3,0,1]
    if (L == 8) v = max(v, other(v, std::integral_constant<int, 0x141>{}));   // row_half_mirror
    return v;
}

__device__ __forceinline__ uint32_t magnitude(float v) { return __float_as_uint(v) & 0x7FFFFFFFu; }

// Packs the block of which each of LANES<T> adjacent lanes holds E<T> values:
// its code, and in `bytes` the lane's elements.
template <class T>
__device__ __forceinline__ int pack_block(float (&v)[E<T>], uint32_t (&bytes)[E<T> / 4]) {
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < E<T>; ++j) m = max(m, magnitude(v[j]));
    m = group_max<LANES<T>>(m);
    if (m > LARGEST<T>) {   // the same in all lanes of the block, and rare
        m = 0;
#pragma unroll
        for (int j = 0; j < E<T>; ++j) {
            if (magnitude(v[j]) >= 0x7F800000u) {
                v[j] = __uint_as_float(0x7FC00000u);
            } else {
                const float most = __uint_as_float(LARGEST<T>);
                v[j] = fminf(fmaxf(v[j], -most), most);
                m = max(m, magnitude(v[j]));
            }
        }
        m = group_max<LANES<T>>(m);
    }
    // m = 2^(exponent - 127) (1 + fraction): up to 1.75 it fits under 448 = 1.75 2^8
    const int code = max((int)(m >> 23) - 8 + ((m & 0x7FFFFFu) > 0x600000u), 1);
    const float inverse = __uint_as_float((uint32_t)(254 - code) << 23);
#pragma unroll
    for (int w = 0; w < E<T> / 4; ++w) {
        int b = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * w] * inverse, v[4 * w + 1] * inverse, 0, false);
        bytes[w] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(v[4 * w + 2] * inverse, v[4 * w + 3] * inverse, b, true);
    }
    return code;
}

// Writes a piece and, from the block's first lane, its scale; the last block's
// also the zeros behind it.  k: the piece's first column.
template <class T>
__device__ __forceinline__ void store(uint8_t* data, uint8_t* scales, int k, int dim, const uint32_t (&bytes)[E<T> / 4],
                                      int code) {
    __builtin_memcpy(data + k, bytes, E<T>);
    if (k % BLOCK != 0) return;
    const int b = k / BLOCK;
    scales[b] = (uint8_t)code;
    if (k + BLOCK >= dim)
        for (int i = b + 1; i % 4 != 0; ++i) scales[i] = 0;
}

__device__ __forceinline__ float scale_of(int code) {
    return __uint_as_float(code == 0 ? 0x00400000u : code == 255 ? 0x7FC00000u : (uint32_t)code << 23);
}

// The values of E<T> elements under a scale.
template <class T>
__device__ __forceinline__ void values(const uint32_t (&bytes)[E<T> / 4], int code, float (&v)[E<T>]) {
    const float s = scale_of(code);
#pragma unroll
    for (int w = 0; w < E<T> / 4; ++w) {
        const auto a = __builtin_amdgcn_cvt_pk_f32_fp8((int)bytes[w], false);
        const auto b = __builtin_amdgcn_cvt_pk_f32_fp8((int)bytes[w], true);
        v[4 * w] = a[0] * s;
        v[4 * w + 1] = a[1] * s;
        v[4 * w + 2] = b[0] * s;
        v[4 * w + 3] = b[1] * s;
    }
}

// The values of E<T> elements at column k of a row.
template <class T>
__device__ __forceinline__ void load(const uint8_t* data, const uint8_t* scales, int k, float (&v)[E<T>]) {
    uint32_t bytes[E<T> / 4];
    __builtin_memcpy(bytes, data + k, E<T>);
    values<T>(bytes, scales[k / BLOCK], v);
}

}  // namespace mx8
}  // namespace msp
