// rows.hpp — rows that lanes or a workgroup hold in registers while they are
// summed over, as layer norm and the root-mean-square norm do.
//
// L lanes share a row, NV pieces of 16 bytes each: the fewest lanes that hold
// the row (so a wave takes 64 / L rows at once), a whole wave from 64 pieces on
// and a workgroup of 256 beyond 256 pieces.
#pragma once

#include "nn.hpp"

#include <algorithm>
#include <type_traits>

namespace msp {
namespace rows {

constexpr int THREADS = 256;

// Sum over the L threads of a row: lanes of a wave, or the whole workgroup
// (L == THREADS; then every thread of the workgroup must call it).
template <int L>
__device__ __forceinline__ float row_sum(float v, float* red) {
    if (L <= 64) return group_sum<L <= 64 ? L : 64>(v);
    v = group_sum<64>(v);
    __syncthreads();   // the previous sum has been read
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    return (red[0] + red[1]) + (red[2] + red[3]);
}

// A row's pieces, read ahead while the row before is computed, then settled
// (read_piece, settle_piece).  Only rows that the fewest lanes (MIN) hold may
// be less than a piece.
template <class T, int L, int NV, int MIN, class A>
__device__ __forceinline__ void read_row(const void* base, int64_t stride, int64_t row, const A& a, int lane,
                                         piece_t<T> (&p)[NV]) {
    const T* at = static_cast<const T*>(base) + min(row, a.rows - 1) * stride;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int k = (i * L + lane) * E<T>;
        p[i] = L == MIN && a.dim < E<T> ? load_piece(at, k, a.dim) : read_piece(at, k, a.dim);
    }
}
template <class T, int L, int NV, int MIN, class A>
__device__ __forceinline__ void settle_row(int64_t row, const A& a, int lane, piece_t<T> (&p)[NV]) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int k = (i * L + lane) * E<T>;
        if (L == MIN && a.dim < E<T>) p[i] = row < a.rows ? p[i] : piece_t<T>{};
        else p[i] = settle_piece<T>(p[i], k, a.dim, row < a.rows);
    }
}

// Rows of at least AHEAD_PIECES are read ahead.  With fewer, a wave has several
// rows under way at once and the occupancy is worth more: backward over 900k
// rows of 60 bf16 76 us without, 81 us with; over 40k rows of 1500 215 and 81.
constexpr int AHEAD_PIECES = 64;

// Calls f with (L, NV) as integral constants for a row of `dim`, L at least MIN.
template <class T, int MIN, class F>
void with_shape(int dim, F&& f) {
    const int c = std::max(MIN, (dim + E<T> - 1) / E<T>);
#define SHAPE(l, nv)                                                                                    \
    do {                                                                                                \
        if constexpr (l >= MIN) f(std::integral_constant<int, l>{}, std::integral_constant<int, nv>{}); \
    } while (0)
    if (c <= 1) SHAPE(1, 1);
    else if (c <= 2) SHAPE(2, 1);
    else if (c <= 4) SHAPE(4, 1);
    else if (c <= 8) SHAPE(8, 1);
    else if (c <= 16) SHAPE(16, 1);
    else if (c <= 32) SHAPE(32, 1);
    else if (c <= 64) SHAPE(64, 1);
    else if (c <= 128) SHAPE(64, 2);
    else if (c <= 256) SHAPE(64, 4);
    else if (c <= 512) SHAPE(256, 2);
    else if (c <= 1024) SHAPE(256, 4);
    else if constexpr (sizeof(T) == 4) SHAPE(256, 8);
#undef SHAPE
}

inline int grid_for(int64_t rows, int rows_per_group, int most) {
    const int64_t g = (rows + rows_per_group - 1) / rows_per_group;
    return (int)std::min<int64_t>(g, most);
}

}  // namespace rows
}  // namespace msp
