// linear.hpp — the linear layer, forward and backward:
//
//   z = x W^T + b    y = residual + a(z)    a: identity, SiLU, GELU (tanh form)
//   dz = dy a'(z)    dx = dz W    dW = dz^T x    db = sum over rows of dz
//
// Products run on 16x16 matrix instructions with 32-bit sums, fragments as
// ffn.hpp lays them out: lane (q, r) has elements q E .. q E + E - 1 of row r in
// a block of KB indices.  A wave takes 32 columns of the result (outputs) as two
// tiles, tile s with
//
//   column(s, r) = (r / 4) 8 + 4 s + r % 4
//
// as its row r, so that the result leaves in each lane eight adjacent columns of
// one row: a 16-byte piece or two to add bias and residual to and to store.
//
// x and W in mx8 become bfloat16 fragments, which hold e4m3 times a power of two
// exactly (down to 2^-126; smaller counts as 0).  gfx950's scaled instruction,
// which takes 8 bits as they are, drops bits of small products: a sum of 128 was
// up to 1.5e-4 of its terms' magnitudes off, where 32-bit sums stay within 6e-8.
// The layer is bound by memory at the widths it is used at, so that the rate of
// twice as many operations would not show.
#pragma once

#include "ffn.hpp"
#include "mx8.hpp"

namespace msp {
namespace linear {

using ffn::ceil_div;
using ffn::KB;
using ffn::mma;

constexpr int COLS = 32;   // columns of a wave's step

// What is multiplied: the matrices' own type, bfloat16 for mx8.
template <class T, bool MX>
struct Operand {
    typedef T type;
};
template <class T>
struct Operand<T, true> {
    typedef __bf16 type;
};

__device__ __forceinline__ int column(int s, int r) { return (r >> 2) * 8 + 4 * s + (r & 3); }

// Eight values of mx8 as bfloat16: the conversion multiplies by the scale (a float)
// in one instruction a pair.
__device__ __forceinline__ piece_t<__bf16> from_mx8(const uint32_t (&bytes)[2], int code) {
    const float s = mx8::scale_of(code);
    piece_t<__bf16> o;
#pragma unroll
    for (int w = 0; w < 2; ++w) {
        const auto a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)bytes[w], s, false);
        const auto b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)bytes[w], s, true);
        __builtin_memcpy((char*)&o + 8 * w, &a, 4);
        __builtin_memcpy((char*)&o + 8 * w + 4, &b, 4);
    }
    return o;
}

// The piece of lane group q in block kb of a row of x, as it is read and as the
// products take it.  The last piece of a row that E does not divide is read so that it
// ends with the row, and so are pieces behind it: W has zeros in the place of
// what was there before (w_piece), so that x needs no mask.
template <class T, bool MX>
struct XPiece {
    piece_t<T> v;
    template <bool TINY>   // whether a row may be less than a piece
    __device__ __forceinline__ void read(const LinearArgs& a, int64_t row, int kb, int q) {
        const T* at = static_cast<const T*>(a.x) + row * a.x_stride;
        v = TINY && a.inner < E<T> ? load_piece(at, kb * KB<T> + q * E<T>, a.inner)
                                   : read_piece(at, kb * KB<T> + q * E<T>, a.inner);
    }
    __device__ __forceinline__ piece_t<T> taken() const { return v; }
};
template <class T>
struct XPiece<T, true> {
    uint32_t bytes[2];
    int code;
    template <bool TINY>
    __device__ __forceinline__ void read(const LinearArgs& a, int64_t row, int kb, int q) {
        const int64_t ds = mx8::data_stride(a.inner);
        kb = min(kb, (int)(ds / 32) - 1);
        __builtin_memcpy(bytes, static_cast<const uint8_t*>(a.x) + row * ds + kb * 32 + q * 8, 8);
        code = a.x_scales[row * mx8::scale_stride(a.inner) + kb];
    }
    __device__ __forceinline__ piece_t<__bf16> taken() const { return from_mx8(bytes, code); }
};

// The piece of a row of W that meets it, W^T where TRANS, zero beyond the matrix.
// ENDS: the last piece ends with the row, as x is read.
template <class T, bool MX, bool TRANS, bool ENDS = true>
__device__ __forceinline__ piece_t<typename Operand<T, MX>::type> w_piece(const LinearArgs& a, int row, int kb, int q) {
    using C = typename Operand<T, MX>::type;
    const int at = min(row, a.outer - 1);
    piece_t<C> v;
    if constexpr (MX) {
        if (kb * 32 >= a.inner) return piece_t<C>{};
        uint32_t bytes[2];
        __builtin_memcpy(bytes, static_cast<const uint8_t*>(a.w) + at * mx8::data_stride(a.inner) + kb * 32 + q * 8, 8);
        v = from_mx8(bytes, a.w_scales[at * mx8::scale_stride(a.inner) + kb]);
    } else {
        const int k = kb * KB<T> + q * E<T>, from = ENDS ? max(min(k, a.inner - E<T>), 0) : k;
        if constexpr (TRANS) {
            const T* w = static_cast<const T*>(a.w) + at;
#pragma unroll
            for (int j = 0; j < E<T>; ++j) v[j] = w[min(from + j, a.inner - 1) * a.w_stride];
        } else {
            v = load_piece(static_cast<const T*>(a.w) + at * a.w_stride, from, a.inner);
        }
#pragma unroll
        for (int j = 0; j < E<T>; ++j)
            if (from + j < k || from + j >= a.inner) v[j] = (T)0.f;
    }
    return row < a.outer ? v : piece_t<C>{};
}

// a(v) = v / (1 + 2^p), p = -log2(e) times the sigmoid's argument (ffn::act with one
// product less).
template <int ACT>
__device__ __forceinline__ float activated(float v) {
    if (ACT == LINEAR_NONE) return v;
    const float p = ACT == LINEAR_SILU ? v * -ffn::LOG2E
                                       : v * fmaf(v * v, -ffn::LOG2E * ffn::GELU_B, -ffn::LOG2E * ffn::GELU_A);
    return v * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(p));
}
// The same by an argument: branches where ACT is ANY.
constexpr int ANY = -1;
template <int ACT, int N>
__device__ __forceinline__ void activate(int act, float (&v)[N]) {
    if (ACT == ANY ? act == LINEAR_SILU : ACT == LINEAR_SILU) {
#pragma unroll
        for (int j = 0; j < N; ++j) v[j] = activated<LINEAR_SILU>(v[j]);
    } else if (ACT == ANY ? act == LINEAR_GELU : ACT == LINEAR_GELU) {
#pragma unroll
        for (int j = 0; j < N; ++j) v[j] = activated<LINEAR_GELU>(v[j]);
    }
}

// a'(v); large GELU arguments as in ffn::act_grad.
template <int ACT>
__device__ __forceinline__ float slope(float v) {
    if (ACT == LINEAR_NONE) return 1.f;
    if (ACT == LINEAR_SILU) {
        const float s = ffn::sigmoid_fast(v);
        return fmaf(v * s, 1.f - s, s);
    }
    const float s = ffn::sigmoid_fast(v * fmaf(v * v, ffn::GELU_B, ffn::GELU_A));
    return fmaf(v * s * (1.f - s), fmaf(fminf(v * v, 1e38f), 3.f * ffn::GELU_B, ffn::GELU_A), s);
}

// Eight columns from `col` < n on of a row, zeros from n on, in 32 bits.  Where 8
// divides n all eight are there.
template <class T>
__device__ __forceinline__ void load8(const T* row, int col, int n, float (&v)[8]) {
#pragma unroll
    for (int h = 0; h < 8 / E<T>; ++h) {
        piece_t<T> p = {};
        if (n % 8 == 0) __builtin_memcpy(&p, row + col + h * E<T>, 16);
        else if (col + h * E<T> < n) p = load_piece(row, col + h * E<T>, n);
#pragma unroll
        for (int j = 0; j < E<T>; ++j) v[h * E<T> + j] = (float)p[j];
    }
}
// v's elements with infinities as the type's largest number where FINITE: z as it is kept
// for the backward pass.  a'(z) is 1 or 0 from far smaller arguments on, but of an
// infinity it would be NaN (infinity times 0), as would z packed into 8 bits.  Of the types
// only float16 ends where sums may be; NaN stays.
template <bool FINITE, class T>
__device__ __forceinline__ piece_t<T> kept(piece_t<T> v) {
    if constexpr (FINITE && std::is_same<T, _Float16>::value) {
        typedef uint16_t u16x8 __attribute__((ext_vector_type(8)));
        u16x8 w;
        __builtin_memcpy(&w, &v, 16);
#pragma unroll
        for (int j = 0; j < 8; ++j) w[j] -= (w[j] & 0x7FFF) == 0x7C00;   // the number before infinity
        __builtin_memcpy(&v, &w, 16);
    }
    return v;
}
template <bool FINITE = false, class T>
__device__ __forceinline__ void store8(T* row, int col, int n, const float (&v)[8]) {
#pragma unroll
    for (int h = 0; h < 8 / E<T>; ++h) {
        piece_t<T> p;
#pragma unroll
        for (int j = 0; j < E<T>; ++j) p[j] = (T)v[h * E<T> + j];
        p = kept<FINITE, T>(p);
        if (n % 8 == 0) __builtin_memcpy(row + col + h * E<T>, &p, 16);
        else if (col + h * E<T> < n) store_piece(row, col + h * E<T>, n, p);
    }
}
// The same by a type that is an argument.
__device__ __forceinline__ void load8(const void* base, int dtype, int64_t stride, int64_t row, int col, int n,
                                      float (&v)[8]) {
    if (dtype == 0) load8(static_cast<const float*>(base) + row * stride, col, n, v);
    else if (dtype == 1) load8(static_cast<const _Float16*>(base) + row * stride, col, n, v);
    else load8(static_cast<const __bf16*>(base) + row * stride, col, n, v);
}

// What follows the product: v are the eight columns from col on of row, bias
// included; C is the products' type, Y the result's.
template <class C, class Y>
__device__ __forceinline__ void finish(const LinearArgs& a, int64_t row, int col, float (&v)[8]) {
    if (col >= a.outer) return;
    if (a.z) store8<true>(static_cast<C*>(a.z) + row * a.z_stride, col, a.outer, v);
    activate<ANY>(a.act, v);
    if (a.residual) {
        float r[8];
        load8(static_cast<const Y*>(a.residual) + row * a.residual_stride, col, a.outer, r);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] += r[j];
    }
    store8(static_cast<Y*>(a.y) + row * a.y_stride, col, a.outer, v);
}

// Stores of 16 rows in whole 128-byte lines.  Lane (q, r) holds two pieces of row
// r, at columns ca and cb; lanes r and r ^ 8 change one, so that the first store is
// all of rows 0 .. 7 and the second all of rows 8 .. 15.  (1.09M x 64 -> 256
// without an activation: 182 us in the 64-byte parts that a piece a lane makes, 145
// in lines.)
template <class T>
__device__ __forceinline__ void store_lines(void* base, int64_t stride, int64_t row0, int64_t rows, int ca, int cb,
                                            int n, piece_t<T> pa, piece_t<T> pb) {
    typedef int i32x4 __attribute__((ext_vector_type(4)));
    i32x4 wa, wb, first, second;
    __builtin_memcpy(&wa, &pa, 16);
    __builtin_memcpy(&wb, &pb, 16);
#pragma unroll
    for (int j = 0; j < 4; ++j) {   // row_ror:8 into lanes 8 .. 15, and into lanes 0 .. 7
        first[j] = __builtin_amdgcn_update_dpp(wa[j], wb[j], 0x128, 0xF, 0xC, false);
        second[j] = __builtin_amdgcn_update_dpp(wb[j], wa[j], 0x128, 0xF, 0x3, false);
    }
    __builtin_memcpy(&pa, &first, 16);
    __builtin_memcpy(&pb, &second, 16);
    const int r = threadIdx.x & 15, col = r < 8 ? ca : cb;
    const int64_t row = row0 + (r & 7);
    if (col >= n) return;
    T* at = static_cast<T*>(base) + row * stride;
    if (n % 8 == 0) {
        if (row < rows) __builtin_memcpy(at + col, &pa, 16);
        if (row + 8 < rows) __builtin_memcpy(at + 8 * stride + col, &pb, 16);
    } else {
        if (row < rows) store_piece(at, col, n, pa);
        if (row + 8 < rows) store_piece(at + 8 * stride, col, n, pb);
    }
}
// Blocks of columns whose results a wave stores at once: as many as make lines.
template <class Y>
constexpr int LINE = sizeof(Y) == 4 ? 1 : 2;

// The columns col .. col + 7 of each of N blocks, of which the first `live` are there.
template <bool FINITE, class T, int N>
__device__ __forceinline__ void store16(void* base, int64_t stride, int64_t row0, int64_t rows, int col, int n,
                                        int live, const float (&v)[N][8]) {
    piece_t<T> p[N][8 / E<T>];
#pragma unroll
    for (int b = 0; b < N; ++b)
#pragma unroll
        for (int j = 0; j < 8; ++j) p[b][j / E<T>][j % E<T>] = (T)v[b][j];
#pragma unroll
    for (int b = 0; b < N; ++b)
#pragma unroll
        for (int h = 0; h < 8 / E<T>; ++h) p[b][h] = kept<FINITE, T>(p[b][h]);
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int b = 0; b < N; ++b)
            if (b < live)
                store_lines<T>(base, stride, row0, rows, col + b * COLS, col + b * COLS + 4, n, p[b][0], p[b][1]);
    } else if constexpr (N == 2) {
        store_lines<T>(base, stride, row0, rows, col, live >= 2 ? col + COLS : n, n, p[0][0], p[1][0]);
    } else {
        const int64_t row = row0 + (threadIdx.x & 15);
        T* at = static_cast<T*>(base) + row * stride;
        if (row < rows && col < n) {
            if (n % 8 == 0) __builtin_memcpy(at + col, &p[0][0], 16);
            else store_piece(at, col, n, p[0][0]);
        }
    }
}

// finish for a wave's 16 rows and N blocks of columns, of which the first `live` are there;
// col is the lane's in the first.  All lanes must be active.
template <class C, class Y, int ACT, int N>
__device__ __forceinline__ void finish16(const LinearArgs& a, int64_t row0, int col, int live, float (&v)[N][8]) {
    if (a.z) store16<true, C>(a.z, a.z_stride, row0, a.rows, col, a.outer, live, v);
#pragma unroll
    for (int b = 0; b < N; ++b) activate<ACT>(a.act, v[b]);
    if (a.residual) {
        const int64_t row = min(row0 + (threadIdx.x & 15), a.rows - 1);
        const Y* at = static_cast<const Y*>(a.residual) + row * a.residual_stride;
#pragma unroll
        for (int b = 0; b < N; ++b) {
            if (col + b * COLS >= a.outer || b >= live) continue;
            float r[8];
            load8(at, col + b * COLS, a.outer, r);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[b][j] += r[j];
        }
    }
    store16<false, Y>(a.y, a.y_stride, row0, a.rows, col, a.outer, live, v);
}

// The bias of eight columns, zeros for none; it is of x's type, 32-bit beside mx8.
template <class T, bool MX>
__device__ __forceinline__ void bias8(const LinearArgs& a, int col, float (&v)[8]) {
    using B = typename std::conditional<MX, float, T>::type;
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = 0.f;
    if (a.bias && col < a.outer) load8(static_cast<const B*>(a.bias), col, a.outer, v);
}

// 16 R rows and 32 columns a workgroup, whose waves share the contraction (wave
// w takes blocks w, w + WAVES, ...) and join their sums in LDS in a fixed order.
// Bound by latency: two reads from memory and the join (8 x 256 -> 1000 bf16: 4.1 us).
constexpr int FEW_TILES = 4;
// Eight waves for a single row tile: 1000 inputs are then read in one go (4 x 1000 ->
// 1000 bf16: 5.6 us, 6.7 with four; up to 256 inputs the same).  Four tiles of eight
// waves would leave room for two workgroups a CU.
template <int R>
constexpr int FEW_WAVES = R == 1 ? 8 : 4;
template <class T, class Y, bool MX, bool TRANS, int R>
__global__ __launch_bounds__(64 * FEW_WAVES<R>) void k_linear_few(LinearArgs a) {
    using C = typename Operand<T, MX>::type;
    __shared__ f32x4 part[FEW_WAVES<R>][R][2][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, q = lane >> 4, r = lane & 15;
    const int blocks = (a.outer + COLS - 1) / COLS, kbs = (a.inner + KB<C> - 1) / KB<C>;
    const int64_t row0 = (int64_t)(blockIdx.x / blocks) * 16 * R;
    const int col0 = (int)(blockIdx.x % blocks) * COLS;
    f32x4 acc[R][2] = {};
    constexpr int U = 4;   // blocks whose reads are under way at once
    for (int kb0 = wave; kb0 < kbs; kb0 += U * FEW_WAVES<R>) {
        XPiece<T, MX> x[U][R] = {};
        piece_t<C> w[U][2] = {};
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int kb = kb0 + u * FEW_WAVES<R>;
            if (kb >= kbs) break;
#pragma unroll
            for (int s = 0; s < 2; ++s) w[u][s] = w_piece<T, MX, TRANS>(a, col0 + column(s, r), kb, q);
#pragma unroll
            for (int i = 0; i < R; ++i) x[u][i].template read<true>(a, min(row0 + 16 * i + r, a.rows - 1), kb, q);
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int i = 0; i < R; ++i)
#pragma unroll
                for (int s = 0; s < 2; ++s) acc[i][s] = mma(w[u][s], x[u][i].taken(), acc[i][s]);
    }
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
        for (int s = 0; s < 2; ++s) part[wave][i][s][lane] = acc[i][s];
    __syncthreads();
    float bias[8];
    bias8<T, MX>(a, col0 + q * 8, bias);
#pragma unroll
    for (int i = 0; i < R; ++i) {
        if (i % FEW_WAVES<R> != wave) continue;
        const int64_t row = row0 + 16 * i + r;
        float v[8];
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            f32x4 t = part[0][i][s][lane];
#pragma unroll
            for (int p = 1; p < FEW_WAVES<R>; ++p) t += part[p][i][s][lane];
#pragma unroll
            for (int j = 0; j < 4; ++j) v[4 * s + j] = t[j] + bias[4 * s + j];
        }
        if (row < a.rows) finish<C, Y>(a, row, col0 + q * 8, v);
    }
}

// Weights in LDS for all of the contraction (DK blocks) and the columns of a
// slice; 16 waves a CU go through rows, 16 R at a time, without a barrier, and read
// the next rows' x ahead.  Workgroups of one XCD share an L2: the slices of the same
// rows run on one.  Bound by HBM, and by the vector unit where there is an activation
// (1.09M x 64 -> 256 bf16: 145 us without, 4.8 TB/s, 154 to 160 with GELU, vector unit 83%;
// 500k x 256 -> 256 from 8 bits 112 us, 3.4 TB/s; 120k x 45 -> 192 f32
// GELU 39 us).  With two workgroups of 12 waves or 16
// the registers of a wave do not suffice (214 us -> 366 and more at an earlier step).
template <class T, class Y, bool MX, bool TRANS, int ACT, int DK, int R>
__global__ __launch_bounds__(1024) __attribute__((amdgpu_waves_per_eu(4, 4))) void k_linear_all(
    LinearArgs a, int slices, int slice_blocks) {
    using C = typename Operand<T, MX>::type;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    piece_t<C>* w = reinterpret_cast<piece_t<C>*>(lds);
    float* bias = reinterpret_cast<float*>(lds + slice_blocks * 2 * DK * 1024);
    const int lane = threadIdx.x & 63, q = lane >> 4, r = lane & 15, waves = blockDim.x >> 6;
    const int slice = (int)(blockIdx.x / 8 % slices);
    const int64_t group = blockIdx.x / 8 / slices * 8 + blockIdx.x % 8;
    const int64_t groups = gridDim.x / slices;
    const int first = slice * slice_blocks, blocks = min(slice_blocks, (a.outer + COLS - 1) / COLS - first);
#pragma unroll 4
    for (int i = threadIdx.x; i < blocks * 2 * DK * 64; i += blockDim.x) {
        const int f = i >> 6, kb = f % DK, s = f / DK % 2, cb = f / DK / 2;
        w[i] = w_piece<T, MX, TRANS>(a, (first + cb) * COLS + column(s, i & 15), kb, (i >> 4) & 3);
    }
    for (int i = threadIdx.x; i < blocks * COLS; i += blockDim.x) {
        using B = typename std::conditional<MX, float, T>::type;
        bias[i] = a.bias ? (float)static_cast<const B*>(a.bias)[min(first * COLS + i, a.outer - 1)] : 0.f;
    }
    __syncthreads();
    const int64_t tiles = (a.rows + 16 * R - 1) / (16 * R), step = groups * waves;
    // neighbours in a workgroup, but few tiles to as many CUs
    int64_t t = tiles >= step ? group * waves + (threadIdx.x >> 6) : group + (threadIdx.x >> 6) * groups;
    XPiece<T, MX> next[R][DK];
    auto read = [&](int64_t tile) {
#pragma unroll
        for (int i = 0; i < R; ++i)
#pragma unroll
            for (int kb = 0; kb < DK; ++kb)
                next[i][kb].template read<DK == 1>(a, min(tile * 16 * R + 16 * i + r, a.rows - 1), kb, q);
    };
    read(t);
    piece_t<C> x[R][DK];
    auto take = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < R; ++i)
#pragma unroll
            for (int kb = 0; kb < DK; ++kb) x[i][kb] = next[i][kb].taken();
    };
    if (!MX) take();
    for (; t < tiles; t += step) {
        if (MX) take();
        read(t + step);
        constexpr int N = LINE<Y>;
        for (int cb = 0; cb < blocks; cb += N) {
            f32x4 acc[R][N][2];   // starts as the bias
#pragma unroll
            for (int b = 0; b < N; ++b) {
                const int at = min(cb + b, blocks - 1);
#pragma unroll
                for (int s = 0; s < 2; ++s) {
                    __builtin_memcpy(&acc[0][b][s], bias + at * COLS + q * 8 + 4 * s, 16);
#pragma unroll
                    for (int i = 1; i < R; ++i) acc[i][b][s] = acc[0][b][s];
                }
                const piece_t<C>* wb = w + at * 2 * DK * 64 + lane;
#pragma unroll
                for (int kb = 0; kb < DK; ++kb)
#pragma unroll
                    for (int s = 0; s < 2; ++s) {
                        const piece_t<C> wf = wb[(s * DK + kb) * 64];
#pragma unroll
                        for (int i = 0; i < R; ++i) acc[i][b][s] = mma(wf, x[i][kb], acc[i][b][s]);
                    }
            }
            // the next rows are waited for before the last stores, which the wait would include (1M
            // x 128 -> 64 bf16 with a residual 151 -> 134 us; 8 bits, which convert here, 117 -> 120)
            if (!MX && cb + N >= blocks) take();
#pragma unroll
            for (int i = 0; i < R; ++i) {
                float v[N][8];
#pragma unroll
                for (int b = 0; b < N; ++b)
#pragma unroll
                    for (int j = 0; j < 8; ++j) v[b][j] = acc[i][b][j / 4][j % 4];
                finish16<C, Y, ACT>(a, t * 16 * R + 16 * i, (first + cb) * COLS + q * 8, blocks - cb, v);
            }
        }
    }
}

// Fragments of the weights, zero beyond the matrix: for a slice of NB column blocks
// after the other, block after block of the contraction (kbs of them), the slice's
// 2 NB tiles.
template <class T, bool MX, bool TRANS>
__global__ __launch_bounds__(256) void k_linear_pack(LinearArgs a, int nb, int kbs,
                                                     piece_t<typename Operand<T, MX>::type>* out, int64_t pieces) {
    using C = typename Operand<T, MX>::type;
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= pieces) return;
    const int lane = (int)(i & 63), live = (a.inner + KB<C> - 1) / KB<C>;
    const int64_t f = i >> 6;
    const int t = (int)(f % (2 * nb)), kb = (int)(f / (2 * nb) % kbs), slice = (int)(f / (2 * nb) / kbs);
    const int row = (slice * nb + t / 2) * COLS + column(t % 2, lane & 15);
    piece_t<C> v = {};
    if (kb < live) v = w_piece<T, MX, TRANS>(a, row, kb, lane >> 4);
    out[i] = v;
}

// Packed weights streamed through two areas of LDS, KC blocks of the contraction at
// a time; a wave holds the sums of 16 R rows and a slice of NB column blocks.  x is
// read two steps ahead: a step's products take less than a read from memory does.
// (65536 x 1000 -> 200 f16: 49 us, 3.7 TB/s, matrix unit 26%; one step ahead 81.)
template <class T, class Y, bool MX, int NB, int R, int KC>
__global__ __launch_bounds__(512) void k_linear_stream(LinearArgs a,
                                                       const piece_t<typename Operand<T, MX>::type>* packed, int slices,
                                                       int steps) {
    using C = typename Operand<T, MX>::type;
    constexpr int F = KC * 2 * NB;   // fragments of a step
    __shared__ piece_t<C> w[2][F * 64];
    const int lane = threadIdx.x & 63, q = lane >> 4, r = lane & 15, waves = blockDim.x >> 6;
    const int slice = (int)(blockIdx.x / 8 % slices);
    const int64_t group = blockIdx.x / 8 / slices * 8 + blockIdx.x % 8;
    const int64_t row0 = (group * waves + (threadIdx.x >> 6)) * 16 * R;
    packed += (int64_t)slice * steps * F * 64;
    XPiece<T, MX> next[2][R][KC];
    auto read = [&](int step, XPiece<T, MX> (&to)[R][KC]) {
        step = min(step, steps - 1);
#pragma unroll
        for (int i = 0; i < R; ++i)
#pragma unroll
            for (int c = 0; c < KC; ++c)
                to[i][c].template read<false>(a, min(row0 + 16 * i + r, a.rows - 1), step * KC + c, q);
    };
    f32x4 acc[R][2 * NB];   // starts as the bias
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        float bias[8];
        bias8<T, MX>(a, (slice * NB + b) * COLS + q * 8, bias);
#pragma unroll
        for (int i = 0; i < R; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) acc[i][2 * b + j / 4][j % 4] = bias[j];
    }
    read(0, next[0]);
    ffn::fetch<C>(packed, w[0], F);
    asm volatile("" ::: "memory");
    read(1, next[1]);
    for (int step0 = 0; step0 < steps; step0 += 2)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int step = step0 + h;
            if (step >= steps) break;
            // the step's weights are there when at most the reads of x that followed them are
            // under way: one a piece at least
            asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(R * KC) : "memory");
            piece_t<C> x[R][KC];
#pragma unroll
            for (int i = 0; i < R; ++i)
#pragma unroll
                for (int c = 0; c < KC; ++c) x[i][c] = next[h][i][c].taken();
            if (step + 1 < steps) ffn::fetch<C>(packed + (int64_t)(step + 1) * F * 64, w[h ^ 1], F);
            asm volatile("" ::: "memory");
            read(step + 2, next[h]);
            const piece_t<C>* at = w[h] + lane;
#pragma unroll
            for (int c = 0; c < KC; ++c)
#pragma unroll
                for (int f = 0; f < 2 * NB; ++f) {
                    const piece_t<C> wf = at[(c * 2 * NB + f) * 64];
#pragma unroll
                    for (int i = 0; i < R; ++i) acc[i][f] = mma(wf, x[i][c], acc[i][f]);
                }
            ffn::read_ahead<1, R * ffn::MFMAS<C>, F, 4>();
        }
    constexpr int N = LINE<Y>;
#pragma unroll
    for (int b = 0; b < NB; b += N)
#pragma unroll
        for (int i = 0; i < R; ++i) {
            float v[N][8] = {};
#pragma unroll
            for (int h = 0; h < N; ++h)
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (b + h < NB) v[h][j] = acc[i][b + h < NB ? 2 * (b + h) + j / 4 : 0][j % 4];
            finish16<C, Y, ANY>(a, row0 + 16 * i, (slice * NB + b) * COLS + q * 8, NB - b, v);
        }
}

constexpr int64_t CUS = 256;
constexpr int64_t LDS_BYTES = 160 * 1024;
constexpr int ALL_BLOCKS = 8;   // of the contraction, up to which the weights stay in LDS

// How a product is launched, by its sizes: by k_linear_few up to so many of its
// workgroups that the others' start costs more.  (bf16, us: 256 -> 512 over 8000 rows
// 21 and 29, 16000 38 and 23; 64 -> 256 over 16000 15 and 21, 32000 26 and 19; 1000 ->
// 200 over 8000 28 and 38, 16000 48 and 39; 1000 -> 1000 over 2000 22 and 45, 8000 77
// and 47.)
struct Shape {
    int kbs;            // blocks of the contraction
    int blocks;         // of columns
    int slices, nb;     // of columns, and blocks of a slice
    int steps;          // streamed: of KC blocks of the contraction
    int64_t packed;     // streamed: bytes of the packed weights
    bool few, all;
};
constexpr int KC = 2;
template <class C>
Shape shape(int64_t rows, int inner, int outer) {
    Shape p{};
    p.kbs = (int)ceil_div(inner, KB<C>);
    p.blocks = (int)ceil_div(outer, COLS);
    p.few = ceil_div(rows, 16 * FEW_TILES) * p.blocks <= (inner > 512 ? 1024 : 2048);
    p.all = !p.few && p.kbs <= ALL_BLOCKS;
    if (p.all) {
        if (p.kbs == 5 || p.kbs == 7) ++p.kbs;   // kernels there are for 1 to 4, 6 and 8
        const int most = (int)(LDS_BYTES / (p.kbs * 2048 + COLS * 4));
        p.slices = (int)ceil_div(p.blocks, most);
        p.nb = (int)ceil_div(p.blocks, p.slices);
    } else if (!p.few) {
        const int64_t most = 8;
        p.slices = (int)ceil_div(p.blocks, most);
        p.nb = (int)ceil_div(p.blocks, p.slices);
        p.steps = (int)ceil_div(p.kbs, KC);
        p.packed = (int64_t)p.slices * p.steps * KC * 2 * p.nb * 1024;
    }
    return p;
}

// Rows from `at` on.
template <class T, bool MX>
LinearArgs rows_from(const LinearArgs& a, int64_t at, int64_t rows) {
    LinearArgs p = a;
    const int64_t size = sizeof(T), ysize = a.y_dtype == 0 ? 4 : 2;
    p.rows = rows;
    p.x = static_cast<const char*>(a.x) + at * (MX ? mx8::data_stride(a.inner) : a.x_stride * size);
    if (MX) p.x_scales = a.x_scales + at * mx8::scale_stride(a.inner);
    if (a.residual) p.residual = static_cast<const char*>(a.residual) + at * a.residual_stride * ysize;
    p.y = static_cast<char*>(a.y) + at * a.y_stride * ysize;
    if (a.z) p.z = static_cast<char*>(a.z) + at * a.z_stride * size;
    return p;
}

// One launch: 2048 workgroups at most, or the tail's 1024 rows.
template <class T, class Y, bool MX, bool TRANS>
void few_product(hipStream_t s, const LinearArgs& a) {
    auto launch = [&](auto r) {
        constexpr int R = r();
        const int64_t groups = ceil_div(a.rows, 16 * R) * ceil_div(a.outer, COLS);
        k_linear_few<T, Y, MX, TRANS, R><<<(unsigned)groups, 64 * FEW_WAVES<R>, 0, s>>>(a);
    };
    if (a.rows <= 16) launch(std::integral_constant<int, 1>{});
    else launch(std::integral_constant<int, FEW_TILES>{});
}

template <class T, class Y, bool MX, bool TRANS, int ACT, int DK>
void all_product(hipStream_t s, const LinearArgs& a, const Shape& p) {
    constexpr int R = DK <= 4 ? 2 : 1;
    const size_t bytes = (size_t)p.nb * (2 * DK * 1024 + COLS * 4);
    const int per_cu = std::min<int>(2, LDS_BYTES / bytes), most_waves = 16 / per_cu;
    const int64_t tiles = ceil_div(a.rows, 16 * R), most = std::max<int64_t>(per_cu * CUS / p.slices / 8, 1) * 8;
    const int64_t groups = std::min(ceil_div(tiles, 8) * 8, most);   // a multiple of 8, as the kernel numbers them
    k_linear_all<T, Y, MX, TRANS, ACT, DK, R>
        <<<(unsigned)(groups * p.slices), 64 * most_waves, bytes, s>>>(a, p.slices, p.nb);
}

// Rows that a streamed product leaves to k_linear_few: the start of a last round of
// workgroups that would take as long as a full one (65543 x 1000 -> 200 f16: 86 us
// with seven rows in a round of their own).
constexpr int64_t STREAM_ROWS = 16 * 2 * 8;   // of a workgroup
inline int64_t tail_rows(int64_t rows, int slices) {
    const int64_t round = STREAM_ROWS * std::max<int64_t>(CUS / slices, 1), rest = rows % round;
    return rows > round && rest <= 1024 ? rest : 0;
}

template <class T, class Y, bool MX, int NB>
void stream_product(hipStream_t s, const LinearArgs& a, const Shape& p) {
    using C = typename Operand<T, MX>::type;
    const piece_t<C>* packed = reinterpret_cast<const piece_t<C>*>(a.ws);
    constexpr int R = 2, WAVES = 8;
    static_assert(STREAM_ROWS == 16 * R * WAVES, "rows of a workgroup");
    const int64_t most = (int64_t(1) << 22) / p.slices / 8 * 8 * STREAM_ROWS;   // fewer than 2^32 threads
    for (int64_t at = 0; at < a.rows; at += most) {
        const LinearArgs part = rows_from<T, MX>(a, at, std::min(most, a.rows - at));
        const int64_t groups = ceil_div(ceil_div(part.rows, STREAM_ROWS), 8) * 8;
        k_linear_stream<T, Y, MX, NB, R, KC>
            <<<(unsigned)(groups * p.slices), 64 * WAVES, 0, s>>>(part, packed, p.slices, p.steps);
    }
}

// TRANS: W^T in W's place, and no activation.
template <class T, class Y, bool MX, bool TRANS>
void product(hipStream_t s, const LinearArgs& a) {
    using C = typename Operand<T, MX>::type;
    const Shape p = shape<C>(a.rows, a.inner, a.outer);
    if (p.few) return few_product<T, Y, MX, TRANS>(s, a);
    if (p.all) {
        auto all = [&](auto dk) {
            if constexpr (!TRANS) {
                if (a.act == LINEAR_SILU) return all_product<T, Y, MX, TRANS, LINEAR_SILU, dk()>(s, a, p);
                if (a.act == LINEAR_GELU) return all_product<T, Y, MX, TRANS, LINEAR_GELU, dk()>(s, a, p);
            }
            all_product<T, Y, MX, TRANS, LINEAR_NONE, dk()>(s, a, p);
        };
        switch (p.kbs) {
#define BLOCKS(n) case n: return all(std::integral_constant<int, n>{})
            BLOCKS(1);
            BLOCKS(2);
            BLOCKS(3);
            BLOCKS(4);
            BLOCKS(6);
            BLOCKS(8);
#undef BLOCKS
        }
    }
    const int64_t pieces = p.packed / 16;
    piece_t<C>* packed = reinterpret_cast<piece_t<C>*>(a.ws);
    k_linear_pack<T, MX, TRANS><<<(unsigned)ceil_div(pieces, 256), 256, 0, s>>>(a, p.nb, p.steps * KC, packed, pieces);
    const int64_t tail = tail_rows(a.rows, p.slices);
    const LinearArgs main = rows_from<T, MX>(a, 0, a.rows - tail);
    if (tail) few_product<T, Y, MX, TRANS>(s, rows_from<T, MX>(a, a.rows - tail, tail));
    switch (p.nb) {
#define BLOCKS(n) case n: return stream_product<T, Y, MX, n>(s, main, p)
        BLOCKS(1);
        BLOCKS(2);
        BLOCKS(3);
        BLOCKS(4);
        BLOCKS(5);
        BLOCKS(6);
        BLOCKS(7);
        BLOCKS(8);
#undef BLOCKS
    }
}

template <class C>
int64_t product_workspace(int64_t rows, int inner, int outer) {
    return shape<C>(rows, inner, outer).packed;
}

// ---------------------------------------------------------------- backward

// dz = dy a'(z) in T, and the sums of its columns over each workgroup's rows.
// tx threads along a row, eight columns each; 256 / tx rows at once.
template <class T, bool MX>
__global__ __launch_bounds__(256) void k_linear_dz(LinearGradArgs a, T* dz, float* part, int tx,
                                                   int64_t rows_per_group) {
    __shared__ float sums[256][8];
    const int lane = threadIdx.x & (tx - 1), sub = threadIdx.x / tx, rb = 256 / tx;
    const int64_t first = (int64_t)blockIdx.x * rows_per_group, last = min(first + rows_per_group, a.rows);
    for (int base = 0; base < a.outer; base += tx * 8) {
        const int col = base + lane * 8;
        float sum[8] = {};
        if (col < a.outer)
            for (int64_t row = first + sub; row < last; row += rb) {
                float v[8];
                load8(a.dy, a.y_dtype, a.dy_stride, row, col, a.outer, v);
                if (a.act != LINEAR_NONE) {
                    float z[8];
                    if constexpr (MX) {
                        const uint8_t* data = static_cast<const uint8_t*>(a.z) + row * mx8::data_stride(a.outer);
                        uint32_t bytes[2];
                        __builtin_memcpy(bytes, data + col, 8);
                        mx8::values<__bf16>(bytes, a.z_scales[row * mx8::scale_stride(a.outer) + col / 32], z);
                    } else {
                        load8(static_cast<const T*>(a.z) + row * a.z_stride, col, a.outer, z);
                    }
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        v[j] *= a.act == LINEAR_SILU ? slope<LINEAR_SILU>(z[j]) : slope<LINEAR_GELU>(z[j]);
                }
#pragma unroll
                for (int j = 0; j < 8; ++j) sum[j] += v[j];
                if (dz) store8(dz + row * a.outer, col, a.outer, v);
            }
        if (!part) continue;
        __syncthreads();
#pragma unroll
        for (int j = 0; j < 8; ++j) sums[threadIdx.x][j] = sum[j];
        __syncthreads();
        for (int c = threadIdx.x; c < tx * 8; c += 256) {
            if (base + c >= a.outer) continue;
            float t = 0.f;
            for (int p = 0; p < rb; ++p) t += sums[p * tx + c / 8][c % 8];
            part[(int64_t)blockIdx.x * a.outer + base + c] = t;
        }
    }
}

// Adds `groups` partial rows of n1 + n2 numbers into two results, either of which
// may be null: 32 columns a workgroup at once, 32 threads a column.
template <class T>
__global__ __launch_bounds__(1024) void k_linear_fold(const float* part, int groups, int64_t n1, int64_t n2, T* out1,
                                                      T* out2) {
    __shared__ float red[32][33];
    const int sl = threadIdx.x >> 5;
    const int64_t n = n1 + n2;
    for (int64_t at = (int64_t)blockIdx.x * 32; at < n; at += (int64_t)gridDim.x * 32) {
        const int64_t col = at + (threadIdx.x & 31);
        float t = 0.f;
        if (col < n)
#pragma unroll 8
            for (int g = sl; g < groups; g += 32) t += part[g * n + col];
        red[sl][threadIdx.x & 31] = t;
        __syncthreads();
        if (sl == 0 && col < n) {
            t = 0.f;
            for (int q = 0; q < 32; ++q) t += red[q][threadIdx.x & 31];
            if (col < n1) {
                if (out1) out1[col] = (T)t;
            } else if (out2) {
                out2[col - n1] = (T)t;
            }
        }
        __syncthreads();
    }
}
// The same for few groups: a thread a column.
template <class T>
__global__ __launch_bounds__(256) void k_linear_fold_few(const float* part, int groups, int64_t n1, int64_t n2, T* out1,
                                                         T* out2) {
    const int64_t n = n1 + n2;
    for (int64_t col = (int64_t)blockIdx.x * 256 + threadIdx.x; col < n; col += (int64_t)gridDim.x * 256) {
        float t = 0.f;
#pragma unroll 8
        for (int g = 0; g < groups; ++g) t += part[g * n + col];
        if (col < n1) {
            if (out1) out1[col] = (T)t;
        } else if (out2) {
            out2[col - n1] = (T)t;
        }
    }
}
// Up to 32 groups leave most of k_linear_fold's threads without work (8 groups of 1000 x
// 1000: 70 us, 6.9 this way), and more of them make a thread's sum long.
template <class T>
void fold(hipStream_t s, const float* part, int groups, int64_t n1, int64_t n2, void* out1, void* out2) {
    const int64_t n = n1 + n2;
    if (groups <= 32)
        k_linear_fold_few<T><<<(unsigned)std::min<int64_t>(ceil_div(n, 256), 1 << 14), 256, 0, s>>>(
            part, groups, n1, n2, static_cast<T*>(out1), static_cast<T*>(out2));
    else
        k_linear_fold<T><<<(unsigned)std::min<int64_t>(ceil_div(n, 32), 1 << 20), 1024, 0, s>>>(
            part, groups, n1, n2, static_cast<T*>(out1), static_cast<T*>(out2));
}

// Where piece c of row rho of a block of rows lies (ffn::slot): rho = perm(s, r).
template <class T>
__device__ __forceinline__ int staged(int rho, int c) {
    return ffn::slot<T>(c / 4, rho % E<T> / 4, c % 4, rho / E<T> * 4 + rho % 4);
}

// dW, db and more in one pass over dy, z and x: a workgroup's registers hold dW, or a
// part of it: 16 waves, WN x WK of them, HN x HK tiles of 16 x 16 each.  Two blocks of
// KB rows at a time go through LDS: dz is made of dy and z on the way in, its sums
// over rows stay in registers, dW takes both operands through transposing reads, and
// dx takes dz's rows and W^T, which stays in LDS.  A SIMD has four waves: two multiply
// a step and then make dz of the next, two do it in the other order, so that
// vector and matrix units work at once.  A wave's tiles are WN (WK) apart and tiles
// beyond the matrix are left out, so that the matrix units share what there is.
//   500k x 64 -> 256 bf16 SiLU: 136 us, 4.7 TB/s (8 waves a workgroup: 153)
//   120k x 48 -> 192 f32 GELU from 8 bits: 96 us, 46 TFLOP/s: dz by itself takes 42, dx 24
//   and dW 30, and little of the one passes behind the other
constexpr int RB = 2;
constexpr int BWD_WAVES = 16, BWD_THREADS = 64 * BWD_WAVES;
template <int N, int K>
struct BwdShape {
    static constexpr int n = N, k = K;
    static constexpr int WN = N >= 256 ? 8 : N * 2 <= K ? (N == 64 ? 2 : 4) : 4, WK = BWD_WAVES / WN;
    static constexpr int HN = N / 16 / WN, HK = K / 16 / WK;
};
// Pieces of a matrix on their way in, the same columns of many rows.
template <class T, bool MX>
struct Kept {
    const T* at;   // the piece in row 0; the last ends with the row
    __device__ __forceinline__ Kept(const void* base, const uint8_t*, int col, int n)
        : at(static_cast<const T*>(base) + max(min(col, n - E<T>), 0)) {}
    struct Raw {
        piece_t<T> v;
    };
    // offset: the row's, in elements
    __device__ __forceinline__ void read(Raw& r, int64_t offset, int64_t, int n) const {
        if (n >= E<T>) __builtin_memcpy(&r.v, at + offset, 16);
        else r.v = load_piece(at + offset, 0, n);
    }
    // the piece itself, zeros from n on where it begins before n
    static __device__ __forceinline__ piece_t<T> piece(const Raw& r, int col, int n) {
        if (n % E<T> == 0 || n < E<T>) return r.v;
        asm volatile("");   // a branch, so that widths of whole pieces are spared the moves
        return col > n - E<T> ? moved_down<T>(r.v, E<T> - n % E<T>) : r.v;
    }
    static __device__ __forceinline__ void values(const Raw& r, int col, int n, float (&f)[E<T>]) {
        const piece_t<T> p = piece(r, col, n);
#pragma unroll
        for (int j = 0; j < E<T>; ++j) f[j] = (float)p[j];
    }
    static __device__ __forceinline__ int64_t scale_offset(int64_t, int) { return 0; }
    static __device__ __forceinline__ int64_t stride(int64_t s, int) { return s; }
};
template <class T>
struct Kept<T, true> {
    const uint8_t *at, *scale;
    __device__ __forceinline__ Kept(const void* base, const uint8_t* scales, int col, int n) {
        col = min(col, (int)mx8::data_stride(n) - E<T>);
        at = static_cast<const uint8_t*>(base) + col;
        scale = scales + col / mx8::BLOCK;
    }
    struct Raw {
        uint32_t bytes[E<T> / 4];
        int code;
    };
    __device__ __forceinline__ void read(Raw& r, int64_t offset, int64_t scale_offset, int) const {
        __builtin_memcpy(r.bytes, at + offset, E<T>);
        r.code = scale[scale_offset];
    }
    static __device__ __forceinline__ void values(const Raw& r, int col, int n, float (&f)[E<T>]) {
        mx8::values<T>(r.bytes, r.code, f);
        if (n % E<T> != 0)   // zeros by the format, NaN where their block's scale is
#pragma unroll
            for (int j = 0; j < E<T>; ++j)
                if (col + j >= n) f[j] = 0.f;
    }
    static __device__ __forceinline__ piece_t<T> piece(const Raw& r, int col, int n) {
        float f[E<T>];
        values(r, col, n, f);
        piece_t<T> o;
#pragma unroll
        for (int j = 0; j < E<T>; ++j) o[j] = (T)f[j];
        return o;
    }
    static __device__ __forceinline__ int64_t scale_offset(int64_t row, int n) { return row * mx8::scale_stride(n); }
    static __device__ __forceinline__ int64_t stride(int64_t, int n) { return mx8::data_stride(n); }
};

// Columns of dx that one task makes, and where they are: two tiles of 16-bit results
// side by side (column), one of 32-bit ones, so that a lane has a piece.
template <class T>
constexpr int TASK = 4 * E<T>;
template <class T>
__device__ __forceinline__ int dx_column(int tile, int r) {
    return sizeof(T) == 4 ? tile * 16 + r : tile / 2 * COLS + column(tile % 2, r);
}

template <class T>
__host__ __device__ inline int dx_tiles(int inner) {
    return (inner + TASK<T> - 1) / TASK<T> * (TASK<T> / 16);
}

// Calls f with the least number of tiles that there is code for, MOST (2 or 4) or half of
// four, that holds n.
template <int MOST, class F>
__device__ __forceinline__ void with_live(int n, F&& f) {
    if constexpr (MOST == 4)
        if (n <= 2) return f(std::integral_constant<int, 2>{});
    f(std::integral_constant<int, MOST>{});
}

template <class T, class S, int ACT, bool ZMX, bool XMX>
__global__ __launch_bounds__(BWD_THREADS) __attribute__((amdgpu_waves_per_eu(4, 4))) void k_linear_bwd(
    LinearGradArgs a, T* dz, float* part, int tiles, int ktiles_all) {
    constexpr int STEP = RB * KB<T>;
    constexpr int NB = S::n / KB<T>, KBS = S::k / KB<T>, NP = NB * 4, KP = KBS * 4, RT = STEP / 16;
    constexpr int PD = STEP * NP / BWD_THREADS > 0 ? STEP * NP / BWD_THREADS : 1;
    constexpr int PX = STEP * KP / BWD_THREADS > 0 ? STEP * KP / BWD_THREADS : 1;
    constexpr int HT = ffn::HT<T>, TT = TASK<T> / 16;   // tiles of a block, of a task
    extern __shared__ __attribute__((aligned(16))) char lds[];
    // the part of dW that is the workgroup's; dx is made where that is all of it
    const int part_of = (int)(blockIdx.x % tiles), n0 = part_of / ktiles_all * S::n, k0 = part_of % ktiles_all * S::k;
    const int64_t group = blockIdx.x / tiles, groups = gridDim.x / tiles;
    const int width = min(a.outer - n0, S::n), depth = min(a.inner - k0, S::k);
    // live blocks of outputs and inputs, tiles of them, pieces of a block of rows
    const int nbs = (width + KB<T> - 1) / KB<T>, ntiles = nbs * HT, nblock = nbs * KB<T> * 4;
    const int kbs = (depth + KB<T> - 1) / KB<T>, ktiles = kbs * HT, kblock = kbs * KB<T> * 4;
    piece_t<T>* w = reinterpret_cast<piece_t<T>*>(lds);
    piece_t<T>* ld = w + (a.dx ? dx_tiles<T>(a.inner) * nbs * 64 : 0);   // two steps of dz
    piece_t<T>* lx = ld + 2 * RB * nblock;                              // and of x
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, q = lane >> 4, r = lane & 15;
    const int wn = wave % S::WN, wk = wave / S::WN;   // so that a SIMD has waves of every wk
    if (a.dx) {
        LinearArgs t{};   // W^T [inner, outer]
        t.w = a.w;
        t.w_stride = a.w_stride;
        t.inner = a.outer;
        t.outer = a.inner;
#pragma unroll 2
        for (int i = tid; i < dx_tiles<T>(a.inner) * nbs * 64; i += BWD_THREADS) {
            const int f = i >> 6;
            w[i] = w_piece<T, false, true, false>(t, dx_column<T>(f / nbs, i & 15), f % nbs, (i >> 4) & 3);
        }
    }
    // pieces behind the matrices stay zero
    for (int i = tid; i < 2 * RB * (nblock + kblock); i += BWD_THREADS) ld[i] = piece_t<T>{};
    __syncthreads();
    const int64_t steps = (a.rows + STEP - 1) / STEP;
    const int cd = tid % NP * E<T>, cx = tid % KP * E<T>;
    const Kept<T, false> fy(a.dy, nullptr, n0 + cd, a.outer);
    const Kept<T, ZMX> fz(a.z, a.z_scales, n0 + cd, a.outer);
    const Kept<T, XMX> fx(a.x, a.x_scales, k0 + cx, a.inner);
    typename Kept<T, false>::Raw dy[PD];
    typename Kept<T, ZMX>::Raw z[PD];
    typename Kept<T, XMX>::Raw x[PX];
    const int64_t zstride = fz.stride(a.z_stride, a.outer), xstride = fx.stride(a.x_stride, a.inner);
    const int rd = min(tid / NP, STEP - 1), rx = min(tid / KP, STEP - 1);
    // rows of a whole step are the step's, uniform, and the thread's
    auto read = [&](int64_t b) __attribute__((always_inline)) {
        const int64_t row0 = b * STEP;
        const bool whole = row0 + STEP <= a.rows;
#pragma unroll
        for (int p = 0; p < PD; ++p) {
            if (whole) {
                const int64_t row = row0 + p * (BWD_THREADS / NP);
                fy.read(dy[p], row * a.dy_stride + rd * a.dy_stride, 0, a.outer);
                if (ACT != LINEAR_NONE)
                    fz.read(z[p], row * zstride + rd * zstride,
                            fz.scale_offset(row, a.outer) + fz.scale_offset(rd, a.outer), a.outer);
            } else {
                const int64_t row = min(row0 + rd + p * (BWD_THREADS / NP), a.rows - 1);
                fy.read(dy[p], row * a.dy_stride, 0, a.outer);
                if (ACT != LINEAR_NONE) fz.read(z[p], row * zstride, fz.scale_offset(row, a.outer), a.outer);
            }
        }
#pragma unroll
        for (int p = 0; p < PX; ++p) {
            if (whole) {
                const int64_t row = row0 + p * (BWD_THREADS / KP);
                fx.read(x[p], row * xstride + rx * xstride,
                        fx.scale_offset(row, a.inner) + fx.scale_offset(rx, a.inner), a.inner);
            } else {
                const int64_t row = min(row0 + rx + p * (BWD_THREADS / KP), a.rows - 1);
                fx.read(x[p], row * xstride, fx.scale_offset(row, a.inner), a.inner);
            }
        }
    };
    f32x4 acc[S::HN][S::HK] = {};
    float db[E<T>] = {};
    int first = 0;
    // dz and x of step b into LDS
    auto form = [&](int64_t b, int turn) __attribute__((always_inline)) {
        piece_t<T>* bd = ld + turn * RB * nblock;
        piece_t<T>* bx = lx + turn * RB * kblock;
        const int live = (int)min(a.rows - b * STEP, (int64_t)STEP);
#pragma unroll
        for (int p = 0; p < PD; ++p) {
            const int rho = tid / NP + p * (BWD_THREADS / NP);
            float v[E<T>];
            fy.values(dy[p], n0 + cd, a.outer, v);
            if (ACT != LINEAR_NONE) {
                float f[E<T>];
                fz.values(z[p], n0 + cd, a.outer, f);
#pragma unroll
                for (int j = 0; j < E<T>; ++j) v[j] *= slope<ACT>(f[j]);
            }
            if (live < STEP)
#pragma unroll
                for (int j = 0; j < E<T>; ++j) v[j] = rho < live ? v[j] : 0.f;
            piece_t<T> o;
#pragma unroll
            for (int j = 0; j < E<T>; ++j) {
                if (STEP * NP >= BWD_THREADS || rho < STEP) db[j] += v[j];
                o[j] = (T)v[j];
            }
            if (rho < STEP && cd < width) {
                bd[rho / KB<T> * nblock + staged<T>(rho % KB<T>, tid % NP)] = o;
                if (dz && k0 == 0 && rho < live) store_piece(dz + (b * STEP + rho) * a.outer, n0 + cd, a.outer, o);
            }
        }
#pragma unroll
        for (int p = 0; p < PX; ++p) {
            const int rho = tid / KP + p * (BWD_THREADS / KP);
            piece_t<T> o = fx.piece(x[p], k0 + cx, a.inner);
            if (rho >= live) o = piece_t<T>{};
            if (rho < STEP && cx < depth) bx[rho / KB<T> * kblock + staged<T>(rho % KB<T>, tid % KP)] = o;
        }
    };
    // the products of step b
    auto multiply = [&](int64_t b, int turn) __attribute__((always_inline)) {
        const piece_t<T>* bd = ld + turn * RB * nblock;
        const piece_t<T>* bx = lx + turn * RB * kblock;
        if (a.dweight)
            // straight code for each number of tiles along the inputs that a wave may have
            with_live<S::HK>((ktiles - wk + S::WK - 1) / S::WK, [&](auto live) __attribute__((always_inline)) {
                constexpr int HK = decltype(live)::value;
#pragma unroll
                for (int h = 0; h < RB; ++h) {
                    piece_t<T> ds[S::HN], xs[HK];
#pragma unroll
                    for (int j = 0; j < HK; ++j)
                        xs[j] = ffn::by_dim<T>(bx + h * kblock, min(j * S::WK + wk, ktiles - 1));
#pragma unroll
                    for (int i = 0; i < S::HN; ++i)
                        ds[i] = ffn::by_dim<T>(bd + h * nblock, min(i * S::WN + wn, ntiles - 1));
#pragma unroll
                    for (int i = 0; i < S::HN; ++i)
                        if (i * S::WN + wn < ntiles)
#pragma unroll
                            for (int j = 0; j < HK; ++j) acc[i][j] = mma(ds[i], xs[j], acc[i][j]);
                }
            });
        if (a.dx) {
            // tasks go round the waves from step to step
            const int tasks = dx_tiles<T>(a.inner) / TT * RT;
            for (int t = (wave + first) % BWD_WAVES; t < tasks; t += BWD_WAVES) {
                const int task = t / RT, tile = t % RT;   // columns, and 16 rows
                const piece_t<T>* rows = bd + tile / HT * nblock;
                f32x4 o[TT] = {};
                auto some = [&](int kb, auto count) __attribute__((always_inline)) {   // reads go out together
                    constexpr int U = decltype(count)::value;
                    piece_t<T> fd[U], fw[U][TT];
#pragma unroll
                    for (int u = 0; u < U; ++u) {
                        fd[u] = ffn::by_row<T>(rows, (kb + u) * HT + tile % HT);
#pragma unroll
                        for (int s = 0; s < TT; ++s) fw[u][s] = w[((task * TT + s) * nbs + kb + u) * 64 + lane];
                    }
#pragma unroll
                    for (int u = 0; u < U; ++u)
#pragma unroll
                        for (int s = 0; s < TT; ++s) o[s] = mma(fw[u][s], fd[u], o[s]);
                };
                constexpr int U = TT == 1 ? 4 : S::HN * S::HK <= 4 ? 2 : 1;   // by the registers left
                int kb = 0;
                for (; kb + U <= nbs; kb += U) some(kb, std::integral_constant<int, U>{});
                for (; kb < nbs; ++kb) some(kb, std::integral_constant<int, 1>{});
                piece_t<T> v;
#pragma unroll
                for (int j = 0; j < E<T>; ++j) v[j] = (T)o[j / 4][j % 4];
                const int64_t row = b * STEP + tile / HT * KB<T> + ffn::perm<T>(tile % HT, r);
                const int col = task * TASK<T> + q * E<T>;
                if (row < a.rows && col < a.inner)
                    store_piece(static_cast<T*>(a.dx) + row * a.dx_stride, col, a.inner, v);
            }
            first += tasks;
        }
    };
    int turn = 0;
    read(group);
    form(group, 0);
    read(group + groups);
    for (int64_t b = group; b < steps; b += groups, turn ^= 1) {
        // one barrier a step: the other buffers' readers have passed it
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        const int64_t next = b + groups;
        auto advance = [&]() __attribute__((always_inline)) {
            if (next < steps) form(next, turn ^ 1);
            read(next + groups);
        };
        if (wave >= BWD_WAVES / 2) advance();
        multiply(b, turn);
        if (wave < BWD_WAVES / 2) advance();
    }
    if (!part) return;
    const int64_t n = a.dweight ? (int64_t)a.outer * a.inner : 0;
    part += group * (n + a.outer);
    // lane (q, r): dW rows 4 q .. of the tile, column r
    if (a.dweight)
#pragma unroll
        for (int i = 0; i < S::HN; ++i)
#pragma unroll
            for (int j = 0; j < S::HK; ++j) {
                const int fi = i * S::WN + wn, fj = j * S::WK + wk;
                const int kk = k0 + fj / HT * KB<T> + ffn::perm<T>(fj % HT, r);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int nn = n0 + fi / HT * KB<T> + ffn::perm<T>(fi % HT, 4 * q + e);
                    if (nn < a.outer && kk < a.inner) part[(int64_t)nn * a.inner + kk] = acc[i][j][e];
                }
            }
    if (k0 != 0) return;   // all threads
    __syncthreads();
    float* sums = reinterpret_cast<float*>(lds);   // [BWD_THREADS / NP][columns]
#pragma unroll
    for (int j = 0; j < E<T>; ++j) sums[tid / NP * (NP * E<T>) + cd + j] = db[j];
    __syncthreads();
    for (int c = tid; c < width; c += BWD_THREADS) {
        float t = 0.f;
        for (int p = 0; p < BWD_THREADS / NP; ++p) t += sums[p * NP * E<T> + c];
        part[n + n0 + c] = t;
    }
}

// How a backward call is split.  dy of another type than the products' becomes dz
// by itself first (own_dz).  Where a workgroup holds all of dW, and W^T beside it in
// LDS, one pass makes all gradients; else the pass makes dW in parts, dz goes to
// memory where an activation stands before it, and dx is a product of its own.
struct Plan {
    bool own_dz, all;
    int n, k;                 // of a part of dW
    int tiles, ktiles, groups;
    int dz_tx, dz_groups;
    int64_t dz_rows;
    size_t lds;
    int64_t dz_bytes, db_bytes, dw_bytes, dx_bytes;
    int64_t bytes() const { return dz_bytes + db_bytes + dw_bytes + dx_bytes; }
};
template <class T>
Plan plan(int64_t rows, int inner, int outer, int act, bool same_type) {
    Plan p{};
    auto aligned = [](int64_t n) { return (n + 15) / 16 * 16; };
    p.own_dz = !same_type;
    p.all = !p.own_dz && (sizeof(T) == 4 ? (outer <= 256 && inner <= 64) || (outer <= 64 && inner <= 256)
                                         : (outer <= 256 && inner <= 128) || (outer <= 128 && inner <= 256));
    // the shapes that there is code for
    if (inner <= 64) p.n = 256, p.k = 64;
    else if (outer <= 64) p.n = 64, p.k = 256;
    else if (sizeof(T) == 4) p.n = 256, p.k = 64;
    else if (inner <= 128 || outer > 128) p.n = 256, p.k = 128;
    else p.n = 128, p.k = 256;
    p.ktiles = (int)ceil_div(inner, p.k);
    p.tiles = (int)ceil_div(outer, p.n) * p.ktiles;
    p.groups = (int)std::min<int64_t>(ceil_div(rows, RB * KB<T>), std::max<int64_t>(CUS / p.tiles, 1));
    const int64_t n = ceil_div(std::min(outer, p.n), KB<T>) * KB<T>, k = ceil_div(std::min(inner, p.k), KB<T>) * KB<T>;
    // W^T, two steps of dz and x; the sums of db at the end
    const int64_t held = (p.all ? n * dx_tiles<T>(inner) * 16 : 0) + 2 * RB * KB<T> * (n + k);
    p.lds = (size_t)std::max<int64_t>(held * sizeof(T), BWD_THREADS * E<T> * 4);
    p.dw_bytes = aligned((int64_t)p.groups * ((int64_t)outer * inner + outer) * 4);
    if (p.own_dz) {
        p.dz_tx = 1;
        while (p.dz_tx < 256 && p.dz_tx * 8 < outer) p.dz_tx *= 2;
        p.dz_rows = std::max<int64_t>(ceil_div(rows, 1024), 4 * 256 / p.dz_tx);
        p.dz_groups = (int)ceil_div(rows, p.dz_rows);
        p.db_bytes = aligned((int64_t)p.dz_groups * outer * 4);
    }
    if (p.own_dz || (!p.all && act != LINEAR_NONE)) p.dz_bytes = aligned(rows * outer * (int64_t)sizeof(T));
    if (!p.all) p.dx_bytes = product_workspace<T>(rows, outer, inner);
    return p;
}

// dW, db (from dz as it is before it is rounded) and, by the plan, dx or dz.
template <class T>
void pass(hipStream_t s, const LinearGradArgs& a, const Plan& p, T* dz, float* part) {
    const unsigned grid = (unsigned)(p.groups * p.tiles);
    auto launch = [&](auto shape) {
        using S = decltype(shape);
        auto run = [&](auto act, auto zmx) {
            auto with = [&](auto xmx) {
                k_linear_bwd<T, S, act(), zmx(), xmx()>
                    <<<grid, BWD_THREADS, p.lds, s>>>(a, dz, part, p.tiles, p.ktiles);
            };
            if (a.x_scales) with(std::true_type{});
            else with(std::false_type{});
        };
        auto kept = [&](auto act) {
            if (a.z_scales) run(act, std::true_type{});
            else run(act, std::false_type{});
        };
        if (a.act == LINEAR_NONE) run(std::integral_constant<int, LINEAR_NONE>{}, std::false_type{});
        else if (a.act == LINEAR_SILU) kept(std::integral_constant<int, LINEAR_SILU>{});
        else kept(std::integral_constant<int, LINEAR_GELU>{});
    };
    if (p.k == 64) launch(BwdShape<256, 64>{});
    else if (p.n == 64) launch(BwdShape<64, 256>{});
    else if constexpr (sizeof(T) == 2) {
        if (p.k == 128) launch(BwdShape<256, 128>{});
        else launch(BwdShape<128, 256>{});
    }
}

template <class T>
void backward(hipStream_t s, LinearGradArgs a) {
    const Plan p = plan<T>(a.rows, a.inner, a.outer, a.act, a.y_dtype == a.dtype);
    T* dz = p.dz_bytes ? reinterpret_cast<T*>(a.ws) : nullptr;
    float* db_part = reinterpret_cast<float*>(a.ws + p.dz_bytes);
    float* part = reinterpret_cast<float*>(a.ws + p.dz_bytes + p.db_bytes);
    const bool dx = a.dx && a.rows > 0;
    if (p.own_dz) {
        float* sums = a.dbias ? db_part : nullptr;
        T* taken = dx || a.dweight ? dz : nullptr;
        if (p.dz_groups > 0) {
            if (a.z_scales) k_linear_dz<T, true><<<p.dz_groups, 256, 0, s>>>(a, taken, sums, p.dz_tx, p.dz_rows);
            else k_linear_dz<T, false><<<p.dz_groups, 256, 0, s>>>(a, taken, sums, p.dz_tx, p.dz_rows);
        }
        if (sums) fold<T>(s, sums, p.dz_groups, a.outer, 0, a.dbias, nullptr);
        a.dy = dz;
        a.dy_stride = a.outer;
        a.act = LINEAR_NONE;
        a.z = nullptr;
        a.z_scales = nullptr;
        a.dbias = nullptr;
    }
    LinearGradArgs g = a;
    if (!p.all) g.dx = nullptr;
    const bool sums = a.dweight || a.dbias, makes_dz = dz && !p.own_dz && dx;
    if (p.groups > 0 && (sums || makes_dz || g.dx)) pass<T>(s, g, p, makes_dz ? dz : nullptr, sums ? part : nullptr);
    if (sums) fold<T>(s, part, p.groups, a.dweight ? (int64_t)a.outer * a.inner : 0, a.outer, a.dweight, a.dbias);
    if (p.all || !dx) return;
    LinearArgs d{};
    d.rows = a.rows;
    d.inner = a.outer;
    d.outer = a.inner;
    d.x = dz ? dz : a.dy;
    d.x_stride = dz ? a.outer : a.dy_stride;
    d.w = a.w;
    d.w_stride = a.w_stride;
    d.act = LINEAR_NONE;
    d.y = a.dx;
    d.y_stride = a.dx_stride;
    d.y_dtype = a.dtype;
    d.ws = a.ws + p.dz_bytes + p.db_bytes + p.dw_bytes;
    product<T, T, false, true>(s, d);
}

}  // namespace linear

// One translation unit per type and direction.
template <class T, class Y, bool MX>
void linear_forward(hipStream_t s, const LinearArgs& a);
template <class T>
void linear_backward(hipStream_t s, const LinearGradArgs& a);

}  // namespace msp
