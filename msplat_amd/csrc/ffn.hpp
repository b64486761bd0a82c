// ffn.hpp — the gated feed-forward block, forward and backward:
//
//   g = x Wg^T   u = x Wu^T   h = a(g) * u   y = h Wd^T
//   dh = dy Wd   du = dh a(g)   dg = dh u a'(g)   dx = dg Wg + du Wu
//   dWg = dg^T x   dWu = du^T x   dWd = dy^T h
//
// a(v) = v sigmoid(z(v)), with z = v (SiLU) or z = 2 sqrt(2/pi) (v + 0.044715
// v^3) (GELU in its tanh form).  The rows are many and the width is at most
// 256, so g, u and h (rows x hidden) never go to memory: 12 bytes a hidden
// unit and row would cost more than the 6 dim operations that make them again.
//
// All products run on 16x16 matrix instructions with 32-bit sums.  Indices
// are taken in blocks of KB = 4 E (one 16-byte piece in each of the four
// 16-lane groups q = lane / 16): operand fragments hold, in lane (q, r = lane
// % 16), elements q E .. q E + E - 1 of row r.  A result holds, in lane (q,
// r), rows 4 q .. 4 q + 3 of column r.  Let tile s of a block take as its row
// r the block's index
//
//   perm(s, r) = (r / 4) E + 4 s + r % 4,
//
// then the HT = E / 4 result tiles of a block, side by side, are in each lane
// the elements q E .. q E + E - 1 of the block: the operand fragment of the
// next product.  So h goes from the first two products to the third in
// registers, and so do dg, du and h to the gradients.
//
// Weights are packed into fragments (1 KB each, zero beyond the matrices) by a
// small kernel first: each is used in up to three orders, and the pack takes
// up every width and stride.  In 16-bit types h, dg and du are rounded to the
// type for the next product, as the type's own matrix instructions take them;
// the error is of the size of the output's own rounding.
#pragma once

#include "nn.hpp"

#include <algorithm>
#include <type_traits>

namespace msp {
namespace ffn {

template <class T>
constexpr int HT = E<T> / 4;   // 16-row tiles of a block
template <class T>
constexpr int KB = 4 * E<T>;   // indices of a block

template <class T>
__device__ __forceinline__ int perm(int s, int r) {
    return (r >> 2) * E<T> + 4 * s + (r & 3);
}

__device__ __forceinline__ f32x4 mma(piece_t<__bf16> a, piece_t<__bf16> b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mma(piece_t<_Float16> a, piece_t<_Float16> b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mma(piece_t<float> a, piece_t<float> b, f32x4 c) {
#pragma unroll
    for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], b[i], c, 0, 0, 0);
    return c;
}

// The result tiles of a block as one piece.
template <class T>
__device__ __forceinline__ piece_t<T> join(const f32x4* t) {
    piece_t<T> o;
#pragma unroll
    for (int j = 0; j < E<T>; ++j) o[j] = (T)t[j / 4][j % 4];
    return o;
}

constexpr float LOG2E = 1.44269504088896341f;
constexpr float GELU_A = 1.59576912160573071f;             // 2 sqrt(2/pi)
constexpr float GELU_B = 0.0713548162726009f;              // 0.044715 * GELU_A

__device__ __forceinline__ float sigmoid_fast(float z) {
    return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(z * -LOG2E));
}
template <bool GELU>
__device__ __forceinline__ float act(float g) {
    return g * sigmoid_fast(GELU ? g * fmaf(g * g, GELU_B, GELU_A) : g);
}
// h, dg and du of one hidden unit, in place of g, u and dh.
template <bool GELU>
__device__ __forceinline__ void act_grad(float& g, float& u, float& dh) {
    const float s = sigmoid_fast(GELU ? g * fmaf(g * g, GELU_B, GELU_A) : g);
    const float a = g * s;
    const float da = fmaf(GELU ? a * fmaf(g * g, 3.f * GELU_B, GELU_A) : a, 1.f - s, s);
    const float h = a * u;
    g = dh * u * da;   // dg
    u = dh * a;        // du
    dh = h;            // h
}

// Fragments of the weights, block of hidden units after block: in a block the
// matrices in order, DK * HT fragments each.  Rows x contraction index:
// forward  0 Wg (hidden x dim)  1 Wu  2 Wd (dim x hidden)
// backward 0 Wg  1 Wu  2 Wd^T (hidden x dim)  3 Wg^T (dim x hidden)  4 Wu^T
template <class T>
__global__ __launch_bounds__(256) void k_ffn_pack(FfnArgs a, int dk, int hblocks, int mats, piece_t<T>* out) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int lane = (int)(i & 63), r = lane & 15, q = lane >> 4;
    const int64_t f = i >> 6;
    const int s = (int)(f % HT<T>), kb = (int)(f / HT<T> % dk);
    const int64_t bm = f / (HT<T> * dk);
    const int m = (int)(bm % mats), b = (int)(bm / mats);
    if (b >= hblocks) return;
    const bool hidden_rows = m < 2 || (mats == 5 && m == 2);
    const bool down = m == 2;
    const T* w = static_cast<const T*>(down ? a.w_down : (m == 1 || m == 4) ? a.w_up : a.w_gate);
    const int64_t stride = down ? a.down_stride : (m == 1 || m == 4) ? a.up_stride : a.gate_stride;
    piece_t<T> v = {};
#pragma unroll
    for (int j = 0; j < E<T>; ++j) {
        const int h = b * KB<T> + (hidden_rows ? perm<T>(s, r) : q * E<T> + j);
        const int d = kb * KB<T> + (hidden_rows ? q * E<T> + j : perm<T>(s, r));
        if (h < a.hidden && d < a.dim) v[j] = down ? w[d * stride + h] : w[h * stride + d];
    }
    out[i] = v;
}

// Copies n fragments (1 KB each) from memory to LDS without registers in
// between; a wave takes every waves-th.  They have arrived after the next
// __syncthreads.
template <class T>
__device__ __forceinline__ void fetch(const piece_t<T>* src, piece_t<T>* lds, int n) {
    const int lane = threadIdx.x & 63, waves = blockDim.x >> 6;
    for (int f = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); f < n; f += waves)
        __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(src + f * 64 + lane),
                                         (__attribute__((address_space(3))) void*)(lds + f * 64), 16, 0, 0);
}

// The pieces of R rows' operand fragments, in two steps (read_piece,
// settle_piece).  Only a width of one block may be less than a piece.
template <class T, int DK, int R>
__device__ __forceinline__ void read_rows(const void* base, int64_t stride, int64_t row0, int64_t rows, int dim, int q,
                                          piece_t<T> (&f)[R][DK]) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const T* row = static_cast<const T*>(base) + min(row0 + 16 * r, rows - 1) * stride;
#pragma unroll
        for (int kb = 0; kb < DK; ++kb)
            f[r][kb] = DK == 1 && dim < E<T> ? load_piece(row, q * E<T>, dim) : read_piece(row, kb * KB<T> + q * E<T>, dim);
    }
}
template <class T, int DK, int R>
__device__ __forceinline__ void settle_rows(int64_t row0, int64_t rows, int dim, int q, piece_t<T> (&f)[R][DK]) {
    if (DK == 1 && dim < E<T>) return;
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int kb = 0; kb < DK; ++kb)
            f[r][kb] = settle_piece<T>(f[r][kb], kb * KB<T> + q * E<T>, dim, row0 + 16 * r < rows);
}
template <class T, int DK, int R>
__device__ __forceinline__ void load_rows(const void* base, int64_t stride, int64_t row0, int64_t rows, int dim, int q,
                                          piece_t<T> (&f)[R][DK]) {
    read_rows<T, DK, R>(base, stride, row0, rows, dim, q, f);
    settle_rows<T, DK, R>(row0, rows, dim, q, f);
}

template <class T, int DK, int R>
__device__ __forceinline__ void store_rows(void* base, int64_t stride, int64_t row0, int64_t rows, int dim, int q,
                                           const f32x4 (&acc)[R][DK * HT<T>]) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int64_t row = row0 + 16 * r;
        if (row >= rows) continue;
#pragma unroll
        for (int kb = 0; kb < DK; ++kb) {
            const int k = kb * KB<T> + q * E<T>;
            if (k < dim) store_piece(static_cast<T*>(base) + row * stride, k, dim, join<T>(&acc[r][kb * HT<T>]));
        }
    }
}

// The two steps of a block of hidden units for R tiles of 16 rows: h from x,
// then its part of y.
template <class T, int DK, int R, bool GELU>
__device__ __forceinline__ void fwd_up(const piece_t<T>* up, const piece_t<T> (&xf)[R][DK], piece_t<T> (&h)[R]) {
    constexpr int F = DK * HT<T>;
    const int lane = threadIdx.x & 63;
    f32x4 g[R][HT<T>] = {}, u[R][HT<T>] = {};
#pragma unroll
    for (int f = 0; f < F; ++f) {
        const piece_t<T> wg = up[f * 64 + lane], wu = up[(F + f) * 64 + lane];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            g[r][f % HT<T>] = mma(wg, xf[r][f / HT<T>], g[r][f % HT<T>]);
            u[r][f % HT<T>] = mma(wu, xf[r][f / HT<T>], u[r][f % HT<T>]);
        }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
#pragma unroll
        for (int j = 0; j < E<T>; ++j) g[r][j / 4][j % 4] = act<GELU>(g[r][j / 4][j % 4]) * u[r][j / 4][j % 4];
        h[r] = join<T>(g[r]);
    }
}
template <class T, int F, int R>
__device__ __forceinline__ void fwd_down(const piece_t<T>* down, const piece_t<T> (&h)[R], f32x4 (&acc)[R][F]) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int f = 0; f < F; ++f) {
        const piece_t<T> wd = down[f * 64 + lane];
#pragma unroll
        for (int r = 0; r < R; ++r) acc[r][f] = mma(wd, h[r], acc[r][f]);
    }
}

// dg and du from x and dy, then their part of dx.
template <class T, int DK, int R, bool GELU>
__device__ __forceinline__ void dx_up(const piece_t<T>* up, const piece_t<T> (&xf)[R][DK], const piece_t<T> (&df)[R][DK],
                                      piece_t<T> (&dg)[R], piece_t<T> (&du)[R]) {
    constexpr int F = DK * HT<T>;
    const int lane = threadIdx.x & 63;
    f32x4 g[R][HT<T>] = {}, u[R][HT<T>] = {}, dh[R][HT<T>] = {};
#pragma unroll
    for (int f = 0; f < F; ++f) {
        const piece_t<T> wg = up[f * 64 + lane], wu = up[(F + f) * 64 + lane], wd = up[(2 * F + f) * 64 + lane];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            g[r][f % HT<T>] = mma(wg, xf[r][f / HT<T>], g[r][f % HT<T>]);
            u[r][f % HT<T>] = mma(wu, xf[r][f / HT<T>], u[r][f % HT<T>]);
            dh[r][f % HT<T>] = mma(wd, df[r][f / HT<T>], dh[r][f % HT<T>]);
        }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
#pragma unroll
        for (int j = 0; j < E<T>; ++j) {
            float vg = g[r][j / 4][j % 4], vu = u[r][j / 4][j % 4], vh = dh[r][j / 4][j % 4];
            act_grad<GELU>(vg, vu, vh);
            g[r][j / 4][j % 4] = vg;
            u[r][j / 4][j % 4] = vu;
        }
        dg[r] = join<T>(g[r]);
        du[r] = join<T>(u[r]);
    }
}
template <class T, int F, int R>
__device__ __forceinline__ void dx_down(const piece_t<T>* down, const piece_t<T> (&dg)[R], const piece_t<T> (&du)[R],
                                        f32x4 (&acc)[R][F]) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int f = 0; f < F; ++f) {
        const piece_t<T> wg = down[f * 64 + lane], wu = down[(F + f) * 64 + lane];
#pragma unroll
        for (int r = 0; r < R; ++r) acc[r][f] = mma(wu, du[r], mma(wg, dg[r], acc[r][f]));
    }
}

// A wave takes R tiles of 16 rows and walks the hidden units block by block.
// The workgroup's waves share a block's weights in LDS, in two areas: while
// one of the two steps of a block computes, the other's weights arrive.
template <class T, int DK, int R, int WAVES, bool GELU>
__global__ __launch_bounds__(64 * WAVES) void k_ffn_fwd(FfnArgs a, const piece_t<T>* packed, int hblocks) {
    constexpr int F = DK * HT<T>;
    __shared__ piece_t<T> up[2 * F * 64], down[F * 64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, q = lane >> 4;
    const int64_t row0 = ((int64_t)blockIdx.x * WAVES + wave) * (16 * R) + (lane & 15);
    fetch<T>(packed, up, 2 * F);
    piece_t<T> xf[R][DK], h[R];
    load_rows<T, DK, R>(a.x, a.x_stride, row0, a.rows, a.dim, q, xf);
    f32x4 acc[R][F] = {};
    __syncthreads();
    for (int b = 0; b < hblocks; ++b) {
        fetch<T>(packed + ((int64_t)b * 3 * F + 2 * F) * 64, down, F);
        fwd_up<T, DK, R, GELU>(up, xf, h);
        __syncthreads();
        if (b + 1 < hblocks) fetch<T>(packed + (int64_t)(b + 1) * 3 * F * 64, up, 2 * F);
        fwd_down<T, F, R>(down, h, acc);
        __syncthreads();
    }
    store_rows<T, DK, R>(a.out, a.out_stride, row0, a.rows, a.dim, q, acc);
}

template <class T, int DK, int R, int WAVES, bool GELU>
__global__ __launch_bounds__(64 * WAVES) void k_ffn_dx(FfnArgs a, const piece_t<T>* packed, int hblocks) {
    constexpr int F = DK * HT<T>;
    __shared__ piece_t<T> up[3 * F * 64], down[2 * F * 64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, q = lane >> 4;
    const int64_t row0 = ((int64_t)blockIdx.x * WAVES + wave) * (16 * R) + (lane & 15);
    fetch<T>(packed, up, 3 * F);
    piece_t<T> xf[R][DK], df[R][DK], dg[R], du[R];
    load_rows<T, DK, R>(a.x, a.x_stride, row0, a.rows, a.dim, q, xf);
    load_rows<T, DK, R>(a.dy, a.dy_stride, row0, a.rows, a.dim, q, df);
    f32x4 acc[R][F] = {};
    __syncthreads();
    for (int b = 0; b < hblocks; ++b) {
        fetch<T>(packed + ((int64_t)b * 5 * F + 3 * F) * 64, down, 2 * F);
        dx_up<T, DK, R, GELU>(up, xf, df, dg, du);
        __syncthreads();
        if (b + 1 < hblocks) fetch<T>(packed + (int64_t)(b + 1) * 5 * F * 64, up, 3 * F);
        dx_down<T, F, R>(down, dg, du, acc);
        __syncthreads();
    }
    store_rows<T, DK, R>(a.out, a.out_stride, row0, a.rows, a.dim, q, acc);
}

// The same where all packed weights fit in LDS: a workgroup loads them once,
// then its waves walk row tiles on their own, with no barrier that would hold
// all of them at the matrix or at the vector instructions at once.
template <class T, int DK, int R, int WAVES, bool GELU>
__global__ __launch_bounds__(64 * WAVES) void k_ffn_fwd_all(FfnArgs a, const piece_t<T>* packed, int hblocks) {
    constexpr int F = DK * HT<T>;
    extern __shared__ char smem[];
    piece_t<T>* w = reinterpret_cast<piece_t<T>*>(smem);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, q = lane >> 4;
    fetch<T>(packed, w, hblocks * 3 * F);
    __syncthreads();
    const int64_t step = (int64_t)gridDim.x * WAVES;
    int64_t row0 = ((int64_t)blockIdx.x * WAVES + wave) * (16 * R) + (lane & 15);
    piece_t<T> xf[R][DK], xn[R][DK], h[R];
    read_rows<T, DK, R>(a.x, a.x_stride, row0, a.rows, a.dim, q, xn);
    for (; row0 - (lane & 15) < a.rows; row0 += step * (16 * R)) {
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int kb = 0; kb < DK; ++kb) xf[r][kb] = xn[r][kb];
        settle_rows<T, DK, R>(row0, a.rows, a.dim, q, xf);
        read_rows<T, DK, R>(a.x, a.x_stride, row0 + step * (16 * R), a.rows, a.dim, q, xn);
        f32x4 acc[R][F] = {};
        for (int b = 0; b < hblocks; ++b) {
            fwd_up<T, DK, R, GELU>(w + b * 3 * F * 64, xf, h);
            fwd_down<T, F, R>(w + (b * 3 + 2) * F * 64, h, acc);
        }
        store_rows<T, DK, R>(a.out, a.out_stride, row0, a.rows, a.dim, q, acc);
    }
}

template <class T, int DK, int R, int WAVES, bool GELU>
__global__ __launch_bounds__(64 * WAVES) void k_ffn_dx_all(FfnArgs a, const piece_t<T>* packed, int hblocks) {
    constexpr int F = DK * HT<T>;
    extern __shared__ char smem[];
    piece_t<T>* w = reinterpret_cast<piece_t<T>*>(smem);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, q = lane >> 4;
    fetch<T>(packed, w, hblocks * 5 * F);
    __syncthreads();
    for (int64_t t = (int64_t)blockIdx.x * WAVES + wave; t * (16 * R) < a.rows; t += (int64_t)gridDim.x * WAVES) {
        const int64_t row0 = t * (16 * R) + (lane & 15);
        piece_t<T> xf[R][DK], df[R][DK], dg[R], du[R];
        load_rows<T, DK, R>(a.x, a.x_stride, row0, a.rows, a.dim, q, xf);
        load_rows<T, DK, R>(a.dy, a.dy_stride, row0, a.rows, a.dim, q, df);
        f32x4 acc[R][F] = {};
        for (int b = 0; b < hblocks; ++b) {
            dx_up<T, DK, R, GELU>(w + b * 5 * F * 64, xf, df, dg, du);
            dx_down<T, F, R>(w + (b * 5 + 3) * F * 64, dg, du, acc);
        }
        store_rows<T, DK, R>(a.out, a.out_stride, row0, a.rows, a.dim, q, acc);
    }
}

// Few rows: a workgroup takes R tiles of 16 rows, and its waves share out the
// hidden units; the waves' parts of y are added in LDS, half of the waves onto
// the other half until one is left, in the same order every time.  Weights
// come from the L2 cache into registers, each read once a workgroup.
template <class T, int F, int R, int WAVES>
__device__ __forceinline__ void add_waves(f32x4 (&acc)[R][F], f32x4* lds) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int n = WAVES / 2; n >= 1; n /= 2) {
        f32x4* mine = lds + (int64_t)(wave % n) * R * F * 64 + lane;
        if (wave >= n && wave < 2 * n) {
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int f = 0; f < F; ++f) mine[(r * F + f) * 64] = acc[r][f];
        }
        __syncthreads();
        if (wave < n) {
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int f = 0; f < F; ++f) acc[r][f] += mine[(r * F + f) * 64];
        }
        __syncthreads();
    }
}

// The forward reads the weights as they are: all three matrices' fragments lie
// along their rows.
template <class T, int DK, int R, int WAVES, bool GELU>
__global__ __launch_bounds__(64 * WAVES) void k_ffn_fwd_few(FfnArgs a, int hblocks) {
    constexpr int F = DK * HT<T>;
    __shared__ f32x4 sums[WAVES / 2 * R * F * 64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, q = lane >> 4, i = lane & 15;
    const int64_t row0 = (int64_t)blockIdx.x * (16 * R) + i;
    piece_t<T> xf[R][DK], h[R];
    load_rows<T, DK, R>(a.x, a.x_stride, row0, a.rows, a.dim, q, xf);
    f32x4 acc[R][F] = {};
    for (int b = wave; b < hblocks; b += WAVES) {
        piece_t<T> wg[F], wu[F], wd[F];
#pragma unroll
        for (int s = 0; s < HT<T>; ++s) {
            const int u = b * KB<T> + perm<T>(s, i), at = min(u, a.hidden - 1);
            const T* pg = static_cast<const T*>(a.w_gate) + at * a.gate_stride;
            const T* pu = static_cast<const T*>(a.w_up) + at * a.up_stride;
#pragma unroll
            for (int kb = 0; kb < DK; ++kb) {
                wg[kb * HT<T> + s] = load_piece(pg, kb * KB<T> + q * E<T>, a.dim);
                wu[kb * HT<T> + s] = load_piece(pu, kb * KB<T> + q * E<T>, a.dim);
                if (u >= a.hidden) wg[kb * HT<T> + s] = wu[kb * HT<T> + s] = piece_t<T>{};
            }
        }
#pragma unroll
        for (int f = 0; f < F; ++f) {
            const int d = f / HT<T> * KB<T> + perm<T>(f % HT<T>, i);
            wd[f] = load_piece(static_cast<const T*>(a.w_down) + min(d, a.dim - 1) * a.down_stride, b * KB<T> + q * E<T>, a.hidden);
            if (d >= a.dim) wd[f] = piece_t<T>{};
        }
        f32x4 g[R][HT<T>] = {}, u[R][HT<T>] = {};
#pragma unroll
        for (int f = 0; f < F; ++f)
#pragma unroll
            for (int r = 0; r < R; ++r) {
                g[r][f % HT<T>] = mma(wg[f], xf[r][f / HT<T>], g[r][f % HT<T>]);
                u[r][f % HT<T>] = mma(wu[f], xf[r][f / HT<T>], u[r][f % HT<T>]);
            }
#pragma unroll
        for (int r = 0; r < R; ++r) {
#pragma unroll
            for (int j = 0; j < E<T>; ++j) g[r][j / 4][j % 4] = act<GELU>(g[r][j / 4][j % 4]) * u[r][j / 4][j % 4];
            h[r] = join<T>(g[r]);
        }
#pragma unroll
        for (int f = 0; f < F; ++f)
#pragma unroll
            for (int r = 0; r < R; ++r) acc[r][f] = mma(wd[f], h[r], acc[r][f]);
    }
    add_waves<T, F, R, WAVES>(acc, sums);
    if (wave == 0) store_rows<T, DK, R>(a.out, a.out_stride, row0, a.rows, a.dim, q, acc);
}

template <class T, int DK, int R, int WAVES, bool GELU>
__global__ __launch_bounds__(64 * WAVES) void k_ffn_dx_few(FfnArgs a, const piece_t<T>* packed, int hblocks) {
    constexpr int F = DK * HT<T>;
    __shared__ f32x4 sums[WAVES / 2 * R * F * 64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, q = lane >> 4;
    const int64_t row0 = (int64_t)blockIdx.x * (16 * R) + (lane & 15);
    piece_t<T> xf[R][DK], df[R][DK], dg[R], du[R];
    load_rows<T, DK, R>(a.x, a.x_stride, row0, a.rows, a.dim, q, xf);
    load_rows<T, DK, R>(a.dy, a.dy_stride, row0, a.rows, a.dim, q, df);
    f32x4 acc[R][F] = {};
    for (int b = wave; b < hblocks; b += WAVES) {
        const piece_t<T>* w = packed + (int64_t)b * 5 * F * 64;
        dx_up<T, DK, R, GELU>(w, xf, df, dg, du);
        dx_down<T, F, R>(w + 3 * F * 64, dg, du, acc);
    }
    add_waves<T, F, R, WAVES>(acc, sums);
    if (wave == 0) store_rows<T, DK, R>(a.out, a.out_stride, row0, a.rows, a.dim, q, acc);
}

// A block of KB rows of x (or dy) in LDS, as operand fragments rows x dim: the
// piece of row perm(s, r), elements (4 kb + c) E ..., lies at slot(kb, s, c, r),
// whose order of rows turns with c so that by_dim's reads spread over the banks.
template <class T>
__device__ __forceinline__ int slot(int kb, int s, int c, int r) {
    return (kb * HT<T> + s) * 64 + c * 16 + (r ^ (sizeof(T) == 4 ? c : (c & 1) * 4));
}
template <class T>
__device__ __forceinline__ piece_t<T> by_row(const piece_t<T>* rows, int f) {
    const int lane = threadIdx.x & 63;
    return rows[slot<T>(0, 0, lane >> 4, lane & 15) + f * 64];
}
// The fragment dim x rows of 16 columns from 16 dt on, whose elements are
// consecutive rows: 16-bit types through the transposing LDS read, in which
// the lanes 4 k + i / 4 of 16 give lane i element i % 4 of their 8 bytes.
template <class T>
__device__ __forceinline__ piece_t<T> by_dim(const piece_t<T>* rows, int dt) {
    const int lane = threadIdx.x & 63, q = lane >> 4, j = lane & 15;
    piece_t<T> o;
    if constexpr (sizeof(T) == 2) {
        typedef short s16x4 __attribute__((ext_vector_type(4)));
        typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
        const char* base = reinterpret_cast<const char*>(rows + slot<T>(0, 0, (j & 3) >> 1, q * 4 + (j >> 2))) + (j & 1) * 8;
        base += (dt >> 1) * (2 * 64 * 16) + (dt & 1) * (2 * 16 * 16);
        s16x4 h[2];
#pragma unroll
        for (int s = 0; s < 2; ++s) h[s] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(base + s * 64 * 16));
        __builtin_memcpy(&o, h, 16);
    } else {
        const float* base = reinterpret_cast<const float*>(rows + dt * 64);
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = base[slot<T>(0, 0, j >> 2, q * 4 + e) * 4 + (j & 3)];
    }
    return o;
}

// Weight gradients: a wave owns NH tiles of 16 hidden units, keeps their
// weights and their rows of the three gradients in registers and walks a
// group's rows. The workgroup's waves share each block of rows in LDS, two
// blocks in turn: the next is on its way while one is computed.  Sums go to
// part[group][tile][matrix][dim tile][lane].
constexpr int DW_WAVES = 4;
// Tiles of hidden units a wave of the weight gradient takes, and waves a SIMD,
// by registers: 12 a tile and 16 columns of sums, as many again for 16-bit
// weights' halves.
template <class T>
constexpr int dw_tiles(int dk) {
    return sizeof(T) == 2 && dk <= 4 ? 2 : 1;
}
template <class T>
constexpr int dw_occupancy(int dk, int nh) {
    return dk * nh * (int)sizeof(T) <= 8 ? 2 : 1;
}

template <class T, int DK, int NH, int WAVES, bool GELU>
__global__ __launch_bounds__(64 * WAVES, WAVES / 4 * dw_occupancy<T>(DK, NH)) void k_ffn_dw(
    FfnArgs a, const piece_t<T>* packed, int hblocks, int slices, int64_t blocks_per_group, f32x4* part) {
    constexpr int F = DK * HT<T>;
    constexpr int ITEMS = (2 * F + WAVES - 1) / WAVES;   // pieces a thread brings
    __shared__ piece_t<T> xy[2][2 * F * 64];             // x, then dy
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int slice = blockIdx.x % slices, group = blockIdx.x / slices;
    const int tile0 = (slice * WAVES + wave) * NH, tiles = slices * WAVES * NH;
    piece_t<T> wg[NH][DK], wu[NH][DK], wd[NH][DK];
#pragma unroll
    for (int n = 0; n < NH; ++n) {
        const int b = (tile0 + n) / HT<T>, s = (tile0 + n) % HT<T>;
#pragma unroll
        for (int kb = 0; kb < DK; ++kb) {
            wg[n][kb] = wu[n][kb] = wd[n][kb] = piece_t<T>{};
            if (b < hblocks) {
                const piece_t<T>* p = packed + ((int64_t)b * 5 * F + kb * HT<T> + s) * 64 + lane;
                wg[n][kb] = p[0];
                wu[n][kb] = p[F * 64];
                wd[n][kb] = p[2 * F * 64];
            }
        }
    }
    f32x4 acc[3][NH][F] = {};
    const int64_t first = group * blocks_per_group * KB<T>;
    const int64_t last = min(a.rows, first + blocks_per_group * KB<T>);

    // a thread's pieces of a block: read, and on the next turn put into LDS
    piece_t<T> in[ITEMS];
    auto load = [&](int64_t row0) {
#pragma unroll
        for (int k = 0; k < ITEMS; ++k) {
            int i = k * 64 * WAVES + threadIdx.x;
            const bool y = i >= F * 64;
            i -= y ? F * 64 : 0;
            if (2 * F % WAVES != 0 && i >= F * 64) continue;
            const int64_t row = min(row0 + i / (DK * 4), a.rows - 1);
            const T* p = static_cast<const T*>(y ? a.dy : a.x) + row * (y ? a.dy_stride : a.x_stride);
            const int c = i % (DK * 4) * E<T>;
            in[k] = DK == 1 && a.dim < E<T> ? load_piece(p, c, a.dim) : read_piece(p, c, a.dim);
        }
    };
    auto store = [&](piece_t<T>* to, int64_t row0) {
#pragma unroll
        for (int k = 0; k < ITEMS; ++k) {
            int i = k * 64 * WAVES + threadIdx.x;
            const bool y = i >= F * 64;
            i -= y ? F * 64 : 0;
            if (2 * F % WAVES != 0 && i >= F * 64) continue;
            const int w = i / (DK * 4), ch = i % (DK * 4);   // w = perm(s, r)
            const int s = HT<T> == 2 ? (w >> 2) & 1 : 0, r = w / E<T> * 4 + (w & 3);
            piece_t<T> v = in[k];
            if (DK == 1 && a.dim < E<T>) v = row0 + w < last ? v : piece_t<T>{};
            else v = settle_piece<T>(v, ch * E<T>, a.dim, row0 + w < last);
            to[(y ? F * 64 : 0) + slot<T>(ch >> 2, s, ch & 3, r)] = v;
        }
    };
    load(first);
    store(xy[0], first);
    load(first + KB<T>);
    __syncthreads();
    int cur = 0;
    for (int64_t row0 = first; row0 < last; row0 += KB<T>, cur ^= 1) {
        store(xy[cur ^ 1], row0 + KB<T>);
        load(row0 + 2 * KB<T>);
        const piece_t<T>*x = xy[cur], *y = xy[cur] + F * 64;
        f32x4 g[NH][HT<T>] = {}, u[NH][HT<T>] = {}, h[NH][HT<T>] = {};
#pragma unroll
        for (int f = 0; f < F; ++f) {
            const piece_t<T> px = by_row<T>(x, f), py = by_row<T>(y, f);
#pragma unroll
            for (int n = 0; n < NH; ++n) {
                g[n][f % HT<T>] = mma(px, wg[n][f / HT<T>], g[n][f % HT<T>]);
                u[n][f % HT<T>] = mma(px, wu[n][f / HT<T>], u[n][f % HT<T>]);
                h[n][f % HT<T>] = mma(py, wd[n][f / HT<T>], h[n][f % HT<T>]);
            }
        }
        piece_t<T> pg[NH], pu[NH], ph[NH];
#pragma unroll
        for (int n = 0; n < NH; ++n) {
#pragma unroll
            for (int j = 0; j < E<T>; ++j) {
                float vg = g[n][j / 4][j % 4], vu = u[n][j / 4][j % 4], vh = h[n][j / 4][j % 4];
                act_grad<GELU>(vg, vu, vh);
                g[n][j / 4][j % 4] = vg;
                u[n][j / 4][j % 4] = vu;
                h[n][j / 4][j % 4] = vh;
            }
            pg[n] = join<T>(g[n]);
            pu[n] = join<T>(u[n]);
            ph[n] = join<T>(h[n]);
        }
#pragma unroll
        for (int f = 0; f < F; ++f) {
            const piece_t<T> px = by_dim<T>(x, f), py = by_dim<T>(y, f);
#pragma unroll
            for (int n = 0; n < NH; ++n) {
                acc[0][n][f] = mma(pg[n], px, acc[0][n][f]);
                acc[1][n][f] = mma(pu[n], px, acc[1][n][f]);
                acc[2][n][f] = mma(ph[n], py, acc[2][n][f]);
            }
        }
        __syncthreads();
    }
#pragma unroll
    for (int n = 0; n < NH; ++n)
#pragma unroll
        for (int m = 0; m < 3; ++m)
#pragma unroll
            for (int f = 0; f < F; ++f)
                part[((((int64_t)group * tiles + tile0 + n) * 3 + m) * F + f) * 64 + lane] = acc[m][n][f];
}

// Adds the groups' sums in a fixed order and writes the gradients: a workgroup
// per fragment, 16 waves over the groups.  A lane has four consecutive hidden
// units of one column.
template <class T>
__global__ __launch_bounds__(1024) void k_ffn_fold(FfnArgs a, const f32x4* part, int groups, int tiles, int fr) {
    __shared__ f32x4 red[16][64];
    const int lane = threadIdx.x & 63, sl = threadIdx.x >> 6;
    const int64_t per = (int64_t)tiles * 3 * fr * 64, i = (int64_t)blockIdx.x * 64 + lane;
    f32x4 t = {};
#pragma unroll 4
    for (int g = sl; g < groups; g += 16) t += part[g * per + i];
    red[sl][lane] = t;
    __syncthreads();
    if (sl != 0) return;
#pragma unroll
    for (int k = 1; k < 16; ++k) t += red[k][lane];
    const int f = blockIdx.x % fr, m = blockIdx.x / fr % 3, tile = blockIdx.x / fr / 3;
    const int d = f * 16 + (lane & 15);
    const int h0 = tile / HT<T> * KB<T> + perm<T>(tile % HT<T>, (lane >> 4) * 4);
    if (d >= a.dim) return;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        if (h0 + k >= a.hidden) return;
        if (m == 0) static_cast<T*>(a.dw_gate)[(int64_t)(h0 + k) * a.dim + d] = (T)t[k];
        if (m == 1) static_cast<T*>(a.dw_up)[(int64_t)(h0 + k) * a.dim + d] = (T)t[k];
        if (m == 2) static_cast<T*>(a.dw_down)[(int64_t)d * a.hidden + h0 + k] = (T)t[k];
    }
}

// Blocks of the width that a kernel is made for, for a width of `dim`.
template <class T>
inline int dim_blocks(int dim) {
    const int n = (dim + KB<T> - 1) / KB<T>;
    constexpr int made[] = {1, 2, 3, 4, 6, 8, 12, 16};
    for (int m : made)
        if (n <= m) return m;
    return 0;
}
template <class T, class F>
inline void with_blocks(int dim, F&& f) {
#define BLOCKS(n) \
    case n: f(std::integral_constant<int, n>{}); break
    switch (dim_blocks<T>(dim)) {
        BLOCKS(1);
        BLOCKS(2);
        BLOCKS(3);
        BLOCKS(4);
        BLOCKS(6);
        BLOCKS(8);
        default:
            if constexpr (sizeof(T) == 4) {
                if (dim_blocks<T>(dim) == 12) f(std::integral_constant<int, 12>{});
                else f(std::integral_constant<int, 16>{});
            }
    }
#undef BLOCKS
}

// How the weight gradient is split: NH hidden tiles a wave, workgroups over
// slices of hidden tiles and over groups of rows, as many of them as are
// resident at once.
struct Split {
    int nh, slices, groups, tiles;
    int64_t blocks_per_group;
};
template <class T>
inline Split dw_split(int64_t rows, int dim, int hidden) {
    Split p;
    const int dk = dim_blocks<T>(dim);
    const int tiles = (hidden + KB<T> - 1) / KB<T> * HT<T>;
    p.nh = tiles > DW_WAVES ? dw_tiles<T>(dk) : 1;
    p.slices = (tiles + DW_WAVES * p.nh - 1) / (DW_WAVES * p.nh);
    p.tiles = p.slices * DW_WAVES * p.nh;
    const int64_t blocks = (rows + KB<T> - 1) / KB<T>;
    int64_t groups = 1024 / DW_WAVES * dw_occupancy<T>(dk, p.nh) / p.slices;
    groups = groups < 1 ? 1 : groups;
    groups = groups > (blocks + 3) / 4 ? (blocks + 3) / 4 : groups;
    p.blocks_per_group = groups ? (blocks + groups - 1) / groups : 0;
    p.groups = p.blocks_per_group ? (int)((blocks + p.blocks_per_group - 1) / p.blocks_per_group) : 0;
    return p;
}

template <class T>
size_t packed_bytes(int dim, int hidden, int mats) {
    return (size_t)((hidden + KB<T> - 1) / KB<T>) * mats * dim_blocks<T>(dim) * HT<T> * 1024;
}

template <class T>
size_t workspace(int64_t rows, int dim, int hidden, bool backward) {
    if (!backward) return packed_bytes<T>(dim, hidden, 3);
    const Split p = dw_split<T>(rows, dim, hidden);
    return packed_bytes<T>(dim, hidden, 5) + (size_t)p.groups * p.tiles * 3 * dim_blocks<T>(dim) * HT<T> * 1024;
}

template <class T>
piece_t<T>* pack(hipStream_t s, const FfnArgs& a, int dk, int hblocks, int mats) {
    piece_t<T>* packed = reinterpret_cast<piece_t<T>*>(a.ws);
    const int64_t n = (int64_t)hblocks * mats * dk * HT<T> * 64;
    k_ffn_pack<T><<<(unsigned)((n + 255) / 256), 256, 0, s>>>(a, dk, hblocks, mats, packed);
    return packed;
}

constexpr int64_t CUS = 256;
constexpr size_t LDS_BYTES = 160 * 1024;
inline unsigned groups_of(int64_t rows, int64_t each) { return (unsigned)((rows + each - 1) / each); }

// Rows up to which a workgroup takes one or two row tiles for all hidden units
// (k_ffn_*_few): as long as every one of them finds a CU free, twice that
// where two fit on one.
inline int64_t few_rows(int fragments) { return 32 * CUS * (fragments <= 4 ? 2 : 1); }

// Workgroups of k_ffn_*_all: as many as are resident at once (16 waves a CU by
// registers), or fewer for fewer rows.
inline unsigned resident_groups(int64_t rows, int64_t each, int waves, size_t lds) {
    const int64_t fit = std::min<int64_t>((int64_t)(LDS_BYTES / lds), 16 / waves) * CUS;
    return (unsigned)std::min<int64_t>(fit, (rows + each - 1) / each);
}

template <class F>
inline void with_act(const FfnArgs& a, F&& f) {
    if (a.gelu) f(std::true_type{});
    else f(std::false_type{});
}

template <class T>
void forward(hipStream_t s, const FfnArgs& a) {
    with_blocks<T>(a.dim, [&](auto dk) {
        with_act(a, [&](auto gelu) {
            constexpr int F = dk() * HT<T>;
            const int hblocks = (a.hidden + KB<T> - 1) / KB<T>;
            if (a.rows <= 16 * CUS) {
                k_ffn_fwd_few<T, dk(), 1, 8, gelu()><<<groups_of(a.rows, 16), 512, 0, s>>>(a, hblocks);
                return;
            }
            if (a.rows <= few_rows(F)) {
                k_ffn_fwd_few<T, dk(), 2, 8, gelu()><<<groups_of(a.rows, 32), 512, 0, s>>>(a, hblocks);
                return;
            }
            const piece_t<T>* packed = pack<T>(s, a, dk(), hblocks, 3);
            const size_t lds = packed_bytes<T>(a.dim, a.hidden, 3);
            if constexpr (F <= 4) {
                if (lds <= LDS_BYTES) {
                    k_ffn_fwd_all<T, dk(), 2, 16, gelu()><<<resident_groups(a.rows, 32 * 16, 16, lds), 1024, lds, s>>>(
                        a, packed, hblocks);
                    return;
                }
            }
            k_ffn_fwd<T, dk(), 2, 8, gelu()><<<groups_of(a.rows, 32 * 8), 512, 0, s>>>(a, packed, hblocks);
        });
    });
}

template <class T, int DK, bool GELU>
void input_gradient(hipStream_t s, const FfnArgs& a, const piece_t<T>* packed, int hblocks) {
    constexpr int F = DK * HT<T>;
    if (a.rows <= 16 * CUS) {
        k_ffn_dx_few<T, DK, 1, 8, GELU><<<groups_of(a.rows, 16), 512, 0, s>>>(a, packed, hblocks);
        return;
    }
    if (a.rows <= few_rows(F)) {
        k_ffn_dx_few<T, DK, 2, 8, GELU><<<groups_of(a.rows, 32), 512, 0, s>>>(a, packed, hblocks);
        return;
    }
    const size_t lds = packed_bytes<T>(a.dim, a.hidden, 5);
    if constexpr (F <= 4) {
        if (lds <= LDS_BYTES) {
            k_ffn_dx_all<T, DK, 2, 8, GELU><<<resident_groups(a.rows, 32 * 8, 8, lds), 512, lds, s>>>(a, packed, hblocks);
            return;
        }
    }
    constexpr int W = F <= 8 ? 8 : 4;
    k_ffn_dx<T, DK, 2, W, GELU><<<groups_of(a.rows, 32 * W), 64 * W, 0, s>>>(a, packed, hblocks);
}

template <class T>
void backward(hipStream_t s, const FfnArgs& a) {
    with_blocks<T>(a.dim, [&](auto dk) {
        constexpr int F = dk() * HT<T>;
        const int hblocks = (a.hidden + KB<T> - 1) / KB<T>;
        const piece_t<T>* packed = pack<T>(s, a, dk(), hblocks, 5);
        if (a.out && a.rows > 0)
            with_act(a, [&](auto gelu) { input_gradient<T, dk(), gelu()>(s, a, packed, hblocks); });
        if (!a.dw_gate) return;
        const Split p = dw_split<T>(a.rows, a.dim, a.hidden);
        f32x4* part = reinterpret_cast<f32x4*>(a.ws + packed_bytes<T>(a.dim, a.hidden, 5));
        auto dw = [&](auto nh) {
            with_act(a, [&](auto gelu) {
                k_ffn_dw<T, dk(), nh(), DW_WAVES, gelu()><<<(unsigned)(p.groups * p.slices), 64 * DW_WAVES, 0, s>>>(
                    a, packed, hblocks, p.slices, p.blocks_per_group, part);
            });
        };
        if (p.groups > 0) {
            if (p.nh == 1) dw(std::integral_constant<int, 1>{});
            else if constexpr (dw_tiles<T>(dk()) == 2) dw(std::integral_constant<int, 2>{});
        }
        k_ffn_fold<T><<<(unsigned)(p.tiles * 3 * F), 1024, 0, s>>>(a, part, p.groups, p.tiles, F);
    });
}

}  // namespace ffn

// One translation unit per type and direction.
template <class T>
void ffn_forward(hipStream_t s, const FfnArgs& a);
template <class T>
void ffn_backward(hipStream_t s, const FfnArgs& a);

}  // namespace msp
