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
    const float slope = GELU ? fmaf(g * g, 3.f * GELU_B, GELU_A) : 1.f;
    const float da = fmaf(a * (1.f - s), slope, s);
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

constexpr int WAVES = 4;

// A wave takes R tiles of 16 rows and walks the hidden units block by block;
// the workgroup's four waves share a block's weights in LDS.
template <class T, int DK, int R, bool GELU>
__global__ __launch_bounds__(64 * WAVES) void k_ffn_fwd(FfnArgs a, const piece_t<T>* packed, int hblocks) {
    constexpr int F = DK * HT<T>;
    __shared__ piece_t<T> lds[3 * F * 64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, q = lane >> 4;
    const int64_t row0 = ((int64_t)blockIdx.x * WAVES + wave) * (16 * R) + (lane & 15);
    piece_t<T> xf[R][DK];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int kb = 0; kb < DK; ++kb) {
            const int64_t row = row0 + 16 * r;
            xf[r][kb] = piece_t<T>{};
            if (row < a.rows)
                xf[r][kb] = load_piece(static_cast<const T*>(a.x) + row * a.x_stride, kb * KB<T> + q * E<T>, a.dim);
        }
    f32x4 acc[R][F] = {};
    for (int b = 0; b < hblocks; ++b) {
        __syncthreads();
        for (int i = threadIdx.x; i < 3 * F * 64; i += 64 * WAVES) lds[i] = packed[(int64_t)b * 3 * F * 64 + i];
        __syncthreads();
        f32x4 g[R][HT<T>] = {}, u[R][HT<T>] = {};
#pragma unroll
        for (int f = 0; f < F; ++f) {
            const piece_t<T> wg = lds[f * 64 + lane], wu = lds[(F + f) * 64 + lane];
#pragma unroll
            for (int r = 0; r < R; ++r) {
                g[r][f % HT<T>] = mma(wg, xf[r][f / HT<T>], g[r][f % HT<T>]);
                u[r][f % HT<T>] = mma(wu, xf[r][f / HT<T>], u[r][f % HT<T>]);
            }
        }
        piece_t<T> h[R];
#pragma unroll
        for (int r = 0; r < R; ++r) {
#pragma unroll
            for (int j = 0; j < E<T>; ++j) g[r][j / 4][j % 4] = act<GELU>(g[r][j / 4][j % 4]) * u[r][j / 4][j % 4];
            h[r] = join<T>(g[r]);
        }
#pragma unroll
        for (int f = 0; f < F; ++f) {
            const piece_t<T> wd = lds[(2 * F + f) * 64 + lane];
#pragma unroll
            for (int r = 0; r < R; ++r) acc[r][f] = mma(wd, h[r], acc[r][f]);
        }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int64_t row = row0 + 16 * r;
        if (row >= a.rows) continue;
#pragma unroll
        for (int kb = 0; kb < DK; ++kb) {
            const int k = kb * KB<T> + q * E<T>;
            if (k < a.dim)
                store_piece(static_cast<T*>(a.out) + row * a.out_stride, k, a.dim, join<T>(&acc[r][kb * HT<T>]));
        }
    }
}

// dx: as the forward, with g, u and dh made from x and dy and two products
// behind them.
template <class T, int DK, int R, bool GELU>
__global__ __launch_bounds__(64 * WAVES) void k_ffn_dx(FfnArgs a, const piece_t<T>* packed, int hblocks) {
    constexpr int F = DK * HT<T>;
    __shared__ piece_t<T> lds[5 * F * 64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, q = lane >> 4;
    const int64_t row0 = ((int64_t)blockIdx.x * WAVES + wave) * (16 * R) + (lane & 15);
    piece_t<T> xf[R][DK], df[R][DK];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int kb = 0; kb < DK; ++kb) {
            const int64_t row = row0 + 16 * r;
            const int k = kb * KB<T> + q * E<T>;
            xf[r][kb] = df[r][kb] = piece_t<T>{};
            if (row < a.rows) {
                xf[r][kb] = load_piece(static_cast<const T*>(a.x) + row * a.x_stride, k, a.dim);
                df[r][kb] = load_piece(static_cast<const T*>(a.dy) + row * a.dy_stride, k, a.dim);
            }
        }
    f32x4 acc[R][F] = {};
    for (int b = 0; b < hblocks; ++b) {
        __syncthreads();
        for (int i = threadIdx.x; i < 5 * F * 64; i += 64 * WAVES) lds[i] = packed[(int64_t)b * 5 * F * 64 + i];
        __syncthreads();
        f32x4 g[R][HT<T>] = {}, u[R][HT<T>] = {}, dh[R][HT<T>] = {};
#pragma unroll
        for (int f = 0; f < F; ++f) {
            const piece_t<T> wg = lds[f * 64 + lane], wu = lds[(F + f) * 64 + lane], wd = lds[(2 * F + f) * 64 + lane];
#pragma unroll
            for (int r = 0; r < R; ++r) {
                g[r][f % HT<T>] = mma(wg, xf[r][f / HT<T>], g[r][f % HT<T>]);
                u[r][f % HT<T>] = mma(wu, xf[r][f / HT<T>], u[r][f % HT<T>]);
                dh[r][f % HT<T>] = mma(wd, df[r][f / HT<T>], dh[r][f % HT<T>]);
            }
        }
        piece_t<T> dg[R], du[R];
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
#pragma unroll
        for (int f = 0; f < F; ++f) {
            const piece_t<T> wg = lds[(3 * F + f) * 64 + lane], wu = lds[(4 * F + f) * 64 + lane];
#pragma unroll
            for (int r = 0; r < R; ++r) acc[r][f] = mma(wu, du[r], mma(wg, dg[r], acc[r][f]));
        }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int64_t row = row0 + 16 * r;
        if (row >= a.rows) continue;
#pragma unroll
        for (int kb = 0; kb < DK; ++kb) {
            const int k = kb * KB<T> + q * E<T>;
            if (k < a.dim)
                store_piece(static_cast<T*>(a.out) + row * a.out_stride, k, a.dim, join<T>(&acc[r][kb * HT<T>]));
        }
    }
}

// Both operand forms of a block of KB rows of x (or dy) in LDS: `by_row`
// fragments (rows x dim) and `by_dim` fragments (dim x rows), whose elements
// are consecutive rows.  A thread takes rows in pairs (16-bit types), so that
// the transposed form is written in 4-byte words.
template <class T, int DK>
__device__ __forceinline__ void stage_rows(const T* src, int64_t stride, int64_t row0, int64_t rows, int dim,
                                           piece_t<T>* by_row, piece_t<T>* by_dim) {
    constexpr int PER = 4 / (int)sizeof(T);   // rows of a 4-byte word
    constexpr int GROUPS = KB<T> / PER;       // 16
    for (int i = threadIdx.x; i < GROUPS * DK * 4; i += blockDim.x) {
        const int rho = (i % GROUPS) * PER, ch = i / GROUPS;
        piece_t<T> p[PER];
#pragma unroll
        for (int e = 0; e < PER; ++e) {
            p[e] = piece_t<T>{};
            if (row0 + rho + e < rows) p[e] = load_piece(src + (row0 + rho + e) * stride, ch * E<T>, dim);
            const int w = rho + e;   // = perm(s, r)
            const int s = HT<T> == 2 ? (w >> 2) & 1 : 0, r = w / E<T> * 4 + (w & 3);
            by_row[((ch >> 2) * HT<T> + s) * 64 + (ch & 3) * 16 + r] = p[e];
        }
        T* t = reinterpret_cast<T*>(by_dim);
#pragma unroll
        for (int j = 0; j < E<T>; ++j) {
            const int d = ch * E<T> + j;
            T* at = t + ((d >> 4) * 64 + rho / E<T> * 16 + (d & 15)) * E<T> + rho % E<T>;
#pragma unroll
            for (int e = 0; e < PER; ++e) at[e] = p[e][j];
        }
    }
}

// Weight gradients: a wave owns NH tiles of 16 hidden units, keeps their
// weights and their rows of the three gradients in registers and walks a
// group's rows; the workgroup's waves share each block of rows in LDS.  Sums
// go to part[group][tile][matrix][dim tile][lane].
template <class T, int DK, int NH, bool GELU>
__global__ __launch_bounds__(64 * WAVES) void k_ffn_dw(FfnArgs a, const piece_t<T>* packed, int hblocks, int slices,
                                                       int64_t blocks_per_group, f32x4* part) {
    constexpr int F = DK * HT<T>;
    __shared__ piece_t<T> xr[F * 64], xd[F * 64], yr[F * 64], yd[F * 64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
    const int slice = blockIdx.x % slices, group = blockIdx.x / slices;
    const int tile0 = (slice * waves + wave) * NH, tiles = slices * waves * NH;
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
    for (int64_t row0 = first; row0 < last; row0 += KB<T>) {
        __syncthreads();
        stage_rows<T, DK>(static_cast<const T*>(a.x), a.x_stride, row0, a.rows, a.dim, xr, xd);
        stage_rows<T, DK>(static_cast<const T*>(a.dy), a.dy_stride, row0, a.rows, a.dim, yr, yd);
        __syncthreads();
        f32x4 g[NH][HT<T>] = {}, u[NH][HT<T>] = {}, h[NH][HT<T>] = {};
#pragma unroll
        for (int f = 0; f < F; ++f) {
            const piece_t<T> x = xr[f * 64 + lane], y = yr[f * 64 + lane];
#pragma unroll
            for (int n = 0; n < NH; ++n) {
                g[n][f % HT<T>] = mma(x, wg[n][f / HT<T>], g[n][f % HT<T>]);
                u[n][f % HT<T>] = mma(x, wu[n][f / HT<T>], u[n][f % HT<T>]);
                h[n][f % HT<T>] = mma(y, wd[n][f / HT<T>], h[n][f % HT<T>]);
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
            const piece_t<T> x = xd[f * 64 + lane], y = yd[f * 64 + lane];
#pragma unroll
            for (int n = 0; n < NH; ++n) {
                acc[0][n][f] = mma(pg[n], x, acc[0][n][f]);
                acc[1][n][f] = mma(pu[n], x, acc[1][n][f]);
                acc[2][n][f] = mma(ph[n], y, acc[2][n][f]);
            }
        }
    }
#pragma unroll
    for (int n = 0; n < NH; ++n)
#pragma unroll
        for (int m = 0; m < 3; ++m)
#pragma unroll
            for (int f = 0; f < F; ++f)
                part[((((int64_t)group * tiles + tile0 + n) * 3 + m) * F + f) * 64 + lane] = acc[m][n][f];
}

// Adds the groups' sums in order and writes the gradients.  A thread has four
// consecutive hidden units of one column.
template <class T>
__global__ __launch_bounds__(256) void k_ffn_fold(FfnArgs a, const f32x4* part, int groups, int tiles, int fr) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t per = (int64_t)tiles * 3 * fr * 64;
    if (i >= per) return;
    f32x4 t = {};
    for (int g = 0; g < groups; ++g) t += part[g * per + i];
    const int lane = (int)(i & 63), f = (int)(i / 64 % fr), m = (int)(i / 64 / fr % 3);
    const int tile = (int)(i / 64 / fr / 3);
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

// How the weight gradient is split: workgroups over slices of hidden tiles
// and over groups of rows, enough of them to fill the GPU.
struct Split {
    int nh, waves, slices, groups, tiles;
    int64_t blocks_per_group;
};
template <class T>
inline Split dw_split(int64_t rows, int dim, int hidden) {
    Split p;
    p.nh = dim_blocks<T>(dim) * (int)sizeof(T) <= 8 && sizeof(T) == 2 ? 2 : 1;
    const int want = ((hidden + KB<T> - 1) / KB<T> * HT<T> + p.nh - 1) / p.nh;
    p.waves = want < WAVES ? want : WAVES;
    p.slices = (want + p.waves - 1) / p.waves;
    p.tiles = p.slices * p.waves * p.nh;
    const int64_t blocks = (rows + KB<T> - 1) / KB<T>;
    int64_t groups = 2048 / (p.slices * p.waves);
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

template <class T>
void forward(hipStream_t s, const FfnArgs& a) {
    with_blocks<T>(a.dim, [&](auto dk) {
        constexpr int R = 2;
        const int hblocks = (a.hidden + KB<T> - 1) / KB<T>;
        const piece_t<T>* packed = pack<T>(s, a, dk(), hblocks, 3);
        const unsigned grid = (unsigned)((a.rows + 16 * R * WAVES - 1) / (16 * R * WAVES));
        if (a.gelu) k_ffn_fwd<T, dk(), R, true><<<grid, 64 * WAVES, 0, s>>>(a, packed, hblocks);
        else k_ffn_fwd<T, dk(), R, false><<<grid, 64 * WAVES, 0, s>>>(a, packed, hblocks);
    });
}

template <class T>
void backward(hipStream_t s, const FfnArgs& a) {
    with_blocks<T>(a.dim, [&](auto dk) {
        constexpr int R = dk() * sizeof(T) <= 8 ? 2 : 1;
        constexpr int F = dk() * HT<T>;
        constexpr int NH = dk() * sizeof(T) <= 8 && sizeof(T) == 2 ? 2 : 1;
        const int hblocks = (a.hidden + KB<T> - 1) / KB<T>;
        const piece_t<T>* packed = pack<T>(s, a, dk(), hblocks, 5);
        if (a.out && a.rows > 0) {
            const unsigned grid = (unsigned)((a.rows + 16 * R * WAVES - 1) / (16 * R * WAVES));
            if (a.gelu) k_ffn_dx<T, dk(), R, true><<<grid, 64 * WAVES, 0, s>>>(a, packed, hblocks);
            else k_ffn_dx<T, dk(), R, false><<<grid, 64 * WAVES, 0, s>>>(a, packed, hblocks);
        }
        if (!a.dw_gate) return;
        const Split p = dw_split<T>(a.rows, a.dim, a.hidden);
        f32x4* part = reinterpret_cast<f32x4*>(a.ws + packed_bytes<T>(a.dim, a.hidden, 5));
        if (p.groups > 0) {
            const unsigned grid = (unsigned)(p.groups * p.slices);
            if (a.gelu) k_ffn_dw<T, dk(), NH, true><<<grid, 64 * p.waves, 0, s>>>(a, packed, hblocks, p.slices, p.blocks_per_group, part);
            else k_ffn_dw<T, dk(), NH, false><<<grid, 64 * p.waves, 0, s>>>(a, packed, hblocks, p.slices, p.blocks_per_group, part);
        }
        const int64_t n = (int64_t)p.tiles * 3 * F * 64;
        k_ffn_fold<T><<<(unsigned)((n + 255) / 256), 256, 0, s>>>(a, part, p.groups, p.tiles, F);
    });
}

}  // namespace ffn

// One translation unit per type and direction.
template <class T>
void ffn_forward(hipStream_t s, const FfnArgs& a);
template <class T>
void ffn_backward(hipStream_t s, const FfnArgs& a);

}  // namespace msp
