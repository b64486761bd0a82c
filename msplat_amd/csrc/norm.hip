// norm.hip — layer norm over the last axis, forward and backward.
//
//   mu = mean(x)   v = mean((x - mu)^2)   r = 1 / sqrt(v + eps)   n = (x - mu) r
//   y  = n w + b
//   dx = r (g - mean(g) - n mean(g n)),  g = dy w
//   dw = sum over rows of dy n,  db = sum over rows of dy
//
// Bound by HBM: a row is read once, kept in registers (rows.hpp) and written
// once.  The variance is the mean of squared differences, a second pass over
// registers, so that it does not cancel.
//   forward, 1.09M rows of 64 bf16: 50 us, 5.8 TB/s (a large copy 5.1)
//   backward, 500k rows of 128 bf16: 71 us, 5.4 TB/s, and 5 us for the sums
//   backward, 120k rows of 45 f32 (180 bytes, off the 16-byte grid): 15 + 4 us
#include "rows.hpp"

namespace msp {
namespace {

using namespace rows;

// Workgroups of the backward: each leaves a partial row.  512 left too few
// reads under way (500k rows of 128 bf16: 105 us, 1024: 71, 2048: 74).
constexpr int MAX_GROUPS = 1024;

template <class T, int L, int NV>
__global__ __launch_bounds__(THREADS) void k_norm_fwd(NormArgs a) {
    constexpr int RB = THREADS / L;   // rows of a workgroup at once
    __shared__ float red[4];
    const int lane = threadIdx.x % L, sub = threadIdx.x / L;
    const float inv = 1.f / (float)a.dim;
    const T* w = static_cast<const T*>(a.weight);
    const T* b = static_cast<const T*>(a.bias);
    piece_t<T> wv[NV], bv[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int k = (i * L + lane) * E<T>;
        if (w) wv[i] = load_piece(w, k, a.dim);
        else wv[i] = (T)1.f;
        if (b) bv[i] = load_piece(b, k, a.dim);
        else bv[i] = (T)0.f;
    }
    const int64_t step = (int64_t)gridDim.x * RB;
    constexpr bool AHEAD = L * NV >= AHEAD_PIECES;
    piece_t<T> next[NV];
    if (AHEAD) read_row<T, L, NV, 1>(a.x, a.x_stride, (int64_t)blockIdx.x * RB + sub, a, lane, next);
    for (int64_t base = (int64_t)blockIdx.x * RB; base < a.rows; base += step) {
        const int64_t row = base + sub;
        const bool live = row < a.rows;
        piece_t<T> p[NV];
        if (!AHEAD) read_row<T, L, NV, 1>(a.x, a.x_stride, row, a, lane, next);
#pragma unroll
        for (int i = 0; i < NV; ++i) p[i] = next[i];
        settle_row<T, L, NV, 1>(row, a, lane, p);
        if (AHEAD) read_row<T, L, NV, 1>(a.x, a.x_stride, row + step, a, lane, next);
        float v[NV][E<T>];
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
#pragma unroll
            for (int j = 0; j < E<T>; ++j) {
                v[i][j] = (float)p[i][j];
                s += v[i][j];
            }
        }
        const float mu = row_sum<L>(s, red) * inv;
        float q = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < E<T>; ++j) {
                v[i][j] -= mu;
                if ((i * L + lane) * E<T> + j < a.dim) q = fmaf(v[i][j], v[i][j], q);
            }
        const float r = 1.f / sqrtf(fmaf(row_sum<L>(q, red), inv, a.eps));
        if (!live) continue;   // no row_sum below: a workgroup's row is live for all or none
        if (lane == 0) {
            if (a.mean) a.mean[row] = mu;
            if (a.rstd) a.rstd[row] = r;
        }
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int k = (i * L + lane) * E<T>;
            piece_t<T> o;
#pragma unroll
            for (int j = 0; j < E<T>; ++j) o[j] = (T)fmaf(v[i][j] * r, (float)wv[i][j], (float)bv[i][j]);
            if (k < a.dim) store_piece(static_cast<T*>(a.out) + row * a.out_stride, k, a.dim, o);
        }
    }
}

// dx of each row; the rows' sums of dy n and dy stay in registers until the
// workgroup ends, are added over its rows in LDS and written as one partial
// row a workgroup (added up by k_norm_fold in a fixed order).
template <class T, int L, int NV>
__global__ __launch_bounds__(THREADS) void k_norm_bwd(NormArgs a) {
    constexpr int RB = THREADS / L, W = L * NV * E<T>;   // W: padded row width
    __shared__ float red[4];
    __shared__ float acc[RB * W];
    const int lane = threadIdx.x % L, sub = threadIdx.x / L;
    const float inv = 1.f / (float)a.dim;
    const T* w = static_cast<const T*>(a.weight);
    float wf[NV][E<T>], dw[NV][E<T>] = {}, db[NV][E<T>] = {};
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int k = (i * L + lane) * E<T>;
        piece_t<T> p;
        if (w) p = load_piece(w, k, a.dim);
        else p = (T)1.f;
#pragma unroll
        for (int j = 0; j < E<T>; ++j) wf[i][j] = (float)p[j];
    }
    const int64_t step = (int64_t)gridDim.x * RB;
    constexpr bool AHEAD = L * NV >= AHEAD_PIECES;
    piece_t<T> nx[NV], nd[NV];
    if (AHEAD) {
        read_row<T, L, NV, 1>(a.x, a.x_stride, (int64_t)blockIdx.x * RB + sub, a, lane, nx);
        read_row<T, L, NV, 1>(a.dy, a.dy_stride, (int64_t)blockIdx.x * RB + sub, a, lane, nd);
    }
    for (int64_t base = (int64_t)blockIdx.x * RB; base < a.rows; base += step) {
        const int64_t row = base + sub;
        const bool live = row < a.rows;
        piece_t<T> px[NV], pd[NV];
        if (!AHEAD) {
            read_row<T, L, NV, 1>(a.x, a.x_stride, row, a, lane, nx);
            read_row<T, L, NV, 1>(a.dy, a.dy_stride, row, a, lane, nd);
        }
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            px[i] = nx[i];
            pd[i] = nd[i];
        }
        settle_row<T, L, NV, 1>(row, a, lane, px);
        settle_row<T, L, NV, 1>(row, a, lane, pd);
        if (AHEAD) {
            read_row<T, L, NV, 1>(a.x, a.x_stride, row + step, a, lane, nx);
            read_row<T, L, NV, 1>(a.dy, a.dy_stride, row + step, a, lane, nd);
        }
        float n[NV][E<T>], g[NV][E<T>];
        float s1 = 0.f, s2 = 0.f;
        const float mu = live ? a.mean[row] : 0.f, r = live ? a.rstd[row] : 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int k = (i * L + lane) * E<T>;
#pragma unroll
            for (int j = 0; j < E<T>; ++j) {
                const bool in = k + j < a.dim;
                const float d = (float)pd[i][j];
                n[i][j] = in ? ((float)px[i][j] - mu) * r : 0.f;
                g[i][j] = d * wf[i][j];
                s1 += g[i][j];
                s2 = fmaf(g[i][j], n[i][j], s2);
                dw[i][j] = fmaf(d, n[i][j], dw[i][j]);
                db[i][j] += d;
            }
        }
        s1 = row_sum<L>(s1, red) * inv;
        s2 = row_sum<L>(s2, red) * inv;
        if (!live || !a.out) continue;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int k = (i * L + lane) * E<T>;
            piece_t<T> o;
#pragma unroll
            for (int j = 0; j < E<T>; ++j) o[j] = (T)(r * (g[i][j] - s1 - n[i][j] * s2));
            if (k < a.dim) store_piece(static_cast<T*>(a.out) + row * a.out_stride, k, a.dim, o);
        }
    }
    if (!a.part) return;
    float* part = a.part + (int64_t)blockIdx.x * 2 * a.dim;
    for (int m = 0; m < 2; ++m) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < E<T>; ++j) acc[sub * W + (i * L + lane) * E<T> + j] = m ? db[i][j] : dw[i][j];
        __syncthreads();
        for (int c = threadIdx.x; c < a.dim; c += THREADS) {
            float t = 0.f;
            for (int q = 0; q < RB; ++q) t += acc[q * W + c];
            part[m * a.dim + c] = t;
        }
    }
}

// Adds the groups' partial rows: 32 columns a workgroup, 32 threads a column.
template <class T>
__global__ __launch_bounds__(1024) void k_norm_fold(const float* part, int groups, int dim, T* dweight, T* dbias) {
    __shared__ float red[32][33];
    const int col = blockIdx.x * 32 + (threadIdx.x & 31), sl = threadIdx.x >> 5;
    float t = 0.f;
    if (col < 2 * dim)
#pragma unroll 8
        for (int g = sl; g < groups; g += 32) t += part[(int64_t)g * 2 * dim + col];
    red[sl][threadIdx.x & 31] = t;
    __syncthreads();
    if (sl == 0 && col < 2 * dim) {
        t = 0.f;
        for (int q = 0; q < 32; ++q) t += red[q][threadIdx.x & 31];
        T* out = col < dim ? dweight : dbias;
        if (out) out[col < dim ? col : col - dim] = (T)t;
    }
}

}  // namespace

void launch_norm_fwd(hipStream_t s, int dtype, const NormArgs& a) {
    with_type(dtype, [&](auto t) {
        using T = decltype(t);
        with_shape<T, 1>(a.dim, [&](auto l, auto nv) {
            k_norm_fwd<T, l(), nv()><<<grid_for(a.rows, THREADS / l(), 4096), THREADS, 0, s>>>(a);
        });
    });
}

int norm_groups(int64_t rows, int dim, int dtype) {
    int g = 0;
    with_type(dtype, [&](auto t) {
        with_shape<decltype(t), 1>(dim, [&](auto l, auto) { g = grid_for(rows, THREADS / l(), MAX_GROUPS); });
    });
    return g;
}

void launch_norm_bwd(hipStream_t s, int dtype, const NormArgs& a, void* dweight, void* dbias) {
    const int groups = norm_groups(a.rows, a.dim, dtype);
    with_type(dtype, [&](auto t) {
        using T = decltype(t);
        if (groups > 0)
            with_shape<T, 1>(a.dim, [&](auto l, auto nv) { k_norm_bwd<T, l(), nv()><<<groups, THREADS, 0, s>>>(a); });
        if (dweight || dbias)
            k_norm_fold<T><<<(2 * a.dim + 31) / 32, 1024, 0, s>>>(a.part, groups, a.dim, static_cast<T*>(dweight),
                                                                  static_cast<T*>(dbias));
    });
}

}  // namespace msp
