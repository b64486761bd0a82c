// rms.hip — root-mean-square norm over the last axis with the residual's
// addition, forward and backward.
//
//   t = x + residual (rounded to the type)   r = 1 / sqrt(mean(t^2) + eps)
//   y = t r w, in the type or in mx8 (mx8.hpp)
//   dx = r (g - n mean(g n)) + dt,  g = dy w,  n = t r
//   dw = sum over rows of dy n
//
// The norm is that of the rounded sum, which is what the backward sees; the
// backward may take the sum from mx8 too.
//
// Bound by HBM: a row is read once, kept in registers (rows.hpp) and written
// once.
//   forward, 1.09M rows of 64 bf16 with a residual: 106 us, 5.2 TB/s (a large copy 5.2)
//   the same into 8 bits, 500k rows of 128: 94 us, 4.8 TB/s
//   backward from 8 bits, 500k rows of 128 bf16: 82 us, 5.5 TB/s, and 5 us for the sums
#include "mx8.hpp"
#include "rows.hpp"

namespace msp {
namespace {

using namespace rows;

// Workgroups of the backward: each leaves a partial row of dw.
constexpr int MAX_GROUPS = 1024;

// Rows in mx8 end with a whole block, so that many lanes are the fewest.
template <class T, bool MX>
constexpr int FEWEST = MX ? mx8::LANES<T> : 1;

template <class T, int L, int NV, bool MX, bool RES>
__global__ __launch_bounds__(THREADS) void k_rms_fwd(RmsArgs a) {
    constexpr int RB = THREADS / L, MIN = FEWEST<T, MX>;
    __shared__ float red[4];
    const int lane = threadIdx.x % L, sub = threadIdx.x / L;
    const float inv = 1.f / (float)a.dim;
    const T* w = static_cast<const T*>(a.weight);
    piece_t<T> wv[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int k = (i * L + lane) * E<T>;
        if (w) wv[i] = load_piece(w, k, a.dim);
        else wv[i] = (T)1.f;
    }
    const int64_t step = (int64_t)gridDim.x * RB;
    constexpr bool AHEAD = L * NV >= AHEAD_PIECES;
    piece_t<T> nx[NV], nr[NV];
    auto read = [&](int64_t row) {
        read_row<T, L, NV, MIN>(a.x, a.x_stride, row, a, lane, nx);
        if (RES) read_row<T, L, NV, MIN>(a.residual, a.residual_stride, row, a, lane, nr);
    };
    if (AHEAD) read((int64_t)blockIdx.x * RB + sub);
    for (int64_t base = (int64_t)blockIdx.x * RB; base < a.rows; base += step) {
        const int64_t row = base + sub;
        const bool live = row < a.rows;
        piece_t<T> p[NV];
        if (!AHEAD) read(row);
#pragma unroll
        for (int i = 0; i < NV; ++i) p[i] = nx[i];
        settle_row<T, L, NV, MIN>(row, a, lane, p);
        if (RES) {
            settle_row<T, L, NV, MIN>(row, a, lane, nr);
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int j = 0; j < E<T>; ++j) p[i][j] = (T)((float)p[i][j] + (float)nr[i][j]);
        }
        if (AHEAD) read(row + step);
        float q = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < E<T>; ++j) q = fmaf((float)p[i][j], (float)p[i][j], q);
        const float r = 1.f / sqrtf(fmaf(row_sum<L>(q, red), inv, a.eps));
        // past the sum every read of the row is done, so that its sum may take its place
        if (live) {
            if (lane == 0 && a.rstd) a.rstd[row] = r;
            if (a.total)
#pragma unroll
                for (int i = 0; i < NV; ++i) {
                    const int k = (i * L + lane) * E<T>;
                    if (k < a.dim) store_piece(static_cast<T*>(a.total) + row * a.total_stride, k, a.dim, p[i]);
                }
        }
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int k = (i * L + lane) * E<T>;
            float v[E<T>];
#pragma unroll
            for (int j = 0; j < E<T>; ++j) v[j] = (float)p[i][j] * r * (float)wv[i][j];
            if constexpr (MX) {
                uint32_t bytes[E<T> / 4];
                if (k >= a.dim)   // r may be infinite
#pragma unroll
                    for (int j = 0; j < E<T>; ++j) v[j] = 0.f;
                else
#pragma unroll
                    for (int j = 0; j < E<T>; ++j)
                        if (k + j >= a.dim) v[j] = 0.f;
                const int code = mx8::pack_block<T>(v, bytes);
                if (live && k < mx8::data_stride(a.dim))
                    mx8::store<T>(static_cast<uint8_t*>(a.y) + row * mx8::data_stride(a.dim),
                                  a.y_scales + row * mx8::scale_stride(a.dim), k, a.dim, bytes, code);
            } else {
                piece_t<T> o;
#pragma unroll
                for (int j = 0; j < E<T>; ++j) o[j] = (T)v[j];
                if (live && k < a.dim) store_piece(static_cast<T*>(a.y) + row * a.y_stride, k, a.dim, o);
            }
        }
    }
}

// A row's pieces in mx8: their bytes, read ahead like a row of T, and scales.
template <class T, int NV>
struct Packed {
    uint32_t bytes[NV][E<T> / 4];
    uint8_t codes[NV];
};

// dx of each row; the rows' sums of dy n stay in registers until the workgroup
// ends, are added over its rows in LDS and written as one partial row a
// workgroup (added up by k_rms_fold in a fixed order).
template <class T, int L, int NV, bool MX>
__global__ __launch_bounds__(THREADS) void k_rms_bwd(RmsArgs a) {
    constexpr int RB = THREADS / L, W = L * NV * E<T>, MIN = FEWEST<T, MX>;
    __shared__ float red[4];
    __shared__ float acc[RB * W];
    const int lane = threadIdx.x % L, sub = threadIdx.x / L;
    const float inv = 1.f / (float)a.dim;
    const T* w = static_cast<const T*>(a.weight);
    float wf[NV][E<T>], dw[NV][E<T>] = {};
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
    piece_t<T> nt[NV], nd[NV], ng[NV];
    Packed<T, NV> np;
    auto read = [&](int64_t row) {
        if constexpr (MX) {
            const int64_t at = min(row, a.rows - 1);
            const uint8_t* data = static_cast<const uint8_t*>(a.x) + at * mx8::data_stride(a.dim);
            const uint8_t* scales = a.x_scales + at * mx8::scale_stride(a.dim);
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int k = min((i * L + lane) * E<T>, (int)mx8::data_stride(a.dim) - E<T>);
                __builtin_memcpy(np.bytes[i], data + k, E<T>);
                np.codes[i] = scales[k / mx8::BLOCK];
            }
        } else {
            read_row<T, L, NV, MIN>(a.x, a.x_stride, row, a, lane, nt);
        }
        read_row<T, L, NV, MIN>(a.dy, a.dy_stride, row, a, lane, nd);
        if (a.dtotal) read_row<T, L, NV, MIN>(a.dtotal, a.dtotal_stride, row, a, lane, ng);
    };
    if (AHEAD) read((int64_t)blockIdx.x * RB + sub);
    for (int64_t base = (int64_t)blockIdx.x * RB; base < a.rows; base += step) {
        const int64_t row = base + sub;
        const bool live = row < a.rows;
        if (!AHEAD) read(row);
        piece_t<T> pd[NV], pg[NV] = {};
        float n[NV][E<T>], g[NV][E<T>];
        const float r = live ? a.rstd[row] : 0.f;
        if constexpr (!MX) settle_row<T, L, NV, MIN>(row, a, lane, nt);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            pd[i] = nd[i];
            if (a.dtotal) pg[i] = ng[i];
            if constexpr (MX) {
                mx8::values<T>(np.bytes[i], np.codes[i], n[i]);
            } else {
#pragma unroll
                for (int j = 0; j < E<T>; ++j) n[i][j] = (float)nt[i][j];
            }
        }
        settle_row<T, L, NV, MIN>(row, a, lane, pd);
        if (a.dtotal) settle_row<T, L, NV, MIN>(row, a, lane, pg);
        if (AHEAD) read(row + step);
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int k = (i * L + lane) * E<T>;
#pragma unroll
            for (int j = 0; j < E<T>; ++j) {
                const float d = (float)pd[i][j];
                n[i][j] = live && k + j < a.dim ? n[i][j] * r : 0.f;
                g[i][j] = d * wf[i][j];
                s = fmaf(g[i][j], n[i][j], s);
                dw[i][j] = fmaf(d, n[i][j], dw[i][j]);
            }
        }
        s = row_sum<L>(s, red) * inv;
        if (!live || !a.dx) continue;   // no row_sum below: a workgroup's row is live for all or none
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int k = (i * L + lane) * E<T>;
            piece_t<T> o;
#pragma unroll
            for (int j = 0; j < E<T>; ++j) o[j] = (T)fmaf(r, g[i][j] - n[i][j] * s, (float)pg[i][j]);
            if (k < a.dim) store_piece(static_cast<T*>(a.dx) + row * a.dx_stride, k, a.dim, o);
        }
    }
    if (!a.part) return;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < E<T>; ++j) acc[sub * W + (i * L + lane) * E<T> + j] = dw[i][j];
    __syncthreads();
    for (int c = threadIdx.x; c < a.dim; c += THREADS) {
        float t = 0.f;
        for (int q = 0; q < RB; ++q) t += acc[q * W + c];
        a.part[(int64_t)blockIdx.x * a.dim + c] = t;
    }
}

// Adds the groups' partial rows: 32 columns a workgroup, 32 threads a column.
template <class T>
__global__ __launch_bounds__(1024) void k_rms_fold(const float* part, int groups, int dim, T* dweight) {
    __shared__ float red[32][33];
    const int col = blockIdx.x * 32 + (threadIdx.x & 31), sl = threadIdx.x >> 5;
    float t = 0.f;
    if (col < dim)
#pragma unroll 8
        for (int g = sl; g < groups; g += 32) t += part[(int64_t)g * dim + col];
    red[sl][threadIdx.x & 31] = t;
    __syncthreads();
    if (sl == 0 && col < dim) {
        t = 0.f;
        for (int q = 0; q < 32; ++q) t += red[q][threadIdx.x & 31];
        dweight[col] = (T)t;
    }
}

// Calls f with (type, L, NV, whether in mx8) for rows of `dim`.
template <class F>
void with_rms(int dtype, int dim, bool mx, F&& f) {
    with_type(dtype, [&](auto t) {
        using T = decltype(t);
        if (mx)
            with_shape<T, FEWEST<T, true>>((int)mx8::data_stride(dim),
                                           [&](auto l, auto nv) { f(t, l, nv, std::true_type{}); });
        else with_shape<T, 1>(dim, [&](auto l, auto nv) { f(t, l, nv, std::false_type{}); });
    });
}

}  // namespace

void launch_rms_fwd(hipStream_t s, int dtype, const RmsArgs& a) {
    with_rms(dtype, a.dim, a.y_scales != nullptr, [&](auto t, auto l, auto nv, auto mx) {
        const int grid = grid_for(a.rows, THREADS / l(), 4096);
        if (a.residual) k_rms_fwd<decltype(t), l(), nv(), mx(), true><<<grid, THREADS, 0, s>>>(a);
        else k_rms_fwd<decltype(t), l(), nv(), mx(), false><<<grid, THREADS, 0, s>>>(a);
    });
}

int rms_groups(int64_t rows, int dim, int dtype, bool mx) {
    int g = 0;
    with_rms(dtype, dim, mx, [&](auto, auto l, auto, auto) { g = grid_for(rows, THREADS / l(), MAX_GROUPS); });
    return g;
}

void launch_rms_bwd(hipStream_t s, int dtype, const RmsArgs& a, void* dweight) {
    const int groups = rms_groups(a.rows, a.dim, dtype, a.x_scales != nullptr);
    if (groups > 0)
        with_rms(dtype, a.dim, a.x_scales != nullptr, [&](auto t, auto l, auto nv, auto mx) {
            k_rms_bwd<decltype(t), l(), nv(), mx()><<<groups, THREADS, 0, s>>>(a);
        });
    if (dweight)
        with_type(dtype, [&](auto t) {
            using T = decltype(t);
            k_rms_fold<T><<<(a.dim + 31) / 32, 1024, 0, s>>>(a.part, groups, a.dim, static_cast<T*>(dweight));
        });
}

}  // namespace msp
