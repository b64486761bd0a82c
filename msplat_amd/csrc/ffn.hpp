// ffn.hpp — the gated feed-forward block, forward and backward:
//
//   g = x Wg^T   u = x Wu^T   h = a(g) * u   y = h Wd^T
//   dh = dy Wd   du = dh a(g)   dg = dh u a'(g)   dx = dg Wg + du Wu
//   dWg = dg^T x   dWu = du^T x   dWd = dy^T h
//
// a(v) = v sigmoid(z(v)), with z = v (SiLU) or z = 2 sqrt(2/pi) (v + 0.044715
// v^3) (GELU in its tanh form).  The rows are many and the width is at most
// 256, so g, u and h (rows x hidden) never go to memory: 12 bytes a hidden
// unit and row would cost more than the 6 dim operations that make them again (at the
// rates of a large copy and a large library product up to a width of 430).
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
// small kernel first (5 us): each is used in up to three orders, and the pack
// takes up every width and stride.  In 16-bit types h, dg and du are rounded to
// the type for the next product, as the type's own matrix instructions take
// them; the error is of the size of the output's own rounding (1.4 of it in
// all), within the type's range: in float16 a hidden unit beyond 65504 becomes
// infinite though the output may not be, and a dg or du below 6e-5 loses bits
// and below 3e-8 is zero, though a sum of many rows of it may not be.
//
// What bounds it: the activations go through the vector unit and the products
// through the matrix unit, of which a SIMD has one each and a wave uses one at a
// time.  The two overlap in part (a probe with four waves a SIMD: 24 matrix
// instructions 404 cycles, the activations of as many rows 550, both 782: 43% of
// the matrix cycles pass behind vector ones).  At 64 features the activations
// are the larger half, at 256 an eighth.  64-256-64 below: the matrix unit is
// busy in 36% of the cycles, the vector unit in 59% (without issuing matrix
// instructions, 9%); what hides the rest of the one behind the other is open.
//   64-256-64 bf16 forward over 1.09M rows: 129-139 us, 770-830 TFLOP/s
//   256-1024-256 bf16 forward over 229k rows: 335 us, 1075 TFLOP/s (a library
//   product of 8192^3 reaches 1111)
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

// A block of KB rows of a matrix [rows, dim] as fragments rows x dim: the piece
// of row perm(s, r), elements (4 kb + c) E ..., lies at slot(kb, s, c, r).  The
// order of rows turns with c so that by_dim's reads spread over LDS's banks;
// in 16-bit types groups of four rows change places so that by_row's 16-byte
// reads, which the hardware takes as lanes 0-3, 12-15, 20-23, 24-27 and so on,
// stay free of conflicts too.
template <class T>
__device__ __forceinline__ int slot(int kb, int s, int c, int r) {
    return (kb * HT<T> + s) * 64 + c * 16 + (r ^ (sizeof(T) == 4 ? c : (-c & 3) * 4));
}
// Fragment f = kb HT + s, rows x dim.
template <class T>
__device__ __forceinline__ piece_t<T> by_row(const piece_t<T>* block, int f) {
    const int lane = threadIdx.x & 63;
    return block[slot<T>(0, 0, lane >> 4, lane & 15) + f * 64];
}
// Fragment f = kb HT + s, dim x rows, of a block in LDS: column kb KB + perm(s,
// r), elements consecutive rows.  16-bit types take the transposing LDS read,
// in which lane 4 k + c of 16 brings 4 elements of row k and lane i gets
// element i % 4 of the lanes 4 k + i / 4.
template <class T>
__device__ __forceinline__ piece_t<T> by_dim(const piece_t<T>* block, int f) {
    const int lane = threadIdx.x & 63, q = lane >> 4, j = lane & 15;
    piece_t<T> o;
    if constexpr (sizeof(T) == 2) {
        typedef short s16x4 __attribute__((ext_vector_type(4)));
        typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
        const char* base = reinterpret_cast<const char*>(block + slot<T>(0, 0, j & 3, q * 4 + (j >> 2)));
        s16x4 h[2];
#pragma unroll
        for (int t = 0; t < 2; ++t)
            h[t] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(base + ((f >> 1) * 2 + t) * 1024 + (f & 1) * 8));
        __builtin_memcpy(&o, h, 16);
    } else {
        const float* base = reinterpret_cast<const float*>(block + f * 64);
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = base[slot<T>(0, 0, j >> 2, q * 4 + e) * 4 + (j & 3)];
    }
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
    // a' = s + a (1 - s) z'.  GELU's z' grows as g g, but from |g| of about 20 on
    // a (1 - s) is 0 and a' is s: z' is kept finite (g g overflows from 2e19 on) and
    // comes last (a z' overflows from 1e13 on).
    const float s = sigmoid_fast(GELU ? g * fmaf(g * g, GELU_B, GELU_A) : g);
    const float a = g * s;
    const float da =
        GELU ? fmaf(a * (1.f - s), fmaf(fminf(g * g, 1e38f), 3.f * GELU_B, GELU_A), s) : fmaf(a, 1.f - s, s);
    const float h = a * u;
    g = dh * u * da;   // dg
    u = dh * a;        // du
    dh = h;            // h
}

// Fragments of the weights, block of hidden units after block: in a block the
// matrices in order, DK * HT fragments each.  Rows x contraction index:
// forward  0 Wg (hidden x dim)  1 Wu  2 Wd (dim x hidden)
// backward 0 Wg  1 Wu  2 Wd^T (hidden x dim), and for few rows
//          3 Wg^T (dim x hidden)  4 Wu^T
template <class T>
__global__ __launch_bounds__(256) void k_ffn_pack(FfnArgs a, bool backward, int dk, int hblocks,
                                                  int mats, piece_t<T>* out) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int lane = (int)(i & 63), r = lane & 15, q = lane >> 4;
    const int64_t f = i >> 6;
    const int s = (int)(f % HT<T>), kb = (int)(f / HT<T> % dk);
    const int64_t bm = f / (HT<T> * dk);
    const int m = (int)(bm % mats), b = (int)(bm / mats);
    if (b >= hblocks) return;
    // rows x contraction index of the fragment; the matrix as it lies has
    // outer x inner
    const bool hidden_rows = m < 2 || (backward && m == 2), down = m == 2, along = hidden_rows != down;
    const T* w = static_cast<const T*>(down ? a.w_down : (m == 1 || m == 4) ? a.w_up : a.w_gate);
    const int64_t stride = down ? a.down_stride : (m == 1 || m == 4) ? a.up_stride : a.gate_stride;
    const int row = (hidden_rows ? b : kb) * KB<T> + perm<T>(s, r), at = (hidden_rows ? kb : b) * KB<T> + q * E<T>;
    const int rows = hidden_rows ? a.hidden : a.dim, n = hidden_rows ? a.dim : a.hidden;
    const int safe = min(row, rows - 1);
    piece_t<T> v;
    if (along && n >= E<T>) {
        v = settle_piece<T>(read_piece(w + safe * stride, at, n), at, n, row < rows);
    } else {   // all reads go out before the first is looked at
#pragma unroll
        for (int j = 0; j < E<T>; ++j) {
            const int k = min(at + j, n - 1);
            v[j] = along ? w[safe * stride + k] : w[k * stride + safe];
        }
#pragma unroll
        for (int j = 0; j < E<T>; ++j)
            if (row >= rows || at + j >= n) v[j] = (T)0.f;
    }
    out[f * 64 + slot<T>(0, 0, q, r)] = v;
}

// Copies n fragments (1 KB each) from memory to LDS without registers in
// between; a wave takes every waves-th.  They are there after fetched().
template <class T>
__device__ __forceinline__ void fetch(const piece_t<T>* src, piece_t<T>* lds, int n) {
    const int lane = threadIdx.x & 63, waves = blockDim.x >> 6;
    for (int f = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); f < n; f += waves)
        __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(src + f * 64 + lane),
                                         (__attribute__((address_space(3))) void*)(lds + f * 64), 16, 0, 0);
}

// Waits for the wave's own fetches, then for the workgroup.
__device__ __forceinline__ void fetched() {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
}

// The pieces of R rows' operand fragments, in two steps (read_piece,
// settle_piece).  TINY: rows are less than a piece.
template <class T, int DK, int R, bool TINY>
__device__ __forceinline__ void read_rows(const void* base, int64_t stride, int64_t row0, int64_t rows, int dim, int q,
                                          piece_t<T> (&f)[R][DK]) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const T* row = static_cast<const T*>(base) + min(row0 + 16 * r, rows - 1) * stride;
#pragma unroll
        for (int kb = 0; kb < DK; ++kb)
            f[r][kb] = TINY ? load_piece(row, q * E<T>, dim) : read_piece(row, kb * KB<T> + q * E<T>, dim);
    }
}
template <class T, int DK, int R, bool TINY>
__device__ __forceinline__ void settle_rows(int64_t row0, int64_t rows, int dim, int q, piece_t<T> (&f)[R][DK]) {
    if (TINY) return;
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int kb = 0; kb < DK; ++kb)
            f[r][kb] = settle_piece<T>(f[r][kb], kb * KB<T> + q * E<T>, dim, row0 + 16 * r < rows);
}
template <class T, int DK, int R, bool TINY>
__device__ __forceinline__ void load_rows(const void* base, int64_t stride, int64_t row0, int64_t rows, int dim, int q,
                                          piece_t<T> (&f)[R][DK]) {
    read_rows<T, DK, R, TINY>(base, stride, row0, rows, dim, q, f);
    settle_rows<T, DK, R, TINY>(row0, rows, dim, q, f);
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

// Order of issue for a step of `groups` groups of LDS reads and the matrix
// instructions that take them: reads run `ahead` groups in front, so that
// their latency passes behind matrix work.  (The compiler by itself reads a
// group, waits, and multiplies.)
template <int READS, int MFMAS, int GROUPS, int AHEAD>
__device__ __forceinline__ void read_ahead() {
    constexpr int A = AHEAD < GROUPS ? AHEAD : GROUPS;
    __builtin_amdgcn_sched_group_barrier(0x100, READS * A, 0);
#pragma unroll
    for (int g = 0; g < GROUPS - A; ++g) {
        __builtin_amdgcn_sched_group_barrier(0x8, MFMAS, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, READS, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x8, MFMAS * A, 0);
}
template <class T>
constexpr int MFMAS = sizeof(T) == 4 ? 4 : 1;   // matrix instructions of an mma

// The two steps of a block of hidden units for R tiles of 16 rows: h from x,
// then its part of y.
template <class T, int DK, int R, bool GELU>
__device__ __forceinline__ void fwd_up(const piece_t<T>* up, const piece_t<T> (&xf)[R][DK], piece_t<T> (&h)[R]) {
    constexpr int F = DK * HT<T>;
    f32x4 g[R][HT<T>] = {}, u[R][HT<T>] = {};
#pragma unroll
    for (int f = 0; f < F; ++f) {
        const piece_t<T> wg = by_row<T>(up, f), wu = by_row<T>(up, F + f);
#pragma unroll
        for (int r = 0; r < R; ++r) {
            g[r][f % HT<T>] = mma(wg, xf[r][f / HT<T>], g[r][f % HT<T>]);
            u[r][f % HT<T>] = mma(wu, xf[r][f / HT<T>], u[r][f % HT<T>]);
        }
    }
    read_ahead<2, 2 * R * MFMAS<T>, F, 2>();
#pragma unroll
    for (int r = 0; r < R; ++r) {
#pragma unroll
        for (int j = 0; j < E<T>; ++j) g[r][j / 4][j % 4] = act<GELU>(g[r][j / 4][j % 4]) * u[r][j / 4][j % 4];
        h[r] = join<T>(g[r]);
    }
}
template <class T, int F, int R>
__device__ __forceinline__ void fwd_down(const piece_t<T>* down, const piece_t<T> (&h)[R], f32x4 (&acc)[R][F]) {
#pragma unroll
    for (int f = 0; f < F; ++f) {
        const piece_t<T> wd = by_row<T>(down, f);
#pragma unroll
        for (int r = 0; r < R; ++r) acc[r][f] = mma(wd, h[r], acc[r][f]);
    }
    read_ahead<1, R * MFMAS<T>, F, 2>();
}

// dg and du from x and dy, then their part of dx.
template <class T, int DK, int R, bool GELU>
__device__ __forceinline__ void dx_up(const piece_t<T>* up, const piece_t<T> (&xf)[R][DK], const piece_t<T> (&df)[R][DK],
                                      piece_t<T> (&dg)[R], piece_t<T> (&du)[R]) {
    constexpr int F = DK * HT<T>;
    f32x4 g[R][HT<T>] = {}, u[R][HT<T>] = {}, dh[R][HT<T>] = {};
#pragma unroll
    for (int f = 0; f < F; ++f) {
        const piece_t<T> wg = by_row<T>(up, f), wu = by_row<T>(up, F + f), wd = by_row<T>(up, 2 * F + f);
#pragma unroll
        for (int r = 0; r < R; ++r) {
            g[r][f % HT<T>] = mma(wg, xf[r][f / HT<T>], g[r][f % HT<T>]);
            u[r][f % HT<T>] = mma(wu, xf[r][f / HT<T>], u[r][f % HT<T>]);
            dh[r][f % HT<T>] = mma(wd, df[r][f / HT<T>], dh[r][f % HT<T>]);
        }
    }
    read_ahead<3, 3 * R * MFMAS<T>, F, 2>();
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
// With TURN the fragments dim x hidden are those of Wg and Wu themselves, in
// LDS; else they were packed too.
template <class T, int F, int R, bool TURN>
__device__ __forceinline__ void dx_down(const piece_t<T>* down, const piece_t<T> (&dg)[R], const piece_t<T> (&du)[R],
                                        f32x4 (&acc)[R][F]) {
#pragma unroll
    for (int f = 0; f < F; ++f) {
        const piece_t<T> wg = TURN ? by_dim<T>(down, f) : by_row<T>(down, f);
        const piece_t<T> wu = TURN ? by_dim<T>(down + F * 64, f) : by_row<T>(down, F + f);
#pragma unroll
        for (int r = 0; r < R; ++r) acc[r][f] = mma(wu, du[r], mma(wg, dg[r], acc[r][f]));
    }
    if (TURN) read_ahead<sizeof(T) == 4 ? 8 : 4, 2 * R * MFMAS<T>, F, 2>();
}

// A wave takes R tiles of 16 rows and walks the hidden units block by block.
// The workgroup's waves share a block's weights in LDS, in two areas: while
// one is computed with, the next block's weights arrive in the other.
template <class T, int DK, int R, int WAVES, bool GELU, bool TINY>
__global__ __launch_bounds__(64 * WAVES) void k_ffn_fwd(FfnArgs a, const piece_t<T>* packed, int hblocks, int mats) {
    constexpr int F = DK * HT<T>;
    __shared__ piece_t<T> even[3 * F * 64], odd[3 * F * 64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, q = lane >> 4;
    const int64_t row0 = ((int64_t)blockIdx.x * (blockDim.x >> 6) + wave) * (16 * R) + (lane & 15);
    fetch<T>(packed, even, 3 * F);
    piece_t<T> xf[R][DK];
    load_rows<T, DK, R, TINY>(a.x, a.x_stride, row0, a.rows, a.dim, q, xf);
    f32x4 acc[R][F] = {};
    auto block = [&](int b, const piece_t<T>* w, piece_t<T>* next) {
        fetched();
        if (b + 1 < hblocks) fetch<T>(packed + (int64_t)(b + 1) * mats * F * 64, next, 3 * F);
        piece_t<T> h[R];
        fwd_up<T, DK, R, GELU>(w, xf, h);
        fwd_down<T, F, R>(w + 2 * F * 64, h, acc);
    };
    for (int b = 0; b < hblocks; b += 2) {
        block(b, even, odd);
        if (b + 1 < hblocks) block(b + 1, odd, even);
    }
    store_rows<T, DK, R>(a.out, a.out_stride, row0, a.rows, a.dim, q, acc);
}

template <class T, int DK, int R, int WAVES, bool GELU, bool TINY>
__global__ __launch_bounds__(64 * WAVES) void k_ffn_dx(FfnArgs a, const piece_t<T>* packed, int hblocks, int mats) {
    constexpr int F = DK * HT<T>;
    __shared__ piece_t<T> even[3 * F * 64], odd[3 * F * 64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, q = lane >> 4;
    const int64_t row0 = ((int64_t)blockIdx.x * (blockDim.x >> 6) + wave) * (16 * R) + (lane & 15);
    fetch<T>(packed, even, 3 * F);
    piece_t<T> xf[R][DK], df[R][DK];
    load_rows<T, DK, R, TINY>(a.x, a.x_stride, row0, a.rows, a.dim, q, xf);
    load_rows<T, DK, R, TINY>(a.dy, a.dy_stride, row0, a.rows, a.dim, q, df);
    f32x4 acc[R][F] = {};
    auto block = [&](int b, const piece_t<T>* w, piece_t<T>* next) {
        fetched();
        if (b + 1 < hblocks) fetch<T>(packed + (int64_t)(b + 1) * mats * F * 64, next, 3 * F);
        piece_t<T> dg[R], du[R];
        dx_up<T, DK, R, GELU>(w, xf, df, dg, du);
        dx_down<T, F, R, true>(w, dg, du, acc);
    };
    for (int b = 0; b < hblocks; b += 2) {
        block(b, even, odd);
        if (b + 1 < hblocks) block(b + 1, odd, even);
    }
    store_rows<T, DK, R>(a.out, a.out_stride, row0, a.rows, a.dim, q, acc);
}

// The same where all packed weights fit in LDS: a workgroup loads them once,
// then its waves walk row tiles on their own, with no barrier that would hold
// all of them at the matrix or at the vector instructions at once.  (64-256-64
// bf16 over 1.09M rows, a call: streamed 165 us, resident 152; backward
// over 500k rows 246 and 241.)
template <class T, int DK, int R, int WAVES, bool GELU, bool TINY>
__global__ __launch_bounds__(64 * WAVES) void k_ffn_fwd_all(FfnArgs a, const piece_t<T>* packed, int hblocks) {
    constexpr int F = DK * HT<T>;
    extern __shared__ char smem[];
    piece_t<T>* w = reinterpret_cast<piece_t<T>*>(smem);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, q = lane >> 4;
    fetch<T>(packed, w, hblocks * 3 * F);
    fetched();
    const int64_t waves = blockDim.x >> 6, step = gridDim.x * waves;
    int64_t row0 = ((int64_t)wave * gridDim.x + blockIdx.x) * (16 * R) + (lane & 15);   // CUs differ by a tile at most
    piece_t<T> xf[R][DK], xn[R][DK], h[R];
    read_rows<T, DK, R, TINY>(a.x, a.x_stride, row0, a.rows, a.dim, q, xn);
    for (; row0 - (lane & 15) < a.rows; row0 += step * (16 * R)) {
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int kb = 0; kb < DK; ++kb) xf[r][kb] = xn[r][kb];
        settle_rows<T, DK, R, TINY>(row0, a.rows, a.dim, q, xf);
        read_rows<T, DK, R, TINY>(a.x, a.x_stride, row0 + step * (16 * R), a.rows, a.dim, q, xn);
        f32x4 acc[R][F] = {};
        for (int b = 0; b < hblocks; ++b) {
            fwd_up<T, DK, R, GELU>(w + b * 3 * F * 64, xf, h);
            fwd_down<T, F, R>(w + (b * 3 + 2) * F * 64, h, acc);
        }
        store_rows<T, DK, R>(a.out, a.out_stride, row0, a.rows, a.dim, q, acc);
    }
}

template <class T, int DK, int R, int WAVES, bool GELU, bool TINY>
__global__ __launch_bounds__(64 * WAVES) void k_ffn_dx_all(FfnArgs a, const piece_t<T>* packed, int hblocks) {
    constexpr int F = DK * HT<T>;
    extern __shared__ char smem[];
    piece_t<T>* w = reinterpret_cast<piece_t<T>*>(smem);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, q = lane >> 4;
    fetch<T>(packed, w, hblocks * 3 * F);
    fetched();
    const int64_t waves = blockDim.x >> 6;
    for (int64_t t = (int64_t)wave * gridDim.x + blockIdx.x; t * (16 * R) < a.rows; t += gridDim.x * waves) {
        const int64_t row0 = t * (16 * R) + (lane & 15);
        piece_t<T> xf[R][DK], df[R][DK], dg[R], du[R];
        load_rows<T, DK, R, TINY>(a.x, a.x_stride, row0, a.rows, a.dim, q, xf);
        load_rows<T, DK, R, TINY>(a.dy, a.dy_stride, row0, a.rows, a.dim, q, df);
        f32x4 acc[R][F] = {};
        for (int b = 0; b < hblocks; ++b) {
            dx_up<T, DK, R, GELU>(w + b * 3 * F * 64, xf, df, dg, du);
            dx_down<T, F, R, true>(w + b * 3 * F * 64, dg, du, acc);
        }
        store_rows<T, DK, R>(a.out, a.out_stride, row0, a.rows, a.dim, q, acc);
    }
}

// Few rows: a workgroup takes R tiles of 16 rows, and its waves share out the
// hidden units; the waves' parts of y are added in LDS, half of the waves onto
// the other half until one is left, in the same order every time.  Weights
// come from the L2 cache into registers, each read once a workgroup.  (128-512
// bf16 forward, 256 rows: streamed 25 us a call, this way 15; 8192 rows 21.5 and
// 19; 256-1024 over 64 rows 80 and 23.)
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

// Where the row tiles are so few that CUs would be left over, `splits`
// workgroups share a tile's hidden units too and leave their 32-bit parts for
// k_ffn_join.  The forward reads the weights as they are: all three matrices'
// fragments lie along their rows.
template <class T, int F, int R>
__device__ __forceinline__ void leave_part(const f32x4 (&acc)[R][F], int splits, int split, f32x4* part) {
    f32x4* at = part + ((int64_t)(blockIdx.x / splits) * splits + split) * R * F * 64 + (threadIdx.x & 63);
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int f = 0; f < F; ++f) at[(r * F + f) * 64] = acc[r][f];
}

// Adds a tile's parts in order: a wave per tile of 16 rows and block of
// columns.
template <class T>
__global__ __launch_bounds__(64) void k_ffn_join(FfnArgs a, const f32x4* part, int splits, int tiles_each, int dk) {
    const int lane = threadIdx.x, kb = blockIdx.x % dk, fr = dk * HT<T>;
    const int64_t t = blockIdx.x / dk;   // tile of 16 rows
    const f32x4* at = part + ((t / tiles_each * splits * tiles_each + t % tiles_each) * fr + kb * HT<T>) * 64 + lane;
    f32x4 sum[HT<T>] = {};
    for (int s = 0; s < splits; ++s)
#pragma unroll
        for (int h = 0; h < HT<T>; ++h) sum[h] += at[((int64_t)s * tiles_each * fr + h) * 64];
    const int64_t row = t * 16 + (lane & 15);
    const int k = kb * KB<T> + (lane >> 4) * E<T>;
    if (row < a.rows && k < a.dim) store_piece(static_cast<T*>(a.out) + row * a.out_stride, k, a.dim, join<T>(sum));
}

template <class T, int DK, int R, int WAVES, bool GELU, bool TINY>
__global__ __launch_bounds__(64 * WAVES) void k_ffn_fwd_few(FfnArgs a, int hblocks, int splits, f32x4* part) {
    constexpr int F = DK * HT<T>;
    __shared__ f32x4 sums[WAVES / 2 * R * F * 64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, q = lane >> 4, i = lane & 15;
    const int split = blockIdx.x % splits;
    const int64_t row0 = (int64_t)(blockIdx.x / splits) * (16 * R) + i;
    piece_t<T> xf[R][DK], h[R];
    read_rows<T, DK, R, TINY>(a.x, a.x_stride, row0, a.rows, a.dim, q, xf);
    f32x4 acc[R][F] = {};
    bool first = true;
    for (int b = split * WAVES + wave; b < hblocks; b += splits * WAVES) {
        // every read of the block goes out before the first piece is looked at
        // (wide blocks: every read of a step)
        piece_t<T> wg[F], wu[F], wd[F];
#pragma unroll
        for (int f = 0; f < F; ++f) {
            const int64_t u = min(b * KB<T> + perm<T>(f % HT<T>, i), a.hidden - 1);
            const T* pg = static_cast<const T*>(a.w_gate) + u * a.gate_stride;
            const T* pu = static_cast<const T*>(a.w_up) + u * a.up_stride;
            const int k = f / HT<T> * KB<T> + q * E<T>;
            wg[f] = TINY ? load_piece(pg, k, a.dim) : read_piece(pg, k, a.dim);
            wu[f] = TINY ? load_piece(pu, k, a.dim) : read_piece(pu, k, a.dim);
        }
        auto read_down = [&]() {
#pragma unroll
            for (int f = 0; f < F; ++f) {
                const int64_t d = min(f / HT<T> * KB<T> + perm<T>(f % HT<T>, i), a.dim - 1);
                wd[f] = read_piece(static_cast<const T*>(a.w_down) + d * a.down_stride, b * KB<T> + q * E<T>, a.hidden);
            }
        };
        if (F <= 8) read_down();
        __builtin_amdgcn_sched_barrier(0);
        if (first) settle_rows<T, DK, R, TINY>(row0, a.rows, a.dim, q, xf);
        first = false;
#pragma unroll
        for (int f = 0; f < F; ++f) {
            const bool live = b * KB<T> + perm<T>(f % HT<T>, i) < a.hidden;
            const int k = f / HT<T> * KB<T> + q * E<T>;
            if (TINY) {
                if (!live) wg[f] = wu[f] = piece_t<T>{};
            } else {
                wg[f] = settle_piece<T>(wg[f], k, a.dim, live);
                wu[f] = settle_piece<T>(wu[f], k, a.dim, live);
            }
        }
        f32x4 g[R][HT<T>] = {}, u[R][HT<T>] = {};
#pragma unroll
        for (int f = 0; f < F; ++f)
#pragma unroll
            for (int r = 0; r < R; ++r) {
                g[r][f % HT<T>] = mma(wg[f], xf[r][f / HT<T>], g[r][f % HT<T>]);
                u[r][f % HT<T>] = mma(wu[f], xf[r][f / HT<T>], u[r][f % HT<T>]);
            }
        if (F > 8) {
            __builtin_amdgcn_sched_barrier(0);
            read_down();
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
#pragma unroll
            for (int j = 0; j < E<T>; ++j) g[r][j / 4][j % 4] = act<GELU>(g[r][j / 4][j % 4]) * u[r][j / 4][j % 4];
            h[r] = join<T>(g[r]);
        }
#pragma unroll
        for (int f = 0; f < F; ++f) {
            const int d = f / HT<T> * KB<T> + perm<T>(f % HT<T>, i);
            wd[f] = settle_piece<T>(wd[f], b * KB<T> + q * E<T>, a.hidden, d < a.dim);
#pragma unroll
            for (int r = 0; r < R; ++r) acc[r][f] = mma(wd[f], h[r], acc[r][f]);
        }
    }
    add_waves<T, F, R, WAVES>(acc, sums);
    if (wave != 0) return;
    if (splits > 1) leave_part<T, F, R>(acc, splits, split, part);
    else store_rows<T, DK, R>(a.out, a.out_stride, row0, a.rows, a.dim, q, acc);
}

template <class T, int DK, int R, int WAVES, bool GELU, bool TINY>
__global__ __launch_bounds__(64 * WAVES) void k_ffn_dx_few(FfnArgs a, const piece_t<T>* packed, int hblocks, int splits,
                                                            f32x4* part) {
    constexpr int F = DK * HT<T>;
    __shared__ f32x4 sums[WAVES / 2 * R * F * 64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, q = lane >> 4;
    const int split = blockIdx.x % splits;
    const int64_t row0 = (int64_t)(blockIdx.x / splits) * (16 * R) + (lane & 15);
    piece_t<T> xf[R][DK], df[R][DK], dg[R], du[R];
    load_rows<T, DK, R, TINY>(a.x, a.x_stride, row0, a.rows, a.dim, q, xf);
    load_rows<T, DK, R, TINY>(a.dy, a.dy_stride, row0, a.rows, a.dim, q, df);
    f32x4 acc[R][F] = {};
    for (int b = split * WAVES + wave; b < hblocks; b += splits * WAVES) {
        const piece_t<T>* w = packed + (int64_t)b * 5 * F * 64;
        dx_up<T, DK, R, GELU>(w, xf, df, dg, du);
        dx_down<T, F, R, false>(w + 3 * F * 64, dg, du, acc);
    }
    add_waves<T, F, R, WAVES>(acc, sums);
    if (wave != 0) return;
    if (splits > 1) leave_part<T, F, R>(acc, splits, split, part);
    else store_rows<T, DK, R>(a.out, a.out_stride, row0, a.rows, a.dim, q, acc);
}

// Weight gradients: a wave owns NH tiles of 16 hidden units, keeps their
// weights and their rows of the three gradients in registers and walks a
// group's rows. The workgroup's waves share each block of rows in LDS, two
// blocks in turn: the next is on its way while one is computed.  Sums go to
// part[group][tile][matrix][dim tile][lane].  Bound as the forward; wide blocks
// run one wave a SIMD, whose waits nothing covers.  (64-256 bf16 over 500k rows:
// 130 us, 256-1024 over 229k rows: 844, 855 TFLOP/s.)
constexpr int DW_WAVES = 4;
// Tiles of hidden units a wave of the weight gradient takes, and waves a SIMD,
// by registers: 24 a tile and block of columns for weights and sums.  (Two
// tiles at three blocks: 96-384 1073 us against 1033; two waves a SIMD at six
// blocks spill: 192-768 2160 us against 1728.)
template <class T>
constexpr int dw_tiles(int dk) {
    return sizeof(T) == 2 && dk <= 2 ? 2 : 1;
}
template <class T>
constexpr int dw_occupancy(int dk, int nh) {
    const int n = dk * nh;
    return n == 1 ? 4 : n == 2 ? 3 : n <= 5 ? 2 : 1;
}

template <class T, int DK, int NH, int WAVES, bool GELU, bool TINY>
__global__ __launch_bounds__(64 * WAVES, WAVES / 4 * dw_occupancy<T>(DK, NH)) void k_ffn_dw(
    FfnArgs a, const piece_t<T>* packed, int hblocks, int mats, int slices, int64_t blocks_per_group, f32x4* part) {
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
                const piece_t<T>* p = packed + ((int64_t)b * mats * F + kb * HT<T> + s) * 64;
                wg[n][kb] = by_row<T>(p, 0);
                wu[n][kb] = by_row<T>(p, F);
                wd[n][kb] = by_row<T>(p, 2 * F);
            }
        }
    }
    f32x4 acc[3][NH][F] = {};
    const int64_t first = group * blocks_per_group * KB<T>;
    const int64_t last = min(a.rows, first + blocks_per_group * KB<T>);

    // A thread's pieces of a block: read, and on the next turn put into LDS.
    // The last block of all is read so that it ends with the rows (the order
    // of rows in a block does not matter), and rows before it count as zero.
    piece_t<T> in[ITEMS];
    int64_t off[ITEMS];
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) {
        int i = k * 64 * WAVES + threadIdx.x;
        const bool y = i >= F * 64;
        i -= y ? F * 64 : 0;
        const int64_t row = min((int64_t)(i / (DK * 4)), a.rows - 1);
        off[k] = row * (y ? a.dy_stride : a.x_stride) + (TINY ? 0 : min(i % (DK * 4) * E<T>, a.dim - E<T>));
    }
    const int64_t final_block = a.rows > KB<T> ? a.rows - KB<T> : 0;
    auto load = [&](int64_t row0) {
        const int64_t from = min(row0, final_block);
        const T* xb = static_cast<const T*>(a.x) + from * a.x_stride;
        const T* yb = static_cast<const T*>(a.dy) + from * a.dy_stride;
#pragma unroll
        for (int k = 0; k < ITEMS; ++k) {
            const int i = k * 64 * WAVES + threadIdx.x;
            if (2 * F % WAVES != 0 && i >= 2 * F * 64) continue;
            const T* p = (i >= F * 64 ? yb : xb) + off[k];
            if (TINY) in[k] = load_piece(p, i % 4 * E<T>, a.dim);
            else __builtin_memcpy(&in[k], p, 16);
        }
    };
    auto store = [&](piece_t<T>* to, int64_t row0) {
        const int64_t from = min(row0, final_block);
        const bool whole = from == row0 && row0 + KB<T> <= last && a.dim == DK * KB<T>;
#pragma unroll
        for (int k = 0; k < ITEMS; ++k) {
            int i = k * 64 * WAVES + threadIdx.x;
            if (2 * F % WAVES != 0 && i >= 2 * F * 64) continue;
            const bool y = i >= F * 64;
            i -= y ? F * 64 : 0;
            const int w = i / (DK * 4), ch = i % (DK * 4);   // w = perm(s, r)
            const int s = HT<T> == 2 ? (w >> 2) & 1 : 0, r = w / E<T> * 4 + (w & 3);
            piece_t<T> v = in[k];
            if (!whole) {
                const bool live = from + w >= row0 && from + w < last;
                if (TINY) v = live ? v : piece_t<T>{};
                else v = settle_piece<T>(v, ch * E<T>, a.dim, live);
            }
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
        read_ahead<2, 3 * NH * MFMAS<T>, F, 2>();
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
        read_ahead<sizeof(T) == 4 ? 8 : 4, 3 * NH * MFMAS<T>, F, 2>();
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
    const int d = f / HT<T> * KB<T> + perm<T>(f % HT<T>, lane & 15);
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
    constexpr int made[] = {1, 2, 3, 4, 5, 6, 7, 8, 10, 12, 14, 16};
    for (int m : made)
        if (n <= m) return m;
    return 0;
}
// Calls f with the number of blocks and whether rows are less than a piece.
template <class T, class F>
inline void with_blocks(int dim, F&& f) {
    if (dim < E<T>) return f(std::integral_constant<int, 1>{}, std::true_type{});
#define BLOCKS(n) \
    case n: return f(std::integral_constant<int, n>{}, std::false_type{})
    switch (dim_blocks<T>(dim)) {
        BLOCKS(1);
        BLOCKS(2);
        BLOCKS(3);
        BLOCKS(4);
        BLOCKS(5);
        BLOCKS(6);
        BLOCKS(7);
        BLOCKS(8);
    }
    if constexpr (sizeof(T) == 4) {
        switch (dim_blocks<T>(dim)) {
            BLOCKS(10);
            BLOCKS(12);
            BLOCKS(14);
            BLOCKS(16);
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
    // four blocks of rows at least, or one where that leaves CUs without work
    const int64_t most = std::max(1, 1024 / DW_WAVES * dw_occupancy<T>(dk, p.nh) / p.slices);
    const int64_t groups = std::min(most, std::max((blocks + 3) / 4, std::min<int64_t>(blocks, 256 / p.slices)));
    p.blocks_per_group = groups ? (blocks + groups - 1) / groups : 0;
    p.groups = p.blocks_per_group ? (int)((blocks + p.blocks_per_group - 1) / p.blocks_per_group) : 0;
    return p;
}

template <class T>
size_t packed_bytes(int dim, int hidden, int mats) {
    return (size_t)((hidden + KB<T> - 1) / KB<T>) * mats * dim_blocks<T>(dim) * HT<T> * 1024;
}

template <class T>
piece_t<T>* pack(hipStream_t s, const FfnArgs& a, bool backward, int dk, int hblocks, int mats) {
    piece_t<T>* packed = reinterpret_cast<piece_t<T>*>(a.ws);
    const int64_t n = (int64_t)hblocks * mats * dk * HT<T> * 64;
    k_ffn_pack<T><<<(unsigned)((n + 255) / 256), 256, 0, s>>>(a, backward, dk, hblocks, mats, packed);
    return packed;
}

constexpr int64_t CUS = 256;
constexpr size_t LDS_BYTES = 160 * 1024;
inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Rows up to which a workgroup takes one or two row tiles for all hidden units
// (k_ffn_*_few): as long as every one of them finds a CU free, twice that
// where two fit on one; two tiles of wide blocks do not fit in registers.
// (256-1024 bf16 forward over 8192 rows: 117 us this way, 60 streamed.)
inline int64_t few_rows(int fragments) { return fragments <= 4 ? 64 * CUS : fragments <= 8 ? 32 * CUS : 16 * CUS; }

// Launch shape of the kernels whose waves take `tile` rows each: `most` waves
// a workgroup, fewer where that would leave CUs without one.
struct Shape {
    unsigned groups, threads;
};
inline Shape shape_of(int64_t rows, int tile, int most, int64_t max_groups) {
    const int64_t tiles = ceil_div(rows, tile);
    const int64_t waves = std::min<int64_t>(most, ceil_div(tiles, CUS));
    return {(unsigned)std::min(ceil_div(tiles, waves), max_groups), (unsigned)(64 * waves)};
}

// Rows that the streaming kernels leave to the few-row ones: the start of a
// last round of workgroups that would hold the GPU as long as a full one.
inline int64_t tail_rows(int64_t rows, int64_t per_round) {
    const int64_t rest = rows % per_round;
    return rows > per_round && rest <= 16 * CUS ? rest : 0;
}
inline FfnArgs rows_from(FfnArgs a, int64_t from, size_t size) {
    auto at = [&](const void* p, int64_t stride) { return p ? static_cast<const char*>(p) + from * stride * size : nullptr; };
    a.x = at(a.x, a.x_stride);
    a.dy = at(a.dy, a.dy_stride);
    a.out = const_cast<char*>(at(a.out, a.out_stride));
    a.rows -= from;
    return a;
}

// Calls f with a's rows in parts that a launch of the streaming kernels can take:
// it has fewer than 2^32 threads, and those are up to four a row.
template <class F>
inline void in_parts(const FfnArgs& a, size_t size, F&& f) {
    constexpr int64_t most = int64_t(1) << 29;
    for (int64_t at = 0; at < a.rows; at += most) {
        FfnArgs part = rows_from(a, at, size);
        part.rows = std::min(part.rows, most);
        f(part);
    }
}

// Bytes of a call's workspace: packed weights, parts that the few-row kernels
// leave (at most one workgroup a CU shares its tile), the weight gradient's
// sums.
template <class T>
size_t join_bytes(int dim) {
    return (size_t)CUS * dim_blocks<T>(dim) * HT<T> * 1024;
}
template <class T>
size_t workspace(int64_t rows, int dim, int hidden, bool backward) {
    if (!backward) return packed_bytes<T>(dim, hidden, 3) + join_bytes<T>(dim);
    const Split p = dw_split<T>(rows, dim, hidden);
    return packed_bytes<T>(dim, hidden, 5) + join_bytes<T>(dim) +
           (size_t)p.groups * p.tiles * 3 * dim_blocks<T>(dim) * HT<T> * 1024;
}

template <class F>
inline void with_act(const FfnArgs& a, F&& f) {
    if (a.gelu) f(std::true_type{});
    else f(std::false_type{});
}

// Row tiles of a wave in the streaming kernels, and with eight waves a
// workgroup the workgroups of a CU, by registers and LDS.
// (bf16 forward, one tile and two: 96-384 over 1.09M rows 288 us and 327,
// 128-512 over 300k 137 and 137, 192-768 over 100k 117 and 103, 224-896 over 300k
// 393 and 325, 256-1024 505 and 415.  The backward, whose input gradient holds
// twice the fragments: 128-512 over 500k rows 795 and 775, 112-300 527 and 539,
// 96-384 over 1.09M 1039 and 1049, 256-1024 over 229k 1398 and 2047.)
template <class T>
constexpr int fwd_tiles(int fragments) {
    return sizeof(T) == 4 || fragments <= 8 ? 1 : 2;
}
template <class T>
constexpr int dx_tiles(int fragments) {
    return sizeof(T) == 2 && fragments == 8 ? 2 : 1;
}
constexpr int per_cu(int fragments) { return fragments <= 8 ? 2 : 1; }

// How the few-row kernels are launched: tiles of a workgroup, workgroups, and
// the workgroups that share a tile, where a wave would have more than three
// blocks of hidden units: so many that none has a second while CUs are free.
// (256-1024 bf16 forward over 64 rows: 32 blocks, 33 us on two workgroups a
// tile, 20 + 4.7 for the join on four.  128-512 over 256 rows, 16 blocks: 15.0
// on one, 10.0 + 3.9 on two.)
struct Few {
    int tiles, splits;
    unsigned groups;
};
template <class T>
inline Few few_plan(int64_t rows, int hidden) {
    Few p;
    p.tiles = rows <= 16 * CUS ? 1 : 2;
    const int64_t row_groups = ceil_div(rows, 16 * p.tiles), blocks = ceil_div(hidden, KB<T>);
    p.splits = blocks > 24 ? (int)std::max<int64_t>(1, std::min(CUS / row_groups, ceil_div(blocks, 8))) : 1;
    p.groups = (unsigned)(row_groups * p.splits);
    return p;
}
template <class T>
void few_join(hipStream_t s, const FfnArgs& a, const Few& p, const f32x4* part) {
    if (p.splits == 1) return;
    const int dk = dim_blocks<T>(a.dim);
    k_ffn_join<T><<<(unsigned)(ceil_div(a.rows, 16) * dk), 64, 0, s>>>(a, part, p.splits, p.tiles, dk);
}

template <class T, int DK, bool GELU, bool TINY>
void few_forward(hipStream_t s, const FfnArgs& a, int hblocks, f32x4* part) {
    const Few p = few_plan<T>(a.rows, a.hidden);
    if (p.tiles == 1) k_ffn_fwd_few<T, DK, 1, 8, GELU, TINY><<<p.groups, 512, 0, s>>>(a, hblocks, p.splits, part);
    else if constexpr (DK * HT<T> <= 8)
        k_ffn_fwd_few<T, DK, 2, 8, GELU, TINY><<<p.groups, 512, 0, s>>>(a, hblocks, p.splits, part);
    few_join<T>(s, a, p, part);
}

template <class T>
void forward(hipStream_t s, const FfnArgs& a) {
    with_blocks<T>(a.dim, [&](auto dk, auto tiny) {
        with_act(a, [&](auto gelu) {
            constexpr int F = dk() * HT<T>, R = fwd_tiles<T>(F), W = 8;
            const int hblocks = (a.hidden + KB<T> - 1) / KB<T>;
            f32x4* part = reinterpret_cast<f32x4*>(a.ws + packed_bytes<T>(a.dim, a.hidden, 3));
            // the few-row kernel reads the weights as they are, in whole pieces
            const bool pieces = a.hidden >= E<T>;
            if (a.rows <= few_rows(F) && pieces) return few_forward<T, dk(), gelu(), tiny()>(s, a, hblocks, part);
            const piece_t<T>* packed = pack<T>(s, a, false, dk(), hblocks, 3);
            const size_t lds = packed_bytes<T>(a.dim, a.hidden, 3);
            if constexpr (F <= 4) {
                if (lds <= LDS_BYTES) {
                    constexpr int RA = sizeof(T) == 4 ? 1 : 2;
                    const Shape g = shape_of(a.rows, 16 * RA, 16, CUS);
                    k_ffn_fwd_all<T, dk(), RA, 16, gelu(), tiny()><<<g.groups, g.threads, lds, s>>>(a, packed, hblocks);
                    return;
                }
            }
            FfnArgs main = a;
            const int64_t tail = pieces ? tail_rows(a.rows, 16 * R * W * per_cu(F) * CUS) : 0;
            if (tail) few_forward<T, dk(), gelu(), tiny()>(s, rows_from(a, a.rows - tail, sizeof(T)), hblocks, part);
            main.rows -= tail;
            // two tiles a wave only where that still gives every SIMD a wave
            in_parts(main, sizeof(T), [&](const FfnArgs& part) {
                if (R == 2 && part.rows >= 32 * 4 * CUS) {
                    const Shape g = shape_of(part.rows, 16 * R, W, INT32_MAX);
                    k_ffn_fwd<T, dk(), R, W, gelu(), tiny()><<<g.groups, g.threads, 0, s>>>(part, packed, hblocks, 3);
                } else {
                    const Shape g = shape_of(part.rows, 16, W, INT32_MAX);
                    k_ffn_fwd<T, dk(), 1, W, gelu(), tiny()><<<g.groups, g.threads, 0, s>>>(part, packed, hblocks, 3);
                }
            });
        });
    });
}

template <class T, int DK, bool GELU, bool TINY>
void few_dx(hipStream_t s, const FfnArgs& a, const piece_t<T>* packed, int hblocks, f32x4* part) {
    const Few p = few_plan<T>(a.rows, a.hidden);
    if (p.tiles == 1) k_ffn_dx_few<T, DK, 1, 8, GELU, TINY><<<p.groups, 512, 0, s>>>(a, packed, hblocks, p.splits, part);
    else if constexpr (DK * HT<T> <= 8)
        k_ffn_dx_few<T, DK, 2, 8, GELU, TINY><<<p.groups, 512, 0, s>>>(a, packed, hblocks, p.splits, part);
    few_join<T>(s, a, p, part);
}

// How the input's gradient is made: few rows, resident weights, or streamed
// weights with a tail of few rows; the few-row kernel needs five matrices.
template <class T>
struct DxPlan {
    int64_t tail;
    int mats;
    bool all;
};
template <class T>
DxPlan<T> dx_plan(const FfnArgs& a, int fragments) {
    if (a.rows <= few_rows(fragments)) return {a.rows, 5, false};
    if (fragments <= 4 && packed_bytes<T>(a.dim, a.hidden, 3) <= LDS_BYTES) return {0, 3, true};
    const int64_t tail = tail_rows(a.rows, 16 * dx_tiles<T>(fragments) * 8 * per_cu(fragments) * CUS);
    return {tail, tail ? 5 : 3, false};
}

template <class T, int DK, bool GELU, bool TINY>
void input_gradient(hipStream_t s, const FfnArgs& a, const DxPlan<T>& plan, const piece_t<T>* packed, int hblocks,
                    f32x4* part) {
    constexpr int F = DK * HT<T>, W = 8;
    if (plan.tail) few_dx<T, DK, GELU, TINY>(s, rows_from(a, a.rows - plan.tail, sizeof(T)), packed, hblocks, part);
    if (plan.tail == a.rows) return;
    if constexpr (F <= 4) {
        if (plan.all) {
            const size_t lds = packed_bytes<T>(a.dim, a.hidden, 3);
            const Shape g = shape_of(a.rows, 16, 16, CUS);
            k_ffn_dx_all<T, DK, 1, 16, GELU, TINY><<<g.groups, g.threads, lds, s>>>(a, packed, hblocks);
            return;
        }
    }
    FfnArgs main = a;
    main.rows -= plan.tail;
    constexpr int R = dx_tiles<T>(F);
    in_parts(main, sizeof(T), [&](const FfnArgs& p) {
        if (R == 2 && p.rows >= 32 * 4 * CUS) {
            const Shape g = shape_of(p.rows, 16 * R, W, INT32_MAX);
            k_ffn_dx<T, DK, R, W, GELU, TINY><<<g.groups, g.threads, 0, s>>>(p, packed, hblocks, plan.mats);
        } else {
            const Shape g = shape_of(p.rows, 16, W, INT32_MAX);
            k_ffn_dx<T, DK, 1, W, GELU, TINY><<<g.groups, g.threads, 0, s>>>(p, packed, hblocks, plan.mats);
        }
    });
}

template <class T>
void backward(hipStream_t s, const FfnArgs& a) {
    with_blocks<T>(a.dim, [&](auto dk, auto tiny) {
        constexpr int F = dk() * HT<T>;
        const int hblocks = (a.hidden + KB<T> - 1) / KB<T>;
        const DxPlan<T> plan = dx_plan<T>(a, F);
        const int mats = plan.mats;
        const piece_t<T>* packed = pack<T>(s, a, true, dk(), hblocks, mats);
        if (a.out && a.rows > 0)
            with_act(a, [&](auto gelu) {
                f32x4* part = reinterpret_cast<f32x4*>(a.ws + packed_bytes<T>(a.dim, a.hidden, 5));
                input_gradient<T, dk(), gelu(), tiny()>(s, a, plan, packed, hblocks, part);
            });
        if (!a.dw_gate) return;
        const Split p = dw_split<T>(a.rows, a.dim, a.hidden);
        f32x4* part = reinterpret_cast<f32x4*>(a.ws + packed_bytes<T>(a.dim, a.hidden, 5) + join_bytes<T>(a.dim));
        auto dw = [&](auto nh) {
            with_act(a, [&](auto gelu) {
                k_ffn_dw<T, dk(), nh(), DW_WAVES, gelu(), tiny()><<<(unsigned)(p.groups * p.slices), 64 * DW_WAVES, 0, s>>>(
                    a, packed, hblocks, mats, p.slices, p.blocks_per_group, part);
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
