// Layer norm of rows and its backward pass:
//   mu = sum x / D, rstd = 1 / sqrt(sum (x - mu)^2 / D + eps), h = (x - mu) rstd
//   y = h gamma + beta
//   g = dy gamma:  dx = rstd (g - sum g / D - h sum(g h) / D)
//   dgamma = sum over the rows of dy h, dbeta = sum over the rows of dy
// x, y and their gradients are fp32 or bf16 (T), everything else fp32: a bf16
// value is rounded once, as it is stored.
//
// Bound by HBM: x is read once (the row stays in registers between the mean, the
// variance about it and the output), y written once; backward x, dy read once.
#pragma once

#include "common.hpp"

namespace vh {

struct NormArgs {
    const void *x, *dy;
    void *y, *dx;
    int64_t ldx, lddy, ldy, lddx;  // elements
    const float *gamma, *beta;     // beta may be null
    float2 *stats;                 // [rows] (mu, rstd); forward: may be null
    float *part;                   // backward: [workgroups][2][dim] sums of dgamma and dbeta, or null
    int64_t rows;
    int dim;
    float eps;
};

// N consecutive elements (16 bytes, or 8) of any element's alignment: the hardware
// takes such an access as one, also across lines.  n: how many of them belong to
// the row; the others are 0 and not touched.
template <int N>
struct Vec {
    float v[N];
};
template <typename T, int N>
struct Packed {
    typedef T type __attribute__((ext_vector_type(N), aligned(sizeof(T))));
};
template <int N, typename T>
VH_DEVICE Vec<N> ldv(const T *p, int n) {
    Vec<N> r = {};
    if (n >= N) {
        const typename Packed<T, N>::type a = *reinterpret_cast<const typename Packed<T, N>::type *>(p);
#pragma unroll
        for (int e = 0; e < N; e++) r.v[e] = (float)a[e];
    } else {
#pragma unroll
        for (int e = 0; e < N; e++)
            if (e < n) r.v[e] = (float)p[e];
    }
    return r;
}
template <int N, typename T>
VH_DEVICE void stv(T *p, const Vec<N> &v, int n) {
    if (n >= N) {
        typename Packed<T, N>::type a;
#pragma unroll
        for (int e = 0; e < N; e++) a[e] = (T)v.v[e];
        *reinterpret_cast<typename Packed<T, N>::type *>(p) = a;
    } else {
#pragma unroll
        for (int e = 0; e < N; e++)
            if (e < n) p[e] = (T)v.v[e];
    }
}

// Sums over a row's LANES lanes: a wave, or a workgroup of LANES / 64 waves by
// way of LDS (red: two arrays of 16 in turn, so that one barrier a sum is enough).
template <int LANES, int K>
VH_DEVICE void row_sums(float (&v)[K], float *red, int &turn) {
#pragma unroll
    for (int k = 0; k < K; k++) v[k] = wave_sum(v[k]);
    if constexpr (LANES > 64) {
        constexpr int WAVES = LANES / 64;
        float *r = red + turn * 2 * WAVES;
        turn ^= 1;
        if ((threadIdx.x & 63) == 0)
#pragma unroll
            for (int k = 0; k < K; k++) r[k * WAVES + (threadIdx.x >> 6)] = v[k];
        __syncthreads();
#pragma unroll
        for (int k = 0; k < K; k++) {
            v[k] = 0.0f;
#pragma unroll
            for (int w = 0; w < WAVES; w++) v[k] += r[k * WAVES + w];
        }
    }
}

// LANES lanes per row (64: a wave, ROWS rows a workgroup; else the workgroup), NV
// vectors of N elements each.
template <int LANES>
struct NormShape {
    static constexpr int ROWS = LANES == 64 ? 8 : 1;
    static constexpr int THREADS = LANES * ROWS;
};
template <typename T, int LANES, int N, int NV>
static __global__ __launch_bounds__(NormShape<LANES>::THREADS) void layernorm_kernel(NormArgs a) {
    constexpr int ROWS = NormShape<LANES>::ROWS;
    __shared__ float red[4 * (LANES / 64)];
    int turn = 0;
    const int64_t row = (int64_t)blockIdx.x * ROWS + (LANES == 64 ? (int)threadIdx.x >> 6 : 0);
    const int lane = (int)threadIdx.x % LANES;
    if (row >= a.rows) return;  // whole waves, or none
    const T *x = static_cast<const T *>(a.x) + row * a.ldx;
    T *y = static_cast<T *>(a.y) + row * a.ldy;
    Vec<N> v[NV];
    float sum[1] = {0.0f};
#pragma unroll
    for (int i = 0; i < NV; i++) {
        const int c = (lane + LANES * i) * N;
        v[i] = ldv<N>(x + c, a.dim - c);
#pragma unroll
        for (int e = 0; e < N; e++) sum[0] += v[i].v[e];
    }
    row_sums<LANES>(sum, red, turn);
    const float mu = sum[0] / (float)a.dim;
    float sq[1] = {0.0f};
#pragma unroll
    for (int i = 0; i < NV; i++) {
        const int c = (lane + LANES * i) * N;
#pragma unroll
        for (int e = 0; e < N; e++) {
            v[i].v[e] -= mu;
            if (c + e < a.dim) sq[0] = __builtin_fmaf(v[i].v[e], v[i].v[e], sq[0]);
        }
    }
    row_sums<LANES>(sq, red, turn);
    const float rstd = 1.0f / sqrtf(sq[0] / (float)a.dim + a.eps);
    if (a.stats && lane == 0) a.stats[row] = make_float2(mu, rstd);
#pragma unroll
    for (int i = 0; i < NV; i++) {
        const int c = (lane + LANES * i) * N;
        const Vec<N> g = ldv<N>(a.gamma + c, a.dim - c);
        Vec<N> b = {};
        if (a.beta) b = ldv<N>(a.beta + c, a.dim - c);
#pragma unroll
        for (int e = 0; e < N; e++) v[i].v[e] = __builtin_fmaf(v[i].v[e] * rstd, g.v[e], b.v[e]);
        stv<N>(y + c, v[i], a.dim - c);
    }
}

// A workgroup takes every gridDim-th row (or eight), and keeps its rows' sums of
// dgamma and dbeta in registers: a lane's columns are the same in every row.
template <typename T, int LANES, int N, int NV>
static __global__ __launch_bounds__(NormShape<LANES>::THREADS) void layernorm_backward_kernel(NormArgs a) {
    constexpr int ROWS = NormShape<LANES>::ROWS, COLS = LANES * N * NV;
    __shared__ float red[4 * (LANES / 64)];
    __shared__ float cols[ROWS > 1 ? 2 * COLS : 1];
    int turn = 0;
    const int lane = (int)threadIdx.x % LANES, sub = LANES == 64 ? (int)threadIdx.x >> 6 : 0;
    Vec<N> dg[NV] = {}, db[NV] = {};
    for (int64_t row = (int64_t)blockIdx.x * ROWS + sub; row < a.rows; row += (int64_t)gridDim.x * ROWS) {
        const T *x = static_cast<const T *>(a.x) + row * a.ldx, *dy = static_cast<const T *>(a.dy) + row * a.lddy;
        T *dx = static_cast<T *>(a.dx) + row * a.lddx;
        const float2 st = a.stats[row];
        Vec<N> h[NV], g[NV];
        float sum[2] = {0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const int c = (lane + LANES * i) * N;
            h[i] = ldv<N>(x + c, a.dim - c);
            g[i] = ldv<N>(dy + c, a.dim - c);
        }
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const int c = (lane + LANES * i) * N;
            const Vec<N> w = ldv<N>(a.gamma + c, a.dim - c);
#pragma unroll
            for (int e = 0; e < N; e++) {  // past the row's end g is 0
                h[i].v[e] = (h[i].v[e] - st.x) * st.y;
                if (c + e >= a.dim) h[i].v[e] = 0.0f;
                dg[i].v[e] = __builtin_fmaf(g[i].v[e], h[i].v[e], dg[i].v[e]);
                db[i].v[e] += g[i].v[e];
                g[i].v[e] *= w.v[e];
                sum[0] += g[i].v[e];
                sum[1] = __builtin_fmaf(g[i].v[e], h[i].v[e], sum[1]);
            }
        }
        row_sums<LANES>(sum, red, turn);
        const float c1 = sum[0] / (float)a.dim, c2 = sum[1] / (float)a.dim;
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const int c = (lane + LANES * i) * N;
#pragma unroll
            for (int e = 0; e < N; e++) g[i].v[e] = st.y * (g[i].v[e] - c1 - h[i].v[e] * c2);
            stv<N>(dx + c, g[i], a.dim - c);
        }
    }
    if (!a.part) return;
    float *part = a.part + (int64_t)blockIdx.x * 2 * a.dim;
    if constexpr (ROWS > 1) {  // the waves' sums, one after the other
        for (int w = 0; w < ROWS; w++) {
            if (sub == w)
#pragma unroll
                for (int i = 0; i < NV; i++)
#pragma unroll
                    for (int e = 0; e < N; e++) {
                        const int c = (i * N + e) * 64 + lane;  // a column's place: its own lane's
                        if (w) {
                            dg[i].v[e] += cols[c];
                            db[i].v[e] += cols[COLS + c];
                        }
                        cols[c] = dg[i].v[e];
                        cols[COLS + c] = db[i].v[e];
                    }
            __syncthreads();
        }
        if (sub != ROWS - 1) return;
    }
#pragma unroll
    for (int i = 0; i < NV; i++) {
        const int c = (lane + LANES * i) * N;
        stv<N>(part + c, dg[i], a.dim - c);
        stv<N>(part + a.dim + c, db[i], a.dim - c);
    }
}

// Column sums of the workgroups' parts [parts][2 dim]: 64 columns x 16 rows a
// workgroup.  out: dgamma, then dbeta (either may be null).
static __global__ __launch_bounds__(1024) void layernorm_columns_kernel(const float *part, int parts, int dim,
                                                                         float *dgamma, float *dbeta) {
    __shared__ float sums[16][64];
    const int i = (int)threadIdx.x & 63, c = (int)blockIdx.x * 64 + i, w = (int)threadIdx.x >> 6;
    float sum = 0.0f;
    if (c < 2 * dim) {
#pragma unroll 8
        for (int p = w; p < parts; p += 16) sum += part[(int64_t)p * 2 * dim + c];
    }
    sums[w][i] = sum;
    __syncthreads();
    if (w || c >= 2 * dim) return;
#pragma unroll
    for (int k = 1; k < 16; k++) sum += sums[k][i];
    float *out = c < dim ? dgamma : dbeta;
    if (out) out[c < dim ? c : c - dim] = sum;
}

}  // namespace vh
