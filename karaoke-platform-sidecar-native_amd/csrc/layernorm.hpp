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

// N consecutive elements of any element's alignment, 16 bytes in one access (the
// hardware takes it as one, also across lines).
template <int N>
struct Vec {
    float v[N];
};
template <typename T, int N>
struct Packed {
    typedef T type __attribute__((ext_vector_type(N), aligned(sizeof(T))));
};
template <int N, typename T>
VH_DEVICE Vec<N> ldv(const T *p) {
    Vec<N> r;
    const typename Packed<T, N>::type a = *reinterpret_cast<const typename Packed<T, N>::type *>(p);
#pragma unroll
    for (int e = 0; e < N; e++) r.v[e] = (float)a[e];
    return r;
}
template <int N, typename T>
VH_DEVICE void stv(T *p, const Vec<N> &v) {
    typename Packed<T, N>::type a;
#pragma unroll
    for (int e = 0; e < N; e++) a[e] = (T)v.v[e];
    *reinterpret_cast<typename Packed<T, N>::type *>(p) = a;
}

// A row's lanes: LANES of a wave (16 or 64: THREADS / LANES rows a workgroup), or
// the whole workgroup; NV vectors of N elements each.  Lane l's i-th vector covers
// columns (l + LANES i) N .. + N - 1; the row's last one is moved back to end with
// the row, so that no access is partial (a branch to single elements there made the
// backward pass of 1023 columns 1.7 times that of 1024): the columns it shares with
// its neighbour count there only, and are written twice, with the same value.
template <int LANES, int N, int NV>
struct NormShape {
    static constexpr int THREADS = LANES > 512 ? LANES : LANES > 64 ? LANES : 512;
    static constexpr int ROWS = LANES > 64 ? 1 : THREADS / LANES;
    static constexpr int COLUMNS = LANES * N * NV;
    VH_DEVICE static int lane() { return (int)threadIdx.x % LANES; }
    VH_DEVICE static int row() { return LANES > 64 ? 0 : (int)threadIdx.x / LANES; }
    VH_DEVICE static int column(int i) { return (lane() + LANES * i) * N; }
};

// Sums over a row's lanes, by way of LDS where they are a workgroup (red: two
// arrays in turn, so that one barrier a sum is enough).
template <int LANES, int K>
VH_DEVICE void row_sums(float (&v)[K], float *red, int &turn) {
#pragma unroll
    for (int k = 0; k < K; k++)
#pragma unroll
        for (int o = (LANES < 64 ? LANES : 64) / 2; o > 0; o >>= 1) v[k] += __shfl_xor(v[k], o, 64);
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

template <typename T, int LANES, int N, int NV>
static __global__ __launch_bounds__((NormShape<LANES, N, NV>::THREADS)) void layernorm_kernel(NormArgs a) {
    using S = NormShape<LANES, N, NV>;
    __shared__ float red[LANES > 64 ? 4 * (LANES / 64) : 1];
    int turn = 0;
    const int64_t row = (int64_t)blockIdx.x * S::ROWS + S::row();
    if (row >= a.rows) return;  // all of a row's lanes, and no barrier below where these are not a workgroup
    const T *x = static_cast<const T *>(a.x) + row * a.ldx;
    T *y = static_cast<T *>(a.y) + row * a.ldy;
    Vec<N> v[NV];
    float sum[1] = {0.0f};
#pragma unroll
    for (int i = 0; i < NV; i++) {
        const int c = S::column(i), at = min(c, a.dim - N);
        if (c < a.dim) {
            v[i] = ldv<N>(x + at);
#pragma unroll
            for (int e = 0; e < N; e++) sum[0] += at + e >= c ? v[i].v[e] : 0.0f;
        }
    }
    row_sums<LANES>(sum, red, turn);
    const float mu = sum[0] / (float)a.dim;
    float sq[1] = {0.0f};
#pragma unroll
    for (int i = 0; i < NV; i++) {
        const int c = S::column(i), at = min(c, a.dim - N);
        if (c < a.dim) {
#pragma unroll
            for (int e = 0; e < N; e++) {
                v[i].v[e] -= mu;
                sq[0] = __builtin_fmaf(v[i].v[e], at + e >= c ? v[i].v[e] : 0.0f, sq[0]);
            }
        }
    }
    row_sums<LANES>(sq, red, turn);
    const float rstd = 1.0f / sqrtf(sq[0] / (float)a.dim + a.eps);
    if (a.stats && S::lane() == 0) a.stats[row] = make_float2(mu, rstd);
#pragma unroll
    for (int i = 0; i < NV; i++) {
        const int c = S::column(i), at = min(c, a.dim - N);
        if (c < a.dim) {
            const Vec<N> g = ldv<N>(a.gamma + at);
            Vec<N> b = {};
            if (a.beta) b = ldv<N>(a.beta + at);
#pragma unroll
            for (int e = 0; e < N; e++) v[i].v[e] = __builtin_fmaf(v[i].v[e] * rstd, g.v[e], b.v[e]);
            stv<N>(y + at, v[i]);
        }
    }
}

// A workgroup takes every gridDim-th row (or ROWS of them), and keeps its rows' sums
// of dgamma and dbeta in registers: a lane's columns are the same in every row.
template <typename T, int LANES, int N, int NV>
static __global__ __launch_bounds__((NormShape<LANES, N, NV>::THREADS)) void layernorm_backward_kernel(NormArgs a) {
    using S = NormShape<LANES, N, NV>;
    __shared__ float red[LANES > 64 ? 4 * (LANES / 64) : 1];
    __shared__ float cols[LANES > 64 ? 1 : 2 * S::COLUMNS];
    int turn = 0;
    Vec<N> dg[NV] = {}, db[NV] = {}, w[NV] = {};
#pragma unroll
    for (int i = 0; i < NV; i++) {
        const int c = S::column(i);
        if (c < a.dim) w[i] = ldv<N>(a.gamma + min(c, a.dim - N));
    }
    for (int64_t row = (int64_t)blockIdx.x * S::ROWS + S::row(); row < a.rows; row += (int64_t)gridDim.x * S::ROWS) {
        const T *x = static_cast<const T *>(a.x) + row * a.ldx, *dy = static_cast<const T *>(a.dy) + row * a.lddy;
        T *dx = static_cast<T *>(a.dx) + row * a.lddx;
        const float2 st = a.stats[row];
        Vec<N> h[NV], g[NV];
        float sum[2] = {0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const int c = S::column(i), at = min(c, a.dim - N);
            if (c < a.dim) {
                h[i] = ldv<N>(x + at);
                g[i] = ldv<N>(dy + at);
            }
        }
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const int c = S::column(i), at = min(c, a.dim - N);
            if (c < a.dim) {
#pragma unroll
                for (int e = 0; e < N; e++) {
                    const float own = at + e >= c ? g[i].v[e] : 0.0f;
                    h[i].v[e] = (h[i].v[e] - st.x) * st.y;
                    dg[i].v[e] = __builtin_fmaf(own, h[i].v[e], dg[i].v[e]);
                    db[i].v[e] += own;
                    g[i].v[e] *= w[i].v[e];
                    sum[0] = __builtin_fmaf(own, w[i].v[e], sum[0]);
                    sum[1] = __builtin_fmaf(own * w[i].v[e], h[i].v[e], sum[1]);
                }
            }
        }
        row_sums<LANES>(sum, red, turn);
        const float c1 = sum[0] / (float)a.dim, c2 = sum[1] / (float)a.dim;
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const int c = S::column(i), at = min(c, a.dim - N);
            if (c < a.dim) {
#pragma unroll
                for (int e = 0; e < N; e++) g[i].v[e] = st.y * (g[i].v[e] - c1 - h[i].v[e] * c2);
                stv<N>(dx + at, g[i]);
            }
        }
    }
    if (!a.part) return;
    float *part = a.part + (int64_t)blockIdx.x * 2 * a.dim;
    if constexpr (LANES <= 64) {
        // the rows of a wave, then the waves one after the other
        const int wave = (int)threadIdx.x >> 6, lane = (int)threadIdx.x & 63;
#pragma unroll
        for (int i = 0; i < NV; i++)
#pragma unroll
            for (int e = 0; e < N; e++)
#pragma unroll
                for (int o = LANES; o < 64; o <<= 1) {
                    dg[i].v[e] += __shfl_xor(dg[i].v[e], o, 64);
                    db[i].v[e] += __shfl_xor(db[i].v[e], o, 64);
                }
        for (int v = 0; v < S::THREADS / 64; v++) {
            if (wave == v && lane < LANES)
#pragma unroll
                for (int i = 0; i < NV; i++)
#pragma unroll
                    for (int e = 0; e < N; e++) {
                        const int c = (i * N + e) * LANES + lane;  // a column's place: its own lane's
                        if (v) {
                            dg[i].v[e] += cols[c];
                            db[i].v[e] += cols[S::COLUMNS + c];
                        }
                        cols[c] = dg[i].v[e];
                        cols[S::COLUMNS + c] = db[i].v[e];
                    }
            __syncthreads();
        }
        if (wave != S::THREADS / 64 - 1 || lane >= LANES) return;
    }
#pragma unroll
    for (int i = 0; i < NV; i++) {
        const int c = S::column(i), at = min(c, a.dim - N);
#pragma unroll
        for (int e = 0; e < N; e++)
            if (c < a.dim && at + e >= c) {
                part[at + e] = dg[i].v[e];
                part[a.dim + at + e] = db[i].v[e];
            }
    }
}

// Column sums of the workgroups' parts [parts][2 dim]: 16 columns x 64 rows a
// workgroup, so that a thread's loads (8 of 512 parts) are all under way at once.
static __global__ __launch_bounds__(1024) void layernorm_columns_kernel(const float *part, int parts, int dim,
                                                                         float *dgamma, float *dbeta) {
    __shared__ float sums[16][16];
    const int tid = (int)threadIdx.x, i = tid & 15, c = (int)blockIdx.x * 16 + i;
    float sum = 0.0f;
    if (c < 2 * dim) {
#pragma unroll 8
        for (int p = tid >> 4; p < parts; p += 64) sum += part[(int64_t)p * 2 * dim + c];
    }
    sum += __shfl_xor(sum, 16, 64);
    sum += __shfl_xor(sum, 32, 64);
    if ((tid & 63) < 16) sums[tid >> 6][i] = sum;
    __syncthreads();
    if (tid >= 16 || c >= 2 * dim) return;
#pragma unroll
    for (int k = 1; k < 16; k++) sum += sums[k][i];
    float *out = c < dim ? dgamma : dbeta;
    if (out) out[c < dim ? c : c - dim] = sum;
}

}  // namespace vh
