// Rotary positions: a head's dims in pairs (a, b), pair i of position p turned by
// p theta_i and scaled, (a c - b s, a s + b c) with (c, s) from a table; the gradient
// by the transpose, (a c + b s, b c - a s).
//
// Bound by HBM: x read once, y written once, a table row (4 dim bytes) a token, which
// its heads share: 32768 tokens of 8 heads of 64 there and back in fp32 58 us (4.8 TB/s), in
// bf16 30 (4.8), with an input that stays in the last-level cache 48 and 24; 6408 of them 14
// and 11 us; a single token 2.5 us of kernel, the call a launch.
#pragma once

#include "common.hpp"

namespace vh {

// A rotation as the kernels take it; no table: none.
struct Rotation {
    const float *table;  // [positions][dim / 2][2]
    int dim, interleaved, positions;
};

// Each product and sum rounded by itself, so that what is quantised afterwards does
// not depend on which of them the compiler joins.
VH_DEVICE void turn_pair(float &a, float &b, float c, float s) {
#pragma clang fp contract(off)
    const float u = a * c - b * s, w = a * s + b * c;
    a = u;
    b = w;
}

// Row of the table for a position; null: it has none.
VH_DEVICE const float *rotation_row(const Rotation &r, int64_t position) {
    return position >= 0 && position < r.positions ? r.table + position * r.dim : nullptr;
}

// n / d for n below 2^31 by a multiplication (d from 1; Granlund and Montgomery's
// division by invariant integers).
struct Divisor {
    uint32_t d, m, shift;
};
inline Divisor divisor(uint32_t d) {
    uint32_t l = 0;
    while (((uint64_t)1 << l) < d) l++;
    return {d, (uint32_t)((((uint64_t)1 << 32) * (((uint64_t)1 << l) - d)) / d + 1), l};
}
VH_DEVICE uint32_t operator/(uint32_t n, const Divisor &d) { return (uint32_t)(((uint64_t)__umulhi(d.m, n) + n) >> d.shift); }

// N consecutive elements of any element's alignment (the hardware takes 16 bytes in
// one access all the same).
template <typename T, int N>
struct Elements {
    typedef T type __attribute__((ext_vector_type(N), aligned(sizeof(T))));
};
template <int N, typename T>
VH_DEVICE void load_n(const T *p, float (&v)[N]) {
    const typename Elements<T, N>::type a = *reinterpret_cast<const typename Elements<T, N>::type *>(p);
#pragma unroll
    for (int e = 0; e < N; e++) v[e] = (float)a[e];
}
template <int N, typename T>
VH_DEVICE void store_n(T *p, const float (&v)[N]) {
    typename Elements<T, N>::type a;
#pragma unroll
    for (int e = 0; e < N; e++) a[e] = (T)v[e];
    *reinterpret_cast<typename Elements<T, N>::type *>(p) = a;
}

// 8 dims of a head from d on (a multiple of 8), turned by the table's row cs (null: NaN).
// The rotation's dim is a multiple of 16, so they are of one half.
template <typename T>
VH_DEVICE void load_turned8(const Rotation &r, const T *x0, const float *cs, int d, float (&x)[8]) {
    load_n<8>(x0 + d, x);
    if (!r.table || d >= r.dim) return;
    if (!cs) {
#pragma unroll
        for (int e = 0; e < 8; e++) x[e] = __builtin_nanf("");
        return;
    }
    if (r.interleaved) {
        float c[8];
        load_n<8>(cs + d, c);
#pragma unroll
        for (int e = 0; e < 4; e++) turn_pair(x[2 * e], x[2 * e + 1], c[2 * e], c[2 * e + 1]);
        return;
    }
    const int half = r.dim / 2;
    const bool second = d >= half;
    const int pair = second ? d - half : d;
    float c[16], y[8];
    load_n<16>(cs + 2 * pair, c);
    load_n<8>(x0 + (second ? pair : d + half), y);
#pragma unroll
    for (int e = 0; e < 8; e++) {
        if (second) turn_pair(y[e], x[e], c[2 * e], c[2 * e + 1]);
        else turn_pair(x[e], y[e], c[2 * e], c[2 * e + 1]);
    }
}

struct RotaryArgs {
    Rotation r;
    const void *x;
    void *y;
    int64_t xs[3], ys[3];  // elements
    const int *start;
    int length, heads, head_dim;
    int turned, units;     // units of a head that turn 4 pairs, and with those that copy 8 dims
    int blocks, rows;      // workgroups of a sequence, and rows of one
    Divisor per_row, per_head;
};

// 4 pairs of a head from p0 on, `pairs` of them in it.
template <typename T, bool INTERLEAVED, bool BACKWARD>
VH_DEVICE void turn_four(const T *x, T *y, const float *row, int p0, int half, int pairs) {
    const float sign = BACKWARD ? -1.0f : 1.0f;
    if (pairs >= 4) {
        float v[8], cs[8];
        if (row) load_n<8>(row + 2 * p0, cs);
        if constexpr (INTERLEAVED) {
            load_n<8>(x + 2 * p0, v);
        } else {
            float lo[4], hi[4];
            load_n<4>(x + p0, lo);
            load_n<4>(x + half + p0, hi);
#pragma unroll
            for (int e = 0; e < 4; e++) v[2 * e] = lo[e], v[2 * e + 1] = hi[e];
        }
#pragma unroll
        for (int e = 0; e < 4; e++) {
            if (row) turn_pair(v[2 * e], v[2 * e + 1], cs[2 * e], sign * cs[2 * e + 1]);
            else v[2 * e] = v[2 * e + 1] = __builtin_nanf("");
        }
        if constexpr (INTERLEAVED) {
            store_n<8>(y + 2 * p0, v);
        } else {
            float lo[4], hi[4];
#pragma unroll
            for (int e = 0; e < 4; e++) lo[e] = v[2 * e], hi[e] = v[2 * e + 1];
            store_n<4>(y + p0, lo);
            store_n<4>(y + half + p0, hi);
        }
        return;
    }
    for (int i = p0; i < p0 + pairs; i++) {
        const int ia = INTERLEAVED ? 2 * i : i, ib = INTERLEAVED ? 2 * i + 1 : half + i;
        float a = (float)x[ia], b = (float)x[ib];
        if (row) turn_pair(a, b, row[2 * i], sign * row[2 * i + 1]);
        else a = b = __builtin_nanf("");
        y[ia] = (T)a;
        y[ib] = (T)b;
    }
}

template <typename T, bool INTERLEAVED, bool BACKWARD>
static __global__ __launch_bounds__(256) void rotary_kernel(RotaryArgs a) {
    const int s = (int)(blockIdx.x / (uint32_t)a.blocks);
    const int row0 = (int)(blockIdx.x % (uint32_t)a.blocks) * a.rows;
    const uint32_t n = (uint32_t)min(a.rows, a.length - row0) * a.per_row.d;
    const int64_t start = a.start ? a.start[s] : 0;
    const T *xs = static_cast<const T *>(a.x) + s * a.xs[0] + row0 * a.xs[1];
    T *ys = static_cast<T *>(a.y) + s * a.ys[0] + row0 * a.ys[1];
    const int half = a.r.dim / 2;
    for (uint32_t i = threadIdx.x; i < n; i += 256) {
        const uint32_t row = i / a.per_row, in_row = i - row * a.per_row.d;
        const uint32_t head = in_row / a.per_head;
        const int unit = (int)(in_row - head * a.per_head.d);
        const T *x = xs + row * a.xs[1] + head * a.xs[2];
        T *y = ys + row * a.ys[1] + head * a.ys[2];
        if (unit < a.turned) {
            turn_four<T, INTERLEAVED, BACKWARD>(x, y, rotation_row(a.r, start + row0 + row), 4 * unit, half, half - 4 * unit);
        } else {
            const int d = a.r.dim + 8 * (unit - a.turned);
            if (d + 8 <= a.head_dim) {
                float v[8];
                load_n<8>(x + d, v);
                store_n<8>(y + d, v);
            } else {
                for (int e = d; e < a.head_dim; e++) y[e] = x[e];
            }
        }
    }
}

struct RotaryTableArgs {
    float *table;
    int pairs, positions;
    double magnitude;
    double theta[128];
};
static __global__ __launch_bounds__(256) void rotary_table_kernel(RotaryTableArgs a) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= (int64_t)a.positions * a.pairs) return;
    const int64_t p = i / a.pairs;
    double s, c;
    sincos((double)p * a.theta[i - p * a.pairs], &s, &c);
    a.table[2 * i] = (float)(c * a.magnitude);
    a.table[2 * i + 1] = (float)(s * a.magnitude);
}

}  // namespace vh
