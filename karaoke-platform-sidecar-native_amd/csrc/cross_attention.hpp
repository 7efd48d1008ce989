// Attention of queries over keys and values of another length, with a learned
// relative position bias by buckets, and its backward pass.
//
//   x_ij = scale q_i.k_j + table[bucket(j - (start + i))][h]
//   P = softmax over the keys j < klen (causal: j <= start + i)
//   out_i = sum_j P_ij v_j;   a row that sees no key: 0
// and with delta_i = dout_i.out_i, dP_ij = dout_i.v_j, dS = P (dP - delta):
//   dq_i = scale sum_j dS_ij k_j, dk_j = scale sum_i dS_ij q_i, dv_j = sum_i P_ij dout_i
//   (dk and dv summed over the query heads that share the key head), and
//   dtable[b][h] = sum of dS over the pairs whose bucket is b.
//
// T is the type of the tensors, fp32 or bf16.  Every product runs on the matrix
// cores in 32 x 32 tiles with fp32 accumulation, the statistics, the
// exponentials and dS are fp32.  bf16 operands are the tensors as they are;
// P and dS are rounded to bf16 (by up to 2^-8 of themselves, as the outputs are)
// where they enter a product, and nowhere else: scale, bias, statistics and the
// table's gradient see the fp32 values.  A forward that keeps its state for the
// backward pass multiplies v by P in two bf16 pieces (to 2^-16): delta is the
// sum of P dP, and the table's gradient, whose terms cancel in every row, would
// show an error of 2^-8 in it as one of 2e-3 of its own norm.
//
// Operand order (both types).  v_mfma_f32_32x32x16_bf16 takes 8 values of the
// summed index per lane: lane (li = l % 32, lh = l / 32) holds row or column li
// and indexes 8 lh + e of a group of 16.  fp32 runs the same group as eight
// v_mfma_f32_32x32x2_f32, the e-th on every lane's e-th value: the groups' terms
// come in another order, so fragments are loaded alike for both types.  A result
// holds column li and rows 8 (r / 4) + 4 lh + r % 4; its registers 8 st .. 8 st + 7
// are therefore a B operand over rows {16 st + 4 lh + 0..3, 16 st + 8 + 4 lh +
// 0..3}, and the A operand beside it is read from LDS transposed in that order.
#pragma once

#include "attention.hpp"
#include "gemm_bf16.hpp"

namespace vh {

constexpr int CA_D = 64;            // head dims
constexpr int CA_TILE = 32;         // rows of a tile in LDS
constexpr int CA_MAX_BUCKETS = 128;
constexpr int CA_PAD = 63;          // distances past max_distance that the bias window holds on each side

struct CrossTensor {
    char *p;                 // element 0
    int64_t seq, row, head;  // strides in bytes
};

struct CrossArgs {
    CrossTensor q, k, v, out, dout, dq, dk, dv;
    int S, H, KV, Lq, Lk;
    int causal;
    float scale;
    const int *query_lengths, *key_lengths, *query_start;  // [S] or null
    const float *table;                                    // [buckets][H] or null
    int buckets, max_distance, bidirectional;
    float2 *stats;   // [S][H][Lq]: the maximum's place m and -log2 of sum exp(x - m); (0, -inf) without a key
    bf16 *rest;      // bf16: [S][H][Lq][64], out's rounding error, so that delta is exact; null: not kept
    float *delta;    // [S][H][Lq]
    float *dbias_part;  // [S][H][ceil(Lq / 128)][buckets]
    float *dbias;       // [buckets][H]
    // far buckets of one side: bucket near + i begins at distance edge[i]
    int side, near, edges;
    int edge[CA_MAX_BUCKETS];
};

// Bucket of a relative position (key's minus query's).
VH_HOST_DEVICE inline int cross_bucket(const CrossArgs &a, int rel) {
    const int n = rel < 0 ? -rel : a.bidirectional ? rel : 0;
    int b = n;
    if (n >= a.near) {
        b = a.near - 1;
        for (int i = 0; i < a.edges; i++) b += n >= a.edge[i] ? 1 : 0;
    }
    return a.bidirectional && rel > 0 ? b + a.side : b;
}

// --------------------------------------------------------------- operands
template <typename T>
struct Frag;
template <>
struct Frag<bf16> {
    bf16x8 v;
};
template <>
struct Frag<float> {
    floatx4 v[2];
};

VH_DEVICE void frag_mfma(floatx16 &acc, const Frag<bf16> &a, const Frag<bf16> &b) {
    acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.v, b.v, acc, 0, 0, 0);
}
VH_DEVICE void frag_mfma(floatx16 &acc, const Frag<float> &a, const Frag<float> &b) {
#pragma unroll
    for (int e = 0; e < 8; e++)
        acc = __builtin_amdgcn_mfma_f32_32x32x2f32(a.v[e >> 2][e & 3], b.v[e >> 2][e & 3], acc, 0, 0, 0);
}

// 8 consecutive elements of global memory.
VH_DEVICE Frag<bf16> frag_load(const bf16 *p) { return {*reinterpret_cast<const bf16x8 *>(p)}; }
VH_DEVICE Frag<float> frag_load(const float *p) { return {{ld4(p), ld4(p + 4)}}; }

// Registers 8 st .. 8 st + 7 of a result as a B operand.
VH_DEVICE void frag_from(Frag<bf16> &f, const floatx16 &x, int st) {
#pragma unroll
    for (int e = 0; e < 8; e++) f.v[e] = (bf16)x[8 * st + e];
}
// What rounding took from them.
VH_DEVICE void frag_rest(Frag<bf16> &rest, const Frag<bf16> &f, const floatx16 &x, int st) {
#pragma unroll
    for (int e = 0; e < 8; e++) rest.v[e] = (bf16)(x[8 * st + e] - (float)f.v[e]);
}
VH_DEVICE void frag_from(Frag<float> &f, const floatx16 &x, int st) {
#pragma unroll
    for (int e = 0; e < 8; e++) f.v[e >> 2][e & 3] = x[8 * st + e];
}

// A tile of 32 rows of 64 dims in LDS: row r at r * row bytes, its 16-byte chunk
// c in slot c ^ swz(r).  bf16 (128-byte rows: two rows cover the banks once):
// rows 2 p and 2 p + 1 are shifted by p's three bits in reverse, so that the eight
// pairs of 16 rows take eight different slots in a row read, and neighbouring
// pairs, which a transposed read takes together, differ by half a row.  fp32
// (256-byte rows): 16 rows take 16 slots, and rows 4 apart, which the two
// half-waves of a transposed read take together, differ by half a row.
template <typename T>
struct Tile {
    static constexpr int ROW = CA_D * (int)sizeof(T);
    static constexpr int BYTES = CA_TILE * ROW;
    static constexpr int CHUNKS = ROW / 16;
    static constexpr int DMA_ROWS = 1024 / ROW;  // rows of one 1 KB copy
    VH_DEVICE static int swz(int r) {
        if constexpr (sizeof(T) == 2)
            return ((r >> 1) & 1) << 2 | ((r >> 2) & 1) << 1 | ((r >> 3) & 1);
        else
            return (r & 3) | ((r >> 3) & 1) << 2 | ((r >> 2) & 1) << 3;
    }
};

// Row r, dims 16 g + 8 lh .. + 7.
VH_DEVICE Frag<bf16> tile_row(const unsigned char *t, int r, int g, int lh, bf16) {
    using L = Tile<bf16>;
    return {*reinterpret_cast<const bf16x8 *>(t + r * L::ROW + 16 * ((2 * g + lh) ^ L::swz(r)))};
}
VH_DEVICE Frag<float> tile_row(const unsigned char *t, int r, int g, int lh, float) {
    using L = Tile<float>;
    const unsigned char *p = t + r * L::ROW;
    const int c = 4 * g + 2 * lh;
    return {{*reinterpret_cast<const floatx4 *>(p + 16 * (c ^ L::swz(r))),
             *reinterpret_cast<const floatx4 *>(p + 16 * ((c + 1) ^ L::swz(r)))}};
}
// Dim 32 t + li of rows {16 st + 4 lh + 0..3, 16 st + 8 + 4 lh + 0..3}.
VH_DEVICE Frag<bf16> tile_col(const unsigned char *tile, int st, int t, int lane, bf16) {
    using L = Tile<bf16>;
    typedef __fp16 fp16x4 __attribute__((ext_vector_type(4)));
    typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
    typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
    const int lh = lane >> 5, j = lane & 15, dhalf = (lane >> 4) & 1;
    const int row = 16 * st + 4 * lh + (j >> 2);
    const int chunk = 4 * t + 2 * dhalf + ((j & 3) >> 1);
    const unsigned char *base = tile + 8 * (j & 1);
    const unsigned char *a0 = base + row * L::ROW + 16 * (chunk ^ L::swz(row));
    const unsigned char *a1 = base + (row + 8) * L::ROW + 16 * (chunk ^ L::swz(row + 8));
    // 16-bit elements moved as they are (the type only names their size)
    const fp16x4 r0 = __builtin_amdgcn_ds_read_tr16_b64_v4f16((__attribute__((address_space(3))) fp16x4 *)(a0));
    const fp16x4 r1 = __builtin_amdgcn_ds_read_tr16_b64_v4f16((__attribute__((address_space(3))) fp16x4 *)(a1));
    const u32x2 w0 = __builtin_bit_cast(u32x2, r0), w1 = __builtin_bit_cast(u32x2, r1);
    return {__builtin_bit_cast(bf16x8, u32x4{w0[0], w0[1], w1[0], w1[1]})};
}
VH_DEVICE Frag<float> tile_col(const unsigned char *tile, int st, int t, int lane, float) {
    using L = Tile<float>;
    const int li = lane & 31, lh = lane >> 5;
    Frag<float> f;
#pragma unroll
    for (int e = 0; e < 8; e++) {
        const int row = 16 * st + 8 * (e >> 2) + 4 * lh + (e & 3);
        f.v[e >> 2][e & 3] = *reinterpret_cast<const float *>(tile + row * L::ROW +
                                                              16 * ((8 * t + (li >> 2)) ^ L::swz(row)) + 4 * (li & 3));
    }
    return f;
}

// Copies rows row0 .. row0 + 31 of a tensor's sequence and head (base: its row 0)
// into a tile, 1 KB a load, the loads dealt out to the four waves.  Rows past
// `last` are copies of row `last`: what lies behind the valid rows is never read.
template <typename T>
VH_DEVICE void tile_issue(const char *base, int64_t row_bytes, int row0, int last, uint32_t tile_lds, int wave,
                          int lane) {
    using L = Tile<T>;
    const char *sbase = base + (int64_t)row0 * row_bytes;
    constexpr int LOADS = CA_TILE / L::DMA_ROWS / 4;
#pragma unroll
    for (int i = 0; i < LOADS; i++) {
        const int r0 = (LOADS * wave + i) * L::DMA_ROWS;
        const int r = r0 + lane / L::CHUNKS;
        const uint32_t off = (uint32_t)min(r, last - row0) * (uint32_t)row_bytes + 16u * (uint32_t)((lane % L::CHUNKS) ^ L::swz(r));
        lds_dma16s(off, sbase, tile_lds + (uint32_t)(r0 * L::ROW));
    }
}

VH_DEVICE int row_of(int r, int lh) { return 8 * (r >> 2) + 4 * lh + (r & 3); }
VH_DEVICE void zero16(floatx16 &x) {
#pragma unroll
    for (int r = 0; r < 16; r++) x[r] = 0.0f;
}

// LDS accesses of the wave's lanes before and after stay in that order (the
// hardware keeps a wave's; this keeps the compiler's).
VH_DEVICE void wave_order() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

constexpr float CA_LOG2E = 1.4426950408889634f;

VH_DEVICE int cross_length(const int *lengths, int s, int most) {
    return lengths ? max(0, min(lengths[s], most)) : most;
}
// Positions further out than any length act alike.
VH_DEVICE int cross_start(const CrossArgs &a, int s) {
    return a.query_start ? max(-(1 << 30), min(a.query_start[s], 1 << 30)) : 0;
}

// The bias by relative position -max_distance - 63 .. max_distance + 63 (beyond
// max_distance the bucket is the last), so that a 32 x 32 tile that is not
// wholly beyond it looks its pairs up without a clamp.
VH_DEVICE int cross_window(const CrossArgs &a) { return 2 * (a.max_distance + CA_PAD) + 1; }
VH_DEVICE void fill_bias_window(const CrossArgs &a, int h, float *window, int tid) {
    for (int i = tid; i < cross_window(a); i += 256)
        window[i] = a.table[(int64_t)cross_bucket(a, i - a.max_distance - CA_PAD) * a.H + h];
}

// Scores of a tile: x = scale s + bias, -inf where the pair is hidden.  rel0: the
// relative position of register row 0 (lh 0) against the lane's column; step: +1
// where rows are keys, -1 where they are queries.
template <bool BIAS>
VH_DEVICE void scores(const CrossArgs &a, floatx16 &x, const float *window, int tile_lo, int tile_hi, int rel0, int step,
                      int lh) {
    if constexpr (BIAS) {
        const int md = a.max_distance;
        if (tile_hi <= -md || tile_lo >= md) {
            const float b = window[tile_hi <= -md ? CA_PAD : 2 * md + CA_PAD];
#pragma unroll
            for (int r = 0; r < 16; r++) x[r] = __builtin_fmaf(x[r], a.scale, b);
        } else {
            const float *w = window + rel0 + step * 4 * lh + md + CA_PAD;
#pragma unroll
            for (int r = 0; r < 16; r++) x[r] = __builtin_fmaf(x[r], a.scale, w[step * row_of(r, 0)]);
        }
    } else {
#pragma unroll
        for (int r = 0; r < 16; r++) x[r] *= a.scale;
    }
}

// ------------------------------------------------------------------ forward
// Workgroup: 4 waves x 32 queries of one head, tiles of 32 keys.  Per wave and
// tile S^T = K Q^T, so that a lane holds 16 scores of one query, the online
// softmax, and out^T += V^T P^T from the same registers.
// KEEP: statistics, rest, and P in two pieces.
template <typename T, bool BIAS, bool KEEP>
__global__ __launch_bounds__(256, 2) void cross_forward_kernel(CrossArgs a) {
    extern __shared__ __attribute__((aligned(1024))) unsigned char smem[];
    unsigned char *Ks = smem, *Vs = smem + Tile<T>::BYTES;
    float *window = reinterpret_cast<float *>(smem + 2 * Tile<T>::BYTES);

    const int qtiles = (a.Lq + 127) / 128;
    const int task = xcd_swizzle((int)blockIdx.x, (int)gridDim.x);
    const int qt = task % qtiles, h = task / qtiles % a.H, s = task / qtiles / a.H;
    const int tid = (int)threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int li = lane & 31, lh = lane >> 5;
    const int kh = h / (a.H / a.KV);
    const int start = cross_start(a, s);
    const int qlen = cross_length(a.query_lengths, s, a.Lq), klen = cross_length(a.key_lengths, s, a.Lk);
    const int q0 = 128 * qt + 32 * wave, q = q0 + li;
    const bool active = q0 < qlen;
    int keys = klen;  // that any row of the workgroup sees
    if (a.causal) keys = min(keys, start + min(128 * qt + 128, qlen));
    if (128 * qt >= qlen) keys = 0;

    if constexpr (BIAS) {
        fill_bias_window(a, h, window, tid);
        __syncthreads();
    }
    Frag<T> qf[4];
    if (active) {
        const char *qp = a.q.p + s * a.q.seq + (int64_t)min(q, qlen - 1) * a.q.row + h * a.q.head;
#pragma unroll
        for (int g = 0; g < 4; g++) qf[g] = frag_load(reinterpret_cast<const T *>(qp) + 16 * g + 8 * lh);
    }
    floatx16 o[2];
    zero16(o[0]);
    zero16(o[1]);
    float m = -INFINITY, l = 0.0f;
    const char *kp = a.k.p + s * a.k.seq + kh * a.k.head, *vp = a.v.p + s * a.v.seq + kh * a.v.head;
    const uint32_t k_lds = (uint32_t)(uintptr_t)Ks, v_lds = (uint32_t)(uintptr_t)Vs;
    for (int k0 = 0; k0 < keys; k0 += CA_TILE) {
        tile_issue<T>(kp, a.k.row, k0, klen - 1, k_lds, wave, lane);
        tile_issue<T>(vp, a.v.row, k0, klen - 1, v_lds, wave, lane);
        wait_vmcnt<0>();
        __syncthreads();
        if (active && (!a.causal || k0 <= start + q0 + 31)) {
            floatx16 x;
            zero16(x);
#pragma unroll
            for (int g = 0; g < 4; g++) frag_mfma(x, tile_row(Ks, li, g, lh, T()), qf[g]);
            const int lo = k0 - (start + q0 + 31), hi = k0 + 31 - (start + q0);
            scores<BIAS>(a, x, window, lo, hi, k0 - (start + q), 1, lh);
            const int seen = (a.causal ? min(klen, start + q + 1) : klen) - k0;  // rows of the tile that the lane's query sees
            if (k0 + 32 > klen || (a.causal && hi > 0)) {
#pragma unroll
                for (int r = 0; r < 16; r++)
                    if (row_of(r, lh) >= seen) x[r] = -INFINITY;
            }
            float mt = x[0];
#pragma unroll
            for (int r = 1; r < 16; r++) mt = fmaxf(mt, x[r]);
            mt = fmaxf(mt, __shfl_xor(mt, 32, 64));
            const float mn = fmaxf(m, mt);
            const float base = mn == -INFINITY ? 0.0f : mn;  // -inf - -inf is no number
            const float c = __builtin_amdgcn_exp2f((m - base) * CA_LOG2E);
            m = mn;
            l *= c;
#pragma unroll
            for (int r = 0; r < 16; r++) {
                x[r] = __builtin_amdgcn_exp2f((x[r] - base) * CA_LOG2E);
                l += x[r];
                o[0][r] *= c;
                o[1][r] *= c;
            }
#pragma unroll
            for (int st = 0; st < 2; st++) {
                Frag<T> pb;
                frag_from(pb, x, st);
#pragma unroll
                for (int t = 0; t < 2; t++) {
                    const Frag<T> vf = tile_col(Vs, st, t, lane, T());
                    frag_mfma(o[t], vf, pb);
                    if constexpr (KEEP && sizeof(T) == 2) {
                        Frag<T> pr;
                        frag_rest(pr, pb, x, st);
                        frag_mfma(o[t], vf, pr);
                    }
                }
            }
        }
        __syncthreads();
    }
    if (q >= a.Lq) return;
    l += __shfl_xor(l, 32, 64);
    const bool seen = q < qlen && (l > 0.0f || l != l);  // a row of NaN stays one
    const float inv = seen ? 1.0f / l : 0.0f;
    const int64_t row = ((int64_t)s * a.H + h) * a.Lq + q;
    if (KEEP && lh == 0) a.stats[row] = make_float2(seen ? m : 0.0f, seen ? -log2f(l) : -INFINITY);
    T *op = reinterpret_cast<T *>(a.out.p + s * a.out.seq + (int64_t)q * a.out.row + h * a.out.head);
#pragma unroll
    for (int t = 0; t < 2; t++)
#pragma unroll
        for (int rq = 0; rq < 4; rq++) {
            const int d = 32 * t + 8 * rq + 4 * lh;
            floatx4 y;
#pragma unroll
            for (int r = 0; r < 4; r++) y[r] = seen ? o[t][4 * rq + r] * inv : 0.0f;
            st4(op + d, y);
            if constexpr (KEEP && sizeof(T) == 2) {
                const bf16x4 yr = to_bf16x4(y);
#pragma unroll
                for (int r = 0; r < 4; r++) y[r] -= (float)yr[r];
                st4(a.rest + row * CA_D + d, y);
            }
        }
}

// ----------------------------------------------------------------- backward
// dq, delta and the table's gradient: workgroup and tiles as the forward's.
// dbias: a tile's dS are summed along its 63 diagonals in the wave's own LDS by
// ds_add_f32, whose lanes take different diagonals (the half-waves have an array
// each), then each diagonal is added to its bucket's slot of that lane: the order
// of every sum is fixed.  Tiles wholly beyond max_distance have one bucket and
// are summed in registers.
struct DbiasLds {
    float diag[4][2][64];
    float far[4][2];
};
template <typename T, bool BIAS>
__global__ __launch_bounds__(256, 2) void cross_dq_kernel(CrossArgs a) {
    extern __shared__ __attribute__((aligned(1024))) unsigned char smem[];
    unsigned char *Ks = smem, *Vs = smem + Tile<T>::BYTES;
    DbiasLds *db = reinterpret_cast<DbiasLds *>(smem + 2 * Tile<T>::BYTES);
    float *slots = reinterpret_cast<float *>(db + 1);  // [4][buckets][32]
    float *window = slots + 128 * a.buckets;

    const int qtiles = (a.Lq + 127) / 128;
    const int task = xcd_swizzle((int)blockIdx.x, (int)gridDim.x);
    const int qt = task % qtiles, h = task / qtiles % a.H, s = task / qtiles / a.H;
    const int tid = (int)threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int li = lane & 31, lh = lane >> 5;
    const int kh = h / (a.H / a.KV);
    const int start = cross_start(a, s);
    const int qlen = cross_length(a.query_lengths, s, a.Lq), klen = cross_length(a.key_lengths, s, a.Lk);
    const int q0 = 128 * qt + 32 * wave, q = q0 + li;
    const bool active = q0 < qlen;
    int keys = klen;
    if (a.causal) keys = min(keys, start + min(128 * qt + 128, qlen));
    if (128 * qt >= qlen) keys = 0;
    const bool with_dbias = BIAS && a.dbias_part != nullptr;

    if constexpr (BIAS) {
        fill_bias_window(a, h, window, tid);
        if (with_dbias) {
            for (int i = tid; i < 128 * a.buckets; i += 256) slots[i] = 0.0f;
            for (int i = tid; i < 4 * 2 * 64; i += 256) (&db->diag[0][0][0])[i] = 0.0f;
        }
        __syncthreads();
    }
    Frag<T> qf[4], df[4];
    float delta = 0.0f, m = 0.0f, nl = -INFINITY;
    const int64_t row = ((int64_t)s * a.H + h) * a.Lq + min(q, qlen - 1);
    if (active) {
        const int64_t qr = min(q, qlen - 1);
        const T *qp = reinterpret_cast<const T *>(a.q.p + s * a.q.seq + qr * a.q.row + h * a.q.head);
        const T *dp = reinterpret_cast<const T *>(a.dout.p + s * a.dout.seq + qr * a.dout.row + h * a.dout.head);
        const T *op = reinterpret_cast<const T *>(a.out.p + s * a.out.seq + qr * a.out.row + h * a.out.head);
#pragma unroll
        for (int g = 0; g < 4; g++) {
            const int d = 16 * g + 8 * lh;
            qf[g] = frag_load(qp + d);
            df[g] = frag_load(dp + d);
            const Frag<T> of = frag_load(op + d);
            if constexpr (sizeof(T) == 2) {
                const Frag<T> rf = frag_load(a.rest + row * CA_D + d);
#pragma unroll
                for (int e = 0; e < 8; e++) delta += (float)df[g].v[e] * ((float)of.v[e] + (float)rf.v[e]);
            } else {
#pragma unroll
                for (int e = 0; e < 8; e++) delta += df[g].v[e >> 2][e & 3] * of.v[e >> 2][e & 3];
            }
        }
        delta += __shfl_xor(delta, 32, 64);
        const float2 st = a.stats[row];
        m = st.x;
        nl = st.y;
        if (lh == 0 && q < qlen) a.delta[row] = delta;
    }
    floatx16 acc[2];
    zero16(acc[0]);
    zero16(acc[1]);
    float far_lo = 0.0f, far_hi = 0.0f;
    const char *kp = a.k.p + s * a.k.seq + kh * a.k.head, *vp = a.v.p + s * a.v.seq + kh * a.v.head;
    const uint32_t k_lds = (uint32_t)(uintptr_t)Ks, v_lds = (uint32_t)(uintptr_t)Vs;
    for (int k0 = 0; k0 < keys; k0 += CA_TILE) {
        tile_issue<T>(kp, a.k.row, k0, klen - 1, k_lds, wave, lane);
        tile_issue<T>(vp, a.v.row, k0, klen - 1, v_lds, wave, lane);
        wait_vmcnt<0>();
        __syncthreads();
        if (active && (!a.causal || k0 <= start + q0 + 31)) {
            floatx16 x, dp;
            zero16(x);
            zero16(dp);
#pragma unroll
            for (int g = 0; g < 4; g++) {
                frag_mfma(x, tile_row(Ks, li, g, lh, T()), qf[g]);
                frag_mfma(dp, tile_row(Vs, li, g, lh, T()), df[g]);
            }
            const int lo = k0 - (start + q0 + 31), hi = k0 + 31 - (start + q0);
            scores<BIAS>(a, x, window, lo, hi, k0 - (start + q), 1, lh);
            int seen = (a.causal ? min(klen, start + q + 1) : klen) - k0;
            if (q >= qlen) seen = 0;
#pragma unroll
            for (int r = 0; r < 16; r++) {
                const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(x[r] - m, CA_LOG2E, nl));
                x[r] = row_of(r, lh) < seen ? p * (dp[r] - delta) : 0.0f;
            }
            if constexpr (BIAS) {
                if (with_dbias) {
                    const int md = a.max_distance;
                    if (hi <= -md || lo >= md) {
                        float sum = 0.0f;
#pragma unroll
                        for (int r = 0; r < 16; r++) sum += x[r];
                        if (hi <= -md) far_lo += sum;
                        else far_hi += sum;
                    } else {
                        float *w = &db->diag[wave][lh][31 - li + 4 * lh];
#pragma unroll
                        for (int r = 0; r < 16; r++)
                            __hip_atomic_fetch_add(w + row_of(r, 0), x[r], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WAVEFRONT);
                        wave_order();
                        float *d = &db->diag[wave][0][lane];
                        const float v = d[0] + d[64];
                        d[0] = 0.0f;
                        d[64] = 0.0f;
                        const float v1 = __shfl(v, (lane & 31) + 32, 64);
                        if (lane < 32) {  // the second may be the first one's bucket
                            float *sl = slots + wave * a.buckets * 32 + lane;
                            sl[32 * cross_bucket(a, lo + lane)] += v;
                            sl[32 * cross_bucket(a, lo + lane + 32)] += v1;
                        }
                        wave_order();
                    }
                }
            }
#pragma unroll
            for (int st = 0; st < 2; st++) {
                Frag<T> sb;
                frag_from(sb, x, st);
#pragma unroll
                for (int t = 0; t < 2; t++) frag_mfma(acc[t], tile_col(Ks, st, t, lane, T()), sb);
            }
        }
        __syncthreads();
    }
    if constexpr (BIAS) {
        if (with_dbias) {
            far_lo = wave_sum(far_lo);
            far_hi = wave_sum(far_hi);
            if (lane == 0) {
                db->far[wave][0] = far_lo;
                db->far[wave][1] = far_hi;
            }
            __syncthreads();
            for (int b = tid; b < a.buckets; b += 256) {
                float sum = 0.0f;
                for (int w = 0; w < 4; w++) {
                    for (int i = 0; i < 32; i++) sum += slots[(w * a.buckets + b) * 32 + (i + b) % 32];
                    if (b == cross_bucket(a, -a.max_distance)) sum += db->far[w][0];
                    if (b == cross_bucket(a, a.max_distance)) sum += db->far[w][1];
                }
                a.dbias_part[(((int64_t)s * a.H + h) * qtiles + qt) * a.buckets + b] = sum;
            }
        }
    }
    if (q >= a.Lq) return;
    T *out = reinterpret_cast<T *>(a.dq.p + s * a.dq.seq + (int64_t)q * a.dq.row + h * a.dq.head);
#pragma unroll
    for (int t = 0; t < 2; t++)
#pragma unroll
        for (int rq = 0; rq < 4; rq++) {
            floatx4 y;
#pragma unroll
            for (int r = 0; r < 4; r++) y[r] = q < qlen ? acc[t][4 * rq + r] * a.scale : 0.0f;
            st4(out + 32 * t + 8 * rq + 4 * lh, y);
        }
}

// dk and dv: workgroup of 4 waves x 32 keys of one key head, tiles of 32 queries
// of every query head that shares it.  S = Q K^T with the keys as columns, so
// that P and dS are B operands of dv^T += dout^T P and dk^T += Q^T dS as they are.
struct RowStats {
    float m[CA_TILE], nl[CA_TILE], delta[CA_TILE];
};
template <typename T, bool BIAS>
__global__ __launch_bounds__(256, 2) void cross_dkv_kernel(CrossArgs a) {
    extern __shared__ __attribute__((aligned(1024))) unsigned char smem[];
    unsigned char *Qs = smem, *Ds = smem + Tile<T>::BYTES;
    RowStats *rs = reinterpret_cast<RowStats *>(smem + 2 * Tile<T>::BYTES);
    float *window = reinterpret_cast<float *>(rs + 1);

    const int ktiles = (a.Lk + 127) / 128;
    const int task = xcd_swizzle((int)blockIdx.x, (int)gridDim.x);
    const int kt = task % ktiles, kh = task / ktiles % a.KV, s = task / ktiles / a.KV;
    const int tid = (int)threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int li = lane & 31, lh = lane >> 5;
    const int start = cross_start(a, s);
    const int qlen = cross_length(a.query_lengths, s, a.Lq), klen = cross_length(a.key_lengths, s, a.Lk);
    const int k0 = 128 * kt + 32 * wave, key = k0 + li;
    const bool active = k0 < klen;
    // the first query that sees a key of the workgroup
    int first = 0;
    if (a.causal) first = max(0, min(128 * kt - start, qlen)) / CA_TILE * CA_TILE;
    if (128 * kt >= klen) first = qlen;

    Frag<T> kf[4], vf[4];
    if (active) {
        const int64_t kr = min(key, klen - 1);
        const T *kp = reinterpret_cast<const T *>(a.k.p + s * a.k.seq + kr * a.k.row + kh * a.k.head);
        const T *vp = reinterpret_cast<const T *>(a.v.p + s * a.v.seq + kr * a.v.row + kh * a.v.head);
#pragma unroll
        for (int g = 0; g < 4; g++) {
            kf[g] = frag_load(kp + 16 * g + 8 * lh);
            vf[g] = frag_load(vp + 16 * g + 8 * lh);
        }
    }
    floatx16 dk[2], dv[2];
#pragma unroll
    for (int t = 0; t < 2; t++) {
        zero16(dk[t]);
        zero16(dv[t]);
    }
    const uint32_t q_lds = (uint32_t)(uintptr_t)Qs, d_lds = (uint32_t)(uintptr_t)Ds;
    const int G = a.H / a.KV;
    for (int h = kh * G; h < kh * G + G; h++) {
        const char *qp = a.q.p + s * a.q.seq + h * a.q.head, *dp_ = a.dout.p + s * a.dout.seq + h * a.dout.head;
        const int64_t row = ((int64_t)s * a.H + h) * a.Lq;
        if constexpr (BIAS) {
            __syncthreads();  // the last head's window has been read
            fill_bias_window(a, h, window, tid);
        }
        for (int q0 = first; q0 < qlen; q0 += CA_TILE) {
            tile_issue<T>(qp, a.q.row, q0, qlen - 1, q_lds, wave, lane);
            tile_issue<T>(dp_, a.dout.row, q0, qlen - 1, d_lds, wave, lane);
            if (tid < CA_TILE) {
                const int q = min(q0 + tid, qlen - 1);
                const float2 st = a.stats[row + q];
                rs->m[tid] = st.x;
                rs->nl[tid] = q0 + tid < qlen ? st.y : -INFINITY;
                rs->delta[tid] = a.delta[row + q];
            }
            wait_vmcnt<0>();
            __syncthreads();
            if (active && (!a.causal || k0 <= start + q0 + 31)) {
                floatx16 x, dp;
                zero16(x);
                zero16(dp);
#pragma unroll
                for (int g = 0; g < 4; g++) {
                    frag_mfma(x, tile_row(Qs, li, g, lh, T()), kf[g]);
                    frag_mfma(dp, tile_row(Ds, li, g, lh, T()), vf[g]);
                }
                const int lo = k0 - (start + q0 + 31), hi = k0 + 31 - (start + q0);
                scores<BIAS>(a, x, window, lo, hi, key - (start + q0), -1, lh);
                // rows below `hidden` come before the lane's key
                const int hidden = a.causal ? key - start - q0 : -1;
#pragma unroll
                for (int r = 0; r < 16; r++) {
                    const int i = row_of(r, lh);
                    const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(x[r] - rs->m[i], CA_LOG2E, rs->nl[i]));
                    const bool vis = i >= hidden && q0 + i < qlen;
                    x[r] = vis ? p : 0.0f;
                    dp[r] = vis ? p * (dp[r] - rs->delta[i]) : 0.0f;
                }
#pragma unroll
                for (int st = 0; st < 2; st++) {
                    Frag<T> pb, sb;
                    frag_from(pb, x, st);
                    frag_from(sb, dp, st);
#pragma unroll
                    for (int t = 0; t < 2; t++) {
                        frag_mfma(dv[t], tile_col(Ds, st, t, lane, T()), pb);
                        frag_mfma(dk[t], tile_col(Qs, st, t, lane, T()), sb);
                    }
                }
            }
            __syncthreads();
        }
    }
    if (key >= a.Lk) return;
    T *pk = reinterpret_cast<T *>(a.dk.p + s * a.dk.seq + (int64_t)key * a.dk.row + kh * a.dk.head);
    T *pv = reinterpret_cast<T *>(a.dv.p + s * a.dv.seq + (int64_t)key * a.dv.row + kh * a.dv.head);
#pragma unroll
    for (int t = 0; t < 2; t++)
#pragma unroll
        for (int rq = 0; rq < 4; rq++) {
            floatx4 y, z;
#pragma unroll
            for (int r = 0; r < 4; r++) {
                y[r] = key < klen ? dk[t][4 * rq + r] * a.scale : 0.0f;
                z[r] = key < klen ? dv[t][4 * rq + r] : 0.0f;
            }
            st4(pk + 32 * t + 8 * rq + 4 * lh, y);
            st4(pv + 32 * t + 8 * rq + 4 * lh, z);
        }
}

// dtable[b][h]: the workgroups' sums in the order of sequences and query tiles.
static __global__ __launch_bounds__(128) void cross_dbias_kernel(CrossArgs a) {
    const int h = (int)blockIdx.x, b = (int)threadIdx.x;
    if (b >= a.buckets) return;
    const int qtiles = (a.Lq + 127) / 128;
    float sum = 0.0f;
    for (int s = 0; s < a.S; s++)
        for (int t = 0; t < qtiles; t++) sum += a.dbias_part[(((int64_t)s * a.H + h) * qtiles + t) * a.buckets + b];
    a.dbias[(int64_t)b * a.H + h] = sum;
}

}  // namespace vh
