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
// T is the type of the tensors, fp32 or bf16.  Every product runs on the bf16 matrix
// cores in 32 x 32 tiles with fp32 accumulation; the statistics, the exponentials
// and dS are fp32.  fp32 operands are the exact sums of three bf16 pieces each
// (gemm_split.hpp), multiplied in the six products of pieces that reach 2^-24 of
// the whole: six instructions of 32 cycles where the fp32 one takes eight of 64,
// beside 5.5 others a value to split it.  bf16 operands are the tensors as they are;
// P and dS are rounded to bf16 (by up to 2^-8 of themselves, as the outputs are)
// where they enter a product, and nowhere else: scale, bias, statistics and the
// table's gradient see the fp32 values.  delta stands for the sum of P dP, and out
// rounded to bf16, or made of rounded P, would put an error of 2^-8 into it.  So a
// forward that keeps its state for the backward pass multiplies v by P in two bf16
// pieces and keeps what rounding takes from out; with a bias in three pieces, and
// the rest in fp32, since dS sums to 0 over a row and the table's gradient is what
// is left of such sums (14 x 8 x 4089 rows over 60 keys, nearly all in one bucket:
// off by 2.8e-5 of its norm with two pieces and a bf16 rest).
//
// Scores are kept times log2(e): without a bias as s = q.k, the factor scale log2(e)
// being multiplied in the exponential's argument, exp2(s c - m c), one operation a
// score (a negative scale turns q's, or k's, sign instead); with a bias as s c + b
// log2(e), where a finite b stays finite.
//
// Operand order.  v_mfma_f32_32x32x16_bf16 takes 8 values of the summed index per
// lane: lane (li = l % 32, lh = l / 32) holds row or column li and indexes 8 lh + e
// of a group of 16.  A result holds column li and rows 8 (r / 4) + 4 lh + r % 4; its
// registers 8 st .. 8 st + 7 are therefore a B operand over rows {16 st + 4 lh +
// 0..3, 16 st + 8 + 4 lh + 0..3}, and the A operand beside it is read transposed in
// that order.
#pragma once

#include "attention.hpp"
#include "gemm_bf16.hpp"
#include "gemm_split.hpp"

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
    float scale2;    // |scale| log2(e), at least the smallest normal number
    const int *query_lengths, *key_lengths, *query_start;  // [S] or null
    const float *table;                                    // [buckets][H] or null
    int buckets, max_distance, bidirectional;
    // [S][H][Lq], in powers of two: (M, -) with P = exp2(x log2(e) - M); with a bias
    // (m, n) with P = exp2((x log2(e) - m) + n), since one as low as the type goes
    // leaves no bits for n beside it
    float2 *stats;
    void *rest;      // bf16: [S][H][Lq][64], what rounding took from out, in bf16 (with a bias in fp32)
    float *rows;     // backward: [S][H][ceil(Lq / 32)] tiles of RowStats
    // Sums over a part of the keys (forward, dq) or queries (dk, dv), when a row
    // tile's work is split: parts pieces, [part][S][H][Lq][64] and their (m, l);
    // [part][S][KV][Lk][64] for dk, dv, part = head among those that share the
    // keys / kv_heads * kv_parts + piece, a workgroup taking kv_heads of them
    int parts, kv_parts, kv_heads;
    float *part_o;
    float2 *part_ml;
    float *part_dk, *part_dv;
    float *dbias_part;  // [H][dbias_parts][buckets]
    int dbias_parts;    // per head: sequences x row tiles x pieces
    floatx4 *dbias_rows;  // pieces: [H][dbias_parts][32] rows' (sum of dS, probability in either side's far buckets, -)
    float *dbias;       // [buckets][H]
    // far buckets of one side: bucket near + i begins at distance edge[i]
    int side, near, edges;
    float per_octave;  // far buckets in a doubling of the distance
    int edge[CA_MAX_BUCKETS];
};

// Bucket of a distance on its side: its place among the edges, guessed by their
// logarithm and put right by the edges themselves.
VH_HOST_DEVICE inline int side_bucket(const CrossArgs &a, int n) {
    if (n < a.near) return n;
    int i = (int)(log2f((float)n / (float)a.near) * a.per_octave);
    i = i < 0 ? 0 : i > a.edges - 1 ? a.edges - 1 : i;
    while (i > 0 && n < a.edge[i]) i--;
    while (i + 1 < a.edges && n >= a.edge[i + 1]) i++;
    return a.near + i;
}
// Bucket of a relative position (key's minus query's).
VH_HOST_DEVICE inline int cross_bucket(const CrossArgs &a, int rel) {
    const int b = side_bucket(a, rel < 0 ? -rel : a.bidirectional ? rel : 0);
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
// fp32's in three bf16 pieces, the largest first.
struct Pieces {
    bf16x8 p[3];
};
VH_DEVICE void frag_mfma(floatx16 &acc, const Pieces &a, const Pieces &b) {
    constexpr int ia[6] = {2, 0, 1, 1, 0, 0}, ib[6] = {0, 2, 1, 0, 1, 0};  // small products first
#pragma unroll
    for (int i = 0; i < 6; i++)
        acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.p[ia[i]], b.p[ib[i]], acc, 0, 0, 0);
}
// What a product takes for a fragment.
VH_DEVICE const Frag<bf16> &operand(const Frag<bf16> &f) { return f; }
VH_DEVICE Pieces operand(const Frag<float> &f) {
    Pieces o;
    split8(f.v[0], f.v[1], o.p[0], o.p[1], o.p[2]);
    return o;
}
template <typename T>
struct Operand {
    typedef Frag<bf16> type;
};
template <>
struct Operand<float> {
    typedef Pieces type;
};

// 8 consecutive elements of global memory.
VH_DEVICE Frag<bf16> frag_load(const bf16 *p) { return {*reinterpret_cast<const bf16x8 *>(p)}; }
VH_DEVICE Frag<float> frag_load(const float *p) { return {{ld4(p), ld4(p + 4)}}; }

VH_DEVICE void frag_negate(Frag<bf16> &f) { f.v = -f.v; }
VH_DEVICE void frag_negate(Frag<float> &f) {
    f.v[0] = -f.v[0];
    f.v[1] = -f.v[1];
}

// Registers 8 st .. 8 st + 7 of a result as a B operand.
VH_DEVICE void frag_from(Frag<bf16> &f, const floatx16 &x, int st) {
#pragma unroll
    for (int e = 0; e < 8; e++) f.v[e] = (bf16)x[8 * st + e];
}
// What rounding took from them: x becomes it, f its next piece.
VH_DEVICE void frag_rest(Frag<bf16> &f, floatx16 &x, int st) {
#pragma unroll
    for (int e = 0; e < 8; e++) x[8 * st + e] -= (float)f.v[e];
    frag_from(f, x, st);
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

// Which (sequence, head) pair and which of its tiles a workgroup takes.  The pairs
// are dealt out to the 8 XCDs in turn (workgroup i runs on XCD i % 8), so that a
// pair's tiles find their keys in one L2 and a batch's long and short sequences are
// spread evenly; where that leaves the XCDs unequal (few pairs, not a multiple of
// 8), workgroups are taken as they come.  False: none (the last round of pairs).
constexpr bool pairs_by_xcd(int64_t pairs) { return pairs % 8 == 0 || pairs >= 64; }
VH_DEVICE bool pair_task(int pairs, int tiles, int &pair, int &tile) {
    int i = (int)blockIdx.x;
    pair = i / tiles;
    tile = i % tiles;
    if (!pairs_by_xcd(pairs)) return true;
    const int xcd = i % 8;
    i /= 8;
    pair = i / tiles * 8 + xcd;
    tile = i % tiles;
    return pair < pairs;
}

// Where a product's operands come from.  A streamed tile: in LDS, or (fp32) as it
// lies in global memory, rows past `last` (the tile's own count) read as row `last`.
template <typename T>
struct LdsTile {
    const unsigned char *p;
    VH_DEVICE Frag<T> row(int g, int lane) const { return tile_row(p, lane & 31, g, lane >> 5, T()); }
    VH_DEVICE Frag<T> col(int st, int t, int lane) const { return tile_col(p, st, t, lane, T()); }
};
struct GlobalTile {
    const char *p;  // row 0 of the tile, the same in every lane
    uint32_t row_bytes;
    int last;
    VH_DEVICE uint32_t at(int r) const { return (uint32_t)min(r, last) * row_bytes; }
    VH_DEVICE Frag<float> row(int g, int lane) const {
        return frag_load(reinterpret_cast<const float *>(p + (at(lane & 31) + 64u * g + 32u * (lane >> 5))));
    }
    VH_DEVICE Frag<float> col(int st, int t, int lane) const {
        Frag<float> f;
#pragma unroll
        for (int e = 0; e < 8; e++)
            f.v[e >> 2][e & 3] = *reinterpret_cast<const float *>(
                p + (at(16 * st + 8 * (e >> 2) + 4 * (lane >> 5) + (e & 3)) + 128u * t + 4u * (lane & 31)));
        return f;
    }
};
// The operand that stays: 32 rows in registers, or in a tile of LDS.
template <typename T>
struct RegRows {
    typename Operand<T>::type f[4];
    VH_DEVICE const typename Operand<T>::type &get(int g, int) const { return f[g]; }
};
struct LdsPieces {
    const unsigned char *p;  // three bf16 tiles
    VH_DEVICE Pieces get(int g, int lane) const {
        Pieces o;
#pragma unroll
        for (int i = 0; i < 3; i++) o.p[i] = tile_row(p + i * Tile<bf16>::BYTES, lane & 31, g, lane >> 5, bf16()).v;
        return o;
    }
};
// Dims 16 g + 8 lh .. + 7 of row li into them.
VH_DEVICE void put_row(unsigned char *t, int g, int lane, const Pieces &o) {
    using L = Tile<bf16>;
    unsigned char *p = t + (lane & 31) * L::ROW + 16 * ((2 * g + (lane >> 5)) ^ L::swz(lane & 31));
#pragma unroll
    for (int i = 0; i < 3; i++) *reinterpret_cast<bf16x8 *>(p + i * L::BYTES) = o.p[i];
}

// The same pointer, in scalar registers: the wave's lanes all have it.
VH_DEVICE const char *uniform(const void *from) {
    const uint64_t p = (uint64_t)from;
    return reinterpret_cast<const char *>((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(p >> 32)) << 32 |
                                          (uint32_t)__builtin_amdgcn_readfirstlane((int)p));
}

// Copies rows row0 .. row0 + 31 of a tensor's sequence and head (base: its row 0)
// into a tile, 1 KB a load, the loads dealt out to WAVES waves.  Rows past `last`
// are copies of row `last`: what lies behind the rows that count is never read (a
// probability of 0 would not hide a NaN there).
template <typename T, int WAVES>
VH_DEVICE void tile_issue(const char *base, int64_t row_bytes, int row0, int last, uint32_t tile_lds, int wave,
                          int lane) {
    using L = Tile<T>;
    const char *sbase = uniform(base + (int64_t)row0 * row_bytes);
    tile_lds = (uint32_t)__builtin_amdgcn_readfirstlane((int)tile_lds);
    constexpr int LOADS = CA_TILE / L::DMA_ROWS / WAVES;
#pragma unroll
    for (int i = 0; i < LOADS; i++) {
        const int r0 = (LOADS * wave + i) * L::DMA_ROWS;
        const int r = r0 + lane / L::CHUNKS;
        const uint32_t off = (uint32_t)min(r, last - row0) * (uint32_t)row_bytes + 16u * (uint32_t)((lane % L::CHUNKS) ^ L::swz(r));
        lds_dma16s(off, sbase, tile_lds + (uint32_t)(r0 * L::ROW));
    }
}
VH_DEVICE void wait_lds() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

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
    return lengths ? max(0, min(__builtin_amdgcn_readfirstlane(lengths[s]), most)) : most;
}
// Positions further out than any length act alike.
VH_DEVICE int cross_start(const CrossArgs &a, int s) {
    return a.query_start ? max(-(1 << 30), min(__builtin_amdgcn_readfirstlane(a.query_start[s]), 1 << 30)) : 0;
}

// The bias by relative position -max_distance - 63 .. max_distance + 63 (beyond
// max_distance the bucket is the last), so that a 32 x 32 tile that is not
// wholly beyond it looks its pairs up without a clamp.
VH_DEVICE int cross_window(const CrossArgs &a) { return 2 * (a.max_distance + CA_PAD) + 1; }
VH_DEVICE float bias_log2(float b) {
    const float y = b * CA_LOG2E;
    return __builtin_isinf(y) && !__builtin_isinf(b) ? __builtin_copysignf(3.402823466e38f, b) : y;
}
// bias(i, bucket): place i of the window, both sides of every distance at once.
template <typename Fill>
VH_DEVICE void fill_window(const CrossArgs &a, int tid, Fill fill) {
    const int zero = a.max_distance + CA_PAD;
    for (int n = tid; n <= zero; n += 256) {
        const int b = side_bucket(a, n);
        fill(zero - n, b);
        if (n) fill(zero + n, a.bidirectional ? b + a.side : 0);
    }
}
VH_DEVICE void fill_bias_window(const CrossArgs &a, int h, float *window, int tid) {
    fill_window(a, tid, [&](int i, int b) { window[i] = bias_log2(a.table[(int64_t)b * a.H + h]); });
}
VH_DEVICE void fill_bucket_window(const CrossArgs &a, unsigned char *window, int tid) {
    fill_window(a, tid, [&](int i, int b) { window[i] = (unsigned char)b; });
}

// Scores of a tile with the bias.  rel0: the relative position of register row 0
// (lh 0) against the lane's column; step: +1 where rows are keys, -1 where they
// are queries.
VH_DEVICE void add_bias(const CrossArgs &a, floatx16 &x, const float *window, int tile_lo, int tile_hi, int rel0,
                        int step, int lh) {
    const int md = a.max_distance;
    if (tile_hi <= -md || tile_lo >= md) {
        const float b = window[tile_hi <= -md ? CA_PAD : 2 * md + CA_PAD];
#pragma unroll
        for (int r = 0; r < 16; r++) x[r] = __builtin_fmaf(x[r], a.scale2, b);
    } else {
        const float *w = window + rel0 + step * 4 * lh + md + CA_PAD;
#pragma unroll
        for (int r = 0; r < 16; r++) x[r] = __builtin_fmaf(x[r], a.scale2, w[step * row_of(r, 0)]);
    }
}

// ------------------------------------------------------------------ forward
// A wave's 32 query rows as columns: running maximum (of s, or of s c + b with a
// bias), the same in the exponent (0 while the row has seen no key: -inf - -inf is
// no number), sum and out^T.
struct RowState {
    floatx16 o[2];
    float m, mc, l;
    VH_DEVICE void clear() {
        zero16(o[0]);
        zero16(o[1]);
        m = -INFINITY;
        mc = 0.0f;
        l = 0.0f;
    }
    VH_DEVICE float top() const { return m == -INFINITY ? m : mc; }  // the maximum in powers of two
};

// q's fragment g, of the scale's sign.
template <typename T>
VH_DEVICE Frag<T> load_query(const CrossArgs &a, const char *row, int g, int lh) {
    Frag<T> f = frag_load(reinterpret_cast<const T *>(row) + 16 * g + 8 * lh);
    if (a.scale < 0.0f) frag_negate(f);
    return f;
}
// rows of the streamed tile x the held rows, over the head's 64 dims, added to x
template <typename Tile, typename Held>
VH_DEVICE void dot_tile(floatx16 &x, const Tile &tile, const Held &held, int lane) {
#pragma unroll
    for (int g = 0; g < 4; g++) frag_mfma(x, operand(tile.row(g, lane)), held.get(g, lane));
}
template <typename Tile, typename Held>
VH_DEVICE void scores(floatx16 &x, const Tile &tile, const Held &held, int lane) {
    zero16(x);
    dot_tile(x, tile, held, lane);
}

// One tile of keys: x holds its scores on entry; seen: rows of the tile that the
// lane's query sees, -inf past them where mask says that a lane has fewer than 32.
// The maximum is raised only when a tile exceeds it by more than 2^8, which fp32
// sums absorb: the rescaling runs on a few tiles of a row.
template <bool BIAS>
VH_DEVICE void softmax_tile(RowState &st, floatx16 &x, float c, bool mask, int seen, int lh) {
    if (mask) {
#pragma unroll
        for (int r = 0; r < 16; r++)
            if (row_of(r, lh) >= seen) x[r] = -INFINITY;
    }
    float mt = x[0];
#pragma unroll
    for (int r = 1; r < 16; r++) mt = fmaxf(mt, x[r]);
    mt = fmaxf(mt, __shfl_xor(mt, 32, 64));
    const bool grow = BIAS ? mt - 8.0f > st.m : (mt - st.m) * c > 8.0f;
    if (__any(grow)) {
        const float mn = fmaxf(st.m, mt);
        const float mc = mn == -INFINITY ? 0.0f : BIAS ? mn : mn * c;
        const float f = st.m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(BIAS ? st.m - mn : (st.m - mn) * c);
        st.m = mn;
        st.mc = mc;
        st.l *= f;
#pragma unroll
        for (int r = 0; r < 16; r++) {
            st.o[0][r] *= f;
            st.o[1][r] *= f;
        }
    }
#pragma unroll
    for (int r = 0; r < 16; r++) {
        x[r] = __builtin_amdgcn_exp2f(BIAS ? x[r] - st.mc : __builtin_fmaf(x[r], c, -st.mc));
        st.l += x[r];
    }
}
// out^T += V^T P^T.
template <typename T, bool BIAS, bool KEEP, typename Tile>
VH_DEVICE void values_tile(RowState &st, floatx16 &x, const Tile &v, int lane) {
#pragma unroll
    for (int g = 0; g < 2; g++) {
        Frag<T> pb;
        frag_from(pb, x, g);
        typename Operand<T>::type vf[2];
        const auto po = operand(pb);
#pragma unroll
        for (int t = 0; t < 2; t++) {
            vf[t] = operand(v.col(g, t, lane));
            frag_mfma(st.o[t], vf[t], po);
        }
        if constexpr (KEEP && sizeof(T) == 2) {
#pragma unroll
            for (int i = 0; i < (BIAS ? 2 : 1); i++) {
                frag_rest(pb, x, g);
#pragma unroll
                for (int t = 0; t < 2; t++) frag_mfma(st.o[t], vf[t], pb);
            }
        }
    }
}

// Four dims of a finished row: out, and what rounding took from it.
template <typename T, bool BIAS, bool KEEP>
VH_DEVICE void store_out(const CrossArgs &a, T *op, int64_t row, int d, floatx4 y) {
    st4(op + d, y);
    if constexpr (KEEP && sizeof(T) == 2) {
        const bf16x4 yr = to_bf16x4(y);
#pragma unroll
        for (int r = 0; r < 4; r++) y[r] -= (float)yr[r];
        if constexpr (BIAS) st4(static_cast<float *>(a.rest) + row * CA_D + d, y);
        else st4(static_cast<bf16 *>(a.rest) + row * CA_D + d, y);
    }
}
VH_DEVICE float2 row_stats(bool bias, bool seen, float m, float l) {
    if (!seen) return make_float2(bias ? 0.0f : INFINITY, -INFINITY);
    const float n = log2f(l);
    return make_float2(bias ? m : m + n, -n);
}

// A workgroup's four waves are KW groups that take the same ROWS rows and every
// KW-th tile of the other side: twice the workgroups, of half the work, where those
// of 128 rows are few.  A group's RW waves share its tiles, [2] places of two each.
template <typename T, int KW>
struct SharedLds {
    static constexpr int RW = 4 / KW, ROWS = 32 * RW;
    static constexpr int GROUP = 4 * Tile<T>::BYTES;
    static constexpr int RESULTS = KW > 1 ? RW * 64 * (32 * 4 + 8) : 0;  // a group's accumulators, over the tiles
    static constexpr int BYTES = KW * GROUP > RESULTS ? KW * GROUP : RESULTS;
};
// A group's tiles: it takes t = group, group + KW, ... while 32 t < end.
template <int KW>
VH_DEVICE int group_tiles(int end, int group) {
    return max(0, ((max(end, 0) + CA_TILE - 1) / CA_TILE - group + KW - 1) / KW);
}
// Accumulators of the second group's waves for the first's: lane by lane.
VH_DEVICE void give(float *res, int i, int rw, int lane, const floatx16 &x) {
#pragma unroll
    for (int r = 0; r < 16; r++) res[(rw * 32 + 16 * i + r) * 64 + lane] = x[r];
}
VH_DEVICE void take(const float *res, int i, int rw, int lane, floatx16 &x) {
#pragma unroll
    for (int r = 0; r < 16; r++) x[r] += res[(rw * 32 + 16 * i + r) * 64 + lane];
}

// Workgroup: RW waves x 32 queries of one head (KW times), tiles of 32 keys that they
// share, the next one's copies in flight while one is worked on.  Per wave and tile
// S^T = K Q^T, so that a lane holds 16 scores of one query, the online softmax, and
// out^T += V^T P^T from the same registers.  KEEP: statistics, rest, and P in pieces.
// Bound by the VALU (exponentials take four issues each) beside the matrix cores
// where the chip is full: 4 x 16 heads x 4096 rows over 4096 with a bias 347 to 367 us,
// 0.75 to 0.79 PFLOP/s (VALU 83% busy, matrix cores 39%); below, by how evenly the workgroups fill it: 8 x 8 x 801 rows over 1723,
// ragged, 28 us, 0.53.
template <typename T, bool BIAS, bool KEEP, int KW>
__global__ __launch_bounds__(256, sizeof(T) == 2 ? 3 : 2) void cross_forward_kernel(CrossArgs a) {
    using L = SharedLds<T, KW>;
    extern __shared__ __attribute__((aligned(1024))) unsigned char smem[];
    float *window = reinterpret_cast<float *>(smem + L::BYTES);

    const int qtiles = (a.Lq + L::ROWS - 1) / L::ROWS;
    int pair, qt;
    if (!pair_task(a.S * a.H, qtiles, pair, qt)) return;
    const int h = pair % a.H, s = pair / a.H;
    const int tid = (int)threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int li = lane & 31, lh = lane >> 5;
    const int kh = h / (a.H / a.KV);
    const int start = cross_start(a, s);
    const int qlen = cross_length(a.query_lengths, s, a.Lq), klen = cross_length(a.key_lengths, s, a.Lk);
    const int group = wave / L::RW, rw = wave % L::RW;
    const int q0 = L::ROWS * qt + 32 * rw, q = q0 + li;
    const bool active = q0 < qlen;
    int keys = klen;  // that any row of the workgroup sees
    if (a.causal) keys = min(keys, start + min(L::ROWS * (qt + 1), qlen));
    if (L::ROWS * qt >= qlen) keys = 0;

    const char *kp = a.k.p + s * a.k.seq + kh * a.k.head, *vp = a.v.p + s * a.v.seq + kh * a.v.head;
    const unsigned char *tiles = smem + group * L::GROUP;
    const uint32_t lds = (uint32_t)(uintptr_t)smem + (uint32_t)(group * L::GROUP);
    auto issue = [&](int i) {  // the group's i-th tile, if there is one
        const int k0 = CA_TILE * (KW * i + group);
        const uint32_t at = lds + (uint32_t)(i & 1) * 2 * Tile<T>::BYTES;
        if (k0 >= keys) return;
        tile_issue<T, L::RW>(kp, a.k.row, k0, keys - 1, at, rw, lane);
        tile_issue<T, L::RW>(vp, a.v.row, k0, keys - 1, at + Tile<T>::BYTES, rw, lane);
    };
    issue(0);
    if constexpr (BIAS) fill_bias_window(a, h, window, tid);  // read after the loop's first barrier
    RegRows<T> w;
    if (active) {
        const char *qp = a.q.p + s * a.q.seq + (int64_t)min(q, qlen - 1) * a.q.row + h * a.q.head;
#pragma unroll
        for (int g = 0; g < 4; g++) w.f[g] = operand(load_query<T>(a, qp, g, lh));
    }
    RowState st;
    st.clear();
    // the tiles of which the wave sees something, then the others' only for the rest
    // of the workgroup (a branch in the loop would copy every accumulator each time)
    const int steps = group_tiles<KW>(keys, 0);
    const int mine = group_tiles<KW>(!active ? 0 : a.causal ? min(keys, start + q0 + 32) : keys, group);
    int i = 0;
    for (; i < mine; i++) {
        wait_vmcnt<0>();
        __syncthreads();  // this tile is there, and the last one has been read
        issue(i + 1);
        const int k0 = CA_TILE * (KW * i + group);
        const LdsTile<T> K{tiles + (i & 1) * 2 * Tile<T>::BYTES}, V{K.p + Tile<T>::BYTES};
        floatx16 x;
        scores(x, K, w, lane);
        const int lo = k0 - (start + q0 + 31), hi = k0 + 31 - (start + q0);
        if constexpr (BIAS) add_bias(a, x, window, lo, hi, k0 - (start + q), 1, lh);
        softmax_tile<BIAS>(st, x, a.scale2, k0 + 32 > klen || (a.causal && hi > 0),
                           (a.causal ? min(klen, start + q + 1) : klen) - k0, lh);
        values_tile<T, BIAS, KEEP>(st, x, V, lane);
    }
    for (; i < steps; i++) {
        wait_vmcnt<0>();
        __syncthreads();
        issue(i + 1);
    }
    if constexpr (KW == 2) {  // the second group's results joined to the first's
        float *res = reinterpret_cast<float *>(smem);
        float2 *ml = reinterpret_cast<float2 *>(res + L::RW * 32 * 64) + rw * 64 + lane;
        __syncthreads();
        if (group) {
            const float top = st.top();
            give(res, 0, rw, lane, st.o[0]);
            give(res, 1, rw, lane, st.o[1]);
            *ml = make_float2(top, st.l);
        }
        __syncthreads();
        if (group) return;
        const float2 other = *ml;
        const float top = fmaxf(st.top(), other.x), base = top == -INFINITY ? 0.0f : top;
        const float f = __builtin_amdgcn_exp2f(st.top() - base), g = __builtin_amdgcn_exp2f(other.x - base);
        st.l = st.l * f + other.y * g;
        st.mc = base;
#pragma unroll
        for (int t = 0; t < 2; t++) {
            floatx16 o;
            zero16(o);
            take(res, t, rw, lane, o);
#pragma unroll
            for (int r = 0; r < 16; r++) st.o[t][r] = st.o[t][r] * f + o[r] * g;
        }
    }
    if (q >= a.Lq) return;
    const float l = st.l + __shfl_xor(st.l, 32, 64);
    const bool seen = q < qlen && (l > 0.0f || l != l);  // a row of NaN stays one
    const float inv = seen ? 1.0f / l : 0.0f;
    const int64_t row = ((int64_t)s * a.H + h) * a.Lq + q;
    if (KEEP && lh == 0) a.stats[row] = row_stats(BIAS, seen, st.mc, l);
    T *op = reinterpret_cast<T *>(a.out.p + s * a.out.seq + (int64_t)q * a.out.row + h * a.out.head);
#pragma unroll
    for (int t = 0; t < 2; t++)
#pragma unroll
        for (int rq = 0; rq < 4; rq++) {
            floatx4 y;
#pragma unroll
            for (int r = 0; r < 4; r++) y[r] = seen ? st.o[t][4 * rq + r] * inv : 0.0f;
            store_out<T, BIAS, KEEP>(a, op, row, 32 * t + 8 * rq + 4 * lh, y);
        }
}

// The same where that makes too few workgroups: 4 waves take the same 32 rows
// and every fourth tile of keys, each in tiles of its own, so that no wave waits
// for another before the end; a.parts workgroups share a row tile's keys.  PACK:
// a tile's rows are the queries' heads that share the key head, head by head
// within a query, so that single tokens of shared heads fill it.  A wave has one
// place for either tile and starts the next one's copies as soon as it has read the
// last: half the LDS of two places (54 -> 48 us for 8 x 8 x 801 rows over 1723 keys, while
// those were this kernel's; 16 x 32 single tokens over 8192 keys, heads shared by four,
// stream 178 MB in 32.6 us).  fp32's
// forward (DIRECT) reads the streamed operands from global memory as it goes, and
// keeps in LDS the pieces of q, which the waves share, so that registers and LDS
// leave room for four waves on a SIMD.
template <typename T, bool D = false>
struct SplitLds {
    static constexpr bool DIRECT = D;
    static constexpr int WAVE = 2 * Tile<T>::BYTES;
    static constexpr int TILES = DIRECT ? 3 * Tile<bf16>::BYTES : 4 * WAVE;
    static constexpr int PITCH = CA_D + 4;
    static constexpr int RESULTS = 4 * 32 * PITCH * 4 + 4 * 32 * 8;  // the waves' [32][CA_D] and (m, l), over the tiles
    static constexpr int BYTES = TILES > RESULTS ? TILES : RESULTS;
    static constexpr int LOADS = CA_TILE / Tile<T>::DMA_ROWS;  // copies of a tile
};
// Waits until at most the newest N copies are still under way; none where there is
// no next tile.
template <int N>
VH_DEVICE void wait_tile(bool next) {
    if (next) wait_vmcnt<N>();
    else wait_vmcnt<0>();
}

// The bias where a tile's columns belong to several heads: the bucket by relative
// position, and the heads' tables.
struct PackedBias {
    const unsigned char *bucket;  // as the window of one head
    const float *table;           // [heads][buckets], times log2(e)
};
VH_DEVICE void scores_packed(const CrossArgs &a, floatx16 &x, const PackedBias &pb, int tile_lo, int tile_hi, int rel0,
                             int head, int lh) {
    const int md = a.max_distance;
    const float *table = pb.table + head * a.buckets;
    if (tile_hi <= -md || tile_lo >= md) {
        const float b = table[pb.bucket[tile_hi <= -md ? CA_PAD : 2 * md + CA_PAD]];
#pragma unroll
        for (int r = 0; r < 16; r++) x[r] = __builtin_fmaf(x[r], a.scale2, b);
    } else {
        const unsigned char *w = pb.bucket + rel0 + 4 * lh + md + CA_PAD;
#pragma unroll
        for (int r = 0; r < 16; r++) x[r] = __builtin_fmaf(x[r], a.scale2, table[w[row_of(r, 0)]]);
    }
}

template <typename T, bool BIAS, bool KEEP, bool PACK>
__global__ __launch_bounds__(256, sizeof(T) == 4 ? 4 : 2) void cross_forward_split_kernel(CrossArgs a) {
    using L = SplitLds<T, sizeof(T) == 4>;
    extern __shared__ __attribute__((aligned(1024))) unsigned char smem[];
    float *window = reinterpret_cast<float *>(smem + L::BYTES);
    const int G = a.H / a.KV, per = PACK ? G : 1, HH = a.H / per;
    const int rtiles = (int)(((int64_t)a.Lq * per + 31) / 32);
    int pair, tile;
    if (!pair_task(a.S * HH, rtiles * a.parts, pair, tile)) return;
    const int rt = tile % rtiles, part = tile / rtiles, hh = pair % HH, s = pair / HH;
    const int tid = (int)threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int li = lane & 31, lh = lane >> 5;
    const int kh = PACK ? hh : hh / G;
    const int start = cross_start(a, s);
    const int qlen = cross_length(a.query_lengths, s, a.Lq), klen = cross_length(a.key_lengths, s, a.Lk);
    const int q_lo = 32 * rt / per, q_hi = min((32 * rt + 31) / per, qlen - 1);
    const int q = (32 * rt + li) / per, head = PACK ? kh * G + (32 * rt + li) % per : hh;
    const bool active = q_lo < qlen;
    int keys = active ? klen : 0;
    if (a.causal) keys = min(keys, start + q_hi + 1);
    const int tiles = (max(keys, 0) + 31) / 32;
    const int first = (int)((int64_t)tiles * part / a.parts), last = (int)((int64_t)tiles * (part + 1) / a.parts);

    PackedBias pb{reinterpret_cast<const unsigned char *>(window + per * a.buckets), window};
    if constexpr (BIAS) {
        if constexpr (PACK) {
            for (int i = tid; i < per * a.buckets; i += 256)
                window[i] = bias_log2(a.table[(int64_t)(i % a.buckets) * a.H + kh * G + i / a.buckets]);
            fill_bucket_window(a, const_cast<unsigned char *>(pb.bucket), tid);
        } else {
            fill_bias_window(a, hh, window, tid);
        }
        __syncthreads();
    }
    const char *qp = a.q.p + s * a.q.seq + (int64_t)min(q, qlen - 1) * a.q.row + head * a.q.head;
    RowState st;
    st.clear();
    const char *kp = a.k.p + s * a.k.seq + kh * a.k.head, *vp = a.v.p + s * a.v.seq + kh * a.v.head;
    const float c = a.scale2;
    auto weigh = [&](floatx16 &x, int k0) {
        const int lo = k0 - (start + q_hi), hi = k0 + 31 - (start + q_lo);
        if constexpr (BIAS && PACK) scores_packed(a, x, pb, lo, hi, k0 - (start + q), head - kh * G, lh);
        else if constexpr (BIAS) add_bias(a, x, window, lo, hi, k0 - (start + q), 1, lh);
        softmax_tile<BIAS>(st, x, c, k0 + 32 > klen || (a.causal && hi > 0),
                           (a.causal ? min(klen, start + q + 1) : klen) - k0, lh);
    };
    int t = first + wave;
    if constexpr (L::DIRECT) {
        if (active) put_row(smem, wave, lane, operand(load_query<T>(a, qp, wave, lh)));
        __syncthreads();
        const LdsPieces w{smem};
        for (; t < last; t += 4) {
            const int64_t k0 = 32 * t;
            floatx16 x;
            scores(x, GlobalTile{kp + k0 * a.k.row, (uint32_t)a.k.row, keys - 1 - 32 * t}, w, lane);
            weigh(x, 32 * t);
            values_tile<T, BIAS, KEEP>(st, x, GlobalTile{vp + k0 * a.v.row, (uint32_t)a.v.row, keys - 1 - 32 * t}, lane);
        }
    } else {
        RegRows<T> w;
        if (active) {
#pragma unroll
            for (int g = 0; g < 4; g++) w.f[g] = operand(load_query<T>(a, qp, g, lh));
        }
        const LdsTile<T> K{smem + wave * L::WAVE}, V{K.p + Tile<T>::BYTES};
        const uint32_t lds = (uint32_t)(uintptr_t)smem + (uint32_t)(wave * L::WAVE);
        auto issue_k = [&](int t) { tile_issue<T, 1>(kp, a.k.row, 32 * t, keys - 1, lds, 0, lane); };
        auto issue_v = [&](int t) { tile_issue<T, 1>(vp, a.v.row, 32 * t, keys - 1, lds + Tile<T>::BYTES, 0, lane); };
        if (t < last) {
            issue_k(t);
            issue_v(t);
        }
        for (; t < last; t += 4) {
            const bool next = t + 4 < last;
            floatx16 x;
            wait_vmcnt<L::LOADS>();  // K is there, V may be under way
            scores(x, K, w, lane);
            wait_lds();
            if (next) issue_k(t + 4);
            weigh(x, 32 * t);
            wait_tile<L::LOADS>(next);
            values_tile<T, BIAS, KEEP>(st, x, V, lane);
            wait_lds();
            if (next) issue_v(t + 4);
        }
    }

    // the four waves' results joined: row tid / 8, dims 8 (tid % 8) .. + 7
    __syncthreads();
    float *res = reinterpret_cast<float *>(smem);
    float2 *ml = reinterpret_cast<float2 *>(res + 4 * 32 * L::PITCH);
    const float l_wave = st.l + __shfl_xor(st.l, 32, 64);
#pragma unroll
    for (int t = 0; t < 2; t++)
#pragma unroll
        for (int rq = 0; rq < 4; rq++) {
            floatx4 y;
#pragma unroll
            for (int r = 0; r < 4; r++) y[r] = st.o[t][4 * rq + r];
            st4(res + (wave * 32 + li) * L::PITCH + 32 * t + 8 * rq + 4 * lh, y);
        }
    if (lh == 0) ml[wave * 32 + li] = make_float2(st.top(), l_wave);
    __syncthreads();
    const int rr = tid >> 3, d = 8 * (tid & 7);
    const int oq = (32 * rt + rr) / per, oh = PACK ? kh * G + (32 * rt + rr) % per : hh;
    if (oq >= a.Lq) return;
    float m = -INFINITY;
#pragma unroll
    for (int w = 0; w < 4; w++) m = fmaxf(m, ml[w * 32 + rr].x);
    const float base = m == -INFINITY ? 0.0f : m;
    float l = 0.0f;
    floatx4 y[2] = {{0.0f, 0.0f, 0.0f, 0.0f}, {0.0f, 0.0f, 0.0f, 0.0f}};
#pragma unroll
    for (int w = 0; w < 4; w++) {
        const float2 v = ml[w * 32 + rr];
        const float c = __builtin_amdgcn_exp2f(v.x - base);
        l += v.y * c;
#pragma unroll
        for (int e = 0; e < 2; e++) y[e] += ld4(res + (w * 32 + rr) * L::PITCH + d + 4 * e) * c;
    }
    const int64_t row = ((int64_t)s * a.H + oh) * a.Lq + oq;
    if (a.parts > 1) {
        const int64_t at = (int64_t)part * a.S * a.H * a.Lq + row;
        st4(a.part_o + at * CA_D + d, y[0]);
        st4(a.part_o + at * CA_D + d + 4, y[1]);
        if (d == 0) a.part_ml[at] = make_float2(m, l);
        return;
    }
    const bool seen = oq < qlen && (l > 0.0f || l != l);
    const float inv = seen ? 1.0f / l : 0.0f;
    if (KEEP && d == 0) a.stats[row] = row_stats(BIAS, seen, m, l);
    T *op = reinterpret_cast<T *>(a.out.p + s * a.out.seq + (int64_t)oq * a.out.row + oh * a.out.head);
#pragma unroll
    for (int e = 0; e < 2; e++) {
#pragma unroll
        for (int r = 0; r < 4; r++) y[e][r] = seen ? y[e][r] * inv : 0.0f;
        store_out<T, BIAS, KEEP>(a, op, row, d + 4 * e, y[e]);
    }
}

// The pieces of every row joined: 16 lanes a row, 4 dims each, the pieces' loads
// under way together (512 rows of 8 pieces: 4.8 us, most of it the launch).
template <typename T, bool BIAS, bool KEEP>
__global__ __launch_bounds__(256) void cross_join_kernel(CrossArgs a) {
    const int64_t rows = (int64_t)a.S * a.H * a.Lq, row = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4);
    if (row >= rows) return;
    const int d = 4 * ((int)threadIdx.x & 15);
    const int q = (int)(row % a.Lq), h = (int)(row / a.Lq % a.H), s = (int)(row / a.Lq / a.H);
    float m = -INFINITY;
#pragma unroll 8
    for (int p = 0; p < a.parts; p++) m = fmaxf(m, a.part_ml[p * rows + row].x);
    const float base = m == -INFINITY ? 0.0f : m;
    float l = 0.0f;
    floatx4 y = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 8
    for (int p = 0; p < a.parts; p++) {
        const float2 v = a.part_ml[p * rows + row];
        const float c = __builtin_amdgcn_exp2f(v.x - base);
        l += v.y * c;
        y += ld4(a.part_o + (p * rows + row) * CA_D + d) * c;
    }
    const bool seen = q < (a.query_lengths ? a.query_lengths[s] : a.Lq) && (l > 0.0f || l != l);
    const float inv = seen ? 1.0f / l : 0.0f;
    if (KEEP && d == 0) a.stats[row] = row_stats(BIAS, seen, m, l);
#pragma unroll
    for (int r = 0; r < 4; r++) y[r] = seen ? y[r] * inv : 0.0f;
    T *op = reinterpret_cast<T *>(a.out.p + s * a.out.seq + (int64_t)q * a.out.row + h * a.out.head);
    store_out<T, BIAS, KEEP>(a, op, row, d, y);
}

// ----------------------------------------------------------------- backward
// A query tile's statistics and delta: the dq kernels leave them for the dk and dv
// ones, which copy a tile's into LDS beside its q and dout.  Rows past the length
// have no probability.
struct RowStats {
    float m[CA_TILE], n[CA_TILE], delta[CA_TILE];  // delta: its negative
};
static_assert(sizeof(RowStats) == 24 * 16, "24 lanes copy it");
VH_DEVICE RowStats *row_tile(const CrossArgs &a, int s, int h, int t) {
    return reinterpret_cast<RowStats *>(a.rows) + ((int64_t)s * a.H + h) * ((a.Lq + CA_TILE - 1) / CA_TILE) + t;
}

// Copies a tile's into LDS: 24 lanes of a wave, 16 bytes each.
VH_DEVICE void row_tile_issue(const RowStats *from, uint32_t lds, int lane) {
    const char *base = uniform(from);
    lds = (uint32_t)__builtin_amdgcn_readfirstlane((int)lds);
    if (lane < 24) lds_dma16s(16u * (uint32_t)lane, base, lds);
}

// What a wave's 32 query rows need as columns, besides their tiles.
template <typename T>
struct QueryRows {
    RegRows<T> q, dout;
    float delta, m, n;  // delta: its negative
};
// Rows q (clamped into qlen) of head h; their statistics are also left where `leave`.
template <typename T, bool BIAS>
VH_DEVICE void load_rows(const CrossArgs &a, QueryRows<T> &w, int s, int h, int q, int qlen, bool leave, int lane) {
    const int lh = lane >> 5;
    const int64_t qr = min(q, qlen - 1), row = ((int64_t)s * a.H + h) * a.Lq + qr;
    const T *qp = reinterpret_cast<const T *>(a.q.p + s * a.q.seq + qr * a.q.row + h * a.q.head);
    const T *dp = reinterpret_cast<const T *>(a.dout.p + s * a.dout.seq + qr * a.dout.row + h * a.dout.head);
    const T *op = reinterpret_cast<const T *>(a.out.p + s * a.out.seq + qr * a.out.row + h * a.out.head);
    float delta = 0.0f;
#pragma unroll
    for (int g = 0; g < 4; g++) {
        const int d = 16 * g + 8 * lh;
        w.q.f[g] = operand(load_query<T>(a, reinterpret_cast<const char *>(qp), g, lh));
        const Frag<T> df = frag_load(dp + d);
        w.dout.f[g] = operand(df);
        const Frag<T> of = frag_load(op + d);
        if constexpr (sizeof(T) == 2) {
            if constexpr (BIAS) {
                const Frag<float> rf = frag_load(static_cast<const float *>(a.rest) + row * CA_D + d);
#pragma unroll
                for (int e = 0; e < 8; e++) delta += (float)df.v[e] * ((float)of.v[e] + rf.v[e >> 2][e & 3]);
            } else {
                const Frag<bf16> rf = frag_load(static_cast<const bf16 *>(a.rest) + row * CA_D + d);
#pragma unroll
                for (int e = 0; e < 8; e++) delta += (float)df.v[e] * ((float)of.v[e] + (float)rf.v[e]);
            }
        } else {
#pragma unroll
            for (int e = 0; e < 8; e++) delta += df.v[e >> 2][e & 3] * of.v[e >> 2][e & 3];
        }
    }
    delta = -(delta + __shfl_xor(delta, 32, 64));
    float2 st = a.stats[row];
    if (q >= qlen) {  // no probability
        st = make_float2(INFINITY, -INFINITY);
        delta = 0.0f;
    }
    w.m = st.x;
    w.n = st.y;
    w.delta = delta;
    if (leave && lh == 0) {
        RowStats *to = row_tile(a, s, h, q / CA_TILE);
        to->m[lane] = st.x;
        to->n[lane] = st.y;
        to->delta[lane] = delta;
    }
}

// The table's gradient.  A tile's dS are summed along its 63 diagonals: 16 keys at
// a time, the pair of key i and query j is stored at [i - j + 31][i] of the wave's
// own array, whose other places stay 0, and lane d adds up the 16 of diagonal d
// (ds_add_f32 instead, straight into the sums, made the whole kernel 3 times as
// long).  Each diagonal is then added to its bucket's slot of that lane: the order
// of every sum is fixed.  Tiles wholly beyond max_distance have one bucket and are
// summed in registers.
// A row's dS add up to 0, and the far buckets hold most of its keys: there an error
// of delta, dP or P counts as often as there are keys, while the sum itself is only
// what the near buckets leave.  So what a row's dS add up to, r, is taken out of the
// far buckets by their part of the row's probability, r P(far).
constexpr int CA_DIAG = 20;  // pitch: 16-byte reads, and stores of 32 lanes in 32 banks
struct DbiasLds {
    float diag[4][48 * CA_DIAG];
    float far[4][2];
};
struct Dbias {
    DbiasLds *db;
    float *slots;           // [4][buckets][32]
    unsigned char *bucket;  // by relative position, as the bias window
    float lo = 0.0f, hi = 0.0f, near = 0.0f;  // the lane's row's dS
    float p_lo = 0.0f, p_hi = 0.0f;           // its probability in the far buckets
    // behind the tiles: where the gradient is wanted the sums, and the bias window
    VH_DEVICE void lay(const CrossArgs &a, unsigned char *at, float *&window) {
        db = reinterpret_cast<DbiasLds *>(at);
        slots = reinterpret_cast<float *>(db + 1);
        window = slots + 128 * a.buckets;
        bucket = reinterpret_cast<unsigned char *>(window + cross_window(a));
    }
    VH_DEVICE void clear(const CrossArgs &a, int tid) {
        const floatx4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
        for (int i = tid; i < 32 * a.buckets; i += 256) st4(slots + 4 * i, zero);
        for (int i = tid; i < 48 * CA_DIAG; i += 256) st4(&db->diag[0][0] + 4 * i, zero);
        fill_bucket_window(a, bucket, tid);
    }
    VH_DEVICE static float sum16(const floatx16 &x) {
        float sum = 0.0f;
#pragma unroll
        for (int r = 0; r < 16; r++) sum += x[r];
        return sum;
    }
    // p: the probabilities of a tile of relative positions tile_lo .. tile_hi, of
    // which rows `seen` and up are masked
    VH_DEVICE void mass(const CrossArgs &a, const floatx16 &p, int tile_lo, int tile_hi, bool mask, int seen, int lh) {
        const bool below = tile_hi <= -a.max_distance;
        if (!below && tile_lo < a.max_distance) return;
        float sum = 0.0f;
        if (mask) {
#pragma unroll
            for (int r = 0; r < 16; r++) sum += row_of(r, lh) < seen ? p[r] : 0.0f;
        } else {
            sum = sum16(p);
        }
        if (below) p_lo += sum;
        else p_hi += sum;
    }
    // x: dS of a tile whose pairs have the relative positions tile_lo .. tile_hi
    VH_DEVICE void add(const CrossArgs &a, const floatx16 &x, int tile_lo, int tile_hi, int wave, int lane) {
        const int md = a.max_distance, li = lane & 31, lh = lane >> 5;
        if (tile_hi <= -md || tile_lo >= md) {
            const float sum = sum16(x);
            if (tile_hi <= -md) lo += sum;
            else hi += sum;
            return;
        }
        near += sum16(x);
        float *diag = &db->diag[wave][0];
        float sum[2];
#pragma unroll
        for (int g = 0; g < 2; g++) {
            wave_order();
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const int i = row_of(e, lh);  // of the 16
                diag[(i - li + 31) * CA_DIAG + i] = x[8 * g + e];
            }
            wave_order();
            const float *d = diag + min(lane, 46) * CA_DIAG;
            const floatx4 v = (ld4(d) + ld4(d + 4)) + (ld4(d + 8) + ld4(d + 12));
            sum[g] = lane < 47 ? (v[0] + v[1]) + (v[2] + v[3]) : 0.0f;
        }
        // diagonal d of the tile: d of the first 16 keys, d - 16 of the second
        const float up = __shfl(sum[1], (lane - 16) & 63, 64);
        const float v = sum[0] + (lane >= 16 ? up : 0.0f);
        const float v1 = __shfl(v, (lane & 31) + 32, 64);
        wave_order();
        if (lane < 32) {  // the second may be the first one's bucket
            float *sl = slots + wave * a.buckets * 32 + lane;
            const unsigned char *bw = bucket + tile_lo + lane + md + CA_PAD;
            sl[32 * bw[0]] += v;
            sl[32 * bw[lane < 31 ? 32 : 31]] += v1;  // there are 63: the last lane's is 0
        }
        wave_order();
    }
    // the workgroup's sums into part `at` of head h; split: its waves share their
    // rows.  Where several workgroups do, each leaves its part of a row's sum and
    // probabilities, and cross_finish_kernel takes the far buckets' part out.
    VH_DEVICE void finish(const CrossArgs &a, int h, int at, int tid, bool split) {
        const int wave = tid >> 6;
        float rest = near + (lo + hi);
        rest += __shfl_xor(rest, 32, 64);
        if (split) {
            const float low = p_lo + __shfl_xor(p_lo, 32, 64), high = p_hi + __shfl_xor(p_hi, 32, 64);
            wave_order();  // the wave's diagonals are read; rows of (rest, low, high) in their place
            float *row = &db->diag[0][0] + 4 * (tid & 31);
            if ((tid & 63) < 32) st4(row + wave * 48 * CA_DIAG, floatx4{rest, low, high, 0.0f});
            __syncthreads();
            const floatx4 v = (ld4(row) + ld4(row + 48 * CA_DIAG)) + (ld4(row + 96 * CA_DIAG) + ld4(row + 144 * CA_DIAG));
            rest = a.parts == 1 ? v[0] : 0.0f;
            if (a.parts > 1 && tid < 32) a.dbias_rows[((int64_t)h * a.dbias_parts + at) * 32 + tid] = v;
        }
        lo = wave_sum(__builtin_fmaf(-rest, p_lo, lo));
        hi = wave_sum(__builtin_fmaf(-rest, p_hi, hi));
        __syncthreads();  // cleared, where no tile was worked on
        if ((tid & 63) == 0) {
            db->far[wave][0] = lo;
            db->far[wave][1] = hi;
        }
        __syncthreads();
        // wave w's 32 slots of a bucket, a thread each; then the four waves'
        float *sums = &db->diag[0][0];
        for (int i = tid; i < 4 * a.buckets; i += 256) {
            floatx4 v = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int j = 0; j < 8; j++) v += ld4(slots + 32 * i + 4 * ((i + j) & 7));
            sums[i] = (v[0] + v[1]) + (v[2] + v[3]);
        }
        __syncthreads();
        if (tid < a.buckets) {
            float sum = (sums[tid] + sums[a.buckets + tid]) + (sums[2 * a.buckets + tid] + sums[3 * a.buckets + tid]);
            const int zero = a.max_distance + CA_PAD;
            for (int w = 0; w < 4; w++) {
                if (tid == bucket[CA_PAD]) sum += db->far[w][0];
                if (tid == bucket[zero + a.max_distance]) sum += db->far[w][1];
            }
            a.dbias_part[((int64_t)h * a.dbias_parts + at) * a.buckets + tid] = sum;
        }
    }
};

// One tile of keys: dq^T += K^T dS^T, and the table's gradient.  dp: -delta, where
// dP's product begins; have_k() is called before K is read, had_v() when V has been.
template <typename T, bool BIAS, typename Tile, typename Held, typename HaveK, typename HadV>
VH_DEVICE void dq_tile(const CrossArgs &a, const QueryRows<T> &w, const Held &q, const Held &dout, floatx16 dp,
                       floatx16 (&acc)[2], Dbias &db, const float *window, const Tile &K, const Tile &V, int k0, int pos,
                       int pos_lo, int klen, int wave, int lane, HaveK have_k, HadV had_v) {
    const int lh = lane >> 5;
    floatx16 x;
    dot_tile(dp, V, dout, lane);
    had_v();
    have_k();
    scores(x, K, q, lane);
    const int lo = k0 - (pos_lo + 31), hi = k0 + 31 - pos_lo;
    const int seen = (a.causal ? min(klen, pos + 1) : klen) - k0;  // rows of the tile that the lane's query sees
    const bool mask = k0 + 32 > klen || (a.causal && hi > 0);
    if constexpr (BIAS) add_bias(a, x, window, lo, hi, k0 - pos, 1, lh);
#pragma unroll
    for (int r = 0; r < 16; r++)
        x[r] = __builtin_amdgcn_exp2f(BIAS ? (x[r] - w.m) + w.n : __builtin_fmaf(x[r], a.scale2, -w.m));
    if constexpr (BIAS) {
        if (a.dbias_part) db.mass(a, x, lo, hi, mask, seen, lh);
    }
#pragma unroll
    for (int r = 0; r < 16; r++) x[r] *= dp[r];
    if (mask) {
#pragma unroll
        for (int r = 0; r < 16; r++)
            if (row_of(r, lh) >= seen) x[r] = 0.0f;
    }
    if constexpr (BIAS) {
        if (a.dbias_part) db.add(a, x, lo, hi, wave, lane);
    }
#pragma unroll
    for (int g = 0; g < 2; g++) {
        Frag<T> sb;
        frag_from(sb, x, g);
        const auto so = operand(sb);
#pragma unroll
        for (int t = 0; t < 2; t++) frag_mfma(acc[t], operand(K.col(g, t, lane)), so);
    }
}

// dq, delta and the table's gradient: workgroup and tiles as the forward's.  Three
// products a tile; 8 x 8 heads x 1023 rows over 862 keys, ragged, bf16: 28 us, 0.51
// PFLOP/s, at two waves on a SIMD.  Two tiles a step (half the barriers, the second
// one's products beside the first one's exponentials): 27.5 us, and 50.5 for 50 with a
// bias; two groups of two waves: no gain.  Neither is kept.
template <typename T, bool BIAS>
__global__ __launch_bounds__(256, 2) void cross_dq_kernel(CrossArgs a) {
    extern __shared__ __attribute__((aligned(1024))) unsigned char smem[];  // [2] K and V tiles
    float *window;
    Dbias db;
    db.lay(a, smem + 4 * Tile<T>::BYTES, window);

    const int qtiles = (a.Lq + 127) / 128;
    int pair, qt;
    if (!pair_task(a.S * a.H, qtiles, pair, qt)) return;
    const int h = pair % a.H, s = pair / a.H;
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

    const char *kp = a.k.p + s * a.k.seq + kh * a.k.head, *vp = a.v.p + s * a.v.seq + kh * a.v.head;
    const uint32_t lds = (uint32_t)(uintptr_t)smem;
    auto issue = [&](int k0) {
        const uint32_t at = lds + (uint32_t)(k0 / CA_TILE & 1) * 2 * Tile<T>::BYTES;
        tile_issue<T, 4>(kp, a.k.row, k0, keys - 1, at, wave, lane);
        tile_issue<T, 4>(vp, a.v.row, k0, keys - 1, at + Tile<T>::BYTES, wave, lane);
    };
    if (keys > 0) issue(0);
    if constexpr (BIAS) {  // read after the loop's first barrier
        fill_bias_window(a, h, window, tid);
        if (a.dbias_part) db.clear(a, tid);
    }
    QueryRows<T> w;
    if (active) load_rows<T, BIAS>(a, w, s, h, q, qlen, true, lane);
    floatx16 delta;
#pragma unroll
    for (int r = 0; r < 16; r++) delta[r] = w.delta;
    floatx16 acc[2];
    zero16(acc[0]);
    zero16(acc[1]);
    const int mine = !active ? 0 : a.causal ? min(keys, start + q0 + 32) : keys;  // as in the forward
    int k0 = 0;
    for (; k0 < mine; k0 += CA_TILE) {
        wait_vmcnt<0>();
        __syncthreads();
        if (k0 + CA_TILE < keys) issue(k0 + CA_TILE);
        const LdsTile<T> K{smem + (k0 / CA_TILE & 1) * 2 * Tile<T>::BYTES}, V{K.p + Tile<T>::BYTES};
        dq_tile<T, BIAS>(
            a, w, w.q, w.dout, delta, acc, db, window, K, V, k0, start + q, start + q0, klen, wave, lane, [] {}, [] {});
    }
    for (; k0 < keys; k0 += CA_TILE) {
        wait_vmcnt<0>();
        __syncthreads();
        if (k0 + CA_TILE < keys) issue(k0 + CA_TILE);
    }
    if constexpr (BIAS) {
        if (a.dbias_part) db.finish(a, h, s * qtiles + qt, tid, false);
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

// A wave's column of 32 x 64 sums added over the workgroup's four waves: thread
// tid gets dims 8 (tid % 8) .. + 7 of row tid / 8.
template <typename T>
VH_DEVICE void waves_sum(float *res, const floatx16 (&acc)[2], int tid, floatx4 (&y)[2]) {
    using L = SplitLds<T>;
    const int lane = tid & 63, li = lane & 31, lh = lane >> 5, wave = tid >> 6;
    __syncthreads();  // what lay there has been read
#pragma unroll
    for (int t = 0; t < 2; t++)
#pragma unroll
        for (int rq = 0; rq < 4; rq++) {
            floatx4 v;
#pragma unroll
            for (int r = 0; r < 4; r++) v[r] = acc[t][4 * rq + r];
            st4(res + (wave * 32 + li) * L::PITCH + 32 * t + 8 * rq + 4 * lh, v);
        }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < 2; e++) {
        const float *p = res + (tid >> 3) * L::PITCH + 8 * (tid & 7) + 4 * e;
        y[e] = (ld4(p) + ld4(p + 32 * L::PITCH)) + (ld4(p + 64 * L::PITCH) + ld4(p + 96 * L::PITCH));
    }
}

// The same in too few workgroups: as cross_forward_split_kernel.
template <typename T, bool BIAS>
__global__ __launch_bounds__(256, 2) void cross_dq_split_kernel(CrossArgs a) {
    using L = SplitLds<T>;
    extern __shared__ __attribute__((aligned(1024))) unsigned char smem[];
    float *window;
    Dbias db;
    db.lay(a, smem + L::BYTES, window);

    const int rtiles = (a.Lq + 31) / 32;
    int pair, tile;
    if (!pair_task(a.S * a.H, rtiles * a.parts, pair, tile)) return;
    const int rt = tile % rtiles, part = tile / rtiles, h = pair % a.H, s = pair / a.H;
    const int tid = (int)threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int kh = h / (a.H / a.KV);
    const int start = cross_start(a, s);
    const int qlen = cross_length(a.query_lengths, s, a.Lq), klen = cross_length(a.key_lengths, s, a.Lk);
    const int q0 = 32 * rt, q = q0 + (lane & 31);
    int keys = q0 < qlen ? klen : 0;
    if (a.causal) keys = min(keys, start + min(q0 + 32, qlen));
    const int tiles = (max(keys, 0) + 31) / 32;
    const int first = (int)((int64_t)tiles * part / a.parts), last = (int)((int64_t)tiles * (part + 1) / a.parts);

    if constexpr (BIAS) {
        fill_bias_window(a, h, window, tid);
        if (a.dbias_part) db.clear(a, tid);
        __syncthreads();
    }
    QueryRows<T> w;
    if (q0 < qlen) load_rows<T, BIAS>(a, w, s, h, q, qlen, part == 0 && wave == 0, lane);
    floatx16 delta, acc[2];
#pragma unroll
    for (int r = 0; r < 16; r++) delta[r] = w.delta;
    zero16(acc[0]);
    zero16(acc[1]);
    const char *kp = a.k.p + s * a.k.seq + kh * a.k.head, *vp = a.v.p + s * a.v.seq + kh * a.v.head;
    int t = first + wave;
    const LdsTile<T> K{smem + wave * L::WAVE}, V{K.p + Tile<T>::BYTES};
    const uint32_t lds = (uint32_t)(uintptr_t)smem + (uint32_t)(wave * L::WAVE);
    auto issue_k = [&](int t) { tile_issue<T, 1>(kp, a.k.row, 32 * t, keys - 1, lds, 0, lane); };
    auto issue_v = [&](int t) { tile_issue<T, 1>(vp, a.v.row, 32 * t, keys - 1, lds + Tile<T>::BYTES, 0, lane); };
    if (t < last) {
        issue_v(t);
        issue_k(t);
    }
    for (; t < last; t += 4) {
        const bool next = t + 4 < last;
        wait_vmcnt<L::LOADS>();  // V is there, K may be under way
        dq_tile<T, BIAS>(
            a, w, w.q, w.dout, delta, acc, db, window, K, V, 32 * t, start + q, start + q0, klen, wave, lane,
            [&] { wait_tile<L::LOADS>(next); },
            [&] {
                wait_lds();
                if (next) issue_v(t + 4);
            });
        wait_lds();
        if (next) issue_k(t + 4);
    }
    if constexpr (BIAS) {
        if (a.dbias_part) db.finish(a, h, (s * rtiles + rt) * a.parts + part, tid, true);
    }
    floatx4 y[2];
    waves_sum<T>(reinterpret_cast<float *>(smem), acc, tid, y);
    const int oq = q0 + (tid >> 3), d = 8 * (tid & 7);
    if (oq >= a.Lq) return;
#pragma unroll
    for (int e = 0; e < 2; e++)
#pragma unroll
        for (int r = 0; r < 4; r++) y[e][r] = oq < qlen ? y[e][r] * a.scale : 0.0f;
    if (a.parts > 1) {
        float *p = a.part_o + (((int64_t)part * a.S * a.H + (int64_t)s * a.H + h) * a.Lq + oq) * CA_D + d;
        st4(p, y[0]);
        st4(p + 4, y[1]);
        return;
    }
    T *out = reinterpret_cast<T *>(a.dq.p + s * a.dq.seq + (int64_t)oq * a.dq.row + h * a.dq.head) + d;
    st4(out, y[0]);
    st4(out + 4, y[1]);
}

// A wave's 32 keys as columns: fragments g of k (of the scale's sign) and of v, and
// their gradients' sums.
template <typename T>
struct KeyRows {
    RegRows<T> k, v;
};
struct KeySums {
    floatx16 dk[2], dv[2];
    VH_DEVICE void clear() {
#pragma unroll
        for (int t = 0; t < 2; t++) {
            zero16(dk[t]);
            zero16(dv[t]);
        }
    }
};
// The first row of the first tile of queries that sees key k0 (qlen: none does).
VH_DEVICE int first_query(const CrossArgs &a, int k0, int start, int qlen) {
    const int q = a.causal ? max(0, k0 - start) : 0;
    return q < qlen ? q / CA_TILE * CA_TILE : qlen;
}
// Keys that no query sees are copies of the last one that some does.
template <typename T>
VH_DEVICE void load_keys(const CrossArgs &a, KeyRows<T> &w, int s, int kh, int key, int start, int qlen, int klen, int lh) {
    const int end = a.causal ? min(klen, start + qlen) : klen;
    if (end <= 0) return;
    const int64_t kr = min(key, end - 1);
    const T *kp = reinterpret_cast<const T *>(a.k.p + s * a.k.seq + kr * a.k.row + kh * a.k.head);
    const T *vp = reinterpret_cast<const T *>(a.v.p + s * a.v.seq + kr * a.v.row + kh * a.v.head);
#pragma unroll
    for (int g = 0; g < 4; g++) {
        w.k.f[g] = operand(load_query<T>(a, reinterpret_cast<const char *>(kp), g, lh));
        w.v.f[g] = operand(frag_load(vp + 16 * g + 8 * lh));
    }
}

// One tile of queries: S = Q K^T with the keys as columns, so that P and dS are B
// operands of dv^T += dout^T P and dk^T += Q^T dS as they are.  have_q() is called
// before Q is read, had_dout() when dout and the statistics have been.
template <typename T, bool BIAS, typename Tile, typename Held, typename HaveQ, typename HadDout>
VH_DEVICE void dkv_tile(const CrossArgs &a, const Held &k, const Held &v, KeySums &w, const float *window, const Tile &Q,
                        const Tile &D, const RowStats *rs, int q0, int start, int key, int k0, int lane, HaveQ have_q,
                        HadDout had_dout) {
    const int lh = lane >> 5;
    floatx16 x, dp;
#pragma unroll
    for (int r = 0; r < 16; r++) dp[r] = rs->delta[row_of(r, lh)];
    dot_tile(dp, D, v, lane);
    have_q();
    scores(x, Q, k, lane);
    const int lo = k0 - (start + q0 + 31), hi = k0 + 31 - (start + q0);
    if constexpr (BIAS) add_bias(a, x, window, lo, hi, key - (start + q0), -1, lh);
#pragma unroll
    for (int r = 0; r < 16; r++) {
        const int i = row_of(r, lh);
        x[r] = __builtin_amdgcn_exp2f(BIAS ? (x[r] - rs->m[i]) + rs->n[i] : __builtin_fmaf(x[r], a.scale2, -rs->m[i]));
        dp[r] *= x[r];
    }
    if (a.causal && hi > 0) {
        const int hidden = key - start - q0;  // rows below it come before the lane's key
#pragma unroll
        for (int r = 0; r < 16; r++)
            if (row_of(r, lh) < hidden) x[r] = dp[r] = 0.0f;
    }
#pragma unroll
    for (int g = 0; g < 2; g++) {
        Frag<T> pb;
        frag_from(pb, x, g);
        const auto po = operand(pb);
#pragma unroll
        for (int t = 0; t < 2; t++) frag_mfma(w.dv[t], operand(D.col(g, t, lane)), po);
    }
    had_dout();
#pragma unroll
    for (int g = 0; g < 2; g++) {
        Frag<T> sb;
        frag_from(sb, dp, g);
        const auto so = operand(sb);
#pragma unroll
        for (int t = 0; t < 2; t++) frag_mfma(w.dk[t], operand(Q.col(g, t, lane)), so);
    }
}

// dk and dv: workgroup of 4 waves x 32 keys of one key head, tiles of 32 queries
// of every query head that shares it.  Four products a tile; 4 x 12 heads x 1025
// rows over 1025 keys, ragged, with a bias: 51 us, as many as dq's with the table.
template <typename T, bool BIAS>
__global__ __launch_bounds__(256, 2) void cross_dkv_kernel(CrossArgs a) {
    extern __shared__ __attribute__((aligned(1024))) unsigned char smem[];  // [2] Q and dout tiles
    RowStats *rs = reinterpret_cast<RowStats *>(smem + 4 * Tile<T>::BYTES);  // [2]
    float *window = reinterpret_cast<float *>(rs + 2);                       // [2]: of two heads in turn

    const int ktiles = (a.Lk + 127) / 128;
    int pair, kt;
    if (!pair_task(a.S * a.KV, ktiles, pair, kt)) return;
    const int kh = pair % a.KV, s = pair / a.KV;
    const int tid = (int)threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int li = lane & 31, lh = lane >> 5;
    const int start = cross_start(a, s);
    const int qlen = cross_length(a.query_lengths, s, a.Lq), klen = cross_length(a.key_lengths, s, a.Lk);
    const int k0 = 128 * kt + 32 * wave, key = k0 + li;
    const bool active = k0 < klen;
    // the first query that sees a key of the workgroup
    const int first = 128 * kt < klen ? first_query(a, 128 * kt, start, qlen) : qlen;
    // and one of the wave's own: the tiles before it are the other waves' (as in the forward)
    const int mine = active ? first_query(a, k0, start, qlen) : qlen;

    const uint32_t lds = (uint32_t)(uintptr_t)smem, rs_lds = (uint32_t)(uintptr_t)rs;
    const int G = a.H / a.KV;
    auto issue = [&](int h, int q0, int buf) {
        const char *qp = a.q.p + s * a.q.seq + h * a.q.head, *dp = a.dout.p + s * a.dout.seq + h * a.dout.head;
        const uint32_t at = lds + (uint32_t)buf * 2 * Tile<T>::BYTES;
        tile_issue<T, 4>(qp, a.q.row, q0, qlen - 1, at, wave, lane);
        tile_issue<T, 4>(dp, a.dout.row, q0, qlen - 1, at + Tile<T>::BYTES, wave, lane);
        if (wave == 0) row_tile_issue(row_tile(a, s, h, q0 / CA_TILE), rs_lds + (uint32_t)buf * sizeof(RowStats), lane);
    };
    if (first < qlen) issue(kh * G, first, 0);
    KeyRows<T> w;
    load_keys(a, w, s, kh, key, start, qlen, klen, lh);
    KeySums sums;
    sums.clear();
    int buf = 0;
    for (int g = 0; g < G; g++) {
        // the window before last is free: its head's tiles ended a barrier ago
        float *bias = window + (g & 1) * (BIAS ? cross_window(a) : 0);
        if constexpr (BIAS) fill_bias_window(a, kh * G + g, bias, tid);
        auto begin = [&](int q0) {
            wait_vmcnt<0>();
            __syncthreads();
            if (q0 + CA_TILE < qlen) issue(kh * G + g, q0 + CA_TILE, buf ^ 1);
            else if (g + 1 < G) issue(kh * G + g + 1, first, buf ^ 1);
        };
        int q0 = first;
        for (; q0 < mine; q0 += CA_TILE, buf ^= 1) begin(q0);
        for (; q0 < qlen; q0 += CA_TILE, buf ^= 1) {
            begin(q0);
            const LdsTile<T> Q{smem + buf * 2 * Tile<T>::BYTES}, D{Q.p + Tile<T>::BYTES};
            dkv_tile<T, BIAS>(
                a, w.k, w.v, sums, bias, Q, D, rs + buf, q0, start, key, k0, lane, [] {}, [] {});
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
                y[r] = key < klen ? sums.dk[t][4 * rq + r] * a.scale : 0.0f;
                z[r] = key < klen ? sums.dv[t][4 * rq + r] : 0.0f;
            }
            st4(pk + 32 * t + 8 * rq + 4 * lh, y);
            st4(pv + 32 * t + 8 * rq + 4 * lh, z);
        }
}

// The same in too few workgroups: 4 waves take the same 32 keys and every fourth
// tile of the queries of all heads that share them, one head after the other; or,
// where there are too few such workgroups, each head and a.kv_parts pieces of its
// queries are workgroups of their own.  8 x 8 heads over 4 x 862 keys, 1023 rows,
// bf16: 36 us.
template <typename T, bool BIAS>
__global__ __launch_bounds__(256, 2) void cross_dkv_split_kernel(CrossArgs a) {
    using L = SplitLds<T>;
    extern __shared__ __attribute__((aligned(1024))) unsigned char smem[];
    RowStats *stats = reinterpret_cast<RowStats *>(smem + L::BYTES);  // [4]
    float *window = reinterpret_cast<float *>(stats + 4);

    const int ktiles = (a.Lk + 31) / 32, G = a.H / a.KV, HH = a.H / a.kv_heads;
    int pair, tile;
    if (!pair_task(a.S * HH, ktiles * a.kv_parts, pair, tile)) return;
    const int kt = tile % ktiles, part = tile / ktiles, h = pair % HH * a.kv_heads, s = pair / HH;  // h: the first head
    const int tid = (int)threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int lh = lane >> 5, kh = h / G;
    const int start = cross_start(a, s);
    const int qlen = cross_length(a.query_lengths, s, a.Lq), klen = cross_length(a.key_lengths, s, a.Lk);
    const int k0 = 32 * kt, key = k0 + (lane & 31);
    const int tiles = k0 < klen ? (qlen + 31) / 32 : 0;
    const int begin = min(tiles, (first_query(a, k0, start, qlen) + 31) / 32);
    const int each = tiles - begin;  // of a head, the workgroup's numbered head by head
    const int64_t all = (int64_t)each * a.kv_heads;
    const int first = (int)(all * part / a.kv_parts), last = (int)(all * (part + 1) / a.kv_parts);

    if constexpr (BIAS) {
        for (int g = 0; g < a.kv_heads; g++) fill_bias_window(a, h + g, window + g * cross_window(a), tid);
        __syncthreads();
    }
    KeySums sums;
    sums.clear();
    int t = first + wave;
    KeyRows<T> w;
    load_keys(a, w, s, kh, key, start, qlen, klen, lh);
    const LdsTile<T> Q{smem + wave * L::WAVE}, D{Q.p + Tile<T>::BYTES};
    const uint32_t lds = (uint32_t)(uintptr_t)smem + (uint32_t)(wave * L::WAVE);
    RowStats *rs = stats + wave;
    auto issue_q = [&](int t) {
        const char *qp = a.q.p + s * a.q.seq + (h + t / each) * a.q.head;
        tile_issue<T, 1>(qp, a.q.row, 32 * (begin + t % each), qlen - 1, lds, 0, lane);
    };
    auto issue_dout = [&](int t) {
        const char *dp = a.dout.p + s * a.dout.seq + (h + t / each) * a.dout.head;
        tile_issue<T, 1>(dp, a.dout.row, 32 * (begin + t % each), qlen - 1, lds + Tile<T>::BYTES, 0, lane);
        row_tile_issue(row_tile(a, s, h + t / each, begin + t % each), (uint32_t)(uintptr_t)rs, lane);
    };
    if (t < last) {
        issue_dout(t);
        issue_q(t);
    }
    for (; t < last; t += 4) {
        const bool next = t + 4 < last;
        wait_vmcnt<L::LOADS>();  // dout is there, Q may be under way
        dkv_tile<T, BIAS>(
            a, w.k, w.v, sums, BIAS ? window + t / each * cross_window(a) : nullptr, Q, D, rs,
            32 * (begin + t % each), start, key, k0, lane, [&] { wait_vmcnt<0>(); },
            [&] {
                wait_lds();
                if (next) issue_dout(t + 4);
            });
        wait_lds();
        if (next) issue_q(t + 4);
    }
    floatx4 y[2], z[2];
    waves_sum<T>(reinterpret_cast<float *>(smem), sums.dk, tid, y);
    waves_sum<T>(reinterpret_cast<float *>(smem), sums.dv, tid, z);
    const int ok = k0 + (tid >> 3), d = 8 * (tid & 7);
    if (ok >= a.Lk) return;
#pragma unroll
    for (int e = 0; e < 2; e++)
#pragma unroll
        for (int r = 0; r < 4; r++) {
            y[e][r] = ok < klen ? y[e][r] * a.scale : 0.0f;
            z[e][r] = ok < klen ? z[e][r] : 0.0f;
        }
    if (G / a.kv_heads * a.kv_parts > 1) {
        const int64_t at = ((((int64_t)(h % G) / a.kv_heads * a.kv_parts + part) * a.S + s) * a.KV + kh) * a.Lk + ok;
#pragma unroll
        for (int e = 0; e < 2; e++) {
            st4(a.part_dk + at * CA_D + d + 4 * e, y[e]);
            st4(a.part_dv + at * CA_D + d + 4 * e, z[e]);
        }
        return;
    }
    T *pk = reinterpret_cast<T *>(a.dk.p + s * a.dk.seq + (int64_t)ok * a.dk.row + kh * a.dk.head) + d;
    T *pv = reinterpret_cast<T *>(a.dv.p + s * a.dv.seq + (int64_t)ok * a.dv.row + kh * a.dv.head) + d;
#pragma unroll
    for (int e = 0; e < 2; e++) {
        st4(pk + 4 * e, y[e]);
        st4(pv + 4 * e, z[e]);
    }
}

// The pieces added up, in their order: workgroups of one head's bias each, which take
// the longest, then of 16 rows of dq, of dk and of dv.
struct FinishArgs {
    int64_t heads, dq, dkv;  // workgroups of the bias; of dq; of dk (and as many of dv)
};
template <typename T>
VH_DEVICE void sum_parts(const float *part, int parts, int64_t rows, int64_t row, int len, int heads,
                         const CrossTensor &to) {
    if (row >= rows) return;
    const int d = 4 * ((int)threadIdx.x & 15);
    floatx4 y = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 8
    for (int p = 0; p < parts; p++) y += ld4(part + (p * rows + row) * CA_D + d);
    const int64_t i = row % len, h = row / len % heads, s = row / len / heads;
    st4(reinterpret_cast<T *>(to.p + s * to.seq + i * to.row + h * to.head) + d, y);
}
template <typename T>
__global__ __launch_bounds__(256) void cross_finish_kernel(CrossArgs a, FinishArgs f) {
    __shared__ float sums[256], far[4][2];
    const int tid = (int)threadIdx.x, sub = tid >> 4;
    if (blockIdx.x >= f.heads) {
        int64_t block = blockIdx.x - f.heads;
        if (block < f.dq) {
            sum_parts<T>(a.part_o, a.parts, (int64_t)a.S * a.H * a.Lq, block * 16 + sub, a.Lq, a.H, a.dq);
            return;
        }
        block -= f.dq;
        const bool v = block >= f.dkv;
        sum_parts<T>(v ? a.part_dv : a.part_dk, a.H / a.KV / a.kv_heads * a.kv_parts, (int64_t)a.S * a.KV * a.Lk,
                     (block - (v ? f.dkv : 0)) * 16 + sub, a.Lk, a.KV, v ? a.dv : a.dk);
        return;
    }
    const int h = (int)blockIdx.x, lanes = 256 / a.buckets;  // threads that share a bucket
    const int b = tid % a.buckets, l = tid / a.buckets;
    float sum = 0.0f;
    if (l < lanes) {
#pragma unroll 16
        for (int i = l; i < a.dbias_parts; i += lanes)
            sum += a.dbias_part[((int64_t)h * a.dbias_parts + i) * a.buckets + b];
    }
    sums[tid] = sum;
    if (a.parts > 1) {
        // the rows' pieces joined, 8 row tiles at a time and four such loads under way
        // (those past the last are its own, and count for nothing), and what a row's dS
        // add up to times its probability in the far buckets
        const floatx4 *rows = a.dbias_rows + (int64_t)h * a.dbias_parts * 32 + (tid & 31);
        const int tiles = a.dbias_parts / a.parts;
        float lo = 0.0f, hi = 0.0f;
        for (int t0 = tid >> 5; t0 < tiles; t0 += 32) {
            floatx4 v[4] = {};
#pragma unroll 4
            for (int i = 0; i < a.parts; i++)
#pragma unroll
                for (int u = 0; u < 4; u++) v[u] += rows[((int64_t)min(t0 + 8 * u, tiles - 1) * a.parts + i) * 32];
#pragma unroll
            for (int u = 0; u < 4; u++) {
                const float rest = t0 + 8 * u < tiles ? v[u][0] : 0.0f;
                lo = __builtin_fmaf(rest, v[u][1], lo);
                hi = __builtin_fmaf(rest, v[u][2], hi);
            }
        }
        lo = wave_sum(lo);
        hi = wave_sum(hi);
        if ((tid & 63) == 0) {
            far[tid >> 6][0] = lo;
            far[tid >> 6][1] = hi;
        }
    }
    __syncthreads();
    if (tid >= a.buckets) return;
    for (int i = 1; i < lanes; i++) sum += sums[i * a.buckets + b];
    if (a.parts > 1) {
        if (b == cross_bucket(a, -a.max_distance)) sum -= (far[0][0] + far[1][0]) + (far[2][0] + far[3][0]);
        if (b == cross_bucket(a, a.max_distance)) sum -= (far[0][1] + far[1][1]) + (far[2][1] + far[3][1]);
    }
    a.dbias[(int64_t)b * a.H + h] = sum;
}

}  // namespace vh
