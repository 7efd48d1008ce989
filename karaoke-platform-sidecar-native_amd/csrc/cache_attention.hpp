// Attention over a paged cache.
//
//   x_ij = scale q'_i.k_j,  P = softmax over the keys that row i sees,  out_i = sum_j P_ij v_j
//
// with q' = q turned to its position, and out_i = 0 where row i sees no key.  The rows
// of a key head are those of all query heads that share it, token by token: a decoding
// step's single tokens fill a matrix tile with their heads.
//
// A wave has RG groups of 16 rows as columns and walks over the keys in steps of KB = 2
// blocks of 16, each read once, as the page holds it, into registers: S^T = K Q^T and
// O^T = V^T P^T in 16 x 16 x 32 instructions, whose results' lanes (column l % 16, rows
// 4 (l / 16) + 0 .. 3) are where the second product wants P, so nothing passes through
// LDS.  One pass, with the running maximum and sum of the softmax.
//
// Over int8 pages keys and values are whole numbers, exact in fp16 (from the byte by a
// permute and an addition: 0x6400 + u is 1024 + u); a row of q' enters as fp16 times a
// power of two (its largest just below 2^14, so 2^-25 of that is what a small one is
// off by), the block's scale of keys as a factor of the scores.  P, up to 2^4, enters
// times the block's scale of values over the largest one that the row has seen, times 2^10:
// what is below 2^-35 of the largest value that a row sees is lost.  fp32 out: q' and P
// in two fp16 values each.  Over bf16 pages: two bf16 values each, fp32 out: three.
//
// Single tokens are bound by HBM, the cache is read once: 32 of 32 heads on 8 of 128 over
// 16384 keys each, 8 bits, 1.07 GB in 162 us (6.6 TB/s; with loads that stay in the caches
// 185, without asking for the next step's 182).  Chunks over 8 bits are bound by the vector
// instructions, the exponentials and conversions (83% of a busy CU's cycles; the matrix
// instructions 20%): 4 x 517 causal tokens of 16 heads on 4 of 64 over up to 4613 keys 63 us;
// with P's base moved at every larger maximum 74, with keys unbiased 66, with 128 registers and
// four waves a SIMD 144 (spilled).  Over bf16 pages of 128 dims by the matrix cores: 4 x 512
// tokens of 32 heads on 8 over up to 4608 keys are 107 GFLOP, 215 with two operands, in 211 us
// (1.02 PFLOP/s of the 1.1 to 1.2 of a large product).
#pragma once

#include "h2.hpp"
#include "paged_cache.hpp"

namespace vh {

struct CacheAttentionArgs {
    PagedArgs p;
    Rotation r;
    const char *q;
    char *out;
    int64_t qs[3], os[3];  // bytes
    const int *query_lengths, *key_lengths, *start;
    int S, H, group, Lq;   // group: query heads of a key head
    int most, causal;
    float scale2;          // |scale| log2(e), at least the smallest normal number
    int negative;          // the scale is: q' is turned instead
    int tiles;             // workgroups of a (sequence, key head)'s rows
    int by_xcd;            // these pairs are dealt out to the XCDs
    int parts, piece;      // pieces of the keys, and blocks of one
    float *part_o;         // [parts][S][Lq][H][D]
    float2 *part_ml;       // [parts][S][Lq][H]
    Divisor heads;         // group
};

// Operands: I8 pages fp16, else bf16; N of them a value of q' or P.
template <bool I8>
struct Operand16 {
    typedef halfx8 type;
    VH_DEVICE static floatx4 mfma(halfx8 a, halfx8 b, floatx4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
    VH_DEVICE static halfx8 round(const float (&x)[8]) {
        halfx8 h;
#pragma unroll
        for (int e = 0; e < 8; e++) h[e] = (_Float16)x[e];
        return h;
    }
};
template <>
struct Operand16<false> {
    typedef bf16x8 type;
    VH_DEVICE static floatx4 mfma(bf16x8 a, bf16x8 b, floatx4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
    VH_DEVICE static bf16x8 round(const float (&x)[8]) {
        bf16x8 h;
#pragma unroll
        for (int e = 0; e < 8; e++) h[e] = (bf16)x[e];
        return h;
    }
};
// x as the sum of N operands, the largest first.
template <bool I8, int N>
VH_DEVICE void split_n(float (&x)[8], typename Operand16<I8>::type (&o)[N]) {
    // the value rounded to fp32 is what is split: a product that the compiler joins with
    // the conversion, but not with the subtraction, is another one in rare cases, and an
    // fp16 step too large
    if constexpr (N > 1)
#pragma unroll
        for (int e = 0; e < 8; e++) asm("" : "+v"(x[e]));
#pragma unroll
    for (int n = 0; n < N; n++) {
        o[n] = Operand16<I8>::round(x);
        if (n + 1 < N)
#pragma unroll
            for (int e = 0; e < 8; e++) x[e] -= (float)o[n][e];
    }
}

// Four bytes (numbers plus 128) as fp16.
template <bool BIASED = false>
VH_DEVICE void bytes_to_half(uint32_t w, uint32_t &lo, uint32_t &hi) {
    typedef _Float16 halfx2 __attribute__((ext_vector_type(2)));
    const halfx2 bias = {(_Float16)-1152.0f, (_Float16)-1152.0f};
    lo = __builtin_amdgcn_perm(0x64646464u, w, 0x04010400u);
    hi = __builtin_amdgcn_perm(0x64646464u, w, 0x04030402u);
    if constexpr (!BIASED) {
        lo = __builtin_bit_cast(uint32_t, __builtin_bit_cast(halfx2, lo) + bias);
        hi = __builtin_bit_cast(uint32_t, __builtin_bit_cast(halfx2, hi) + bias);
    }
}

// A step's keys or values in registers, as the page holds them.
template <int D, bool I8, int KB>
struct RawBlocks {
    using B = BlockShape<D, I8>;
    u32x4 w[KB][B::UNITS];
    // keys' operand m: dims 32 m .. of block b's, of 8 bits BIASED by 1152
    template <bool BIASED>
    VH_DEVICE typename Operand16<I8>::type key(int b, int m) const {
        if constexpr (I8) {
            u32x4 o;
            uint32_t lo, hi;
            bytes_to_half<BIASED>(w[b][m / 2][2 * (m % 2)], lo, hi);
            o[0] = lo;
            o[1] = hi;
            bytes_to_half<BIASED>(w[b][m / 2][2 * (m % 2) + 1], lo, hi);
            o[2] = lo;
            o[3] = hi;
            return __builtin_bit_cast(halfx8, o);
        } else {
            return __builtin_bit_cast(bf16x8, w[b][m]);
        }
    }
    // values' operand for dims DT i + t, of blocks 2 c and 2 c + 1
    VH_DEVICE typename Operand16<I8>::type value(int c, int t) const {
        u32x4 o;
#pragma unroll
        for (int h = 0; h < 2; h++) {
            if constexpr (I8) {
                uint32_t lo, hi;
                bytes_to_half(w[2 * c + h][t / 4][t % 4], lo, hi);
                o[2 * h] = lo;
                o[2 * h + 1] = hi;
            } else {
                o[2 * h] = w[2 * c + h][t / 2][2 * (t % 2)];
                o[2 * h + 1] = w[2 * c + h][t / 2][2 * (t % 2) + 1];
            }
        }
        return __builtin_bit_cast(typename Operand16<I8>::type, o);
    }
};

VH_DEVICE float exp2_of(float x) { return __builtin_amdgcn_exp2f(x); }
// The larger one, or a NaN if one is (the other maximum first makes sure that its
// operands are quiet, an instruction each).
VH_DEVICE float larger(float a, float b) { return __builtin_elementwise_maximum(a, b); }
constexpr int CQ_STEP = 2;  // blocks of a step
constexpr float FLT_LEAST = 0x1p-126f;
constexpr float LAZY = 4.0f;  // P up to 2^LAZY: times P_SCALE it is fp16's

// SPLIT: a workgroup's four waves share the rows, each every fourth step of the keys,
// and join; else each wave has rows of its own.  Three waves a SIMD hold fp32's 32 rows of 64
// dims over 8 bits, with 4 registers spilled: 4 x 300 tokens of 16 heads on 4 over 2613 keys
// 40.5 us, with two waves and 184 registers 43.
template <typename T, int D, bool I8, int RG, bool SPLIT>
static __global__ __launch_bounds__(256, D == 64 && I8 ? 3 : 2) void cache_attention_kernel(CacheAttentionArgs a) {
    using B = BlockShape<D, I8>;
    using Op = Operand16<I8>;
    // of q' and P.  bf16 out over 8 bits one operand, fp16's 11 bits, three more than out's: an
    // error of 1.69e-3 of the norm, with two 1.66e-3, which products in fp32 have; 4 x 517 causal
    // tokens 63 us, with two 85.  bf16 out over bf16 pages two, 16 bits: with one, which has no
    // more bits than out, 4 x 512 causal tokens over 4608 keys had an error of 3.0e-3 for 1.66e-3
    // (161 us, with two 211).  fp32 out as many as 22 bits and more take.
    constexpr int DT = B::DT, QS = D / 32, N = sizeof(T) == 2 ? (I8 ? 1 : 2) : I8 ? 2 : 3;
    constexpr int ROWS = 16 * RG * (SPLIT ? 1 : 4);
    constexpr int KB = CQ_STEP, PER_FETCH = 64 / KB;
    // bf16 out: keys enter as 1152 more than they are, and the scores begin so much lower:
    // sums 1152 / 40 times as large, whose fp32 roundings stay below those of fp16 queries
    constexpr bool BIASED = I8 && N == 1;
    // Keys are asked for one step ahead when the last ones are multiplied, values likewise,
    // each in its one place, where two steps at once do not fit the registers: 4 x 512 causal
    // tokens of 32 heads on 8 of 128 over 4608 bf16 keys 211 us, twice kept 885 (74 registers
    // spilled).  Elsewhere two steps are kept: 16 x 2048 tokens of 16 heads on 4 of 64 over as
    // many bf16 keys 338 us against 334.
    constexpr bool ROLLING = !I8 && D == 128 && RG > 1;
    constexpr float P_SCALE = I8 ? 0x1p10f : 1.0f;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int i = lane & 15, g = lane >> 4;
    const int tasks = a.tiles * a.parts;
    int pair = (int)blockIdx.x / tasks, task = (int)blockIdx.x % tasks;
    if (a.by_xcd && !pair_task(a.S * a.p.kv, tasks, pair, task)) return;
    const int s = pair / a.p.kv, head = pair % a.p.kv;
    // causal: a sequence's last rows, which see most, first
    const int tile = a.tiles - 1 - task / a.parts, part = task % a.parts;
    const int rows = a.Lq * a.group, row0 = tile * ROWS + (SPLIT ? 0 : wave * 16 * RG);
    const int qlen = a.query_lengths ? max(0, min(__builtin_amdgcn_readfirstlane(a.query_lengths[s]), a.Lq)) : a.Lq;
    const int keys = a.key_lengths ? max(0, min(__builtin_amdgcn_readfirstlane(a.key_lengths[s]), a.most)) : a.most;
    const int64_t start = a.start ? __builtin_amdgcn_readfirstlane(a.start[s]) : 0;
    auto sees = [&](int token) {  // keys that a row sees
        return a.causal ? (int)max((int64_t)0, min((int64_t)keys, start + token + 1)) : keys;
    };
    const int last_row = min(row0 + 16 * RG, rows) - 1;
    const int last_token = min(last_row / a.group, qlen - 1);  // -1: none, or (no rows) less
    const bool any = row0 < rows && row0 / a.group < qlen;
    const int upto = any ? sees(last_token) : 0, all_see = any ? sees(row0 / a.group) : 0;

    // the wave's rows as columns, made when the first keys are asked for
    typename Op::type qf[RG][QS][N];
    float factor[RG];  // of the scores, in powers of two
    float origin[RG];  // BIASED: what a score begins with, -1152 times the sum of q'
    int limit[RG];     // keys that the lane's row sees
    auto prepare_rows = [&] {
#pragma unroll
        for (int rg = 0; rg < RG; rg++) {
            const int row = min(row0 + 16 * rg + i, rows - 1), token = row / a.heads;
            const T *q = reinterpret_cast<const T *>(a.q + s * a.qs[0] + token * a.qs[1] +
                                                     (head * a.group + row - token * a.group) * a.qs[2]);
            const float *cs = a.r.table ? rotation_row(a.r, start + token) : nullptr;
            limit[rg] = sees(token);
            float x[QS][8];
            float top = 0.0f;
#pragma unroll
            for (int m = 0; m < QS; m++) {
                load_turned8(a.r, q, cs, 64 * (m / 2) + 16 * g + 8 * (m % 2), x[m]);
#pragma unroll
                for (int e = 0; e < 8; e++) top = fmaxf(top, fabsf(x[m][e]));
            }
            factor[rg] = a.scale2;
            if (a.negative)
#pragma unroll
                for (int m = 0; m < QS; m++)
#pragma unroll
                    for (int e = 0; e < 8; e++) x[m][e] = -x[m][e];
            if constexpr (I8) {
                top = fmaxf(top, __shfl_xor(top, 16, 64));
                top = fmaxf(top, __shfl_xor(top, 32, 64));
                const int e2 = h2_exponent(top);
#pragma unroll
                for (int m = 0; m < QS; m++)
#pragma unroll
                    for (int e = 0; e < 8; e++) x[m][e] = __builtin_ldexpf(x[m][e], e2);
                factor[rg] = __builtin_ldexpf(a.scale2, -e2);
            }
#pragma unroll
            for (int m = 0; m < QS; m++) split_n<I8, N>(x[m], qf[rg][m]);
            origin[rg] = 0.0f;
            if constexpr (BIASED) {
#pragma unroll
                for (int m = 0; m < QS; m++)
#pragma unroll
                    for (int e = 0; e < 8; e++) origin[rg] += (float)qf[rg][m][0][e];
                origin[rg] += __shfl_xor(origin[rg], 16, 64);
                origin[rg] += __shfl_xor(origin[rg], 32, 64);
                origin[rg] *= -1152.0f;
            }
        }
    };

    floatx4 o[RG][DT];
    float m_run[RG], l_run[RG];
    float v_top[RG];  // the largest scale of values that the row has seen so far
#pragma unroll
    for (int rg = 0; rg < RG; rg++) {
#pragma unroll
        for (int t = 0; t < DT; t++) o[rg][t] = (floatx4){0, 0, 0, 0};
        m_run[rg] = -INFINITY;
        l_run[rg] = 0.0f;
        v_top[rg] = 0x1p-100f;
    }

    const int block0 = part * a.piece;
    const int block1 = min(block0 + a.piece, (upto + PC_BLOCK - 1) / PC_BLOCK);
    const int steps_all = max(0, (block1 - block0 + KB - 1) / KB);
    const int steps = SPLIT ? max(0, (steps_all - wave + 3) / 4) : steps_all;
    auto block_of = [&](int step) { return block0 + (SPLIT ? wave + 4 * step : step) * KB; };

    // Lane l holds where block l % KB of step fetched + l / KB is, and its scales.
    uint32_t at_lo = 0, at_hi = 0;
    float sk = 0.0f, sv = 0.0f;
    uint64_t there = 0;
    auto fetch = [&](int step) {
        const int block = block_of(step + lane / KB) + lane % KB;
        int page = -1;
        uint32_t column = 0;
        if (block < block1) {
            column = (uint32_t)block / a.p.blocks;
            page = page_of(a.p, s, column);
        }
        const int slot = page >= 0 ? block - (int)(column * a.p.blocks.d) : 0;
        const char *p = block_at(a.p, max(page, 0), head, slot, B::BYTES);
        at_lo = (uint32_t)(uint64_t)p;
        at_hi = (uint32_t)((uint64_t)p >> 32);
        if constexpr (I8) {
            const float2 sc = *reinterpret_cast<const float2 *>(scale_at(a.p, max(page, 0), head, slot));
            sk = page >= 0 ? sc.x : 0.0f;
            sv = page >= 0 ? sc.y : 0.0f;
        }
        there = __ballot(page >= 0);
    };
    auto read_lane = [](uint32_t v, int l) { return (uint32_t)__builtin_amdgcn_readlane((int)v, l); };

    struct Step {
        RawBlocks<D, I8, KB> k, v;
        float sk[KB], sv[KB];
        uint32_t there;
    };
    // By an address that is known to be global memory's (one made of a number is not, and its
    // loads are waited for all together), the same in all lanes but for 16 bytes each.
    auto take = [&](uint64_t at, int offset) {
        typedef const __attribute__((address_space(1))) char *Bytes;
        typedef const __attribute__((address_space(1))) u32x4 *Words;
        const Words from = (Words)((Bytes)at + (uint32_t)(16 * lane) + offset);
        // Past the caches: up to 16 rows each key is read by one wave.  fp32 queries of 128 dims
        // have these loads with more rows too, whose workgroups read the same keys, and lose by
        // it: 512 tokens of 32 heads on 8 over 4608 bf16 keys 191 us, with the others 112
        if constexpr (SPLIT && RG == 1) return __builtin_nontemporal_load(from);
        else return *from;
    };
    auto load_values = [&](Step &st, int step) {
        const int at = step % PER_FETCH * KB;
#pragma unroll
        for (int b = 0; b < KB; b++) {
            const uint64_t from = (uint64_t)read_lane(at_hi, at + b) << 32 | read_lane(at_lo, at + b);
#pragma unroll
            for (int u = 0; u < B::UNITS; u++) st.v.w[b][u] = take(from, B::PART + 1024 * u);
        }
    };
    auto load = [&](Step &st, int step) {  // keys, and values where both are kept twice
        const int at = step % PER_FETCH * KB;
        if (at == 0) fetch(step);
        st.there = (uint32_t)(there >> at) & ((1u << KB) - 1);
#pragma unroll
        for (int b = 0; b < KB; b++) {
            const uint64_t from = (uint64_t)read_lane(at_hi, at + b) << 32 | read_lane(at_lo, at + b);
#pragma unroll
            for (int u = 0; u < B::UNITS; u++) st.k.w[b][u] = take(from, 1024 * u);
            if constexpr (!ROLLING)
#pragma unroll
                for (int u = 0; u < B::UNITS; u++) st.v.w[b][u] = take(from, B::PART + 1024 * u);
            if constexpr (I8) {
                st.sk[b] = __uint_as_float(read_lane(__float_as_uint(sk), at + b));
                st.sv[b] = __uint_as_float(read_lane(__float_as_uint(sv), at + b));
            }
        }
    };

    auto compute = [&](Step &st, int step) {
        const int first = block_of(step) * PC_BLOCK;
        const uint32_t held = st.there;
        const bool whole = first + KB * PC_BLOCK <= all_see && held == (1u << KB) - 1;
        floatx4 x[RG][KB];
#pragma unroll
        for (int rg = 0; rg < RG; rg++)
#pragma unroll
            for (int b = 0; b < KB; b++) x[rg][b] = (floatx4){origin[rg], origin[rg], origin[rg], origin[rg]};
#pragma unroll
        for (int b = 0; b < KB; b++)
#pragma unroll
            for (int m = 0; m < QS; m++) {
                const typename Op::type k = st.k.template key<BIASED>(b, m);
#pragma unroll
                for (int rg = 0; rg < RG; rg++)
#pragma unroll
                    for (int n = N - 1; n >= 0; n--) x[rg][b] = Op::mfma(k, qf[rg][m][n], x[rg][b]);
            }
        if (ROLLING && step + 1 < steps) load(st, step + 1);
        // bf16: what lies behind the keys may be no number, which a probability of 0 does not hide
        if (!I8 && !whole) {
#pragma unroll
            for (int b = 0; b < KB; b++)
#pragma unroll
                for (int u = 0; u < B::UNITS; u++)
#pragma unroll
                    for (int d = 0; d < 4; d++) {
                        // a word holds tokens 4 g + 2 (d % 2) and the next
                        const int key = first + 16 * b + 4 * g + 2 * (d % 2);
                        uint32_t keep = (held >> b & 1) == 0 || key >= upto ? 0u : key + 1 >= upto ? 0xffffu : ~0u;
                        st.v.w[b][u][d] &= keep;
                    }
        }
        // scores to powers of two, s f; their largest in this lane.  A row takes the scales of
        // the blocks that it sees only: what it sees is all that its result depends on
        float f[RG][KB], sv[RG][KB], top[RG];
#pragma unroll
        for (int rg = 0; rg < RG; rg++)
#pragma unroll
            for (int b = 0; b < KB; b++) {
                f[rg][b] = I8 ? factor[rg] * st.sk[b] : factor[rg];
                if constexpr (I8) sv[rg][b] = st.sv[b];
            }
        if (!whole) {
#pragma unroll
            for (int rg = 0; rg < RG; rg++)
#pragma unroll
                for (int b = 0; b < KB; b++) {
                    const int keys_of_block = (held >> b & 1) ? limit[rg] - (first + 16 * b) : 0;
                    if (I8 && keys_of_block <= 0) f[rg][b] = sv[rg][b] = 0.0f;
                    if (f[rg][b] < FLT_LEAST) f[rg][b] = FLT_LEAST;  // 0 times -inf is no number; a NaN stays
#pragma unroll
                    for (int r = 0; r < 4; r++)
                        if (4 * g + r >= keys_of_block) x[rg][b][r] = -INFINITY;
                }
        }
        bool over = false;
#pragma unroll
        for (int rg = 0; rg < RG; rg++) {
            top[rg] = -INFINITY;
#pragma unroll
            for (int b = 0; b < KB; b++) {
                const float most = larger(larger(x[rg][b][0], x[rg][b][1]), larger(x[rg][b][2], x[rg][b][3]));
                top[rg] = larger(top[rg], most * f[rg][b]);
            }
            over |= top[rg] > m_run[rg] + LAZY;
            if constexpr (I8)
#pragma unroll
                for (int b = 0; b < KB; b++) over |= sv[rg][b] > v_top[rg];
        }
        // A row's exponents' base follows its maximum only when that is 2^LAZY beyond it, and its
        // values' unit the largest scale: then all that was summed of the row is rescaled, and
        // that of the others times 1.
        if (__ballot(over)) {
#pragma unroll
            for (int rg = 0; rg < RG; rg++) {
                float m = fmaxf(m_run[rg], top[rg]);
                m = fmaxf(m, __shfl_xor(m, 16, 64));
                m = fmaxf(m, __shfl_xor(m, 32, 64));
                m = m > m_run[rg] + LAZY ? m : m_run[rg];
                const float alpha = m == -INFINITY ? 0.0f : exp2_of(m_run[rg] - m);  // -inf - -inf is no number
                m_run[rg] = m;
                l_run[rg] *= alpha;
                float rescale = alpha;
                if constexpr (I8) {
                    float v_new = v_top[rg];
#pragma unroll
                    for (int b = 0; b < KB; b++) v_new = fmaxf(v_new, sv[rg][b]);
                    rescale *= v_top[rg] / v_new;
                    v_top[rg] = v_new;
                }
#pragma unroll
                for (int t = 0; t < DT; t++) o[rg][t] *= rescale;
            }
        }
        typename Op::type pf[RG][KB / 2][N];
#pragma unroll
        for (int rg = 0; rg < RG; rg++) {
            const float base = m_run[rg] == -INFINITY ? 0.0f : m_run[rg];
            const float inv = I8 ? P_SCALE * __builtin_amdgcn_rcpf(v_top[rg]) : 1.0f;
            float sum = 0.0f;
#pragma unroll
            for (int c = 0; c < KB / 2; c++) {
                float p[8];
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const int b = 2 * c + e / 4;
                    p[e] = exp2_of(__builtin_fmaf(x[rg][b][e % 4], f[rg][b], -base));
                    sum += p[e];
                    if constexpr (I8) p[e] *= sv[rg][b] * inv;
                }
                split_n<I8, N>(p, pf[rg][c]);
            }
            l_run[rg] += sum;
        }
#pragma unroll
        for (int c = 0; c < KB / 2; c++)
#pragma unroll
            for (int t = 0; t < DT; t++) {
                const typename Op::type v = st.v.value(c, t);
#pragma unroll
                for (int rg = 0; rg < RG; rg++)
#pragma unroll
                    for (int n = N - 1; n >= 0; n--) o[rg][t] = Op::mfma(v, pf[rg][c][n], o[rg][t]);
            }
        if (ROLLING && step + 1 < steps) load_values(st, step + 1);
    };

    // the next step's blocks are on their way while one is computed
    Step even, odd;
    if (steps > 0) {
        load(even, 0);
        if constexpr (ROLLING) load_values(even, 0);
    }
    prepare_rows();
    for (int step = 0; step < steps; step += ROLLING ? 1 : 2) {
        if constexpr (ROLLING) {
            compute(even, step);
        } else {
            if (step + 1 < steps) load(odd, step + 1);
            compute(even, step);
            if (step + 1 >= steps) break;
            if (step + 2 < steps) load(even, step + 2);
            compute(odd, step + 1);
        }
    }

    // in the values' own units
    if constexpr (I8)
#pragma unroll
        for (int rg = 0; rg < RG; rg++)
#pragma unroll
            for (int t = 0; t < DT; t++) o[rg][t] *= v_top[rg] / P_SCALE;

    // The waves' sums of the same rows lie in the same lanes: half of the waves give theirs
    // to the others, twice.
    if constexpr (SPLIT) {
        __shared__ floatx4 sums[2][RG * DT][64];
        __shared__ float2 stats[2][RG][64];
#pragma unroll
        for (int half = 2; half > 0; half /= 2) {
            if (wave >= half && wave < 2 * half) {
#pragma unroll
                for (int rg = 0; rg < RG; rg++) {
#pragma unroll
                    for (int t = 0; t < DT; t++) sums[wave - half][rg * DT + t][lane] = o[rg][t];
                    stats[wave - half][rg][lane] = {m_run[rg], l_run[rg]};
                }
            }
            __syncthreads();
            if (wave < half) {
#pragma unroll
                for (int rg = 0; rg < RG; rg++) {
                    const float2 ml = stats[wave][rg][lane];
                    const float m = fmaxf(m_run[rg], ml.x), base = m == -INFINITY ? 0.0f : m;  // -inf - -inf is no number
                    const float mine = exp2_of(m_run[rg] - base), other = exp2_of(ml.x - base);
                    m_run[rg] = m;
                    l_run[rg] = l_run[rg] * mine + ml.y * other;
#pragma unroll
                    for (int t = 0; t < DT; t++) o[rg][t] = o[rg][t] * mine + sums[wave][rg * DT + t][lane] * other;
                }
            }
            if (half > 1) __syncthreads();
        }
        if (wave > 0) return;
    }
#pragma unroll
    for (int rg = 0; rg < RG; rg++) {
        float l = l_run[rg];
        l += __shfl_xor(l, 16, 64);
        l += __shfl_xor(l, 32, 64);
        const int row = row0 + 16 * rg + i;
        if (row >= rows) continue;
        const int token = row / a.heads, h = head * a.group + row - token * a.group;
        float y[4 * DT];  // dims 4 DT g ..
        const bool out = a.parts == 1;
        const float inv = l == 0.0f || token >= qlen ? 0.0f : 1.0f / l;
#pragma unroll
        for (int r = 0; r < 4; r++)
#pragma unroll
            for (int t = 0; t < DT; t++) y[DT * r + t] = !out ? o[rg][t][r] : inv == 0.0f ? 0.0f : o[rg][t][r] * inv;
        if (out) {
            store_n<4 * DT>(reinterpret_cast<T *>(a.out + s * a.os[0] + token * a.os[1] + h * a.os[2]) + 4 * DT * g, y);
        } else {
            const int64_t at = (((int64_t)part * a.S + s) * a.Lq + token) * a.H + h;
            if (l != 0.0f) store_n<4 * DT>(a.part_o + at * D + 4 * DT * g, y);
            if (g == 0) a.part_ml[at] = {m_run[rg], l};
        }
    }
}

// Joins the pieces of the keys: 16 lanes a row, first for the pieces' statistics, then
// for D / 16 dims each.
template <typename T, int D>
static __global__ __launch_bounds__(256) void cache_join_kernel(CacheAttentionArgs a) {
    constexpr int DT = D / 16, MOST = 4;  // pieces of a lane: 64 in all
    const int64_t row = (int64_t)blockIdx.x * 16 + threadIdx.x / 16, rows = (int64_t)a.S * a.Lq * a.H;
    if (row >= rows) return;
    const int lane = threadIdx.x & 15;
    const uint32_t in_tokens = (uint32_t)(row / a.H);
    const int h = (int)(row - (int64_t)in_tokens * a.H), s = (int)(in_tokens / (uint32_t)a.Lq), token = (int)(in_tokens % (uint32_t)a.Lq);
    const int qlen = a.query_lengths ? max(0, min(a.query_lengths[s], a.Lq)) : a.Lq;
    const int keys = a.key_lengths ? max(0, min(a.key_lengths[s], a.most)) : a.most;
    int64_t seen = token < qlen ? keys : 0;
    if (a.causal) seen = max((int64_t)0, min(seen, (a.start ? a.start[s] : 0) + (int64_t)token + 1));
    const int piece = a.piece * PC_BLOCK, parts = (int)((seen + piece - 1) / piece);
    float2 ml[MOST];
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < MOST; i++) {
        ml[i] = {-INFINITY, 0.0f};
        if (lane + 16 * i < parts) ml[i] = a.part_ml[(lane + 16 * i) * rows + row];
        m = fmaxf(m, ml[i].x);
    }
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 16));
    float f[MOST], l = 0.0f;
#pragma unroll
    for (int i = 0; i < MOST; i++) {
        // of a piece that nothing was written for the weight is 0, and what is read there left out
        f[i] = ml[i].y == 0.0f ? 0.0f : exp2_of(ml[i].x - m);
        l += ml[i].y == 0.0f ? 0.0f : ml[i].y * f[i];
    }
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) l += __shfl_xor(l, o, 16);
    float v[DT];
#pragma unroll
    for (int e = 0; e < DT; e++) v[e] = 0.0f;
    const float *from = a.part_o + row * D + DT * lane;
#pragma unroll
    for (int i = 0; i < MOST; i++) {
        for (int p0 = 16 * i; p0 < min(parts, 16 * i + 16); p0 += 4) {
            float x[4][DT];
#pragma unroll
            for (int j = 0; j < 4; j++) load_n<DT>(from + min(p0 + j, parts - 1) * rows * D, x[j]);
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const float w = __shfl(f[i], p0 + j - 16 * i, 16);  // 0 beyond the pieces
#pragma unroll
                for (int e = 0; e < DT; e++) v[e] += w == 0.0f ? 0.0f : x[j][e] * w;
            }
        }
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
    for (int e = 0; e < DT; e++) v[e] = inv == 0.0f ? 0.0f : v[e] * inv;
    store_n<DT>(reinterpret_cast<T *>(a.out + s * a.os[0] + token * a.os[1] + h * a.os[2]) + DT * lane, v);
}

}  // namespace vh
