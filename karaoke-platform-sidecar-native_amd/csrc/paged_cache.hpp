// Pages of keys and values: appending rows (keys turned on the way), reading them
// back, and another order of a batch's tables.
//
// A page holds, for each key head, its blocks of 16 tokens one behind the other: the
// block's keys, then its values, each as 16 * D elements in units of 1 KB that a wave
// takes with one 16-byte load a lane, in the order in which the attention's matrix
// instructions (16 x 16 results, 32 summed) want them, so that it needs no LDS.  Lane
// l = 16 g + i of a wave has, with C the elements of 16 bytes (8 bf16, 16 of 8 bits):
//   keys, unit u:    token i, dims 64 (u C / 16) + 16 g + (u C % 16) + 0 .. C - 1
//   values, unit u:  dims (D / 16) i + (C / 4) u + 0 .. C / 4 - 1, each of tokens 4 g + 0 .. 3
// 8-bit numbers are held plus 128, as bytes from 1 to 255.  Behind the blocks a page of
// 8 bits has the blocks' scales, [head][block] (key's, value's).
#pragma once

#include "rotary.hpp"

namespace vh {

constexpr int PC_BLOCK = 16;

struct PagedArgs {
    char *pool;
    const int *table;
    int64_t page_bytes, scales;  // of a page, and from its start to its scales
    int kv, pages, table_pages, page_blocks;
    Divisor blocks;              // page_blocks
};

template <int D, bool I8>
struct BlockShape {
    static constexpr int C = I8 ? 16 : 8;               // elements of 16 bytes
    static constexpr int PART = 16 * D * (I8 ? 1 : 2);  // bytes of a block's keys, or values
    static constexpr int BYTES = 2 * PART;
    static constexpr int UNITS = PART / 1024;
    static constexpr int DT = D / 16;
};

// Page of a sequence's block; -1: none.
VH_DEVICE int page_of(const PagedArgs &a, int s, uint32_t column) {
    if (column >= (uint32_t)a.table_pages) return -1;
    const int p = a.table[(int64_t)s * a.table_pages + column];
    return p >= 0 && p < a.pages ? p : -1;
}

// Address of a block of a head: its keys, then its values.
VH_DEVICE char *block_at(const PagedArgs &a, int page, int head, int slot, int block_bytes) {
    return a.pool + page * a.page_bytes + ((int64_t)head * a.page_blocks + slot) * block_bytes;
}
VH_DEVICE float *scale_at(const PagedArgs &a, int page, int head, int slot) {
    return reinterpret_cast<float *>(a.pool + page * a.page_bytes + a.scales) + 2 * (head * a.page_blocks + slot);
}

struct CacheRowsArgs {
    PagedArgs p;
    Rotation r;
    char *k, *v;
    int64_t ks[3], vs[3];  // bytes
    const int *start, *lengths;
    int length, tasks;     // rows of a sequence; waves
    Divisor per_sequence, per_block;  // tasks of a sequence and of a block, 2 * kv
};

// A wave's task: 16 tokens' keys or values of a head.
struct CacheTask {
    int s, head, values;
    int64_t first, start;  // positions of the block's first token and of row 0
    int rows, page, slot;
    VH_DEVICE bool take(const CacheRowsArgs &a) {
        const uint32_t t = blockIdx.x * 4 + (uint32_t)__builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
        if (t >= (uint32_t)a.tasks) return false;
        const uint32_t sq = t / a.per_sequence, in = t - sq * a.per_sequence.d, block_of_call = in / a.per_block;
        const int part = (int)(in - block_of_call * a.per_block.d);
        values = part >= a.p.kv;
        head = values ? part - a.p.kv : part;
        s = (int)sq;
        start = max(0, a.start ? __builtin_amdgcn_readfirstlane(a.start[s]) : 0);
        rows = a.lengths ? max(0, min(__builtin_amdgcn_readfirstlane(a.lengths[s]), a.length)) : a.length;
        const uint32_t block = (uint32_t)(start / PC_BLOCK) + block_of_call;
        first = (int64_t)block * PC_BLOCK;
        const uint32_t column = block / a.p.blocks;
        slot = (int)(block - column * a.p.blocks.d);
        page = __builtin_amdgcn_readfirstlane(page_of(a.p, s, column));
        return true;
    }
};

VH_DEVICE uint32_t wave_umax(uint32_t v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = max(v, (uint32_t)__shfl_xor((int)v, o, 64));
    return v;
}

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// The whole number next to x f (at most 127 and a half), plus 128, in the low byte: a
// sum with 3 * 2^22 + 128 is rounded there.
VH_DEVICE uint32_t number_of(float x, float f) {
#pragma clang fp contract(off)
    const float q = x * f;
    return __float_as_uint(q + 12583040.0f);
}
VH_DEVICE uint32_t low_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    return __builtin_amdgcn_perm(b, a, 0x0c0c0400u) | __builtin_amdgcn_perm(d, c, 0x04000c0cu);
}

// A block's tokens: held before the call, in it, or (after it) none.
struct TokenRange {
    int lo, hi;
    VH_DEVICE bool earlier(int t) const { return t < lo; }
    VH_DEVICE bool of_call(int t) const { return t >= lo && t < hi; }
};

// N consecutive floats of LDS, up to 4 at a time aligned.
template <int N>
VH_DEVICE void load_lds(const float *p, float (&v)[N]) {
    typedef float V __attribute__((ext_vector_type(N < 4 ? N : 4)));
#pragma unroll
    for (int e = 0; e < N; e += 4) {
        const V a = *reinterpret_cast<const V *>(p + e);
#pragma unroll
        for (int i = 0; i < (N < 4 ? N : 4); i++) v[e + i] = a[i];
    }
}
// LDS accesses of the wave's lanes before and after stay in that order (the hardware
// keeps a wave's; this keeps the compiler's).
VH_DEVICE void cache_wave_order() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// Rows into a block.  A wave's lanes take units of 16 dims of its tokens, beside each
// other in a row, turn them, and take them up in the block's order by way of a tile of
// LDS; earlier tokens of a block that is not new are rescaled in place.
//
// Bound by HBM: 32000 tokens of 8 heads of 128, bf16 into 8 bits 47 us (4.1 TB/s, where
// a copy reaches 5.0), into bf16 54 us (4.8).  Lanes that read what they hold in the
// block's order, without LDS, took 82 us for 18700 tokens instead of 36: a token's row in
// pieces of 16 bytes; a lane's units one behind the other 40 us; four heads a wave, for
// one reading of the table's row, no less than one.
template <typename T, int D, bool I8>
static __global__ __launch_bounds__(256) void cache_append_kernel(CacheRowsArgs a) {
    using B = BlockShape<D, I8>;
    constexpr int DT = B::DT, NU = D / 64, ROW = D + 4;  // units of a lane; floats of a tile's row, four banks apart
    __shared__ __align__(16) float tiles[4][PC_BLOCK * ROW];
    const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
    float *tile = tiles[threadIdx.x >> 6];
    CacheTask w;
    if (!w.take(a) || w.page < 0) return;
    const TokenRange tokens{(int)max(w.start - w.first, (int64_t)0), (int)min(w.start + w.rows - w.first, (int64_t)PC_BLOCK)};
    if (tokens.lo >= tokens.hi) return;
    const int64_t *strides = w.values ? a.vs : a.ks;
    const char *rows = (w.values ? a.v : a.k) + w.s * strides[0] + (w.first - w.start) * strides[1] + w.head * strides[2];
    // Of 128 dims, in groups of 4, the even groups lie before the odd ones: a value's unit is
    // every other group of a row, all of them in banks of their own so.
    auto column = [](int d) { return D == 64 ? d : (d / 8 + 16 * (d / 4 % 2)) * 4 + d % 4; };
    // the lane's units, all asked for before the first is turned
    typedef typename Elements<T, 8>::type Raw;
    Raw lo[NU], hi[NU];
    float cs[NU][16];
    int at[NU], beside[NU];  // where the unit's two times 8 dims are
    bool mine[NU], turned[NU], off_table[NU];
#pragma unroll
    for (int n = 0; n < NU; n++) {
        const int t = (lane + 64 * n) / (D / 16), u = (lane + 64 * n) % (D / 16);
        mine[n] = tokens.of_call(t);
        turned[n] = !w.values && a.r.table && u < a.r.dim / 16;
        at[n] = D == 128 && w.values ? 8 * u : 16 * u;
        beside[n] = D == 128 && w.values ? 64 + 8 * u : 16 * u + 8;
        if (turned[n] && !a.r.interleaved) {
            at[n] = 8 * u;
            beside[n] = a.r.dim / 2 + 8 * u;
        }
        const T *row = reinterpret_cast<const T *>(rows + (mine[n] ? t : tokens.lo) * strides[1]);
        lo[n] = *reinterpret_cast<const Raw *>(row + at[n]);
        hi[n] = *reinterpret_cast<const Raw *>(row + beside[n]);
        off_table[n] = false;
        if (turned[n]) {
            const float *angles = rotation_row(a.r, w.first + t);
            off_table[n] = !angles;
            load_n<16>((angles ? angles : a.r.table) + 16 * u, cs[n]);
        }
    }
    uint32_t top = 0;
#pragma unroll
    for (int n = 0; n < NU; n++) {
        float x[8], y[8];
#pragma unroll
        for (int e = 0; e < 8; e++) x[e] = (float)lo[n][e], y[e] = (float)hi[n][e];
        if (turned[n]) {
            if (a.r.interleaved) {
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    turn_pair(x[2 * e], x[2 * e + 1], cs[n][2 * e], cs[n][2 * e + 1]);
                    turn_pair(y[2 * e], y[2 * e + 1], cs[n][8 + 2 * e], cs[n][9 + 2 * e]);
                }
            } else {
#pragma unroll
                for (int e = 0; e < 8; e++) turn_pair(x[e], y[e], cs[n][2 * e], cs[n][2 * e + 1]);
            }
            if (off_table[n])
#pragma unroll
                for (int e = 0; e < 8; e++) x[e] = y[e] = __builtin_nanf("");
        }
        if constexpr (I8)
#pragma unroll
            for (int e = 0; e < 8; e++)
                if (mine[n]) top = max(top, max(__float_as_uint(x[e]) & 0x7fffffffu, __float_as_uint(y[e]) & 0x7fffffffu));
        float *to = tile + (lane + 64 * n) / (D / 16) * ROW;
#pragma unroll
        for (int e = 0; e < 8; e += 4) {
            st4(to + column(at[n] + e), (floatx4){x[e], x[e + 1], x[e + 2], x[e + 3]});
            st4(to + column(beside[n] + e), (floatx4){y[e], y[e + 1], y[e + 2], y[e + 3]});
        }
    }
    float inv = 0.0f, earlier = 0.0f;
    if constexpr (I8) {
        top = wave_umax(top);
        float *held = scale_at(a.p, w.page, w.head, w.slot) + w.values;
        float scale = fmaxf(__uint_as_float(top) * (1.0f / 127.0f), 0x1p-100f);
        float old = 0.0f;
        if (tokens.lo) {
            old = *held;
            if (!(old <= scale)) scale = old;
        }
        if (top >= 0x7f800000u) scale = __builtin_nanf("");
        inv = 1.0f / scale;
        earlier = old * inv;
        if (lane == 0) *held = scale;
    }
    cache_wave_order();
    u32x4 *block = reinterpret_cast<u32x4 *>(block_at(a.p, w.page, w.head, w.slot, B::BYTES) + w.values * B::PART) + lane;
    const bool whole = tokens.lo == 0 && tokens.hi == PC_BLOCK;
#pragma unroll
    for (int u = 0; u < B::UNITS; u++) {
        float x[B::C];
        if (w.values) {
#pragma unroll
            for (int r = 0; r < 4; r++) {
                float v[B::C / 4];
                load_lds<B::C / 4>(tile + (4 * g + r) * ROW + column(DT * i + B::C / 4 * u), v);
#pragma unroll
                for (int e = 0; e < B::C / 4; e++) x[4 * e + r] = v[e];
            }
        } else {
#pragma unroll
            for (int e = 0; e < B::C; e += 4) {
                const floatx4 v = ld4(tile + i * ROW + column(64 * (u * B::C / 16) + 16 * g + u * B::C % 16 + e));
#pragma unroll
                for (int j = 0; j < 4; j++) x[e + j] = v[j];
            }
        }
        u32x4 now;
#pragma unroll
        for (int d = 0; d < 4; d++) {
            if constexpr (I8) {
                const float *q = x + 4 * d;
                now[d] = low_bytes(number_of(q[0], inv), number_of(q[1], inv), number_of(q[2], inv), number_of(q[3], inv));
            } else {
                const float *q = x + 2 * d;
                now[d] = (uint32_t)__builtin_bit_cast(uint16_t, (bf16)q[0]) | (uint32_t)__builtin_bit_cast(uint16_t, (bf16)q[1]) << 16;
            }
        }
        if (!whole) {
            u32x4 old = {0, 0, 0, 0};
            if (tokens.lo) old = block[64 * u];
#pragma unroll
            for (int d = 0; d < 4; d++) {
                constexpr int N = I8 ? 4 : 2, BITS = 32 / N;
                constexpr uint32_t MASK = I8 ? 0xffu : 0xffffu;
                uint32_t word = 0;
#pragma unroll
                for (int e = 0; e < N; e++) {
                    const int t = w.values ? 4 * g + (N * d + e) % 4 : i;
                    uint32_t before = old[d] >> (BITS * e) & MASK;
                    if constexpr (I8) before = number_of((float)((int)before - 128), earlier) & MASK;
                    const uint32_t value = tokens.of_call(t) ? now[d] >> (BITS * e) & MASK : tokens.earlier(t) ? before : I8 ? 128u : 0u;
                    word |= value << (BITS * e);
                }
                now[d] = word;
            }
        }
        block[64 * u] = now;
    }
}

// A block's rows, one head's: lanes write what they hold in the block's order (of keys a
// token's 16 dims beside each other, of values D / 16 of four tokens).  Bound by HBM:
// 32000 tokens of 8 heads of 128 to bf16, 47 us from 8 bits (4.2 TB/s), 54 us from bf16.
template <typename T, int D, bool I8>
static __global__ __launch_bounds__(256) void cache_read_kernel(CacheRowsArgs a) {
    using B = BlockShape<D, I8>;
    constexpr int DT = B::DT;
    const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
    CacheTask w;
    if (!w.take(a)) return;
    char *out = w.values ? a.v : a.k;
    if (!out) return;
    float x[4 * DT];
    const bool any = w.page >= 0 && w.first < w.start + w.rows;
    const int page = any ? w.page : 0;
    const u32x4 *block = reinterpret_cast<const u32x4 *>(block_at(a.p, page, w.head, any ? w.slot : 0, B::BYTES) + w.values * B::PART) + lane;
    const float scale = I8 && any ? scale_at(a.p, page, w.head, w.slot)[w.values] : 1.0f;
#pragma unroll
    for (int u = 0; u < B::UNITS; u++) {
        u32x4 from = {0, 0, 0, 0};
        if (any) from = block[64 * u];
#pragma unroll
        for (int e = 0; e < B::C; e++) {
            if constexpr (I8) x[B::C * u + e] = (float)((int)(from[e / 4] >> (8 * (e % 4)) & 0xff) - 128) * scale;
            else x[B::C * u + e] = __uint_as_float(from[e / 2] >> (16 * (e % 2)) << 16);
        }
    }
    const int64_t *strides = w.values ? a.vs : a.ks;
    char *to = out + w.s * strides[0] + w.head * strides[2];
    auto zero_or = [&](int64_t row, float v) { return any && row < w.rows ? v : 0.0f; };
    if (w.values) {
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const int64_t row = w.first + 4 * g + r - w.start;
            if (row < 0 || row >= a.length) continue;
            float v[DT];
#pragma unroll
            for (int e = 0; e < DT; e++) v[e] = zero_or(row, x[4 * e + r]);
            store_n<DT>(reinterpret_cast<T *>(to + row * strides[1]) + DT * i, v);
        }
    } else {
        const int64_t row = w.first + i - w.start;
        if (row < 0 || row >= a.length) return;
#pragma unroll
        for (int n = 0; n < D / 64; n++) {
            float v[16];
#pragma unroll
            for (int e = 0; e < 16; e++) v[e] = zero_or(row, x[16 * n + e]);
            store_n<16>(reinterpret_cast<T *>(to + row * strides[1]) + 64 * n + 16 * g, v);
        }
    }
}

struct ReorderArgs {
    PagedArgs p;
    const int *parents, *lengths, *spare;
    int *table_out, *spare_out;
    int beams, block_bytes, scaled;
};

// A workgroup copies a head's blocks of a row's last page; head 0's writes the row of
// the table too.  Bound by HBM: 256 rows of 8 heads of 128, 8 blocks of 8 bits each, 7 of 8
// rows another's: 19 us (6.0 TB/s).
static __global__ __launch_bounds__(256) void cache_reorder_kernel(ReorderArgs a) {
    const int row = (int)(blockIdx.x / (uint32_t)a.p.kv), head = (int)(blockIdx.x % (uint32_t)a.p.kv);
    const int group = row / a.beams;
    int parent = a.parents[row];
    parent = parent >= 0 && parent < a.beams ? group * a.beams + parent : row;
    const int tokens = a.p.page_blocks * PC_BLOCK;
    const int length = max(0, min(a.lengths[group], a.p.table_pages * tokens));
    const int full = length / tokens, used = length % tokens;
    const int *from = a.p.table + (int64_t)parent * a.p.table_pages, *own = a.p.table + (int64_t)row * a.p.table_pages;
    const bool other = used && parent != row;
    const int source = other ? page_of(a.p, parent, full) : -1, target = a.spare[row];
    const bool moved = source >= 0;
    if (head == 0) {
        int *to = a.table_out + (int64_t)row * a.p.table_pages;
        for (int c = threadIdx.x; c < a.p.table_pages; c += 256)
            to[c] = c < full ? from[c] : c > full || !other ? own[c] : moved ? target : from[c];
        if (threadIdx.x == 0) a.spare_out[row] = moved ? own[full] : target;
    }
    if (!moved || target < 0 || target >= a.p.pages) return;
    const int blocks = (used + PC_BLOCK - 1) / PC_BLOCK;
    const u32x4 *src = reinterpret_cast<const u32x4 *>(block_at(a.p, source, head, 0, a.block_bytes));
    u32x4 *dst = reinterpret_cast<u32x4 *>(block_at(a.p, target, head, 0, a.block_bytes));
    const int n = blocks * a.block_bytes / 16;
    for (int i0 = threadIdx.x; i0 < n; i0 += 8 * 256) {
        u32x4 x[8];
#pragma unroll
        for (int j = 0; j < 8; j++)
            if (i0 + 256 * j < n) x[j] = src[i0 + 256 * j];
#pragma unroll
        for (int j = 0; j < 8; j++)
            if (i0 + 256 * j < n) dst[i0 + 256 * j] = x[j];
    }
    if (a.scaled)
        for (int i = threadIdx.x; i < 2 * blocks; i += 256) scale_at(a.p, target, head, 0)[i] = scale_at(a.p, source, head, 0)[i];
}

}  // namespace vh
