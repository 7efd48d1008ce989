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
    VH_DEVICE static int key_dim(int u, int g) { return 64 * (u * C / 16) + 16 * g + u * C % 16; }
    VH_DEVICE static int value_dim(int u, int i) { return DT * i + C / 4 * u; }
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
    int length, blocks;    // rows of a sequence, and blocks that they may touch
    int64_t tasks;         // sequences * blocks * 2 * kv, a wave each
};

// A wave's task: 16 tokens' keys or values of a head.
struct CacheTask {
    int s, head, values;
    int64_t first, start;  // positions of the block's first token and of row 0
    int rows, page, slot;
    VH_DEVICE bool take(const CacheRowsArgs &a, int wave) {
        int64_t t = (int64_t)blockIdx.x * 4 + wave;
        if (t >= a.tasks) return false;
        const int64_t b = t / (2 * a.p.kv);
        const int in = (int)(t - b * 2 * a.p.kv);
        values = in >= a.p.kv;
        head = values ? in - a.p.kv : in;
        s = (int)(b / a.blocks);
        start = max(0, a.start ? __builtin_amdgcn_readfirstlane(a.start[s]) : 0);
        rows = a.lengths ? max(0, min(__builtin_amdgcn_readfirstlane(a.lengths[s]), a.length)) : a.length;
        const uint32_t block = (uint32_t)(start / PC_BLOCK + (b - (int64_t)s * a.blocks));
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
// LDS accesses of the wave's lanes before and after stay in that order (the hardware
// keeps a wave's; this keeps the compiler's).
VH_DEVICE void cache_wave_order() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// How a block's numbers come from its rows.
struct Quant {
    float inv, earlier;  // 1 / scale, and what the numbers of earlier tokens are multiplied by
    VH_DEVICE static uint32_t number(float q) { return (uint32_t)((int)fminf(fmaxf(__builtin_rintf(q), -127.0f), 127.0f) + 128); }
    VH_DEVICE uint32_t of(float x) const { return number(x * inv); }
    VH_DEVICE uint32_t again(uint32_t byte) const { return number((float)((int)byte - 128) * earlier); }
};
// A block's token: held before the call, in it, or (after it) none.
struct TokenRange {
    int lo, hi;
    VH_DEVICE bool earlier(int t) const { return t < lo; }
    VH_DEVICE bool of_call(int t) const { return t >= lo && t < hi; }
};

// Rows into a block.  A wave turns its rows, in units of 16 dims a lane, into a tile
// of LDS, finds the scale, and writes the block from the tile in the block's order,
// earlier tokens rescaled in place.
template <typename T, int D, bool I8>
static __global__ __launch_bounds__(256) void cache_append_kernel(CacheRowsArgs a) {
    using B = BlockShape<D, I8>;
    constexpr int ROW = D + 4;  // floats: rows four banks apart
    __shared__ __align__(16) float tiles[4][PC_BLOCK * ROW];
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), lane = threadIdx.x & 63;
    CacheTask w;
    if (!w.take(a, wave) || w.page < 0) return;
    const TokenRange tokens{(int)max(w.start - w.first, (int64_t)0), (int)min(w.start + w.rows - w.first, (int64_t)PC_BLOCK)};
    if (tokens.lo >= tokens.hi) return;
    float *tile = tiles[wave];
    const int64_t *strides = w.values ? a.vs : a.ks;
    const char *rows = (w.values ? a.v : a.k) + w.s * strides[0] + (w.first - w.start) * strides[1] + w.head * strides[2];
    const int turned = w.values || !a.r.table ? 0 : a.r.dim / 16;
    const int half = a.r.dim / 2;
    uint32_t top = 0;
#pragma unroll
    for (int n = 0; n < D / 64; n++) {
        const int t = (lane + 64 * n) / (D / 16), u = (lane + 64 * n) % (D / 16);
        if (!tokens.of_call(t)) continue;
        const T *x = reinterpret_cast<const T *>(rows + t * strides[1]);
        float lo[8], hi[8];
        int at = 16 * u, beside = 16 * u + 8;
        if (u < turned && !a.r.interleaved) {
            at = 8 * u;
            beside = half + 8 * u;
        }
        load_n<8>(x + at, lo);
        load_n<8>(x + beside, hi);
        if (u < turned) {
            const float *cs = rotation_row(a.r, w.first + t);
            float c[16];
            if (cs) load_n<16>(cs + 16 * u, c);
#pragma unroll
            for (int e = 0; e < 8; e++) {
                if (!cs) lo[e] = hi[e] = __builtin_nanf("");
                else if (!a.r.interleaved) turn_pair(lo[e], hi[e], c[2 * e], c[2 * e + 1]);
            }
            if (cs && a.r.interleaved) {
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    turn_pair(lo[2 * e], lo[2 * e + 1], c[2 * e], c[2 * e + 1]);
                    turn_pair(hi[2 * e], hi[2 * e + 1], c[8 + 2 * e], c[8 + 2 * e + 1]);
                }
            }
        }
        float *to = tile + t * ROW;
#pragma unroll
        for (int e = 0; e < 8; e += 4) {
            st4(to + at + e, (floatx4){lo[e], lo[e + 1], lo[e + 2], lo[e + 3]});
            st4(to + beside + e, (floatx4){hi[e], hi[e + 1], hi[e + 2], hi[e + 3]});
        }
        if constexpr (I8)
#pragma unroll
            for (int e = 0; e < 8; e++)
                top = max(top, max(__float_as_uint(lo[e]) & 0x7fffffffu, __float_as_uint(hi[e]) & 0x7fffffffu));
    }
    cache_wave_order();
    Quant q{};
    if constexpr (I8) {
        top = wave_umax(top);
        float *held = scale_at(a.p, w.page, w.head, w.slot) + w.values;
        const float old = tokens.lo ? *held : 0.0f;
        float scale = fmaxf(__uint_as_float(top) * (1.0f / 127.0f), 0x1p-100f);
        if (tokens.lo && !(old <= scale)) scale = old;
        if (top >= 0x7f800000u) scale = __builtin_nanf("");
        q.inv = 1.0f / scale;
        q.earlier = old * q.inv;
        cache_wave_order();  // every lane has the old one
        if (lane == 0) *held = scale;
    }
    char *block = block_at(a.p, w.page, w.head, w.slot, B::BYTES) + w.values * B::PART + 16 * lane;
    const int i = lane & 15, g = lane >> 4;
#pragma unroll
    for (int u = 0; u < B::UNITS; u++) {
        u32x4 *place = reinterpret_cast<u32x4 *>(block + 1024 * u);
        u32x4 old = {0, 0, 0, 0}, now;
        if (tokens.lo) old = *place;
        // element e of the lane's 16 bytes: its token and its place in the tile
        const int d0 = w.values ? B::value_dim(u, i) : B::key_dim(u, g);
        float x[B::C];
        if (w.values) {
#pragma unroll
            for (int r = 0; r < 4; r++) {
                float v[B::C / 4];
                load_lds<B::C / 4>(tile + (4 * g + r) * ROW + d0, v);
#pragma unroll
                for (int e = 0; e < B::C / 4; e++) x[4 * e + r] = v[e];
            }
        } else {
            load_lds<B::C>(tile + i * ROW + d0, x);
        }
#pragma unroll
        for (int d = 0; d < 4; d++) {
            uint32_t word = 0;
            constexpr int N = I8 ? 4 : 2, BITS = 32 / N;
#pragma unroll
            for (int e = 0; e < N; e++) {
                const int at = N * d + e, t = w.values ? 4 * g + at % 4 : i;
                const uint32_t before = old[d] >> (BITS * e) & ((1ull << BITS) - 1);
                uint32_t value;
                if constexpr (I8)
                    value = tokens.of_call(t) ? q.of(x[at]) : tokens.earlier(t) ? q.again(before) : 128u;
                else
                    value = tokens.of_call(t) ? (uint32_t)__builtin_bit_cast(uint16_t, (bf16)x[at]) : tokens.earlier(t) ? before : 0u;
                word |= value << (BITS * e);
            }
            now[d] = word;
        }
        *place = now;
    }
}

// A block's rows, by way of the same tile.
template <typename T, int D, bool I8>
static __global__ __launch_bounds__(256) void cache_read_kernel(CacheRowsArgs a) {
    using B = BlockShape<D, I8>;
    constexpr int ROW = D + 4;
    __shared__ __align__(16) float tiles[4][PC_BLOCK * ROW];
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), lane = threadIdx.x & 63;
    CacheTask w;
    if (!w.take(a, wave)) return;
    char *out = w.values ? a.v : a.k;
    if (!out) return;
    float *tile = tiles[wave];
    const bool any = w.page >= 0 && w.first < w.start + w.rows;
    if (any) {
        const char *block = block_at(a.p, w.page, w.head, w.slot, B::BYTES) + w.values * B::PART + 16 * lane;
        const float scale = I8 ? scale_at(a.p, w.page, w.head, w.slot)[w.values] : 1.0f;
        const int i = lane & 15, g = lane >> 4;
#pragma unroll
        for (int u = 0; u < B::UNITS; u++) {
            const u32x4 from = *reinterpret_cast<const u32x4 *>(block + 1024 * u);
            float x[B::C];
#pragma unroll
            for (int e = 0; e < B::C; e++) {
                if constexpr (I8) x[e] = (float)((int)(from[e / 4] >> (8 * (e % 4)) & 0xff) - 128) * scale;
                else x[e] = __uint_as_float(from[e / 2] >> (16 * (e % 2)) << 16);
            }
            const int d0 = w.values ? B::value_dim(u, i) : B::key_dim(u, g);
            if (w.values) {
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    float v[B::C / 4];
#pragma unroll
                    for (int e = 0; e < B::C / 4; e++) v[e] = x[4 * e + r];
                    store_lds<B::C / 4>(tile + (4 * g + r) * ROW + d0, v);
                }
            } else {
                store_lds<B::C>(tile + i * ROW + d0, x);
            }
        }
    }
    cache_wave_order();
    const int64_t *strides = w.values ? a.vs : a.ks;
#pragma unroll
    for (int n = 0; n < D / 64; n++) {
        const int t = (lane + 64 * n) / (D / 16), u = (lane + 64 * n) % (D / 16);
        const int64_t row = w.first + t - w.start;
        if (row < 0 || row >= a.length) continue;
        float x[16];
#pragma unroll
        for (int e = 0; e < 16; e++) x[e] = 0.0f;
        if (any && row < w.rows) load_lds<16>(tile + t * ROW + 16 * u, x);
        store_n<16>(reinterpret_cast<T *>(out + w.s * strides[0] + row * strides[1] + w.head * strides[2]) + 16 * u, x);
    }
}

struct ReorderArgs {
    PagedArgs p;
    const int *parents, *lengths, *spare;
    int *table_out, *spare_out;
    int beams, block_bytes, scaled;
};

// A workgroup copies a head's blocks of a row's last page; head 0's writes the row of
// the table too.
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
    for (int i = threadIdx.x; i < n; i += 256) dst[i] = src[i];
    if (a.scaled)
        for (int i = threadIdx.x; i < 2 * blocks; i += 256) scale_at(a.p, target, head, 0)[i] = scale_at(a.p, source, head, 0)[i];
}

}  // namespace vh
