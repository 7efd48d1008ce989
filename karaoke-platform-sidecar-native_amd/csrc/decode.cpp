// Launchers of the rotary positions, the paged cache with the attention over it, and
// beam search (rotary.hpp, paged_cache.hpp, cache_attention.hpp, beam_search.hpp).
#include "runtime.hpp"

#include <float.h>
#include <math.h>

#include <algorithm>
#include <initializer_list>

#include "beam_search.hpp"
#include "cache_attention.hpp"
#include "paged_cache.hpp"
#include "rotary.hpp"

namespace vh {

constexpr int64_t MAX_GROUPS = UINT32_MAX / 256;  // workgroups of 256 threads in a launch
constexpr int MAX_LENGTH = 1 << 29;
constexpr int MAX_SEQUENCES = 1 << 20;
constexpr int64_t MAX_ROW = 1 << 26;  // bytes between a cache call's rows

static bool type_ok(const char *what, int type) {
    if (type == VH_TYPE_FP32 || type == VH_TYPE_BF16) return true;
    set_error("%s: unsupported type %d", what, type);
    return false;
}
static int64_t type_bytes(int type) { return type == VH_TYPE_BF16 ? 2 : 4; }

static bool groups_ok(const char *what, int64_t groups) {
    if (groups <= MAX_GROUPS) return true;
    set_error("%s: %lld workgroups", what, (long long)groups);
    return false;
}

static bool aligned16(const char *what, std::initializer_list<const void *> pointers) {
    for (const void *p : pointers)
        if ((uintptr_t)p & 15) {
            set_error("%s: a tensor or workspace is not 16-byte aligned", what);
            return false;
        }
    return true;
}

// Whether each of what is written begins where no other of these does.
static bool begins_apart(const char *what, std::initializer_list<const void *> written,
                         std::initializer_list<const void *> read) {
    for (const void *const *w = written.begin(); w != written.end(); w++)
        if (*w && (std::find(read.begin(), read.end(), *w) != read.end() || std::find(w + 1, written.end(), *w) != written.end())) {
            set_error("%s: an output or workspace is at the address of another tensor", what);
            return false;
        }
    return true;
}

// Strides of a tensor [sequences][rows][heads][width] in elements; multiple: of bytes.
static bool strides_ok(const char *what, const char *name, const int64_t *strides, int64_t seqs, int64_t rows, int64_t heads,
                       int width, int64_t size, int64_t multiple, bool written) {
    const int64_t counts[3] = {seqs, rows, heads};  // of one of them the stride counts for nothing
    for (int i = 0; i < 3; i++)
        if (counts[i] > 1 && (strides[i] < 0 || strides[i] * size % multiple || strides[i] > ((int64_t)1 << 46) ||
                              (i == 1 && multiple > 1 && strides[i] * size > MAX_ROW))) {
            set_error("%s: %s's strides %lld, %lld, %lld: none negative, whole multiples of %lld bytes, rows at most %lld apart",
                      what, name, (long long)strides[0], (long long)strides[1], (long long)strides[2], (long long)multiple,
                      (long long)MAX_ROW);
            return false;
        }
    if (written && !strides_apart(strides, seqs, rows, heads, width)) {
        set_error("%s: %s's strides %lld, %lld, %lld let rows overlap, and %s is written", what, name, (long long)strides[0],
                  (long long)strides[1], (long long)strides[2], name);
        return false;
    }
    return true;
}
static bool same_strides(const int64_t *a, const int64_t *b, int64_t seqs, int64_t rows, int64_t heads) {
    return (seqs <= 1 || a[0] == b[0]) && (rows <= 1 || a[1] == b[1]) && (heads <= 1 || a[2] == b[2]);
}
static void to_bytes(int64_t *to, const int64_t *strides, int64_t size) {
    for (int i = 0; i < 3; i++) to[i] = strides[i] * size;
}

// ----------------------------------------------------------- rotary positions
bool rotary_table(hipStream_t s, const vh_rotary_angles *a, int dim, int positions, float *table, KernelTimer *t) {
    const char *what = "vh_rotary_table";
    if (!a || !table || dim < 2 || dim > 256 || dim % 2 || positions < 1) {
        set_error("%s: null angles or table, dim %d (even, 2 to 256) or %d positions", what, dim, positions);
        return false;
    }
    if (!(a->base > 1.0) || !isfinite(a->base) || !(a->factor >= 1.0) || !isfinite(a->factor) || a->original < 0 ||
        !isfinite(a->magnitude) || (a->factor > 1.0 && a->original && !(a->low < a->high && isfinite(a->low) && isfinite(a->high)))) {
        set_error("%s: base %g over 1, factor %g from 1, original %d from 0, low %g under high %g, magnitude %g, all finite",
                  what, a->base, a->factor, a->original, a->low, a->high, a->magnitude);
        return false;
    }
    if ((uintptr_t)table & 15) {
        set_error("%s: the table is not 16-byte aligned", what);
        return false;
    }
    RotaryTableArgs k{table, dim / 2, positions, a->magnitude, {}};
    for (int i = 0; i < dim / 2; i++) {
        const double theta = pow(a->base, -2.0 * i / dim);
        double keep = a->factor > 1.0 ? 0.0 : 1.0;
        if (a->factor > 1.0 && a->original)
            keep = std::min(1.0, std::max(0.0, (a->original * theta / 6.283185307179586 - a->low) / (a->high - a->low)));
        k.theta[i] = theta * (keep + (1.0 - keep) / a->factor);
    }
    const int64_t groups = ((int64_t)positions * (dim / 2) + 255) / 256;
    if (!groups_ok(what, groups)) return false;
    Scope sc(t, s, "rotary_table");
    hipLaunchKernelGGL(rotary_table_kernel, dim3((unsigned)groups), dim3(256), 0, s, k);
    return sync_debug(s, "rotary_table_kernel");
}

// A rotation of heads, its dim a multiple of `multiple`; null: none.
static bool rotation_of(const char *what, const vh_rotary *r, int head_dim, int multiple, Rotation &to) {
    to = {};
    if (!r) return true;
    if (r->dim < 2 || r->dim > 256 || r->dim % multiple || r->dim > head_dim || r->positions < 1 || !r->table ||
        ((uintptr_t)r->table & 15)) {
        set_error("%s: a rotation of %d dims (a multiple of %d, up to 256 and a head's %d) over %d positions, or its table null "
                  "or not 16-byte aligned",
                  what, r->dim, multiple, head_dim, r->positions);
        return false;
    }
    to = {r->table, r->dim, r->interleaved ? 1 : 0, r->positions};
    return true;
}

template <typename T>
static void rotary_launch(hipStream_t s, const RotaryArgs &a, int64_t groups, bool backward) {
    if (a.r.interleaved) {
        if (backward) hipLaunchKernelGGL((rotary_kernel<T, true, true>), dim3((unsigned)groups), dim3(256), 0, s, a);
        else hipLaunchKernelGGL((rotary_kernel<T, true, false>), dim3((unsigned)groups), dim3(256), 0, s, a);
    } else {
        if (backward) hipLaunchKernelGGL((rotary_kernel<T, false, true>), dim3((unsigned)groups), dim3(256), 0, s, a);
        else hipLaunchKernelGGL((rotary_kernel<T, false, false>), dim3((unsigned)groups), dim3(256), 0, s, a);
    }
}

bool rotary_apply(hipStream_t s, const vh_rotary *r, const vh_rotary_rows *rows, const void *x, void *y, bool backward,
                  KernelTimer *t) {
    const char *what = "vh_rotary_apply";
    if (!r || !rows) {
        set_error("%s: null rotation or rows", what);
        return false;
    }
    if (!type_ok(what, rows->type)) return false;
    if (rows->sequences < 0 || rows->sequences > MAX_SEQUENCES || rows->length < 0 || rows->length > MAX_LENGTH || rows->heads < 1 ||
        rows->heads > 65536 || rows->head_dim < 2 || rows->head_dim > 1024) {
        set_error("%s: unsupported %d sequences, length %d, %d heads of %d", what, rows->sequences, rows->length, rows->heads,
                  rows->head_dim);
        return false;
    }
    RotaryArgs a{};
    if (!rotation_of(what, r, rows->head_dim, 2, a.r)) return false;
    const int64_t size = type_bytes(rows->type);
    if (!strides_ok(what, "x", rows->x_strides, rows->sequences, rows->length, rows->heads, rows->head_dim, size, 1, false) ||
        !strides_ok(what, "y", rows->y_strides, rows->sequences, rows->length, rows->heads, rows->head_dim, size, 1, true))
        return false;
    if (!rows->sequences || !rows->length) return true;
    if (!x || !y || ((uintptr_t)x | (uintptr_t)y) % size) {
        set_error("%s: x or y null, or not aligned to an element", what);
        return false;
    }
    if (x == y && !same_strides(rows->x_strides, rows->y_strides, rows->sequences, rows->length, rows->heads)) {
        set_error("%s: in place at other strides: rows would be written before they are read", what);
        return false;
    }
    if (!begins_apart(what, {y}, {r->table, rows->start})) return false;
    a.x = x;
    a.y = y;
    std::copy(rows->x_strides, rows->x_strides + 3, a.xs);
    std::copy(rows->y_strides, rows->y_strides + 3, a.ys);
    a.start = rows->start;
    a.length = rows->length;
    a.heads = rows->heads;
    a.head_dim = rows->head_dim;
    a.turned = (r->dim / 2 + 3) / 4;
    a.units = a.turned + (x == y ? 0 : (rows->head_dim - r->dim + 7) / 8);
    const int per_row = a.heads * a.units;
    a.per_row = divisor((uint32_t)per_row);
    a.per_head = divisor((uint32_t)a.units);
    // two units a thread: 6408 tokens there and back 13.7 us, four 15.1, one 14.0
    a.rows = std::max(1, std::min(rows->length, 512 / per_row));
    a.blocks = (rows->length + a.rows - 1) / a.rows;
    const int64_t groups = (int64_t)a.blocks * rows->sequences;
    if (!groups_ok(what, groups)) return false;
    Scope sc(t, s, "rotary");
    if (rows->type == VH_TYPE_BF16) rotary_launch<bf16>(s, a, groups, backward);
    else rotary_launch<float>(s, a, groups, backward);
    return sync_debug(s, "rotary_kernel");
}

// --------------------------------------------------------------- paged cache
static int64_t block_bytes(const vh_cache *c) { return 2ll * PC_BLOCK * c->head_dim * (c->type == VH_CACHE_INT8 ? 1 : 2); }
static int64_t page_scales(const vh_cache *c) { return (int64_t)c->kv_heads * (c->page_tokens / PC_BLOCK) * block_bytes(c); }
static int64_t page_bytes(const vh_cache *c) {
    const int64_t n = page_scales(c) + (c->type == VH_CACHE_INT8 ? (int64_t)c->kv_heads * (c->page_tokens / PC_BLOCK) * 8 : 0);
    return (n + 255) / 256 * 256;
}
static int64_t capacity(const vh_cache *c) { return (int64_t)c->table_pages * c->page_tokens; }

static bool cache_ok(const char *what, const vh_cache *c) {
    if (!c) {
        set_error("%s: null cache", what);
        return false;
    }
    if ((c->type != VH_CACHE_BF16 && c->type != VH_CACHE_INT8) || (c->head_dim != 64 && c->head_dim != 128) || c->kv_heads < 1 ||
        c->kv_heads > 4096 || c->page_tokens < PC_BLOCK || c->page_tokens > 4096 || c->page_tokens % PC_BLOCK || c->pages < 1) {
        set_error("%s: unsupported cache of type %d, %d heads of %d, %d pages of %d tokens", what, c->type, c->kv_heads, c->head_dim,
                  c->pages, c->page_tokens);
        return false;
    }
    if (c->sequences < 0 || c->sequences > MAX_SEQUENCES || c->table_pages < 0 || capacity(c) > MAX_LENGTH) {
        set_error("%s: unsupported table of %d sequences with %d pages of %d tokens", what, c->sequences, c->table_pages,
                  c->page_tokens);
        return false;
    }
    if (page_bytes(c) > INT32_MAX || (int64_t)c->pages > ((int64_t)1 << 46) / page_bytes(c)) {
        set_error("%s: %d pages of %lld bytes", what, c->pages, (long long)page_bytes(c));
        return false;
    }
    return true;
}

size_t cache_bytes(const vh_cache *c) { return cache_ok("vh_cache_bytes", c) ? (size_t)page_bytes(c) * c->pages : 0; }

// What a call with work needs of the cache.
static bool paged_args(const char *what, const vh_cache *c, PagedArgs &a) {
    if (!c->pool || ((uintptr_t)c->pool & 255) || (!c->table && c->table_pages)) {
        set_error("%s: the pool null or not 256-byte aligned, or the table null", what);
        return false;
    }
    a.pool = static_cast<char *>(c->pool);
    a.table = c->table;
    a.page_bytes = page_bytes(c);
    a.scales = page_scales(c);
    a.kv = c->kv_heads;
    a.pages = c->pages;
    a.table_pages = c->table_pages;
    a.page_blocks = c->page_tokens / PC_BLOCK;
    a.blocks = divisor((uint32_t)a.page_blocks);
    return true;
}

static bool cache_rows_ok(const char *what, const vh_cache *c, const vh_cache_rows *r, bool k, bool v, bool written) {
    if (!cache_ok(what, c)) return false;
    if (!r) {
        set_error("%s: null rows", what);
        return false;
    }
    if (!type_ok(what, r->type)) return false;
    if (r->length < 0 || r->length > MAX_LENGTH) {
        set_error("%s: unsupported length %d", what, r->length);
        return false;
    }
    const int64_t size = type_bytes(r->type);
    return (!k || strides_ok(what, "k", r->k_strides, c->sequences, r->length, c->kv_heads, c->head_dim, size, 16, written)) &&
           (!v || strides_ok(what, "v", r->v_strides, c->sequences, r->length, c->kv_heads, c->head_dim, size, 16, written));
}

static bool cache_rows_args(const char *what, const vh_cache *c, const vh_cache_rows *r, const void *k, const void *v,
                            CacheRowsArgs &a, int64_t &groups) {
    if (!paged_args(what, c, a.p) || !aligned16(what, {k, v})) return false;
    const int64_t size = type_bytes(r->type);
    a.k = const_cast<char *>(static_cast<const char *>(k));
    a.v = const_cast<char *>(static_cast<const char *>(v));
    to_bytes(a.ks, r->k_strides, size);
    to_bytes(a.vs, r->v_strides, size);
    a.start = r->start;
    a.lengths = r->lengths;
    a.length = r->length;
    // from the first block's last token on at worst
    const int64_t blocks = ((int64_t)r->length + (r->start ? 2 * PC_BLOCK - 2 : PC_BLOCK - 1)) / PC_BLOCK;
    const int64_t each = blocks * 2 * c->kv_heads, tasks = each * c->sequences;  // below 2^59
    groups = (tasks + 3) / 4;
    if (!groups_ok(what, groups)) return false;
    a.tasks = (int)tasks;
    a.per_sequence = divisor((uint32_t)each);
    a.per_block = divisor(2u * c->kv_heads);
    return true;
}

template <typename T, int D, bool I8>
static void rows_launch(hipStream_t s, const CacheRowsArgs &a, int64_t groups, bool append) {
    if (append) hipLaunchKernelGGL((cache_append_kernel<T, D, I8>), dim3((unsigned)groups), dim3(256), 0, s, a);
    else hipLaunchKernelGGL((cache_read_kernel<T, D, I8>), dim3((unsigned)groups), dim3(256), 0, s, a);
}
template <typename T>
static void rows_dispatch(hipStream_t s, const vh_cache *c, const CacheRowsArgs &a, int64_t groups, bool append) {
    const bool i8 = c->type == VH_CACHE_INT8;
    if (c->head_dim == 64) i8 ? rows_launch<T, 64, true>(s, a, groups, append) : rows_launch<T, 64, false>(s, a, groups, append);
    else i8 ? rows_launch<T, 128, true>(s, a, groups, append) : rows_launch<T, 128, false>(s, a, groups, append);
}

bool cache_append(hipStream_t s, const vh_cache *c, const vh_cache_rows *r, const vh_rotary *rotary, const void *k, const void *v,
                  KernelTimer *t) {
    const char *what = "vh_cache_append";
    if (!cache_rows_ok(what, c, r, true, true, false)) return false;
    CacheRowsArgs a{};
    if (!rotation_of(what, rotary, c->head_dim, 16, a.r)) return false;
    if (!c->sequences || !r->length) return true;
    if (!k || !v) {
        set_error("%s: null k or v", what);
        return false;
    }
    int64_t groups;
    if (!cache_rows_args(what, c, r, k, v, a, groups) ||
        !begins_apart(what, {c->pool}, {k, v, c->table, r->start, r->lengths, a.r.table}))
        return false;
    Scope sc(t, s, "cache_append");
    if (r->type == VH_TYPE_BF16) rows_dispatch<bf16>(s, c, a, groups, true);
    else rows_dispatch<float>(s, c, a, groups, true);
    return sync_debug(s, "cache_append_kernel");
}

bool cache_read(hipStream_t s, const vh_cache *c, const vh_cache_rows *r, void *k, void *v, KernelTimer *t) {
    const char *what = "vh_cache_read";
    if (!cache_rows_ok(what, c, r, k != nullptr, v != nullptr, true)) return false;
    if (!c->sequences || !r->length || (!k && !v)) return true;
    CacheRowsArgs a{};
    int64_t groups;
    if (!cache_rows_args(what, c, r, k, v, a, groups) || !begins_apart(what, {k, v}, {c->pool, c->table, r->start, r->lengths}))
        return false;
    Scope sc(t, s, "cache_read");
    if (r->type == VH_TYPE_BF16) rows_dispatch<bf16>(s, c, a, groups, false);
    else rows_dispatch<float>(s, c, a, groups, false);
    return sync_debug(s, "cache_read_kernel");
}

bool cache_reorder(hipStream_t s, const vh_cache *c, int beams, const int32_t *parents, const int32_t *lengths, const int32_t *spare,
                   int32_t *table_out, int32_t *spare_out, KernelTimer *t) {
    const char *what = "vh_cache_reorder";
    if (!cache_ok(what, c)) return false;
    if (beams < 1 || c->sequences % beams) {
        set_error("%s: %d sequences in groups of %d beams", what, c->sequences, beams);
        return false;
    }
    if (!c->sequences) return true;
    if (!parents || !lengths || !spare || !spare_out || (!table_out && c->table_pages)) {
        set_error("%s: null parents, lengths, spare, table_out or spare_out", what);
        return false;
    }
    ReorderArgs a{};
    if (!paged_args(what, c, a.p) || !begins_apart(what, {table_out, spare_out, c->pool}, {c->table, parents, lengths, spare}))
        return false;
    a.parents = parents;
    a.lengths = lengths;
    a.spare = spare;
    a.table_out = table_out;
    a.spare_out = spare_out;
    a.beams = beams;
    a.block_bytes = (int)block_bytes(c);
    a.scaled = c->type == VH_CACHE_INT8;
    const int64_t groups = (int64_t)c->sequences * c->kv_heads;
    if (!groups_ok(what, groups)) return false;
    Scope sc(t, s, "cache_reorder");
    hipLaunchKernelGGL(cache_reorder_kernel, dim3((unsigned)groups), dim3(256), 0, s, a);
    return sync_debug(s, "cache_reorder_kernel");
}

// ----------------------------------------------------------- cache attention
// How a call is cut into workgroups: with few rows four waves share them, each every
// fourth step of the keys, else each wave has its own; and into pieces of the keys.
// Measured over int8 pages, bf16 queries:
//   CQ_ROWS   rows of their own from 512 workgroups on: 4 x 512 causal tokens of 32 heads
//             on 8 of 128 over 4608 keys 159 us, from 1024 on 171 (bf16 pages 212 and 237); from
//             256 on, 4 x 517 of 16 heads on 4 of 64 over 4613 take 105 us instead of 63; always
//             shared, 16 x 2048 of 16 on 4 of 64 take 344 instead of 269
//   CQ_PIECES pieces until there are 512 workgroups: 16 single tokens of 32 heads on 8 of
//             64, uneven, up to 8192 keys 24.7 us; until 384, 768, 1024: 27.6, 25.7, 27.2
//   one piece from 256 workgroups on: 32 tokens of 32 heads on 8 of 128 over 16384 keys
//             162 us, in two pieces 168
//   a piece has 512 keys at least: one token of 32 heads on 8 of 128 over 8192 keys 15.8 us,
//             with 256 16.5
struct CacheCut {
    bool split, by_xcd;
    int groups, tiles;  // groups of 16 rows a wave has; workgroups of a (sequence, key head)
    int parts = 1, piece;
    int64_t pairs, grid;
};
constexpr int CQ_MAX_ROWS = 1 << 30;
constexpr int64_t CQ_ROWS = 512, CQ_PIECES = 512;
// Groups of 16 rows of a wave at most: what 256 registers hold.  The 4 x 517 tokens above
// 64 us with two, 75 with four (the registers spill); fp32 over 64 dims 39.5 with two, 43 with
// one; the 4 x 512 tokens over bf16 pages 211 with two, 258 with one.
constexpr int most_groups(int type, int head_dim) { return type == VH_TYPE_FP32 && head_dim == 128 ? 1 : 2; }
static CacheCut cache_cut(const vh_cache *c, const vh_cache_queries *q) {
    CacheCut cut;
    const int rows = q->length * (q->heads / c->kv_heads), most = most_groups(q->type, c->head_dim);
    cut.pairs = (int64_t)c->sequences * c->kv_heads;
    cut.split = rows <= 64 || cut.pairs * ((rows + 64 * most - 1) / (64 * most)) < CQ_ROWS;
    cut.groups = cut.split && rows <= 16 ? 1 : most;
    const int per = 16 * cut.groups * (cut.split ? 1 : 4);
    cut.tiles = (rows + per - 1) / per;
    const int64_t base = cut.pairs * cut.tiles;
    const int blocks = std::max<int>(1, (int)((std::min<int64_t>(q->most_keys, capacity(c)) + PC_BLOCK - 1) / PC_BLOCK));
    const int64_t want = base >= CQ_PIECES / 2 ? 1 : std::min<int64_t>(CQ_PIECES / std::max<int64_t>(base, 1), blocks / 32);
    const int parts = (int)std::max<int64_t>(1, std::min<int64_t>(want, 64));
    cut.piece = ((blocks + parts - 1) / parts + 4 * CQ_STEP - 1) / (4 * CQ_STEP) * (4 * CQ_STEP);  // whole steps of all waves
    cut.parts = (blocks + cut.piece - 1) / cut.piece;
    // (sequence, key head) pairs are dealt out to the XCDs where their rows' workgroups share
    // an L2's keys, and are many: of few, uneven ones the longest would be one XCD's
    cut.by_xcd = cut.pairs >= 64 && cut.tiles > 1;
    cut.grid = (cut.by_xcd ? (cut.pairs + 7) / 8 * 8 : cut.pairs) * cut.tiles * cut.parts;
    return cut;
}
static int64_t query_rows(const vh_cache *c, const vh_cache_queries *q) { return (int64_t)c->sequences * q->length * q->heads; }

static bool queries_ok(const char *what, const vh_cache *c, const vh_cache_queries *q) {
    if (!cache_ok(what, c)) return false;
    if (!q) {
        set_error("%s: null queries", what);
        return false;
    }
    if (!type_ok(what, q->type)) return false;
    if (q->heads < 1 || q->heads > 65536 || q->heads % c->kv_heads || q->length < 0 || q->length > MAX_LENGTH || q->most_keys < 0 ||
        q->most_keys > MAX_LENGTH || (int64_t)q->length * (q->heads / c->kv_heads) > CQ_MAX_ROWS) {
        set_error("%s: unsupported %d heads over %d, length %d over %d keys", what, q->heads, c->kv_heads, q->length, q->most_keys);
        return false;
    }
    if (!isfinite(q->scale)) {
        set_error("%s: the scale is no finite number", what);
        return false;
    }
    const int64_t size = type_bytes(q->type);
    if (!strides_ok(what, "q", q->q_strides, c->sequences, q->length, q->heads, c->head_dim, size, 16, false) ||
        !strides_ok(what, "out", q->out_strides, c->sequences, q->length, q->heads, c->head_dim, size, 16, true))
        return false;
    if (!query_rows(c, q)) return true;
    const CacheCut cut = cache_cut(c, q);
    return groups_ok(what, cut.grid) && groups_ok(what, (query_rows(c, q) + 15) / 16);
}
static size_t piece_bytes(const vh_cache *c, const vh_cache_queries *q, const CacheCut &cut) {
    return cut.parts > 1 ? (size_t)query_rows(c, q) * cut.parts * (c->head_dim * sizeof(float) + sizeof(float2)) : 0;
}
size_t cache_workspace_bytes(const vh_cache *c, const vh_cache_queries *q) {
    if (!queries_ok("vh_cache_workspace_bytes", c, q)) return 0;
    return std::max<size_t>(16, query_rows(c, q) ? piece_bytes(c, q, cache_cut(c, q)) : 0);
}

template <typename T, int D, bool I8>
static void attention_launch(hipStream_t s, const CacheAttentionArgs &a, const CacheCut &cut) {
    constexpr int MOST = most_groups(sizeof(T) == 2 ? VH_TYPE_BF16 : VH_TYPE_FP32, D);
    const dim3 grid((unsigned)cut.grid);
    if (!cut.split) hipLaunchKernelGGL((cache_attention_kernel<T, D, I8, MOST, false>), grid, dim3(256), 0, s, a);
    else if (cut.groups > 1) hipLaunchKernelGGL((cache_attention_kernel<T, D, I8, MOST, true>), grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((cache_attention_kernel<T, D, I8, 1, true>), grid, dim3(256), 0, s, a);
    if (cut.parts == 1) return;
    const int64_t rows = (int64_t)a.S * a.Lq * a.H;
    hipLaunchKernelGGL((cache_join_kernel<T, D>), dim3((unsigned)((rows + 15) / 16)), dim3(256), 0, s, a);
}
template <typename T>
static void attention_dispatch(hipStream_t s, const vh_cache *c, const CacheAttentionArgs &a, const CacheCut &cut) {
    const bool i8 = c->type == VH_CACHE_INT8;
    if (c->head_dim == 64) i8 ? attention_launch<T, 64, true>(s, a, cut) : attention_launch<T, 64, false>(s, a, cut);
    else i8 ? attention_launch<T, 128, true>(s, a, cut) : attention_launch<T, 128, false>(s, a, cut);
}

bool cache_attention(hipStream_t s, const vh_cache *c, const vh_cache_queries *q, const vh_rotary *rotary, const void *qp, void *out,
                     void *workspace, KernelTimer *t) {
    const char *what = "vh_cache_attention";
    if (!queries_ok(what, c, q)) return false;
    CacheAttentionArgs a{};
    if (!rotation_of(what, rotary, c->head_dim, 16, a.r)) return false;
    if (!query_rows(c, q)) return true;
    if (!qp || !out) {
        set_error("%s: null q or out", what);
        return false;
    }
    if (!paged_args(what, c, a.p) || !aligned16(what, {qp, out, workspace})) return false;
    const CacheCut cut = cache_cut(c, q);
    const size_t bytes = piece_bytes(c, q, cut);
    if (bytes && !workspace) {
        set_error("%s: null workspace (vh_cache_workspace_bytes)", what);
        return false;
    }
    const bool in_place = same_strides(q->q_strides, q->out_strides, c->sequences, q->length, q->heads);
    const void *ws = bytes ? workspace : nullptr;
    if (!begins_apart(what, {out, ws}, {c->pool, c->table, q->query_lengths, q->key_lengths, q->start, a.r.table}) ||
        !begins_apart(what, {ws, in_place ? nullptr : out}, {qp}))
        return false;
    const int64_t size = type_bytes(q->type);
    a.q = static_cast<const char *>(qp);
    a.out = static_cast<char *>(out);
    to_bytes(a.qs, q->q_strides, size);
    to_bytes(a.os, q->out_strides, size);
    a.query_lengths = q->query_lengths;
    a.key_lengths = q->key_lengths;
    a.start = q->start;
    a.S = c->sequences;
    a.H = q->heads;
    a.group = q->heads / c->kv_heads;
    a.heads = divisor((uint32_t)a.group);
    a.Lq = q->length;
    a.most = (int)std::min<int64_t>(q->most_keys, capacity(c));
    a.causal = q->causal ? 1 : 0;
    a.scale2 = std::min(std::max(fabsf(q->scale) * 1.4426950408889634f, 0x1p-126f), FLT_MAX);
    a.negative = q->scale < 0.0f;
    a.tiles = cut.tiles;
    a.by_xcd = cut.by_xcd;
    a.parts = cut.parts;
    a.piece = cut.piece;
    a.part_o = static_cast<float *>(workspace);
    a.part_ml = reinterpret_cast<float2 *>(a.part_o + (size_t)query_rows(c, q) * cut.parts * c->head_dim);
    Scope sc(t, s, "cache_attention");
    if (q->type == VH_TYPE_BF16) attention_dispatch<bf16>(s, c, a, cut);
    else attention_dispatch<float>(s, c, a, cut);
    return sync_debug(s, "cache_attention_kernel");
}

// --------------------------------------------------------------- beam search
// A stretch of a beam's logits, the vectors of 8 that a thread takes of it (of bf16 up
// to 8, of fp32 4: the same registers); shorter stretches while there are fewer than
// half as many workgroups as CUs.  32 x 8 beams over 120001 tokens, 16 picks: 28.6 us with
// 8 vectors, 31.2 with 4; 8 x 32 over 32003, 64 picks: 32 and 40; 16 rows of 32003: 12.1
// us, cut down to twice as many workgroups as CUs 12.8 (more lists to join).
struct BeamCut {
    int vectors, stretch, stretches, part_bytes;
};
constexpr int64_t BS_ENOUGH = 128;
static BeamCut beam_cut(const vh_beam *b) {
    constexpr int ONE = BS_THREADS * 8;
    const int64_t rows = std::max<int64_t>(1, (int64_t)b->sequences * b->beams);
    BeamCut cut;
    cut.vectors = b->type == VH_TYPE_BF16 ? 8 : 4;
    while (cut.vectors > 1 && b->vocab <= cut.vectors / 2 * ONE) cut.vectors /= 2;
    while (cut.vectors > 1 && rows * ((b->vocab + cut.vectors * ONE - 1) / (cut.vectors * ONE)) < BS_ENOUGH) cut.vectors /= 2;
    cut.stretches = (b->vocab + cut.vectors * ONE - 1) / (cut.vectors * ONE);
    cut.stretch = ((b->vocab + cut.stretches - 1) / cut.stretches + 7) / 8 * 8;
    cut.part_bytes = (int)(sizeof(BeamPart) + (b->picks + 1) / 2 * 2 * sizeof(BeamPick));
    return cut;
}
static bool beam_ok(const char *what, const vh_beam *b) {
    if (!b) {
        set_error("%s: null beam", what);
        return false;
    }
    if (!type_ok(what, b->type)) return false;
    if (b->sequences < 0 || b->sequences > MAX_SEQUENCES || b->beams < 1 || b->beams > BS_MAX_BEAMS || b->vocab < 1 ||
        b->vocab > 1 << 24 || b->picks < 1 || b->picks > BS_MAX_PICKS || b->picks > (int64_t)b->beams * b->vocab ||
        b->end_token < -1 || b->end_token >= b->vocab) {
        set_error("%s: unsupported %d sequences of %d beams (1 to %d) over %d tokens (1 to 2^24), %d picks (1 to %d), end token %d",
                  what, b->sequences, b->beams, BS_MAX_BEAMS, b->vocab, b->picks, BS_MAX_PICKS, b->end_token);
        return false;
    }
    const int64_t counts[2] = {b->sequences, b->beams};
    for (int i = 0; i < 2; i++)
        if (counts[i] > 1 && (b->strides[i] < 0 || b->strides[i] > ((int64_t)1 << 46))) {
            set_error("%s: the logits' strides %lld, %lld: none negative", what, (long long)b->strides[0], (long long)b->strides[1]);
            return false;
        }
    return groups_ok(what, (int64_t)b->sequences * b->beams * beam_cut(b).stretches);
}
static size_t beam_bytes(const vh_beam *b) {
    const BeamCut cut = beam_cut(b);
    return (size_t)b->sequences * b->beams * cut.stretches * cut.part_bytes;
}
size_t beam_workspace_bytes(const vh_beam *b) {
    return beam_ok("vh_beam_workspace_bytes", b) ? std::max<size_t>(16, beam_bytes(b)) : 0;
}

template <typename T>
static void beam_launch(hipStream_t s, const BeamArgs &a, int vectors, int64_t groups) {
    const dim3 grid((unsigned)groups), threads(BS_THREADS);
    if (vectors == 1) hipLaunchKernelGGL((beam_stretch_kernel<T, 1>), grid, threads, 0, s, a);
    else if (vectors == 2) hipLaunchKernelGGL((beam_stretch_kernel<T, 2>), grid, threads, 0, s, a);
    else if (vectors == 4 || sizeof(T) == 4) hipLaunchKernelGGL((beam_stretch_kernel<T, 4>), grid, threads, 0, s, a);
    else hipLaunchKernelGGL((beam_stretch_kernel<T, sizeof(T) == 4 ? 4 : 8>), grid, threads, 0, s, a);
}

bool beam_select(hipStream_t s, const vh_beam *b, const void *logits, const float *scores, const int32_t *ended, int32_t *tokens,
                 int32_t *parents, float *new_scores, int32_t *new_ended, void *workspace, KernelTimer *t) {
    const char *what = "vh_beam_select";
    if (!beam_ok(what, b)) return false;
    if (ended && b->end_token < 0) {
        set_error("%s: ended beams without an end token", what);
        return false;
    }
    if (!b->sequences) return true;
    if (!logits || !scores || !tokens || !parents || !new_scores || !workspace) {
        set_error("%s: null logits, scores, tokens, parents, new_scores or workspace", what);
        return false;
    }
    if ((uintptr_t)logits % type_bytes(b->type) || ((uintptr_t)workspace & 15)) {
        set_error("%s: the logits are not aligned to an element, or the workspace to 16 bytes", what);
        return false;
    }
    if (!begins_apart(what, {tokens, parents, new_scores, new_ended, workspace}, {logits, scores, ended})) return false;
    const BeamCut cut = beam_cut(b);
    BeamArgs a{};
    a.logits = logits;
    a.seq_stride = b->strides[0];
    a.beam_stride = b->strides[1];
    a.scores = scores;
    a.ended = ended;
    a.tokens = tokens;
    a.parents = parents;
    a.new_scores = new_scores;
    a.new_ended = new_ended;
    a.parts = static_cast<char *>(workspace);
    a.S = b->sequences;
    a.B = b->beams;
    a.V = b->vocab;
    a.picks = b->picks;
    a.end_token = b->end_token;
    a.stretches = cut.stretches;
    a.stretch = cut.stretch;
    a.part_bytes = cut.part_bytes;
    a.per_list = divisor((uint32_t)a.picks);
    a.per_beam = divisor((uint32_t)a.stretches);
    Scope sc(t, s, "beam_select");
    const int64_t groups = (int64_t)a.S * a.B * a.stretches;
    if (b->type == VH_TYPE_BF16) beam_launch<bf16>(s, a, cut.vectors, groups);
    else beam_launch<float>(s, a, cut.vectors, groups);
    if (!sync_debug(s, "beam_stretch_kernel")) return false;
    hipLaunchKernelGGL(beam_join_kernel, dim3((unsigned)a.S), dim3(BS_JOIN), 0, s, a);
    return sync_debug(s, "beam_join_kernel");
}

}  // namespace vh
