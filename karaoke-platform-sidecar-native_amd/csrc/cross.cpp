// Launchers of the layer norm and of the attention over another sequence's
// states (layernorm.hpp, cross_attention.hpp).
#include "runtime.hpp"

#include <float.h>
#include <math.h>

#include <algorithm>
#include <initializer_list>
#include <utility>

#include "cross_attention.hpp"
#include "layernorm.hpp"

namespace vh {

constexpr int64_t MAX_THREADS = UINT32_MAX;  // of a launch

// --------------------------------------------------------------- layer norm
constexpr int LN_MAX_DIM = 16384;
// A row's lanes.  Forward: 16 of a wave while 32 elements of bf16, 16 of fp32, a lane
// hold the row (four rows share a reduction; 49662 x 384 bf16 17 us against a wave's
// 19, 16000 x 256 5.5 against 7.7); backward, whose sums for the weights fill the
// registers, up to 128 columns (49662 x 384 bf16 61 us against 51).  A wave up to
// 2048 columns, 256 up to 8192 (2400 of them bf16 75 us against 1024 lanes' 91),
// then 1024; the next more where rows of these are too few to fill the chip (800 x
// 1500 bf16 16 us against 19).
static int layernorm_lanes(int type, int64_t rows, int dim, bool backward) {
    const bool few = rows < 4096;
    if (dim <= 16 || (dim <= (backward ? 128 : type == VH_TYPE_BF16 ? 512 : 256) && !few)) return 16;
    if (dim <= 512 || (dim <= 2048 && !few)) return 64;
    return dim <= 8192 ? 256 : 1024;
}
// Workgroups of the backward pass: each keeps its rows' weight gradients, so more
// of them are more sums to add up afterwards.
static int layernorm_parts(int64_t rows, int dim) {
    const int lanes = layernorm_lanes(VH_TYPE_FP32, rows, dim, true), per = lanes > 64 ? 1 : 512 / lanes;
    return (int)std::min<int64_t>((rows + per - 1) / per, 512);
}

static bool layernorm_ok(const char *what, int type, int64_t rows, int dim, std::initializer_list<int64_t> pitches) {
    if ((type != VH_TYPE_FP32 && type != VH_TYPE_BF16) || rows < 0 || rows > INT32_MAX || dim < 1 || dim > LN_MAX_DIM) {
        set_error("%s: unsupported type %d, rows %lld or dim %d (1 to %d)", what, type, (long long)rows, dim,
                  LN_MAX_DIM);
        return false;
    }
    for (int64_t ld : pitches)
        if (ld < dim) {
            set_error("%s: a row pitch of %lld is below dim %d", what, (long long)ld, dim);
            return false;
        }
    return true;
}

size_t layernorm_workspace_bytes(int64_t rows, int dim) {
    if (!layernorm_ok("vh_layernorm_workspace_bytes", VH_TYPE_FP32, rows, dim, {})) return 0;
    return std::max<size_t>(16, (size_t)layernorm_parts(rows, dim) * 2 * dim * sizeof(float));
}

template <typename T, int LANES, int N, int NV>
static void layernorm_launch(hipStream_t s, const NormArgs &a, bool backward, int parts) {
    using S = NormShape<LANES, N, NV>;
    if (backward) {
        hipLaunchKernelGGL((layernorm_backward_kernel<T, LANES, N, NV>), dim3((unsigned)parts), dim3(S::THREADS), 0, s, a);
        return;
    }
    constexpr int64_t MOST = MAX_THREADS / S::THREADS * S::ROWS;  // rows of a launch
    for (int64_t row = 0; row < a.rows; row += MOST) {
        NormArgs b = a;
        b.rows = std::min(MOST, a.rows - row);
        b.x = static_cast<const T *>(a.x) + row * a.ldx;
        b.y = static_cast<T *>(a.y) + row * a.ldy;
        if (a.stats) b.stats = a.stats + row;
        hipLaunchKernelGGL((layernorm_kernel<T, LANES, N, NV>), dim3((unsigned)((b.rows + S::ROWS - 1) / S::ROWS)),
                           dim3(S::THREADS), 0, s, b);
    }
}
// E: the lane's elements, in loads of 16 bytes.
template <typename T, int LANES, int E>
static void layernorm_elements(hipStream_t s, const NormArgs &a, bool backward, int parts) {
    constexpr int N = 16 / sizeof(T);
    layernorm_launch<T, LANES, N, E / N>(s, a, backward, parts);
}
template <typename T>
static void layernorm_dispatch(hipStream_t s, const NormArgs &a, bool backward, int parts) {
    const int type = sizeof(T) == 2 ? VH_TYPE_BF16 : VH_TYPE_FP32;
    const int d = a.dim, lanes = layernorm_lanes(type, a.rows, d, backward), e = (d + lanes - 1) / lanes;
    if (d < (int)(16 / sizeof(T))) layernorm_launch<T, 16, 1, 1>(s, a, backward, parts);
    else if (lanes == 16) {
        if (e <= 8) layernorm_elements<T, 16, 8>(s, a, backward, parts);
        else if (e <= 16) layernorm_elements<T, 16, 16>(s, a, backward, parts);
        else if (e <= 24) layernorm_elements<T, 16, 24>(s, a, backward, parts);
        else layernorm_elements<T, 16, 32>(s, a, backward, parts);
    } else if (lanes == 64) {
        if (e <= 8) layernorm_elements<T, 64, 8>(s, a, backward, parts);
        else if (e <= 16) layernorm_elements<T, 64, 16>(s, a, backward, parts);
        else if (e <= 24) layernorm_elements<T, 64, 24>(s, a, backward, parts);
        else layernorm_elements<T, 64, 32>(s, a, backward, parts);
    } else if (lanes == 256) {
        if (e <= 8) layernorm_elements<T, 256, 8>(s, a, backward, parts);
        else if (e <= 16) layernorm_elements<T, 256, 16>(s, a, backward, parts);
        else layernorm_elements<T, 256, 32>(s, a, backward, parts);
    } else {
        layernorm_elements<T, 1024, 16>(s, a, backward, parts);
    }
}

// In place: row for row.
static bool in_place_ok(const char *what, int64_t rows, const void *to, int64_t ld, const void *from, int64_t ldf) {
    if (to != from || ld == ldf || rows <= 1) return true;
    set_error("%s: in place at pitches of %lld and %lld: rows would be written before they are read", what, (long long)ld,
              (long long)ldf);
    return false;
}

bool layernorm(hipStream_t s, const LayerNorm &n, KernelTimer *t) {
    if (!layernorm_ok("vh_layernorm", n.type, n.rows, n.dim, {n.ldx, n.ldy})) return false;
    if (!(n.eps >= 0.0f) || isinf(n.eps) || !n.gamma || (n.rows && (!n.x || !n.y))) {
        set_error("vh_layernorm: null x, gamma or y, or an eps that is no number from 0 up");
        return false;
    }
    if (!in_place_ok("vh_layernorm", n.rows, n.y, n.ldy, n.x, n.ldx)) return false;
    if (!n.rows) return true;
    NormArgs a{};
    a.x = n.x; a.y = n.y; a.ldx = n.ldx; a.ldy = n.ldy;
    a.gamma = n.gamma; a.beta = n.beta;
    a.stats = reinterpret_cast<float2 *>(n.stats);
    a.rows = n.rows; a.dim = n.dim; a.eps = n.eps;
    Scope sc(t, s, "layernorm");
    if (n.type == VH_TYPE_BF16) layernorm_dispatch<bf16>(s, a, false, 0);
    else layernorm_dispatch<float>(s, a, false, 0);
    return sync_debug(s, "layernorm_kernel");
}

bool layernorm_backward(hipStream_t s, const LayerNorm &n, KernelTimer *t) {
    if (!layernorm_ok("vh_layernorm_backward", n.type, n.rows, n.dim, {n.ldx, n.ldy, n.lddx})) return false;
    if (!n.gamma || (n.rows && (!n.x || !n.dy || !n.dx || !n.stats))) {
        set_error("vh_layernorm_backward: null dy, x, gamma, stats or dx");
        return false;
    }
    if (!in_place_ok("vh_layernorm_backward", n.rows, n.dx, n.lddx, n.x, n.ldx) ||
        !in_place_ok("vh_layernorm_backward", n.rows, n.dx, n.lddx, n.dy, n.ldy))
        return false;
    const bool weights = n.dgamma || n.dbeta;
    if (weights && (!n.workspace || ((uintptr_t)n.workspace & 15))) {
        set_error("vh_layernorm_backward: the weights' gradients need a 16-byte aligned workspace "
                  "(vh_layernorm_workspace_bytes)");
        return false;
    }
    const int parts = layernorm_parts(n.rows, n.dim);
    Scope sc(t, s, "layernorm_backward");
    if (n.rows) {
        NormArgs a{};
        a.x = n.x; a.dy = n.dy; a.dx = n.dx; a.ldx = n.ldx; a.lddy = n.ldy; a.lddx = n.lddx;
        a.gamma = n.gamma;
        a.stats = reinterpret_cast<float2 *>(n.stats);
        a.part = weights ? static_cast<float *>(n.workspace) : nullptr;
        a.rows = n.rows; a.dim = n.dim;
        if (n.type == VH_TYPE_BF16) layernorm_dispatch<bf16>(s, a, true, parts);
        else layernorm_dispatch<float>(s, a, true, parts);
        if (!sync_debug(s, "layernorm_backward_kernel")) return false;
    }
    if (!weights) return true;
    hipLaunchKernelGGL(layernorm_columns_kernel, dim3((unsigned)(2 * n.dim + 15) / 16), dim3(1024), 0, s,
                       static_cast<const float *>(n.workspace), parts, n.dim, n.dgamma, n.dbeta);
    return sync_debug(s, "layernorm_columns_kernel");
}

// ---------------------------------------------------------- cross attention
// Distances from which the far buckets of a side begin.  Bucket near + i is
// reached at the first whole n with n^far >= max_distance^i near^(far - i), far
// = side - near: the next whole number from near (max_distance / near)^(i / far) on,
// which is taken as whole where it is within a double's roundings.
static int bucket_edges(int side, int near, int max_distance, int *edge) {
    const int far = side - near;
    const double step = log((double)max_distance / near) / far;
    for (int i = 0; i < far; i++) edge[i] = (int)ceil(near * exp(step * i) * (1.0 - 1e-12));
    return far;
}

static bool bias_ok(const char *what, int buckets, int max_distance, int bidirectional) {
    const int side = bidirectional ? buckets / 2 : buckets;
    if (buckets < 2 || buckets > CA_MAX_BUCKETS || (bidirectional && buckets % 2) || side < 2 || max_distance > 4096 ||
        max_distance <= side / 2) {
        set_error("%s: %d buckets (2 to %d, bidirectional: even and from 4) up to a distance of %d (more than the %d "
                  "buckets of single distances, at most 4096)",
                  what, buckets, CA_MAX_BUCKETS, max_distance, side / 2);
        return false;
    }
    return true;
}

static void bias_args(CrossArgs &a, int buckets, int max_distance, int bidirectional) {
    a.buckets = buckets;
    a.max_distance = max_distance;
    a.bidirectional = bidirectional ? 1 : 0;
    a.side = bidirectional ? buckets / 2 : buckets;
    a.near = a.side / 2;
    a.edges = bucket_edges(a.side, a.near, max_distance, a.edge);
    a.per_octave = (float)a.edges / log2f((float)max_distance / (float)a.near);
}

int relative_bucket(int rel, int buckets, int max_distance, int bidirectional) {
    if (!bias_ok("vh_relative_bucket", buckets, max_distance, bidirectional)) return -1;
    CrossArgs a{};
    bias_args(a, buckets, max_distance, bidirectional);
    return cross_bucket(a, std::max(rel, -INT32_MAX));
}

// Whether different (sequence, row, head) have different places: each stride, in
// ascending order, at least what the smaller ones span.
static bool apart(const int64_t *strides, int64_t seqs, int64_t rows, int64_t heads) {
    std::pair<int64_t, int64_t> d[3] = {{strides[0], seqs}, {strides[1], rows}, {strides[2], heads}};
    std::sort(d, d + 3);
    int64_t span = CA_D, stretch;
    for (const auto &[stride, n] : d) {
        if (n <= 1) continue;
        if (stride < span) return false;
        if (__builtin_mul_overflow(stride, n - 1, &stretch) || __builtin_add_overflow(span, stretch, &span)) span = INT64_MAX;
    }
    return true;
}

constexpr int64_t CA_MAX_ROW = 1 << 26;      // bytes of a row stride: 32 rows' offsets fit 32 bits
constexpr int CA_MAX_LENGTH = 1 << 29;

static bool cross_ok(const char *what, const vh_cross *c, bool backward) {
    if (!c) {
        set_error("%s: null layout", what);
        return false;
    }
    if ((c->type != VH_TYPE_FP32 && c->type != VH_TYPE_BF16) || c->sequences < 0 || c->heads < 1 || c->kv_heads < 1 ||
        c->heads > 65536 || c->heads % c->kv_heads || c->query_length < 0 || c->key_length < 0 || c->query_length > CA_MAX_LENGTH ||
        c->key_length > CA_MAX_LENGTH) {
        set_error("%s: unsupported type %d, %d sequences, %d heads over %d, lengths %d and %d", what, c->type,
                  c->sequences, c->heads, c->kv_heads, c->query_length, c->key_length);
        return false;
    }
    if (!isfinite(c->scale)) {
        set_error("%s: the scale is no finite number", what);
        return false;
    }
    if (c->bias_table && !bias_ok(what, c->buckets, c->max_distance, c->bidirectional)) return false;
    const int64_t size = c->type == VH_TYPE_BF16 ? 2 : 4;
    struct {
        const char *name;
        const int64_t *strides;
        int64_t rows, heads;
        bool written;
    } tensors[] = {{"q", c->q_strides, c->query_length, c->heads, backward},
                   {"k", c->k_strides, c->key_length, c->kv_heads, backward},
                   {"v", c->v_strides, c->key_length, c->kv_heads, backward},
                   {"out", c->out_strides, c->query_length, c->heads, true}};
    for (const auto &t : tensors) {
        const int64_t counts[3] = {c->sequences, t.rows, t.heads};  // of one of them the stride counts for nothing
        for (int i = 0; i < 3; i++)
            if (counts[i] > 1 && (t.strides[i] < 0 || t.strides[i] * size % 16 || t.strides[i] > ((int64_t)1 << 46))) {
                set_error("%s: %s's strides %lld, %lld, %lld: none negative, whole multiples of 16 bytes", what, t.name,
                          (long long)t.strides[0], (long long)t.strides[1], (long long)t.strides[2]);
                return false;
            }
        if (t.rows > 1 && t.strides[1] * size > CA_MAX_ROW) {
            set_error("%s: %s's row stride of %lld is over %lld bytes", what, t.name, (long long)t.strides[1],
                      (long long)CA_MAX_ROW);
            return false;
        }
        if (t.written && !apart(t.strides, c->sequences, t.rows, t.heads)) {
            set_error("%s: %s's strides %lld, %lld, %lld let rows overlap, and %s is written", what, t.name,
                      (long long)t.strides[0], (long long)t.strides[1], (long long)t.strides[2],
                      t.name[0] == 'o' ? "out" : "its gradient");
            return false;
        }
    }
    constexpr int64_t MOST = INT32_MAX / 8;
    const int64_t pairs = (int64_t)c->sequences * c->heads;  // below 2^47
    const int64_t tasks = std::min(pairs, MOST + 1) * ((std::max(c->query_length, c->key_length) + 127) / 128 + 1);
    if (tasks > MOST) {
        set_error("%s: %lld workgroups", what, (long long)tasks);
        return false;
    }
    return true;
}

static int64_t cross_rows(const vh_cross *c) { return (int64_t)c->sequences * c->heads * c->query_length; }
static size_t round16(size_t n) { return (n + 15) / 16 * 16; }

size_t cross_saved_bytes(const vh_cross *c) {
    if (!cross_ok("vh_cross_saved_bytes", c, false)) return 0;
    const size_t rows = (size_t)cross_rows(c);
    const size_t rest = c->type == VH_TYPE_BF16 ? (c->bias_table ? sizeof(float) : sizeof(bf16)) * CA_D : 0;
    return std::max<size_t>(16, round16(rows * sizeof(float2)) + rows * rest);
}

constexpr size_t CA_LDS = 160 * 1024;  // of a workgroup
static size_t window_bytes(const vh_cross *c) {
    return c->bias_table ? (size_t)(2 * (c->max_distance + CA_PAD) + 1) * sizeof(float) : 0;
}
// split: the kernels whose four waves share 32 rows; else those of 128 rows in one
// group of waves, or 64 in two.
template <typename T>
static size_t tiles_bytes(bool split, int groups, bool forward) {
    if (!split) return groups == 2 ? SharedLds<T, 2>::BYTES : SharedLds<T, 1>::BYTES;
    return forward && sizeof(T) == 4 ? SplitLds<T, true>::BYTES : SplitLds<T>::BYTES;
}
static size_t tiles_lds(const vh_cross *c, bool split, int groups, bool forward) {
    return c->type == VH_TYPE_BF16 ? tiles_bytes<bf16>(split, groups, forward) : tiles_bytes<float>(split, groups, forward);
}
static size_t dq_lds(const vh_cross *c, bool split) {
    if (!c->bias_table) return tiles_lds(c, split, 1, false);
    return tiles_lds(c, split, 1, false) + window_bytes(c) + sizeof(DbiasLds) + 128 * sizeof(float) * c->buckets + window_bytes(c) / sizeof(float);
}
// heads: that a workgroup takes, one after the other
static size_t dkv_lds(const vh_cross *c, bool split, int heads) {
    return tiles_lds(c, split, 1, false) + (split ? 4 * sizeof(RowStats) + heads * window_bytes(c)
                                                  : 2 * (sizeof(RowStats) + window_bytes(c)));
}
static size_t pack_lds(const vh_cross *c) {
    return tiles_lds(c, true, 1, true) +
           (c->bias_table ? sizeof(float) * c->buckets * (c->heads / c->kv_heads) + window_bytes(c) / sizeof(float) : 0);
}

// How a call is cut into workgroups.  split: the kernels whose four waves share 32
// rows, in `parts` pieces; else those of 128 rows.
struct CrossCut {
    bool split = false, pack = false;
    int parts = 1, heads = 1, waves = 1;  // heads: that a workgroup of dk and dv takes, waves: groups of them in a workgroup
    int64_t pairs = 0, tiles = 0;  // (sequence, head) pairs, and workgroups of each
    int64_t groups() const { return pairs * tiles; }
    int64_t grid() const { return (pairs_by_xcd(pairs) ? (pairs + 7) / 8 * 8 : pairs) * tiles; }
};
// From 1.5 128-row workgroups per CU on, their sharing of tiles wins over even work.
// Both sides in turn, shared against split (8 heads each): forward of 8 x 801 rows over
// 1723 keys, 448 of them, 46 us against 55, fp32 181 against 195; a training step of 6 x
// 1000 over 1000, 384 of them, 103 against 110, but fp32 440 against 419.  At 256 of
// them, 4 x 1000 over 1000, a step in fp32 298 against 283, but bf16 74 against 81, and
// the forward alone, whose 64-row workgroups double their number, 21 against 26 (fp32 71
// against 86): one border for all passes and types costs a fifth there.  The forward's
// are of 64 rows in two groups up to four 128-row ones per CU: 33 us against 36 for 8 x
// 801 ragged rows, even 46 both, 672 of them 58 against 57; backward no gain.  Below, pieces
// of at least 8 tiles (two a wave) until there are about two workgroups per CU (a step
// of 4 x 8 x 801 rows over 389 keys in fp32, 416 workgroups of dk and dv: in one piece
// 124 us, in two 137); for single tokens of 32 tiles until there are four (16 x 32 of
// them over 8192 keys 37.6 us against 37.3 until there are two; many rows so cut, 2 x
// 3841 over 3278, 24.7 against 23.2).
constexpr int64_t CA_ENOUGH = 384, CA_PAIRED = 1024, CA_PIECES = 512, CA_ONE = 256;
static int pieces(int64_t groups, int across, bool few) {
    const int64_t tiles = (across + 31) / 32;
    if (groups <= 0) return 1;
    int64_t n = std::min(CA_PIECES / groups, tiles / 8);
    if (few) n = std::max(n, std::min(2 * CA_PIECES / groups, tiles / 32));
    return (int)std::max<int64_t>(1, std::min<int64_t>(n, 64));
}
static CrossCut cross_cut(int64_t pairs, int rows, int pack, int across, bool fits) {
    CrossCut cut;
    cut.pairs = pairs;
    cut.tiles = (rows + 127) / 128;
    if ((cut.groups() >= CA_ENOUGH && rows >= 64) || !fits) return cut;
    cut.split = true;
    cut.pack = pack > 1 && rows < 32;
    if (cut.pack) cut.pairs /= pack;
    cut.tiles = ((int64_t)rows * (cut.pack ? pack : 1) + 31) / 32;
    cut.parts = pieces(cut.groups(), across, rows < 32);
    cut.tiles *= cut.parts;
    return cut;
}
static CrossCut forward_cut(const vh_cross *c, bool keep) {
    const int shared = c->heads / c->kv_heads;
    const bool pack = !keep && (!c->bias_table || pack_lds(c) <= CA_LDS);
    CrossCut cut = cross_cut((int64_t)c->sequences * c->heads, c->query_length, pack ? shared : 1, c->key_length, true);
    if (!cut.split && cut.groups() < CA_PAIRED) {
        cut.waves = 2;
        cut.tiles = (c->query_length + 63) / 64;
    }
    return cut;
}
static CrossCut dq_cut(const vh_cross *c) {
    return cross_cut((int64_t)c->sequences * c->heads, c->query_length, 1, c->key_length, dq_lds(c, true) <= CA_LDS);
}
static CrossCut dkv_cut(const vh_cross *c) {
    CrossCut cut = cross_cut((int64_t)c->sequences * c->kv_heads, c->key_length, 1, c->query_length, true);
    if (!cut.split) return cut;
    // a workgroup takes all heads that share its keys, where their bias windows leave
    // room for two workgroups on a CU (a step with four windows of 800 positions 140 us
    // against 142); else, or where that makes less than one workgroup per CU, the heads
    // are pairs of their own and their sums pieces (56 workgroups: a step 38 us, together
    // 40; 320: together 82 against 88, with a bias 125 against 129, but fp32 276 against
    // 263)
    const int shared = c->heads / c->kv_heads;
    cut.tiles = (c->key_length + 31) / 32;
    cut.heads = shared;
    if (cut.groups() < CA_ONE || dkv_lds(c, true, shared) > CA_LDS / 2 || (int64_t)shared * c->query_length > CA_MAX_LENGTH) {
        cut.pairs *= shared;
        cut.heads = 1;
    }
    cut.parts = pieces(cut.groups(), c->query_length, false);
    cut.tiles *= cut.parts;
    return cut;
}

// The workspace's sections, in bytes from its start.
struct CrossWork {
    CrossCut rows, keys;  // backward: of dq, of dk and dv
    size_t stats = 0, part_o = 0, part_ml = 0, part_dk = 0, part_dv = 0, dbias = 0, dbias_rows = 0, bytes = 0;
    int dbias_parts = 0;
    size_t take(size_t n) {
        const size_t at = bytes;
        bytes += round16(n);
        return at;
    }
};
static CrossWork forward_work(const vh_cross *c, bool keep) {
    CrossWork w;
    w.rows = forward_cut(c, keep);
    if (w.rows.split && w.rows.parts > 1) {
        const size_t rows = (size_t)cross_rows(c) * w.rows.parts;
        w.part_o = w.take(rows * CA_D * sizeof(float));
        w.part_ml = w.take(rows * sizeof(float2));
    }
    return w;
}
static int kv_pieces(const vh_cross *c, const CrossCut &cut) { return cut.split ? c->heads / c->kv_heads / cut.heads * cut.parts : 1; }
static CrossWork backward_work(const vh_cross *c) {
    CrossWork w;
    w.rows = dq_cut(c);
    w.keys = dkv_cut(c);
    w.stats = w.take((size_t)c->sequences * c->heads * ((c->query_length + 31) / 32) * sizeof(RowStats));
    if (w.rows.split && w.rows.parts > 1) w.part_o = w.take((size_t)cross_rows(c) * w.rows.parts * CA_D * sizeof(float));
    const int pieces = kv_pieces(c, w.keys);
    if (pieces > 1) {
        const size_t n = (size_t)pieces * c->sequences * c->kv_heads * c->key_length * CA_D * sizeof(float);
        w.part_dk = w.take(n);
        w.part_dv = w.take(n);
    }
    if (c->bias_table) {
        w.dbias_parts = (int)(w.rows.groups() / c->heads);
        w.dbias = w.take((size_t)w.rows.groups() * c->buckets * sizeof(float));
        if (w.rows.parts > 1) w.dbias_rows = w.take((size_t)w.rows.groups() * CA_TILE * sizeof(floatx4));
    }
    return w;
}

// Workgroups of the joining kernels: 16 rows each.
static int64_t join_groups(int64_t rows) { return (rows + 15) / 16; }
static int64_t key_rows(const vh_cross *c) { return (int64_t)c->sequences * c->kv_heads * c->key_length; }

// Whether a call's launches are within the device's.
static bool launches_ok(const char *what, const vh_cross *c, const CrossWork &w, bool backward) {
    int64_t most = std::max(w.rows.grid(), w.rows.parts > 1 ? join_groups(cross_rows(c)) : 0);
    if (backward) {
        most = std::max(most, w.keys.grid());
        most = std::max(most, (w.rows.parts > 1 ? join_groups(cross_rows(c)) : 0) +
                                  (kv_pieces(c, w.keys) > 1 ? 2 * join_groups(key_rows(c)) : 0) + c->heads);
    }
    if (most <= MAX_THREADS / 256) return true;
    set_error("%s: %lld workgroups", what, (long long)most);
    return false;
}

size_t cross_workspace_bytes(const vh_cross *c, bool backward) {
    const char *what = "vh_cross_workspace_bytes";
    if (!cross_ok(what, c, backward)) return 0;
    if (backward) {
        const CrossWork w = backward_work(c);
        return launches_ok(what, c, w, true) ? std::max<size_t>(16, w.bytes) : 0;
    }
    const CrossWork w = forward_work(c, false), keep = forward_work(c, true);
    return launches_ok(what, c, w, false) && launches_ok(what, c, keep, false) ? std::max<size_t>({16, w.bytes, keep.bytes}) : 0;
}

static CrossTensor cross_tensor(const void *p, const int64_t *strides, int64_t size) {
    return {const_cast<char *>(static_cast<const char *>(p)), strides[0] * size, strides[1] * size, strides[2] * size};
}

static CrossArgs cross_args(const vh_cross *c, const CrossBuffers &b) {
    CrossArgs a{};
    const int64_t size = c->type == VH_TYPE_BF16 ? 2 : 4;
    a.q = cross_tensor(b.q, c->q_strides, size);
    a.k = cross_tensor(b.k, c->k_strides, size);
    a.v = cross_tensor(b.v, c->v_strides, size);
    a.out = cross_tensor(b.out, c->out_strides, size);
    a.dout = cross_tensor(b.dout, c->out_strides, size);
    a.dq = cross_tensor(b.dq, c->q_strides, size);
    a.dk = cross_tensor(b.dk, c->k_strides, size);
    a.dv = cross_tensor(b.dv, c->v_strides, size);
    a.S = c->sequences; a.H = c->heads; a.KV = c->kv_heads;
    a.Lq = c->query_length; a.Lk = c->key_length;
    a.causal = c->causal ? 1 : 0;
    a.scale = c->scale;
    a.scale2 = std::max(fabsf(c->scale) * 1.4426950408889634f, FLT_MIN);  // 0 times a hidden score is no number
    a.query_lengths = c->query_lengths; a.key_lengths = c->key_lengths; a.query_start = c->query_start;
    a.table = c->bias_table;
    if (a.table) bias_args(a, c->buckets, c->max_distance, c->bidirectional);
    a.stats = static_cast<float2 *>(b.saved);
    if (b.saved && c->type == VH_TYPE_BF16) a.rest = static_cast<char *>(b.saved) + round16((size_t)cross_rows(c) * sizeof(float2));
    return a;
}

static bool aligned(const char *what, std::initializer_list<const void *> pointers) {
    for (const void *p : pointers)
        if ((uintptr_t)p & 15) {
            set_error("%s: a tensor, saved or workspace is not 16-byte aligned", what);
            return false;
        }
    return true;
}

// Whether each of what is written begins where none of the others and none of what
// is still read does.
static bool written_apart(const char *what, std::initializer_list<const void *> written,
                          std::initializer_list<const void *> read) {
    for (const void *const *w = written.begin(); w != written.end(); w++)
        if (*w && (std::find(read.begin(), read.end(), *w) != read.end() || std::find(w + 1, written.end(), *w) != written.end())) {
            set_error("%s: an output, saved or workspace is at the address of another tensor", what);
            return false;
        }
    return true;
}
static bool same_layout(const int64_t *a, const int64_t *b, int64_t seqs, int64_t rows, int64_t heads) {
    return (seqs <= 1 || a[0] == b[0]) && (rows <= 1 || a[1] == b[1]) && (heads <= 1 || a[2] == b[2]);
}

template <typename F>
static void launch(F kernel, int64_t groups, size_t lds, hipStream_t s, const CrossArgs &a) {
    hipLaunchKernelGGL(kernel, dim3((unsigned)groups), dim3(256), lds, s, a);
}

template <typename T, bool BIAS, int KW>
static void forward_shared(hipStream_t s, const CrossArgs &a, int64_t grid, size_t lds) {
    if (a.stats) launch(cross_forward_kernel<T, BIAS, true, KW>, grid, lds, s, a);
    else launch(cross_forward_kernel<T, BIAS, false, KW>, grid, lds, s, a);
}
template <typename T, bool BIAS>
static void forward_launch(hipStream_t s, const vh_cross *c, const CrossArgs &a, const CrossCut &cut) {
    const bool keep = a.stats != nullptr;
    const size_t lds = tiles_lds(c, cut.split, cut.waves, true) + window_bytes(c);
    if (!cut.split) {
        if (cut.waves == 2) forward_shared<T, BIAS, 2>(s, a, cut.grid(), lds);
        else forward_shared<T, BIAS, 1>(s, a, cut.grid(), lds);
        return;
    }
    if (cut.pack) {
        launch(cross_forward_split_kernel<T, BIAS, false, true>, cut.grid(), pack_lds(c), s, a);
    } else if (keep) {
        launch(cross_forward_split_kernel<T, BIAS, true, false>, cut.grid(), lds, s, a);
    } else {
        launch(cross_forward_split_kernel<T, BIAS, false, false>, cut.grid(), lds, s, a);
    }
    if (cut.parts == 1) return;
    const int64_t groups = (cross_rows(c) + 15) / 16;
    if (keep) launch(cross_join_kernel<T, BIAS, true>, groups, 0, s, a);
    else launch(cross_join_kernel<T, BIAS, false>, groups, 0, s, a);
}

bool cross_attention(hipStream_t s, const vh_cross *c, const CrossBuffers &b, KernelTimer *t) {
    const char *what = "vh_cross_attention";
    if (!cross_ok(what, c, false)) return false;
    if (cross_rows(c) == 0) return true;
    if (!b.q || !b.out || (c->key_length && (!b.k || !b.v))) {
        set_error("%s: null q, k, v or out", what);
        return false;
    }
    if (!aligned(what, {b.q, b.k, b.v, b.out, b.saved, b.workspace})) return false;
    CrossArgs a = cross_args(c, b);
    const CrossWork w = forward_work(c, a.stats != nullptr);
    if (!launches_ok(what, c, w, false)) return false;
    if (w.bytes && !b.workspace) {
        set_error("%s: null workspace (vh_cross_workspace_bytes)", what);
        return false;
    }
    // a row of q is read by the workgroups that write its out, before they do
    const bool as_q = same_layout(c->out_strides, c->q_strides, c->sequences, c->query_length, c->heads);
    const void *ws = w.bytes ? b.workspace : nullptr, *k = c->key_length ? b.k : nullptr, *v = c->key_length ? b.v : nullptr;
    if (!written_apart(what, {b.out, b.saved, ws}, {k, v, c->bias_table}) ||
        !written_apart(what, {b.saved, ws, as_q ? nullptr : b.out}, {b.q}))
        return false;
    a.parts = w.rows.parts;
    a.part_o = reinterpret_cast<float *>(static_cast<char *>(b.workspace) + w.part_o);
    a.part_ml = reinterpret_cast<float2 *>(static_cast<char *>(b.workspace) + w.part_ml);
    Scope sc(t, s, "cross_attention");
    if (c->type == VH_TYPE_BF16)
        a.table ? forward_launch<bf16, true>(s, c, a, w.rows) : forward_launch<bf16, false>(s, c, a, w.rows);
    else a.table ? forward_launch<float, true>(s, c, a, w.rows) : forward_launch<float, false>(s, c, a, w.rows);
    return sync_debug(s, "cross_forward_kernel");
}

template <typename T, bool BIAS>
static void dq_launch(hipStream_t s, const vh_cross *c, const CrossArgs &a, const CrossCut &cut) {
    if (cut.split) launch(cross_dq_split_kernel<T, BIAS>, cut.grid(), dq_lds(c, true), s, a);
    else launch(cross_dq_kernel<T, BIAS>, cut.grid(), dq_lds(c, false), s, a);
}

template <typename T, bool BIAS>
static void dkv_launch(hipStream_t s, const vh_cross *c, const CrossArgs &a, const CrossCut &cut) {
    const size_t lds = dkv_lds(c, cut.split, cut.heads);
    if (cut.split) launch(cross_dkv_split_kernel<T, BIAS>, cut.grid(), lds, s, a);
    else launch(cross_dkv_kernel<T, BIAS>, cut.grid(), lds, s, a);
}

bool cross_attention_backward(hipStream_t s, const vh_cross *c, const CrossBuffers &b, KernelTimer *t) {
    const char *what = "vh_cross_attention_backward";
    if (!cross_ok(what, c, true)) return false;
    if ((b.dk != nullptr) != (b.dv != nullptr)) {
        set_error("%s: dk and dv are given together, or neither", what);
        return false;
    }
    if (b.dbias && !c->bias_table) {
        set_error("%s: dbias without a bias table", what);
        return false;
    }
    const bool rows = cross_rows(c) > 0, keys = (int64_t)c->sequences * c->key_length > 0;
    if ((rows && (!b.q || !b.out || !b.saved || !b.dout || !b.dq)) || ((rows || b.dk) && keys && (!b.k || !b.v)) || !b.workspace) {
        set_error("%s: null q, k, v, out, saved, dout, dq or workspace", what);
        return false;
    }
    if (!aligned(what, {b.q, b.k, b.v, b.out, b.saved, b.workspace, b.dout, b.dq, b.dk, b.dv})) return false;
    CrossArgs a = cross_args(c, b);
    const CrossWork w = backward_work(c);
    if (!launches_ok(what, c, w, true)) return false;
    // Tensors without rows have no address.  dq's kernel reads k and v anywhere, and of q,
    // dout and out a row where it writes it; dk's and dv's read q and dout anywhere, and of k
    // and v a row where they write it: there a gradient may take its input's place.
    auto if_rows = [&](const void *p) { return rows ? p : nullptr; };
    auto if_keys = [&](const void *p) { return keys ? p : nullptr; };
    const bool as_out = same_layout(c->q_strides, c->out_strides, c->sequences, c->query_length, c->heads);
    const bool as_v = same_layout(c->k_strides, c->v_strides, c->sequences, c->key_length, c->kv_heads);
    const void *q = if_rows(b.q), *k = if_keys(b.k), *v = if_keys(b.v), *out = if_rows(b.out), *dout = if_rows(b.dout);
    const void *saved = if_rows(b.saved), *dq = if_rows(b.dq), *dk = if_keys(b.dk), *dv = if_keys(b.dv);
    if (!written_apart(what, {dq, dk, dv, b.dbias, b.workspace}, {saved}) ||
        !written_apart(what, {b.workspace}, {q, k, v, out, dout, c->bias_table}) ||
        !written_apart(what, {dq}, {k, v, c->bias_table, as_out ? nullptr : out, dk || !as_out ? dout : nullptr, dk ? q : nullptr}) ||
        !written_apart(what, {dk, dv}, {q, dout, c->bias_table}) || (!as_v && (!written_apart(what, {dk}, {v}) || !written_apart(what, {dv}, {k}))))
        return false;
    auto at = [&](size_t n) { return reinterpret_cast<float *>(static_cast<char *>(b.workspace) + n); };
    a.rows = at(w.stats);
    a.parts = w.rows.parts;
    a.kv_parts = w.keys.parts;
    a.kv_heads = w.keys.heads;
    a.part_o = at(w.part_o);
    a.part_dk = at(w.part_dk);
    a.part_dv = at(w.part_dv);
    a.dbias = b.dbias;
    a.dbias_part = b.dbias ? at(w.dbias) : nullptr;
    a.dbias_parts = w.dbias_parts;
    a.dbias_rows = reinterpret_cast<floatx4 *>(at(w.dbias_rows));
    const bool is_bf16 = c->type == VH_TYPE_BF16;
    if (rows) {
        Scope sc(t, s, "cross_attention_dq");
        if (is_bf16) a.table ? dq_launch<bf16, true>(s, c, a, w.rows) : dq_launch<bf16, false>(s, c, a, w.rows);
        else a.table ? dq_launch<float, true>(s, c, a, w.rows) : dq_launch<float, false>(s, c, a, w.rows);
        if (!sync_debug(s, "cross_dq_kernel")) return false;
    }
    const bool dkv = b.dk && keys;
    if (dkv) {
        Scope sc(t, s, "cross_attention_dkv");
        if (is_bf16) a.table ? dkv_launch<bf16, true>(s, c, a, w.keys) : dkv_launch<bf16, false>(s, c, a, w.keys);
        else a.table ? dkv_launch<float, true>(s, c, a, w.keys) : dkv_launch<float, false>(s, c, a, w.keys);
        if (!sync_debug(s, "cross_dkv_kernel")) return false;
    }
    FinishArgs f{};
    if (rows && w.rows.split && w.rows.parts > 1) f.dq = join_groups(cross_rows(c));
    if (dkv && kv_pieces(c, w.keys) > 1) f.dkv = join_groups(key_rows(c));
    f.heads = b.dbias ? c->heads : 0;
    const int64_t groups = f.heads + f.dq + 2 * f.dkv;
    if (!groups) return true;
    Scope sc(t, s, "cross_attention_sums");
    if (is_bf16) hipLaunchKernelGGL(cross_finish_kernel<bf16>, dim3((unsigned)groups), dim3(256), 0, s, a, f);
    else hipLaunchKernelGGL(cross_finish_kernel<float>, dim3((unsigned)groups), dim3(256), 0, s, a, f);
    return sync_debug(s, "cross_finish_kernel");
}

}  // namespace vh
