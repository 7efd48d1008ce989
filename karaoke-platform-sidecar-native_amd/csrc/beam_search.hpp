// One step of beam search: the best continuations of each sequence's beams.
//
//   lse_b = log sum_t exp(x_bt),  candidate (b, t): scores[b] + x_bt - lse_b
//
// in order of (score down, beam, logit down, token).  Within a beam that is the order
// of (x down, token), so the vocabulary is looked through once, in x: a workgroup takes
// a stretch of a beam's logits in registers, adds up its exponentials and finds its
// best `picks`; a second launch joins the stretches of a sequence's beams, in 64 bits.
// The logits are read once: 256 rows of 120001 in bf16, 61 MB, 23 us (2.7 TB/s) and 7 us
// for the join of 16 picks.  Two rounds of workgroups load and then compute; the VALU is
// busy in 68% of the cycles, half of it for the maximum and the exponentials, half for the
// best.  A step of one request is two launches, 4 to 6 us each.  More lists than the join
// compares at one place (a list is a beam's stretch) cost: 64 beams of 64 picks over 131072
// tokens in fp32, 1024 lists, 114 us, over 140003, 1152 lists, 1043.
#pragma once

#include "beam_floor.hpp"
#include "paged_cache.hpp"

namespace vh {

constexpr int BS_THREADS = 256, BS_WAVES = 4;
constexpr int BS_MAX_PICKS = 64, BS_MAX_BEAMS = 64;
constexpr int BS_LIST = 256;  // a wave's candidates

struct BeamPick {
    float x;
    int token;  // -1: none
};
// What a workgroup found of its stretch: the largest logit, the sum of exp(x - largest)
// (a NaN where a logit is), and its best, best first, behind it.
struct BeamPart {
    double sum;
    float top;
    int pad;
};

struct BeamArgs {
    const void *logits;
    int64_t seq_stride, beam_stride;  // elements
    const float *scores;
    const int *ended;
    int *tokens, *parents, *new_ended;
    float *new_scores;
    char *parts;                      // [sequences * beams][stretches] of part_bytes
    int S, B, V, picks, end_token, stretches, stretch, part_bytes;
    Divisor per_list, per_beam;       // picks, stretches
};

// The order of floats as whole numbers; -0 as 0.
VH_DEVICE uint32_t ordered(float x) {
    const uint32_t u = __float_as_uint(x + 0.0f);
    return u ^ ((uint32_t)((int)u >> 31) | 0x80000000u);
}
VH_DEVICE float from_ordered(uint32_t u) { return __uint_as_float(u & 0x80000000u ? u ^ 0x80000000u : ~u); }
// A logit and its token as one number, the better the larger: (logit, token down).
VH_DEVICE uint64_t key_of(float x, int token) { return (uint64_t)ordered(x) << 32 | ~(uint32_t)token; }
VH_DEVICE BeamPick pick_of(uint64_t key) { return {from_ordered((uint32_t)(key >> 32)), (int)~(uint32_t)key}; }

// 8 consecutive logits as they lie in memory, one of them as fp32.
template <typename T>
struct Logits;
template <>
struct Logits<bf16> {
    uint32_t w[4];
    VH_DEVICE float get(int e) const { return __uint_as_float(e & 1 ? w[e / 2] & 0xffff0000u : w[e / 2] << 16); }
    VH_DEVICE float pick(int e) const {  // e not known at compile time
        const uint32_t a = e & 4 ? w[2] : w[0], b = e & 4 ? w[3] : w[1], u = e & 2 ? b : a;
        return __uint_as_float(e & 1 ? u & 0xffff0000u : u << 16);
    }
    VH_DEVICE void load(const bf16 *p) {
        const Elements<uint16_t, 8>::type a = *reinterpret_cast<const Elements<uint16_t, 8>::type *>(p);
#pragma unroll
        for (int e = 0; e < 4; e++) w[e] = (uint32_t)a[2 * e] | (uint32_t)a[2 * e + 1] << 16;
    }
    VH_DEVICE void load_few(const bf16 *p, int n) {
#pragma unroll
        for (int e = 0; e < 4; e++)
            w[e] = (uint32_t)__builtin_bit_cast(uint16_t, p[max(0, 2 * e - 8 + n)]) |
                   (uint32_t)__builtin_bit_cast(uint16_t, p[max(0, 2 * e - 7 + n)]) << 16;
    }
    // the first n as -inf
    VH_DEVICE void leave_out(int n) {
#pragma unroll
        for (int e = 0; e < 8; e++)
            if (e < n) w[e / 2] = e & 1 ? (w[e / 2] & 0xffffu) | 0xff800000u : (w[e / 2] & 0xffff0000u) | 0xff80u;
    }
};
template <>
struct Logits<float> {
    float w[8];
    VH_DEVICE float get(int e) const { return w[e]; }
    VH_DEVICE float pick(int e) const {
        const float a = e & 4 ? w[4] : w[0], b = e & 4 ? w[5] : w[1], c = e & 4 ? w[6] : w[2], d = e & 4 ? w[7] : w[3];
        return e & 2 ? (e & 1 ? d : c) : (e & 1 ? b : a);
    }
    VH_DEVICE void load(const float *p) { load_n<8>(p, w); }
    VH_DEVICE void load_few(const float *p, int n) {
#pragma unroll
        for (int e = 0; e < 8; e++) w[e] = p[max(0, e - 8 + n)];
    }
    VH_DEVICE void leave_out(int n) {
#pragma unroll
        for (int e = 0; e < 8; e++)
            if (e < n) w[e] = -INFINITY;
    }
};

VH_DEVICE double wave_sum_double(double v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}

// Keeps the compiler from holding what it made of the logits up to here, and from
// taking up more of them than a vector at a time: else it unpacks all of a thread's
// logits at once, and spills.
template <typename T>
VH_DEVICE void anew(Logits<T> &x) {
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (auto &w : x.w) asm volatile("" : "+v"(w));
}

// A thread's vector j covers the stretch's logits (j * BS_THREADS + thread) * 8 .. + 7.
// One that reaches beyond the `valid` of the stretch is moved back to end with them, so
// that no load is partial; its first `skip` logits are the vector's before it (8: all of
// it is beyond).  Of a vocabulary of n < 8 the last n are it, the others its first once more.
struct BeamPlace {
    int at, skip;
    VH_DEVICE BeamPlace(int j, int thread, int valid) {
        const int own = (j * BS_THREADS + thread) * 8;
        at = min(own, valid - 8);
        skip = min(own - at, 8);
    }
};

constexpr int BS_VECTORS = 128;
template <typename T>
struct BeamVectors {
    Logits<T> x[BS_VECTORS];
    int at[BS_VECTORS], skip[BS_VECTORS];
};

// A wave's best `most` of NV * 8 logits a lane into list, unordered; how many.  floor: a
// value that `most` of them reach, or -inf.  p: the stretch, x: its vectors, top: theirs.
template <typename T, int NV>
VH_DEVICE int collect(const T *p, bool whole, const Logits<T> (&x)[NV], const float (&top)[NV], int thread, int valid, float floor,
                      int most, uint64_t *list, BeamVectors<T> &some) {
    const int lane = threadIdx.x & 63;
    const uint64_t below = ((uint64_t)1 << lane) - 1;
    int n = 0;
    // The vectors that have such a logit, where few, are put where all lanes see them; of more,
    // those that reach a higher floor, as long as that leaves `most`.
    auto with = [&](uint32_t least) {
        int vectors = 0;
#pragma unroll
        for (int j = 0; j < NV; j++) vectors += __popcll(__ballot(top[j] >= from_ordered(least)));
        return vectors;
    };
    float largest = top[0];
#pragma unroll
    for (int j = 1; j < NV; j++) largest = fmaxf(largest, top[j]);
    const uint32_t lowest = ordered(floor), highest = ordered(wave_max(largest));
    const BeamFloor chosen = beam_floor(lowest, highest, most, BS_VECTORS, with);
    floor = from_ordered(chosen.least);
    const bool few = chosen.vectors <= BS_VECTORS;
    int vectors = 0;
    if (few)
#pragma unroll
    for (int j = 0; j < NV; j++) {
        const bool has = top[j] >= floor;
        const uint64_t m = __ballot(has);
        const int k = vectors + __popcll(m & below);
        if (has && k < BS_VECTORS) {
            const BeamPlace place(j, thread, valid);
            some.x[k] = x[j];
            some.at[k] = place.at;
            some.skip[k] = place.skip;
        }
        vectors += __popcll(m);
    }
    if (few) {
        cache_wave_order();
        for (int i0 = 0; i0 < 8 * vectors; i0 += 64) {
            const int i = i0 + lane, k = min(i / 8, BS_VECTORS - 1), e = i % 8;
            const float v = some.x[k].pick(e);
            const bool has = i < 8 * vectors && v >= floor && e >= some.skip[k];
            const uint64_t m = __ballot(has);
            const int place = n + __popcll(m & below);
            if (has && place < BS_LIST) list[place] = key_of(v, some.at[k] + e);
            n += __popcll(m);
        }
        if (n <= BS_LIST) return n;
    }
    // Too many: hardly any above -inf, many alike, or those of a few lanes all larger than
    // others'.  The value that the most-th best has, between the floor and the largest by
    // halves; those above it, and of its own the first ones.  The logits are read
    // once more, a vector at a time: kept, they would take every call's registers.
    auto again = [&](int j) {
        const BeamPlace place(j, thread, valid);
        Logits<T> v;
        if (whole) v.load(p + place.at);
        else v.load_few(p, valid);
        return v;
    };
    auto reach = [&](uint32_t least) {  // how many do
        int count = 0;
#pragma clang loop unroll(disable)
        for (int j = 0; j < NV; j++) {
            const Logits<T> v = again(j);
            const BeamPlace place(j, thread, valid);
#pragma unroll
            for (int e = 0; e < 8; e++) count += v.get(e) == v.get(e) && ordered(v.get(e)) >= least && e >= place.skip ? 1 : 0;
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) count += __shfl_xor(count, o, 64);
        return count;
    };
    uint32_t best = lowest, high = highest;
    if (lowest == ordered(-INFINITY) && best < high && reach(best + 1) < most) high = best;  // as where few tokens are allowed
    while (best < high) {
        const uint32_t trial = best + (high - best + 1) / 2;
        if (reach(trial) >= most) best = trial;
        else high = trial - 1;
    }
    const float limit = from_ordered(best);
    n = 0;
#pragma clang loop unroll(disable)
    for (int pass = 0; pass < 2; pass++)  // above the limit, then at it while there is room
#pragma clang loop unroll(disable)
        for (int j = 0; j < NV && n < most; j++) {
            const Logits<T> v = again(j);
            const BeamPlace place(j, thread, valid);
            uint32_t mine = 0;
#pragma unroll
            for (int e = 0; e < 8; e++) mine |= (pass ? v.get(e) == limit : v.get(e) > limit) && e >= place.skip ? 1u << e : 0u;
            int upto = __popc(mine);
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
                const int u = __shfl_up(upto, o, 64);
                if (lane >= o) upto += u;
            }
            int k = n + upto - __popc(mine);
            n = min(n + __shfl(upto, 63, 64), most);
#pragma unroll
            for (int e = 0; e < 8; e++)
                if (mine >> e & 1) {
                    if (k < most) list[k] = key_of(v.get(e), place.at + e);
                    k++;
                }
        }
    return n;
}

template <typename T, int NV>
static __global__ __launch_bounds__(BS_THREADS, 5) void beam_stretch_kernel(BeamArgs a) {
    __shared__ __align__(16) uint64_t lists[BS_WAVES][BS_LIST + 2];
    __shared__ BeamVectors<T> some[BS_WAVES];
    __shared__ uint64_t sorted[BS_WAVES][BS_MAX_PICKS];
    __shared__ int counts[BS_WAVES];
    __shared__ float tops[BS_WAVES];
    __shared__ double sums[BS_WAVES];
    const int row = (int)(blockIdx.x / (uint32_t)a.stretches), part = (int)(blockIdx.x % (uint32_t)a.stretches);
    if (a.ended && a.ended[row]) return;  // nothing of it is looked at
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int first = part * a.stretch, valid = min(a.V - first, a.stretch);
    const T *p = static_cast<const T *>(a.logits) + row / a.B * a.seq_stride + row % a.B * a.beam_stride + first;
    Logits<T> x[NV];
#pragma unroll
    for (int j = 0; j < NV; j++) {
        const BeamPlace place(j, (int)threadIdx.x, valid);
        if (NV > 1 || a.V >= 8) x[j].load(p + place.at);
        else x[j].load_few(p, valid);
    }
#pragma unroll
    for (int j = 0; j < NV; j++) {
        const BeamPlace place(j, (int)threadIdx.x, valid);
        if (place.skip) x[j].leave_out(place.skip);
    }
    // the vectors' largest, the lane's, the wave's, and the sum of exponentials (a NaN stays
    // one); in one pass, from the first vector's largest, 256 rows of 120001 took 13% longer:
    // more registers, for the case that this is far too small
    float tops_of[NV], top = -INFINITY;
#pragma unroll
    for (int j = 0; j < NV; j++) {
        anew(x[j]);
        tops_of[j] = -INFINITY;
#pragma unroll
        for (int e = 0; e < 8; e++) tops_of[j] = fmaxf(tops_of[j], x[j].get(e));
        top = fmaxf(top, tops_of[j]);
    }
    const float wtop = wave_max(top);
    // 2^(c x - base), the exponent rounded once, that of wtop, 64 at most, not at all.  From
    // 2^30 on values are the largest or 128 below it, and nothing is left of them in any base.
    // In steps u of 2^-24 the logarithm of the sum is off by: an exponential's own 2, its
    // exponent's rounding ln 2 of its size, in the sum's mean at most log2 of its 4096 terms, and
    // c's 0.23 of as much in base e, 8.4 + 2; a sum of 8 and one of those 15; with |wtop| from
    // 2^20 on that of wtop's own exponent, ln 2 of 64: 28 u < 2^-19, and 73 u < 2^-17
    const float c = fabsf(wtop) < 0x1p30f ? 1.4426950408889634f : 1.0f, base = wtop == -INFINITY ? 0.0f : wtop * c;
    float sum = 0.0f;
#pragma unroll
    for (int j = 0; j < NV; j++) {
        anew(x[j]);
        float eight = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; e++) eight += __builtin_amdgcn_exp2f(__builtin_fmaf(x[j].get(e), c, -base));
        sum += eight;
    }
    const double wsum = wave_sum_double((double)sum) * (wtop == -INFINITY ? 1.0 : exp2(-(double)__builtin_fmaf(wtop, c, -base)));

    // a value that at least `most` of the wave's lanes' largest reach
    const int most = min(a.picks, valid);
    const bool there = (int)threadIdx.x * 8 < valid;
    uint32_t floor = 0;
    const uint32_t mine = there ? ordered(top) : 0;
    for (int bit = 31; bit >= 0; bit--) {
        const uint32_t trial = floor | 1u << bit;
        const int n = __popcll(__ballot(mine >= trial));
        if (n >= most) floor = trial;
        if (n == most) break;
    }
    // what lies below -inf in that order is no number
    const float least = floor <= ordered(-INFINITY) ? -INFINITY : from_ordered(floor);
    int n = collect<T, NV>(p, NV > 1 || a.V >= 8, x, tops_of, (int)threadIdx.x, valid, least, most, lists[wave], some[wave]);
    if (lane < 2) lists[wave][n + lane] = 0;
    cache_wave_order();
    for (int i = lane; i < n; i += 64) {
        const uint64_t mine = lists[wave][i];
        int rank = 0;
        for (int k = 0; k < n; k += 2) rank += (lists[wave][k] > mine) + (lists[wave][k + 1] > mine);
        if (rank < a.picks) sorted[wave][rank] = mine;
    }
    n = min(n, a.picks);
    if (lane == 0) {
        counts[wave] = n;
        tops[wave] = wtop;
        sums[wave] = wsum;
    }
    __syncthreads();
    BeamPart *head = reinterpret_cast<BeamPart *>(a.parts + (int64_t)blockIdx.x * a.part_bytes);
    BeamPick *best = reinterpret_cast<BeamPick *>(head + 1);
    int total = 0;
    for (int w = 0; w < BS_WAVES; w++) total += counts[w];
    // an entry's place: those of the other waves' sorted lists that beat it
    for (int i = threadIdx.x; i < BS_WAVES * a.picks; i += BS_THREADS) {
        const int w = i / a.picks, r = i % a.picks;
        if (r < counts[w]) {
            const uint64_t mine = sorted[w][r];
            int above[BS_WAVES] = {}, rank = 0;  // of its own list: r
            for (int step = BS_MAX_PICKS; step > 0; step /= 2)
#pragma unroll
                for (int o = 0; o < BS_WAVES; o++) {
                    const int at = above[o] + step;
                    const bool more = sorted[o][min(at, BS_MAX_PICKS) - 1] > mine;
                    if (at <= counts[o] && more) above[o] = at;
                }
#pragma unroll
            for (int o = 0; o < BS_WAVES; o++) rank += above[o];
            const BeamPick pick = pick_of(mine);
            if (rank < a.picks) best[rank] = {pick.x, pick.token + first};
        }
        if (i < a.picks && i >= total) best[i] = {0.0f, -1};
    }
    if (wave == 0) {
        const float top = lane < BS_WAVES ? tops[lane] : -INFINITY, all = wave_max(top);
        double s = lane < BS_WAVES ? sums[lane] : 0.0;
        // a wave of nothing but -inf adds nothing, a NaN stays
        if (top != -INFINITY) s *= exp((double)top - (double)all);
        s = wave_sum_double(s);
        if (lane == 0) {
            head->sum = s;
            head->top = all;
        }
    }
}

// Candidates in order: (score down) in `a`, (beam, logit down, token) in `b`, ascending.
struct BeamKey {
    uint64_t a, b;
};
VH_DEVICE bool key_less(const BeamKey &x, const BeamKey &y) { return (x.a < y.a) | ((x.a == y.a) & (x.b < y.b)); }
VH_DEVICE uint64_t score_down(double s) {
    const uint64_t u = (uint64_t)__double_as_longlong(s + 0.0);
    return ~(u ^ ((uint64_t)((int64_t)u >> 63) | 0x8000000000000000ull));
}
VH_DEVICE double score_of(uint64_t a) {
    const uint64_t u = ~a;
    return __longlong_as_double((int64_t)(u & 0x8000000000000000ull ? u ^ 0x8000000000000000ull : ~u));
}

// What the join knows of a beam: 0 as it is, 1 no candidate but -inf, 2 ended.
struct BeamState {
    double lse, score;
    int state, ended;
};
// Candidate r of a sequence's list; (-1, -1): none.
VH_DEVICE BeamPick listed(const BeamArgs &a, int s, int list, int r) {
    const char *p = a.parts + ((int64_t)s * a.B * a.stretches + list) * a.part_bytes;
    return reinterpret_cast<const BeamPick *>(p + sizeof(BeamPart))[r];
}
VH_DEVICE BeamKey candidate(const BeamArgs &a, int list, int r, const BeamState *beams, const BeamPick &pick) {
    const int beam = (int)((uint32_t)list / a.per_beam), in = (list - beam * a.stretches) * a.picks + r;
    const BeamState &st = beams[beam];
    const BeamKey none{~0ull, ~0ull};
    const double score = st.score;
    if (st.state) {  // the end token with the score as it is, then the others in order
        int token = in;
        double v = -INFINITY;
        if (st.state == 2) {
            token = in == 0 ? a.end_token : in - 1 < a.end_token ? in - 1 : in;
            if (in == 0) v = score;
        }
        if (in >= a.picks || token >= a.V) return none;
        return {score_down(v), (uint64_t)beam << 56 | (uint64_t)token};
    }
    if (pick.token < 0) return none;
    const double v = score + ((double)pick.x - st.lse);
    const uint32_t down = v == -INFINITY ? 0u : ~ordered(pick.x);
    return {score_down(v), (uint64_t)beam << 56 | (uint64_t)down << 24 | (uint64_t)pick.token};
}
VH_DEVICE void put_pick(const BeamArgs &a, int s, int place, const BeamKey &key, const BeamState *beams) {
    const int beam = (int)(key.b >> 56), token = (int)(key.b & 0xffffff);
    const int64_t at = (int64_t)s * a.picks + place;
    a.tokens[at] = token;
    a.parents[at] = beam;
    a.new_scores[at] = (float)score_of(key.a);
    if (a.new_ended) a.new_ended[at] = beams[beam].ended || token == a.end_token ? 1 : 0;
}

constexpr int BS_JOIN = 1024;    // threads of the join, and candidates that it sorts at once
constexpr int BS_LISTS = 1024;   // lists whose candidates at one place are compared with one another
constexpr int BS_LEFT = 4096;    // candidates that those leave, at most

// A workgroup joins a sequence's beams.  Every list is in order: where `need` lists have
// their candidate at place r at or before a key, need (r + 1) >= picks, only candidates at
// or before it count.  r is such that need is about a quarter of the lists (64 lists of
// 64: from 4096 candidates left with the heads themselves, 835 us, to some 100).  These
// lists leave at most need * picks candidates, the others r each, BS_LEFT at most, which
// are ranked by counting.  More lists than BS_LISTS are sorted stretch by stretch beside
// the best so far.
static __global__ __launch_bounds__(BS_JOIN) void beam_join_kernel(BeamArgs a) {
    __shared__ __align__(16) BeamKey keys[BS_LEFT];
    __shared__ BeamState beams[BS_MAX_BEAMS];
    __shared__ BeamKey limit;
    __shared__ int left;
    const int s = (int)blockIdx.x, tid = (int)threadIdx.x;
    const int lists = a.B * a.stretches, all = lists * a.picks;
    const int place = min(a.picks, (4 * a.picks + lists - 1) / lists) - 1, need = (a.picks + place) / (place + 1);
    // a thread's candidates, as long as they are few, asked for while the sums are on their way
    auto place_of = [&](int e) {
        const int list = (int)((uint32_t)e / a.per_list);
        return int2{list, e - list * a.picks};
    };
    constexpr int EARLY = 4;
    BeamPick at_place{0.0f, -1}, early[EARLY];
    if (tid < lists) at_place = listed(a, s, tid, place);
#pragma unroll
    for (int k = 0; k < EARLY; k++) {
        early[k] = {0.0f, -1};
        const int2 at = place_of(tid + k * BS_JOIN);
        if (tid + k * BS_JOIN < all) early[k] = listed(a, s, at.x, at.y);
    }
    if (tid == 0) {
        left = 0;
        limit = {~0ull, ~0ull};
    }
    for (int b0 = 0; b0 < a.B; b0 += BS_JOIN / 16) {
        const int b = b0 + tid / 16, lane = tid % 16;
        if (b >= a.B) break;
        const int row = s * a.B + b;
        const float score = a.scores[row];
        const int ended = a.ended ? a.ended[row] : 0;
        int st = ended ? 2 : 0;
        double l = 0.0;
        if (!st) {
            const char *p = a.parts + (int64_t)row * a.stretches * a.part_bytes;
            float top = -INFINITY;
            double sum = 0.0;
            for (int i = lane; i < a.stretches; i += 16) {
                const BeamPart h = *reinterpret_cast<const BeamPart *>(p + (int64_t)i * a.part_bytes);
                // a stretch of nothing but -inf adds nothing, a NaN stays
                const float up = fmaxf(top, h.top);
                if (top != -INFINITY && top != up) sum *= exp((double)top - (double)up);
                sum += h.top == -INFINITY || h.top == up ? h.sum : h.sum * exp((double)h.top - (double)up);
                top = up;
            }
            float all = top;
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) all = fmaxf(all, __shfl_xor(all, o, 16));
            if (top != -INFINITY) sum *= exp((double)top - (double)all);
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 16);
            l = (double)all + log(sum);
            if (!(fabs(l) < INFINITY)) st = 1;
        }
        if (!(fabsf(score) < INFINITY)) st = 1;
        if (lane == 0) beams[b] = {l, (double)score, st, ended};
    }
    __syncthreads();
    if (lists <= BS_LISTS) {
        if (tid < lists) keys[tid] = candidate(a, tid, place, beams, at_place);
        __syncthreads();
        if (tid < lists) {
            const BeamKey mine = keys[tid];
            int rank = 0;
#pragma unroll 4
            for (int i = 0; i < lists; i++) rank += key_less(keys[i], mine) ? 1 : 0;
            if (rank == need - 1 && ~mine.a) limit = mine;  // fewer than need: no limit
        }
        __syncthreads();
        const BeamKey most = limit;
        auto take = [&](int e, const BeamPick &pick) {
            const int2 at = place_of(e);
            const BeamKey key = candidate(a, at.x, at.y, beams, pick);
            if (~key.a && !key_less(most, key)) keys[atomicAdd(&left, 1)] = key;  // in any order: ranked below
        };
#pragma unroll
        for (int k = 0; k < EARLY; k++)
            if (tid + k * BS_JOIN < all) take(tid + k * BS_JOIN, early[k]);
        for (int e = tid + EARLY * BS_JOIN; e < all; e += BS_JOIN) {
            const int2 at = place_of(e);
            take(e, listed(a, s, at.x, at.y));
        }
        __syncthreads();
        const int n = left;
        for (int i = tid; i < n; i += BS_JOIN) {
            const BeamKey mine = keys[i];
            int rank = 0;
#pragma unroll 4
            for (int k = 0; k < n; k++) rank += key_less(keys[k], mine) ? 1 : 0;
            if (rank < a.picks) put_pick(a, s, rank, mine, beams);
        }
        return;
    }
    const BeamKey none{~0ull, ~0ull};
    int held = 0;  // the best so far, in front
    for (int done = 0; done < all;) {
        const int take = min(all - done, BS_JOIN - held);
        for (int i = tid; i < BS_JOIN - held; i += BS_JOIN) {
            const int2 at = place_of(done + i);
            keys[held + i] = i < take ? candidate(a, at.x, at.y, beams, listed(a, s, at.x, at.y)) : none;
        }
        __syncthreads();
        for (int k = 2; k <= BS_JOIN; k *= 2)
            for (int j = k / 2; j > 0; j /= 2) {
                if (tid < BS_JOIN / 2) {
                    const int lo = tid / j * 2 * j + tid % j, hi = lo + j;
                    const bool up = (lo & k) == 0;
                    const BeamKey x = keys[lo], y = keys[hi];
                    if (key_less(y, x) == up) {
                        keys[lo] = y;
                        keys[hi] = x;
                    }
                }
                __syncthreads();
            }
        done += take;
        held = min(a.picks, held + take);
    }
    if (tid < a.picks) put_pick(a, s, tid, keys[tid], beams);
}

}  // namespace vh
