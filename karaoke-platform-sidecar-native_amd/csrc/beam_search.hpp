// One step of beam search: the best continuations of each sequence's beams.
//
//   lse_b = log sum_t exp(x_bt),  candidate (b, t): scores[b] + x_bt - lse_b
//
// in order of (score down, beam, logit down, token).  Within a beam that is the order
// of (x down, token), so the vocabulary is looked through once, in x: a workgroup takes
// a stretch of a beam's logits in registers, adds up its exponentials and finds its
// best `picks`; a second launch joins the stretches of a sequence's beams, in 64 bits.
// Bound by HBM: the logits are read once.
#pragma once

#include "paged_cache.hpp"

namespace vh {

constexpr int BS_THREADS = 1024, BS_WAVES = 16;
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
};

// The order of floats as whole numbers; -0 as 0.
VH_DEVICE uint32_t ordered(float x) {
    const uint32_t u = __float_as_uint(x + 0.0f);
    return u ^ ((uint32_t)((int)u >> 31) | 0x80000000u);
}
VH_DEVICE float from_ordered(uint32_t u) { return __uint_as_float(u & 0x80000000u ? u ^ 0x80000000u : ~u); }
VH_DEVICE bool beats(const BeamPick &a, const BeamPick &b) { return a.x > b.x || (a.x == b.x && a.token < b.token); }

// 8 consecutive logits as they lie in memory, one of them as fp32.
template <typename T>
struct Logits;
template <>
struct Logits<bf16> {
    uint32_t w[4];
    VH_DEVICE float get(int e) const { return __uint_as_float(e & 1 ? w[e / 2] & 0xffff0000u : w[e / 2] << 16); }
    VH_DEVICE void load(const bf16 *p) {
        const Elements<uint16_t, 8>::type a = *reinterpret_cast<const Elements<uint16_t, 8>::type *>(p);
#pragma unroll
        for (int e = 0; e < 4; e++) w[e] = (uint32_t)a[2 * e] | (uint32_t)a[2 * e + 1] << 16;
    }
    VH_DEVICE void load(const bf16 *p, int n) {
#pragma unroll
        for (int e = 0; e < 4; e++) w[e] = 0xff80ff80u;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            if (e >= n) continue;
            const uint32_t v = __builtin_bit_cast(uint16_t, p[e]);
            w[e / 2] = e & 1 ? (w[e / 2] & 0xffffu) | v << 16 : (w[e / 2] & 0xffff0000u) | v;
        }
    }
};
template <>
struct Logits<float> {
    float w[8];
    VH_DEVICE float get(int e) const { return w[e]; }
    VH_DEVICE void load(const float *p) { load_n<8>(p, w); }
    VH_DEVICE void load(const float *p, int n) {
#pragma unroll
        for (int e = 0; e < 8; e++) w[e] = e < n ? p[e] : -INFINITY;
    }
};

VH_DEVICE double wave_sum_double(double v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}

// Keeps the compiler from holding what it made of the logits up to here.
template <typename T, int NV>
VH_DEVICE void anew(Logits<T> (&x)[NV]) {
#pragma unroll
    for (int j = 0; j < NV; j++)
#pragma unroll
        for (auto &w : x[j].w) asm volatile("" : "+v"(w));
}

// A wave's best `most` of NV * 8 logits a lane into list, unordered; how many.
// Lane l's vector j covers the stretch's elements (j * BS_THREADS + thread) * 8 .. + 7,
// `valid` (of the stretch) of them there.  floor: a value that `most` of them reach,
// or -inf.
template <typename T, int NV>
VH_DEVICE int collect(Logits<T> (&x)[NV], int thread, int valid, float floor, int most, BeamPick *list) {
    const uint64_t below = ((uint64_t)1 << (threadIdx.x & 63)) - 1;
    auto at = [&](int j) { return (j * BS_THREADS + thread) * 8; };
    int n = 0;
#pragma unroll
    for (int j = 0; j < NV; j++)
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const float v = x[j].get(e);
            const uint64_t m = __ballot(v >= floor && at(j) + e < valid);
            if (!m) continue;
            const int k = n + __popcll(m & below);
            if ((m >> (threadIdx.x & 63) & 1) && k < BS_LIST) list[k] = {v, at(j) + e};
            n += __popcll(m);
        }
    if (n <= BS_LIST) return n;
    // Too many (many logits alike, or those of one lane all larger than others'): the
    // value that the most-th best has, bit by bit; those above it, and of its own the
    // first ones.
    uint32_t best = 0;
    for (int bit = 31; bit >= 0; bit--) {
        const uint32_t trial = best | 1u << bit;
        int count = 0;
        anew(x);
#pragma unroll
        for (int j = 0; j < NV; j++)
#pragma unroll
            for (int e = 0; e < 8; e++)
                count += __popcll(__ballot(x[j].get(e) == x[j].get(e) && ordered(x[j].get(e)) >= trial && at(j) + e < valid));
        if (count >= most) best = trial;
    }
    const float limit = from_ordered(best);
    n = 0;
    anew(x);
#pragma unroll
    for (int j = 0; j < NV; j++)
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const float v = x[j].get(e);
            const uint64_t m = __ballot(v > limit && at(j) + e < valid);
            if (!m) continue;
            if (m >> (threadIdx.x & 63) & 1) list[n + __popcll(m & below)] = {v, at(j) + e};
            n += __popcll(m);
        }
    int room = most - n;
    anew(x);
#pragma unroll
    for (int j = 0; j < NV; j++) {
        if (room <= 0) break;
        int mine = 0;
#pragma unroll
        for (int e = 0; e < 8; e++) mine += x[j].get(e) == limit && at(j) + e < valid ? 1 : 0;
        int upto = mine;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int v = __shfl_up(upto, o, 64);
            if ((int)(threadIdx.x & 63) >= o) upto += v;
        }
        int k = upto - mine;
        const int all = __shfl(upto, 63, 64);
#pragma unroll
        for (int e = 0; e < 8; e++)
            if (x[j].get(e) == limit && at(j) + e < valid) {
                if (k < room) list[n + k] = {x[j].get(e), at(j) + e};
                k++;
            }
        n += min(all, room);
        room -= all;
    }
    return n;
}

template <typename T, int NV>
static __global__ __launch_bounds__(BS_THREADS) void beam_stretch_kernel(BeamArgs a) {
    __shared__ BeamPick lists[BS_WAVES][BS_LIST];
    __shared__ BeamPick sorted[BS_WAVES][BS_MAX_PICKS];
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
        const int at = (j * BS_THREADS + (int)threadIdx.x) * 8;
        if (at + 8 <= valid) x[j].load(p + at);
        else x[j].load(p + at, max(0, valid - at));
    }
    // the lane's largest, the wave's, and the sum of exponentials (a NaN stays one)
    float top = -INFINITY;
#pragma unroll
    for (int j = 0; j < NV; j++)
#pragma unroll
        for (int e = 0; e < 8; e++) top = fmaxf(top, x[j].get(e));
    const float wtop = wave_max(top);
    const float c = 1.4426950408889634f, base = wtop == -INFINITY ? 0.0f : wtop;
    float sum = 0.0f;
    anew(x);
#pragma unroll
    for (int j = 0; j < NV; j++)
#pragma unroll
        for (int e = 0; e < 8; e++) sum += __builtin_amdgcn_exp2f((x[j].get(e) - base) * c);
    const double wsum = wave_sum_double((double)sum);

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
    anew(x);
    int n = collect<T, NV>(x, (int)threadIdx.x, valid, floor ? from_ordered(floor) : -INFINITY, most, lists[wave]);
    cache_wave_order();
    for (int i = lane; i < n; i += 64) {
        const BeamPick mine = lists[wave][i];
        int rank = 0;
        for (int k = 0; k < n; k++) rank += beats(lists[wave][k], mine) ? 1 : 0;
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
            const BeamPick mine = sorted[w][r];
            int rank = r;
            for (int o = 0; o < BS_WAVES; o++) {
                if (o == w) continue;
                int lo = 0, hi = counts[o];
                while (lo < hi) {
                    const int mid = (lo + hi) / 2;
                    if (beats(sorted[o][mid], mine)) lo = mid + 1;
                    else hi = mid;
                }
                rank += lo;
            }
            if (rank < a.picks) best[rank] = {mine.x, mine.token + first};
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
VH_DEVICE bool key_less(const BeamKey &x, const BeamKey &y) { return x.a < y.a || (x.a == y.a && x.b < y.b); }
VH_DEVICE uint64_t score_down(double s) {
    const uint64_t u = (uint64_t)__double_as_longlong(s + 0.0);
    return ~(u ^ ((uint64_t)((int64_t)u >> 63) | 0x8000000000000000ull));
}
VH_DEVICE double score_of(uint64_t a) {
    const uint64_t u = ~a;
    return __longlong_as_double((int64_t)(u & 0x8000000000000000ull ? u ^ 0x8000000000000000ull : ~u));
}

constexpr int BS_JOIN = 1024;  // candidates sorted at once

// A workgroup joins a sequence's beams: stretch by stretch candidates beside the best
// so far, sorted.
static __global__ __launch_bounds__(512) void beam_join_kernel(BeamArgs a) {
    __shared__ BeamKey keys[BS_JOIN];
    __shared__ double lse[BS_MAX_BEAMS];
    __shared__ int state[BS_MAX_BEAMS];  // 0: as it is, 1: no candidate but -inf, 2: ended
    const int s = (int)blockIdx.x, tid = (int)threadIdx.x;
    if (tid < a.B) {
        const int row = s * a.B + tid;
        const float score = a.scores[row];
        int st = a.ended && a.ended[row] ? 2 : 0;
        double l = 0.0;
        if (!st) {
            const char *p = a.parts + (int64_t)row * a.stretches * a.part_bytes;
            float top = -INFINITY;
            for (int i = 0; i < a.stretches; i++) top = fmaxf(top, reinterpret_cast<const BeamPart *>(p + (int64_t)i * a.part_bytes)->top);
            double sum = 0.0;
            for (int i = 0; i < a.stretches; i++) {
                const BeamPart *h = reinterpret_cast<const BeamPart *>(p + (int64_t)i * a.part_bytes);
                sum += h->top == -INFINITY ? h->sum : h->sum * exp((double)h->top - (double)top);
            }
            l = (double)top + log(sum);
            if (!(fabs(l) < INFINITY)) st = 1;
        }
        if (!(fabsf(score) < INFINITY)) st = 1;
        lse[tid] = l;
        state[tid] = st;
    }
    __syncthreads();
    const int per_beam = a.stretches * a.picks;
    const int all = a.B * per_beam;
    const BeamKey none{~0ull, ~0ull};
    int held = 0;  // the best so far, in front
    for (int done = 0; done < all;) {
        const int take = min(all - done, BS_JOIN - held);
        int size = 64;
        while (size < held + take) size *= 2;
        for (int i = tid; i < size - held; i += 512) {
            BeamKey key = none;
            const int e = done + i;
            if (i < take) {
                const int beam = e / per_beam, in = e % per_beam, row = s * a.B + beam;
                const double score = (double)a.scores[row];
                if (state[beam]) {
                    // the end token with the score as it is, then the others in order
                    int token = in;
                    double v = -INFINITY;
                    if (state[beam] == 2) {
                        token = in == 0 ? a.end_token : in - 1 < a.end_token ? in - 1 : in;
                        if (in == 0) v = score;
                    }
                    if (in < a.picks && token < a.V) key = {score_down(v), (uint64_t)beam << 56 | (uint64_t)token};
                } else {
                    const char *p = a.parts + ((int64_t)row * a.stretches + in / a.picks) * a.part_bytes;
                    const BeamPick pick = reinterpret_cast<const BeamPick *>(p + sizeof(BeamPart))[in % a.picks];
                    if (pick.token >= 0) {
                        const double v = score + ((double)pick.x - lse[beam]);
                        const uint32_t down = v == -INFINITY ? 0u : ~ordered(pick.x);
                        key = {score_down(v), (uint64_t)beam << 56 | (uint64_t)down << 24 | (uint64_t)pick.token};
                    }
                }
            }
            keys[held + i] = key;
        }
        __syncthreads();
        for (int k = 2; k <= size; k *= 2)
            for (int j = k / 2; j > 0; j /= 2) {
                for (int i = tid; i < size / 2; i += 512) {
                    const int lo = i / j * 2 * j + i % j, hi = lo + j;
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
    if (tid < a.picks) {
        const BeamKey key = keys[tid];
        const int beam = (int)(key.b >> 56), token = (int)(key.b & 0xffffff);
        const int64_t at = (int64_t)s * a.picks + tid;
        a.tokens[at] = token;
        a.parents[at] = beam;
        a.new_scores[at] = (float)score_of(key.a);
        if (a.new_ended) a.new_ended[at] = (a.ended && a.ended[s * a.B + beam]) || token == a.end_token ? 1 : 0;
    }
}

}  // namespace vh
