// gfx950 kernels of a beam search: qmh_beam_select (the best continuations over beams and vocabulary) and
// qmh_beam_reorder (the surviving beams' dense states). No reference counterpart.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "qmh_device.h"
#include "qmh_launch.h"
#include "qmh_types.h"

namespace {

// --------------------------------------------------------------------------- select

constexpr int SEL_T = 256;    // threads of the scan
constexpr int SEL_CAP = 256;  // candidates a wave of it lists
constexpr int JOIN_CAP = 1024;
constexpr int SCAN_WAVES = 3 * 1024, SCAN_EPT = 16; // of plan_scan

// The sum of 2^t over N numbers between -1022 and 1022: t = k + f, |f| <= 1/2, and 2^k times a polynomial of degree 8 that
// meets 2^f at the nine Chebyshev points, at most 1.1e-12 of the value from it: far inside the distance of scores that
// decide a choice. Adding 1.5 2^52 rounds to k and leaves it in the low word. The N chains run side by side.
template <int N>
__device__ __forceinline__ double exp2_sum(double (&t)[N]) {
    constexpr double c[8] = {1.531007940249083e-05, 0.00015403455852408237, 0.0013333450567999663, 0.009618129159402626,
                             0.05550410941205934, 0.2402265069581299, 0.6931471805459335, 1.0};
    double s[N], p[N];
#pragma unroll
    for (int j = 0; j < N; j++) s[j] = t[j] + 0x1.8p52;
#pragma unroll
    for (int j = 0; j < N; j++) t[j] = t[j] - (s[j] - 0x1.8p52);
#pragma unroll
    for (int j = 0; j < N; j++) p[j] = 1.3255224888009091e-06;
#pragma unroll
    for (int k = 0; k < 8; k++)
#pragma unroll
        for (int j = 0; j < N; j++) p[j] = __builtin_fma(p[j], t[j], c[k]);
#pragma unroll
    for (int j = 0; j < N; j++) p[j] = __hiloint2double(__double2hiint(p[j]) + (__double2loint(s[j]) << 20), __double2loint(p[j]));
#pragma unroll
    for (int n = N; n > 1; n /= 2)
#pragma unroll
        for (int j = 0; j < n / 2; j++) p[j] += p[j + n / 2];
    return p[0];
}
constexpr double LOG2E = 1.4426950408889634074;

// e^d, d <= 600, and e^-700 below -700
__device__ __forceinline__ double exp_of(double d) {
    double t[1] = {fmax(d, -700.0) * LOG2E};
    return exp2_sum<1>(t);
}

// The sum of e^(x - ref) over N floats, in 64 bits, x at most 600 above ref (finite); values more than 700 below it count as that.
// NEAR is for |ref| up to 2^14: one fused product, with ref2 = ref log2 e rounded (2^-38 at the most) and a limit in floats,
// low = ref - 700. Further out these two no longer fit (x = ref would not give 1, low not be 700 away), so the difference is taken first: two
// 64-bit instructions more a logit.
constexpr float NEAR_REF = 16384.0f;
template <bool NEAR, int N>
__device__ __forceinline__ double exp_sum(const float *x, float ref, float low, double ref2) {
    double t[N];
#pragma unroll
    for (int j = 0; j < N; j++) t[j] = NEAR ? __builtin_fma((double)fmaxf(x[j], low), LOG2E, -ref2) : fmax((double)x[j] - (double)ref, -700.0) * LOG2E;
    return exp2_sum<N>(t);
}

// the order of floats as unsigned numbers, -0 as 0; 0 for -inf and NaN, which are no continuations
__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t u = __float_as_uint(x + 0.0f);
    return x > -__builtin_inff() ? u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u) : 0u;
}
__device__ __forceinline__ float of_key(uint32_t k) { return __uint_as_float((k >> 31) ? k ^ 0x80000000u : ~k); }

// the same for doubles
__device__ __forceinline__ uint64_t key_of_d(double x) {
    const uint64_t u = (uint64_t)__double_as_longlong(x + 0.0);
    return x > -__builtin_inf() ? u ^ ((u >> 63) ? ~0ull : 1ull << 63) : 0ull;
}
__device__ __forceinline__ double of_key_d(uint64_t k) {
    return __longlong_as_double((long long)((k >> 63) ? k ^ (1ull << 63) : ~k));
}

struct scan_head { // a segment of a row: the sum of exp(x - ref) (NaN: the row has no continuation), its largest logit's key
    double sum;
    float ref;
    uint32_t top;
};

// The largest t that at least n <= 64 of a wave's values reach, 0 if there is none above; with LOW, the largest whose LOW
// lowest bits are 0 (a bound for less). Two bits a round, by ballots.
template <int LOW = 0>
__device__ __forceinline__ uint32_t wave_nth(uint32_t v, int n) {
    uint32_t t = 0;
#pragma unroll
    for (int b = 30; b >= LOW; b -= 2) {
        const uint32_t u1 = t | 1u << b, u2 = t | 2u << b, u3 = t | 3u << b;
        const int c1 = __popcll(__ballot(v >= u1)), c2 = __popcll(__ballot(v >= u2)), c3 = __popcll(__ballot(v >= u3));
        t = c3 >= n ? u3 : c2 >= n ? u2 : c1 >= n ? u1 : t;
    }
    return t;
}

// done(c, rank) for each of n candidates: its rank is how many others are before(i, c) it, counted by as many neighbouring
// threads as there are for each (a power of two up to 64). All threads of the workgroup take part.
template <typename B, typename D>
__device__ __forceinline__ void rank_all(int n, int threads, B before, D done) {
    int per = 1;
    while (per < 64 && 2 * per * n <= threads) per *= 2;
    const int tid = threadIdx.x, part = tid & (per - 1);
    for (int c0 = 0; c0 < n; c0 += threads / per) {
        const int c = c0 + tid / per;
        int r = 0;
        if (c < n)
#pragma unroll 8
            for (int i = part; i < n; i += per) r += before(i, c);
        for (int x = 1; x < per; x *= 2) r += __shfl_xor(r, x);
        if (c < n && part == 0) done(c, r);
    }
}

// what a wave wrote to LDS is there for all its lanes
__device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// A wave takes a segment of a row, iters pieces of 64 EPT logits, in one pass with no word to the other waves: the sum of
// exponentials in 64 bits, and the segment's n_out best logits. A piece is in registers while the next one's loads are
// under way. Candidates go to a list in LDS, placed by ballots. What may be one is told by a bound: at first the
// n_out-th largest of the lanes' own maxima (below it nothing is among the best); when the list is cut down to its
// n_out best, the least of them, which only larger logits pass, since later ones lose a tie. Where a piece brings
// more than the list holds (a rising row, repeated values) its own lane maxima raise the bound, and if that does not help
// the exact bound of the piece is searched bit by bit.
// Bound by VALU issue (34 instructions a logit, 14 of them the exponential's 64-bit ones: 21 of the 34 us of 24.6 million f32
// logits) beside the loads (98 MB).
template <typename T, int EPT, int VEC>
__global__ __launch_bounds__(SEL_T) void k_beam_scan(const qmh_beam_args a, scan_head *heads, uint2 *cands, int row0, int iters) {
    constexpr int PIECE = 64 * EPT;
    __shared__ uint2 lists[SEL_T / 64][SEL_CAP];
    const int lane = threadIdx.x & 63, row = row0 + blockIdx.y, n_out = a.n_out;
    const int seg = __builtin_amdgcn_readfirstlane((int)(blockIdx.x * (SEL_T / 64) + (threadIdx.x >> 6)));
    if ((a.done && a.done[row]) || !(a.score[row] > -__builtin_inff())) return; // the join does not look at it
    uint2 *list = lists[threadIdx.x >> 6];
    const int64_t slot = (int64_t)row * (gridDim.x * (SEL_T / 64)) + seg;
    const T *x = (const T *)a.logits + row * a.stride;
    // vectors from the row's start rounded down to a vector: the ones that hold some element of the row
    const int skew = VEC > 1 ? (int)(((uintptr_t)x / sizeof(T)) % VEC) : 0;
    const int64_t first = (int64_t)seg * iters * PIECE - skew;
    int base = first < a.vocab ? (int)first : a.vocab;
    qmh_vec<T, VEC> v[EPT / VEC];
    auto load = [&](int from) {
#pragma unroll
        for (int k = 0; k < EPT / VEC; k++) {
            const int i = from + (k * 64 + lane) * VEC;
            if (i + VEC > 0 && i < a.vocab) v[k] = *(const qmh_vec<T, VEC> *)(x + i);
        }
    };
    load(base);
    float xs[EPT];
    float max = -__builtin_inff(), ref = 0.0f, low = -700.0f; // the segment's maximum; what its exponentials are taken below
    double sum = 0.0, ref2 = 0.0;
    bool near = true;
    float bound = -__builtin_inff(); // logits above it are candidates
    bool bad = false, none = true;
    int n = 0; // candidates in the list
    auto place = [&](uint64_t all) { return (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(all >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)all, 0)); };
    // the largest index that leaves fewer than n_out, and then the next one
    auto lowest = [&](auto count) {
        int last = -1;
        for (int b = 24; b >= 0; b--) last = count(last + (1 << b)) < n_out ? last + (1 << b) : last;
        return last + 1;
    };
    // the list's n_out best, in any order: the n_out-th largest key by ballots, the lowest indexes among those equal to it
    // (by ballots too where it is long: every entry's rank among 250 is a chain of 12 us, this one of 2)
    auto cut = [&]() {
        constexpr int E = SEL_CAP / 64;
        wave_sync();
        if (n > 64) { // what the n_out-th largest of the lanes' best leaves
            uint2 e[E];
            uint32_t best = 0;
#pragma unroll
            for (int j = 0; j < E; j++) {
                e[j] = lane + 64 * j < n ? list[lane + 64 * j] : make_uint2(0, 0);
                best = e[j].x > best ? e[j].x : best;
            }
            const uint32_t u = wave_nth<12>(best, n_out);
            wave_sync();
            n = 0;
#pragma unroll
            for (int j = 0; j < E; j++) {
                const uint64_t all = __ballot(e[j].x >= u && e[j].x);
                if (e[j].x >= u && e[j].x) list[n + place(all)] = e[j];
                n += __popcll(all);
            }
            wave_sync();
        }
        if (n < n_out) return;
        uint32_t t = 0; // stays above 0: n entries have keys
        if (n <= 64) {
            const uint2 e = lane < n ? list[lane] : make_uint2(0, 0);
            t = wave_nth(e.x, n_out);
            bool keep = e.x >= t;
            if (__popcll(__ballot(keep)) > n_out) {
                int r = 0;
                for (int i = 0; i < n; i++) {
                    const uint2 u = list[i];
                    r += (u.x > e.x) | ((u.x == e.x) & (u.y < e.y));
                }
                keep = lane < n && r < n_out;
            }
            const uint64_t all = __ballot(keep);
            wave_sync();
            if (keep) list[place(all)] = e;
        } else {
            uint2 e[E];
#pragma unroll
            for (int j = 0; j < E; j++) e[j] = lane + 64 * j < n ? list[lane + 64 * j] : make_uint2(0, 0);
            auto count = [&](auto in) {
                int c = 0;
#pragma unroll
                for (int j = 0; j < E; j++) c += __popcll(__ballot(in(e[j])));
                return c;
            };
            for (int b = 31; b >= 0; b--) {
                const uint32_t u = t | 1u << b;
                t = count([&](uint2 v) { return v.x >= u; }) >= n_out ? u : t;
            }
            int last = 0x7fffffff;
            if (count([&](uint2 v) { return v.x >= t; }) > n_out) last = lowest([&](int i) {
                return count([&](uint2 v) { return (v.x > t) | ((v.x == t) & ((int)v.y <= i)); });
            });
            wave_sync();
            n = 0;
#pragma unroll
            for (int j = 0; j < E; j++) {
                const bool keep = (e[j].x > t) | ((e[j].x == t) & ((int)e[j].y <= last));
                const uint64_t all = __ballot(keep);
                if (keep) list[n + place(all)] = e[j];
                n += __popcll(all);
            }
        }
        wave_sync();
        n = n_out;
        bound = fmaxf(bound, of_key(t));
    };
    for (int it = 0; it < iters && base < a.vocab; it++, base += PIECE) {
#pragma unroll
        for (int k = 0; k < EPT; k++) xs[k] = qmh_to_f(v[k / VEC].e[k % VEC]);
        if (it + 1 < iters && base + PIECE < a.vocab) load(base + PIECE);
        auto index = [&](int k) { return base + ((k / VEC) * 64 + lane) * VEC + k % VEC; };
        if (base < 0 || base + PIECE > a.vocab) // the row's ends
#pragma unroll
            for (int k = 0; k < EPT; k++)
                if ((uint32_t)index(k) >= (uint32_t)a.vocab) xs[k] = -__builtin_inff();
        float top = xs[0];
#pragma unroll
        for (int k = 1; k < EPT; k++) top = __builtin_elementwise_maximum(top, xs[k]); // NaN if one is
        bad = bad || __any(!(top < __builtin_inff()));
        if (__any(top > max)) {
            // a new maximum: the sums stay in range as long as it is within 600 of the reference
            max = fmaxf(max, qmh_wave_max(top));
            if (max < __builtin_inff() && (none || (double)max > (double)ref + 600.0)) {
                sum *= none ? 0.0 : exp_of((double)ref - (double)max);
                ref = max;
                low = ref - 700.0f;
                ref2 = (double)ref * LOG2E;
                near = !__any(__builtin_fabsf(ref) > NEAR_REF);
                none = false;
            }
        }
        if (near) {
#pragma unroll
            for (int k = 0; k < EPT; k += 4) sum += exp_sum<true, 4>(xs + k, ref, low, ref2);
        } else {
#pragma unroll
            for (int k = 0; k < EPT; k += 4) sum += exp_sum<false, 4>(xs + k, ref, low, ref2);
        }
        // the largest float below the n_out-th largest of the lanes' maxima, if that is more than the bound
        auto raise = [&]() {
            uint32_t mine = 0;
            if (!bad) {
                mine = key_of(top);
            } else { // NaN hides the lane's maximum
#pragma unroll
                for (int k = 0; k < EPT; k++) {
                    const uint32_t q = key_of(xs[k]);
                    mine = q > mine ? q : mine;
                }
            }
            const uint32_t t = wave_nth<12>(mine, n_out);
            if (t > 1) bound = fmaxf(bound, of_key(t - (t == 0x80000000u ? 2 : 1))); // below 0 is not -0
        };
        auto passing = [&]() {
            int c = 0;
#pragma unroll
            for (int k = 0; k < EPT; k++) c += __popcll(__ballot(xs[k] > bound));
            return c;
        };
        auto append = [&](int k, bool take) {
            const uint64_t all = __ballot(take);
            if (all) {
                if (take) list[n + place(all)] = make_uint2(key_of(xs[k]), (uint32_t)index(k));
                n += __popcll(all);
            }
        };
        if (it == 0) raise();
        if (!__any(top > bound) && !bad) continue;
        bool full = n + passing() > SEL_CAP;
        if (full) {
            cut();
            raise();
            full = n + passing() > SEL_CAP;
        }
        if (!full) {
#pragma unroll
            for (int k = 0; k < EPT; k++) append(k, xs[k] > bound);
        } else {
            // the largest key that n_out of the piece's reach, then the lowest indexes among those equal to it
            uint32_t keys[EPT];
#pragma unroll
            for (int k = 0; k < EPT; k++) keys[k] = key_of(xs[k]);
            auto count = [&](auto in) {
                int c = 0;
#pragma unroll
                for (int k = 0; k < EPT; k++) c += __popcll(__ballot(in(k)));
                return c;
            };
            uint32_t from = 0;
            for (int b = 31; b >= 0; b--) {
                const uint32_t t = from | 1u << b;
                from = count([&](int k) { return keys[k] >= t; }) >= n_out ? t : from;
            }
            int last = 0x7fffffff;
            if (count([&](int k) { return keys[k] >= from; }) > n_out) last = lowest([&](int i) {
                return count([&](int k) { return (keys[k] > from) | ((keys[k] == from) & (index(k) <= i)); });
            });
#pragma unroll
            for (int k = 0; k < EPT; k++) append(k, keys[k] && ((keys[k] > from) | ((keys[k] == from) & (index(k) <= last))));
        }
        if (n > SEL_CAP / 2) cut();
    }
    cut();
    if (lane < n_out) cands[slot * n_out + lane] = lane < n ? list[lane] : make_uint2(0, 0);
    sum = qmh_wave_sum_d(sum);
    if (lane == 0) heads[slot] = scan_head{bad ? __builtin_nan("") : none ? 0.0 : sum, ref, key_of(max)};
}

// A group's choice from its rows' segments: each row's log sum (a wave a row), then the n_out best totals as in the scan:
// a bound, what reaches it ranked in LDS. The bound is the n_out-th largest of 64 parts' maxima, a part being one lane of
// every wave; from 64 parts it lets about 64 (1 + 1/2 + ... + 1/64) pass at the most on average, however many candidates there are, as
// long as their best are spread over the parts. Where more than JOIN_CAP reach it (equal totals), one after another. A
// chain of short steps in one workgroup: 5 to 7 us, 4 of them an empty launch's; past 8 beams twice the threads (12 rows of
// 8000 13.2 us with 1024, 14.7 with 512).
// MANY: a segment whose largest total is below the n_out-th largest of these has none of the best. The others are found
// first, by the same bound, and only their candidates are read.
template <bool MANY, int JT>
__global__ __launch_bounds__(JT) void k_beam_join(const qmh_beam_args a, const scan_head *heads, const uint2 *cands, int segs) {
    constexpr int NW = JT / 64, TOPS = MANY ? SCAN_WAVES : 1;
    __shared__ double lse[64], score[64];
    __shared__ uint64_t ckey[JOIN_CAP], bk[NW], rkey[64]; // rkey: the chosen totals, best first
    __shared__ uint32_t cplace[JOIN_CAP], best_of[JT], bf[NW], tops[TOPS];
    __shared__ uint16_t chosen[TOPS];
    __shared__ int ncand, nchosen, listed[64];
    const int g = blockIdx.x, tid = threadIdx.x, w = tid >> 6, lane = tid & 63, K = a.n_beams, n_out = a.n_out;
    if (tid == 0) ncand = nchosen = 0;
    // few beams: several waves a row, each with the row's log sum for itself (MANY: a wave a row)
    const int share = !MANY && K < NW ? NW / K : 1, per = segs * n_out;
    const int b0 = w / share < NW / share ? w / share : K, j0 = (w % share) * 64;
    auto number = [&](int k) { return j0 + 64 * share * k + ((lane + 21 * k + 9 * w) & 63); }; // of a row's candidates: every part gets some of a segment's first
    auto behind = [&](uint64_t all) { return (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(all >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)all, 0)); };
    // the first row's first heads and candidates are asked for at once with its score (of a dead row they are not used)
    double sum0 = 0.0;
    float ref0 = 0.0f;
    uint2 v0[4];
    if (!MANY && b0 < K) {
        const int64_t at = (int64_t)(g * K + b0) * segs;
        if (lane < segs) {
            sum0 = heads[at + lane].sum;
            ref0 = heads[at + lane].ref;
        }
#pragma unroll
        for (int k = 0; k < 4; k++) v0[k] = number(k) < per ? cands[at * n_out + number(k)] : make_uint2(0, 0);
    }
    uint32_t mine = 0;
    for (int b = b0; b < K; b += NW / share) {
        const int row = g * K + b;
        const float sc = a.score[row];
        const bool done = a.done && a.done[row], live = !done && sc > -__builtin_inff();
        double s = __builtin_nan("");
        const scan_head *h = heads + (int64_t)row * segs;
        if (!MANY && live) {
            if (b != b0 && lane < segs) {
                sum0 = h[lane].sum;
                ref0 = h[lane].ref;
            }
            float m = sum0 == 0.0 ? -__builtin_inff() : ref0;
            for (int c = lane + 64; c < segs; c += 64) m = h[c].sum == 0.0 ? m : fmaxf(m, h[c].ref);
            m = qmh_wave_max(m);
            s = sum0 == 0.0 ? 0.0 : sum0 * exp_of((double)ref0 - (double)m);
            for (int c = lane + 64; c < segs; c += 64) { // a sum of 0 has no reference to be in range of
                const double e = h[c].sum;
                if (e != 0.0) s = __builtin_fma(e, exp_of((double)h[c].ref - (double)m), s);
            }
            s = (double)m + log(qmh_wave_sum_d(s));
        }
        if constexpr (MANY) {
            uint32_t *top = tops + b * segs;
            scan_head v[4]; // the first 256 are asked for with the score
            auto load = [&](int c) {
#pragma unroll
                for (int k = 0; k < 4; k++) v[k] = c + 64 * k < segs ? h[c + 64 * k] : scan_head{0.0, 0.0f, 0u};
            };
            load(lane);
            if (live) {
                float m = -__builtin_inff();
                s = 0.0;
                for (int c0 = lane; c0 - lane < segs; c0 += 256) {
                    if (c0 != lane) load(c0);
                    float to = m;
#pragma unroll
                    for (int k = 0; k < 4; k++) to = v[k].sum == 0.0 ? to : fmaxf(to, v[k].ref);
                    to = qmh_wave_max(to);
                    const float ref = to > -__builtin_inff() ? to : 0.0f; // nothing yet: sums of 0
                    if (to > m && m > -__builtin_inff()) s *= exp_of((double)m - (double)ref);
                    m = to;
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        const float r = v[k].sum == 0.0 ? ref : v[k].ref;
                        s = __builtin_fma(v[k].sum, exp_of((double)r - (double)ref), s);
                        if (c0 + 64 * k < segs) top[c0 + 64 * k] = v[k].top;
                    }
                }
                s = (double)m + log(qmh_wave_sum_d(s));
            }
            // the tops become the high words of their totals' ordered keys
            for (int c = lane; c < segs; c += 64) {
                const uint32_t t = live && s == s ? top[c] : 0;
                const uint32_t q = done && c == 0 ? (uint32_t)(key_of_d(sc) >> 32)
                                   : t            ? (uint32_t)(key_of_d((double)sc + ((double)of_key(t) - s)) >> 32)
                                                  : 0;
                top[c] = q;
            }
        }
        if (lane == 0 && w % share == 0) {
            lse[b] = done ? __builtin_inf() : s; // marks a finished row: another's sum is at most 2^24 e^600, or NaN
            score[b] = (double)sc;
        }
    }
    // What the n_out-th largest is not below, from each thread's largest: the n_out-th largest of 64 parts' (one lane of
    // every wave). All threads take part.
    auto bound = [&]() {
        best_of[tid] = mine;
        __syncthreads();
        uint32_t v = 0;
#pragma unroll
        for (int k = 0; k < NW; k++) v = best_of[64 * k + lane] > v ? best_of[64 * k + lane] : v;
        v = wave_nth<12>(v, n_out);
        return v > 1 ? v : 1;
    };
    const int lanes = n_out <= 1 ? 1 : 1 << (32 - __builtin_clz(n_out - 1)); // of a chosen segment: a power of two
    if constexpr (MANY) {
        __syncthreads();
        for (int c = tid; c < K * segs; c += JT) mine = tops[c] > mine ? tops[c] : mine;
        const uint32_t from = bound();
        for (int c0 = 0; c0 < K * segs; c0 += JT) {
            const int c = c0 + tid;
            const bool take = c < K * segs && tops[c] >= from;
            const uint64_t in = __ballot(take);
            int at = 0;
            if (lane == 0 && in) at = atomicAdd(&nchosen, __popcll(in));
            at = __builtin_amdgcn_readfirstlane(at) + behind(in);
            if (take) chosen[at] = (uint16_t)c;
        }
    }
    __syncthreads();
    const int n_chosen = MANY ? nchosen : 0;
    // lanes of them for each chosen segment, four a thread from segment number i on
    auto of_chosen = [&](int i, uint64_t *q, uint32_t *p) {
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const int e = i + ((k * NW + w) * 64 + lane) / lanes, o = (lane + 5 * e) & (lanes - 1); // every part gets some of the first
            q[k] = 0;
            if (e < n_chosen && o < n_out) {
                const int c = chosen[e];
                const uint2 v = cands[((int64_t)g * K * segs + c) * n_out + o];
                const int b = c / segs;
                const double L = lse[b], sc = score[b];
                const bool done = L == __builtin_inf(); // one continuation
                q[k] = done ? o == 0 ? key_of_d(sc) : 0ull : v.x ? key_of_d(sc + ((double)of_key(v.x) - L)) : 0ull;
                p[k] = (uint32_t)(b * a.vocab) + (done ? (uint32_t)a.eos : v.y);
            }
        }
    };
    uint64_t q0[4] = {};
    uint32_t p0[4] = {};
    if constexpr (MANY) of_chosen(0, q0, p0);
    // body(ordered keys of the totals (0: none), places beam * vocab + token), four candidates a lane, all lanes at once
    auto each = [&](auto body) {
        if constexpr (MANY) {
            body(q0, p0);
            for (int i = 4 * JT / lanes; i < n_chosen; i += 4 * JT / lanes) {
                uint64_t q[4];
                uint32_t p[4] = {};
                of_chosen(i, q, p);
                body(q, p);
            }
        } else {
            for (int b = b0; b < K; b += NW / share) {
                const double L = lse[b], sc = score[b];
                uint64_t q[4] = {};
                uint32_t p[4] = {};
                if (L == __builtin_inf()) { // finished
                    if (lane == 0 && w % share == 0) q[0] = key_of_d(sc);
                    p[0] = (uint32_t)(b * a.vocab + a.eos);
                    body(q, p);
                    continue;
                }
                if (L != L) continue;
                const uint2 *c = cands + (int64_t)(g * K + b) * per;
                for (int i = 0; i < per; i += 256 * share) {
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        const int j = i + number(k);
                        const uint2 v = b == b0 && i == 0 ? v0[k] : j < per ? c[j] : make_uint2(0, 0);
                        q[k] = v.x ? key_of_d(sc + ((double)of_key(v.x) - L)) : 0ull;
                        p[k] = (uint32_t)(b * a.vocab) + v.y;
                    }
                    body(q, p);
                }
            }
        }
    };
    mine = 0;
    each([&](const uint64_t *q, const uint32_t *) {
#pragma unroll
        for (int k = 0; k < 4; k++) mine = (uint32_t)(q[k] >> 32) > mine ? (uint32_t)(q[k] >> 32) : mine;
    });
    const uint32_t from = bound();
    each([&](const uint64_t *q, const uint32_t *p) { // places by ballots, one addition to the count a wave
        uint64_t in[4];
        int n = 0;
#pragma unroll
        for (int k = 0; k < 4; k++) {
            in[k] = __ballot((uint32_t)(q[k] >> 32) >= from);
            n += __popcll(in[k]);
        }
        if (!n) return;
        int at = 0;
        if (lane == 0) at = atomicAdd(&ncand, n);
        at = __builtin_amdgcn_readfirstlane(at);
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const int to = at + behind(in[k]);
            if ((in[k] >> lane & 1) && to < JOIN_CAP) {
                ckey[to] = q[k];
                cplace[to] = p[k];
            }
            at += __popcll(in[k]);
        }
    });
    __syncthreads();
    auto write = [&](int o, uint64_t k, uint32_t p) { // every score has been read: out_score may be score
        const int64_t at = (int64_t)g * n_out + o;
        a.out_score[at] = k ? (float)of_key_d(k) : -__builtin_inff();
        a.out_parent[at] = k ? (int)(p / (uint32_t)a.vocab) : -1;
        a.out_token[at] = k ? (int)(p % (uint32_t)a.vocab) : -1;
    };
    const int n = ncand;
    uint64_t below = ~0ull; // what was chosen last: its total, then its place
    int64_t after = -1;
    if (n <= JOIN_CAP) {
        rank_all(
            n, JT, [&](int i, int c) { return (ckey[i] > ckey[c]) | ((ckey[i] == ckey[c]) & (cplace[i] < cplace[c])); }, // no branches: the reads overlap
            [&](int c, int r) {
                if (r < n_out) {
                    rkey[r] = ckey[c];
                    write(r, ckey[c], cplace[c]);
                }
            });
        if (tid >= n && tid < n_out) {
            rkey[tid] = 0;
            write(tid, 0, 0);
        }
    } else for (int o = 0; o < n_out; o++) {
        uint64_t best = 0;
        uint32_t at = 0xffffffffu;
        each([&](const uint64_t *q, const uint32_t *p) {
#pragma unroll
            for (int k = 0; k < 4; k++) {
                if (!q[k] || q[k] > below || (q[k] == below && (int64_t)p[k] <= after)) continue;
                if (q[k] > best || (q[k] == best && p[k] < at)) {
                    best = q[k];
                    at = p[k];
                }
            }
        });
        for (int x = 1; x < 64; x <<= 1) {
            const uint64_t oq = __shfl_xor((unsigned long long)best, x);
            const uint32_t op = __shfl_xor(at, x);
            if (oq > best || (oq == best && op < at)) {
                best = oq;
                at = op;
            }
        }
        __syncthreads();
        if (lane == 0) {
            bk[w] = best;
            bf[w] = at;
        }
        __syncthreads();
        for (int k = 0; k < NW; k++)
            if (bk[k] > best || (bk[k] == best && bf[k] < at)) {
                best = bk[k];
                at = bf[k];
            }
        below = best;
        after = at;
        if (tid == 0) {
            rkey[o] = best;
            write(o, best, at);
        }
    }
    __syncthreads();
    // The scan chose by logits. Where different logits of a row come to one total, the last one chosen, a lower token may not be
    // among the candidates: its logit is at most 2^-26 of the row's score, log sum and total then (a step of a float against
    // one of a double), and its segment has listed n_out that are no less. If some row can have such, the places of that total go to
    // the first of all logits that come to it: 4 rows of 128256 with their best at 0 take 48 us, 12 otherwise. (Rows of log
    // probabilities have one next to 0 each, but not n_out: the count keeps them at 12.)
    const uint64_t last = rkey[n_out - 1];
    bool coarse = false;
    if (last && lane < K) {
        const double L = lse[lane], sc = score[lane], t = of_key_d(last);
        coarse = L > -__builtin_inf() && L < __builtin_inf() && !(fabs((t - sc) + L) > 0x1p-26 * (fabs(L) + fabs(sc) + fabs(t)));
    }
    if (!__any(coarse)) return; // every wave finds the same
    if (n <= JOIN_CAP) {
        if (tid < 64) listed[tid] = 0;
        __syncthreads();
        for (int c = tid; c < n; c += JT)
            if (ckey[c] >= last) atomicAdd(&listed[cplace[c] / (uint32_t)a.vocab], 1);
        __syncthreads();
        if (!__any(coarse && listed[lane] >= n_out)) return;
    }
    int at = __popcll(__ballot(lane < n_out && rkey[lane] > last));
    // the next places, up to n_out, to the lanes that have one, in their order
    auto put = [&](bool in, uint32_t p) {
        const uint64_t all = __ballot(in);
        __syncthreads(); // bf has been read
        if (lane == 0) bf[w] = (uint32_t)__popcll(all);
        __syncthreads();
        int to = at + behind(all);
        for (int k = 0; k < NW; k++) {
            to += k < w ? (int)bf[k] : 0;
            at += (int)bf[k];
        }
        if (in && to < n_out) write(to, last, p);
    };
    for (int b = 0; b < K && at < n_out; b++) {
        const double L = lse[b], sc = score[b];
        const uint32_t p0 = (uint32_t)(b * a.vocab);
        if (L == __builtin_inf()) { // finished
            put(tid == 0 && key_of_d(sc) == last, p0 + (uint32_t)a.eos);
            continue;
        }
        if (!(L > -__builtin_inf())) continue;
        const int64_t row = (int64_t)(g * K + b) * a.stride;
        for (int t0 = 0; t0 < a.vocab && at < n_out; t0 += 8 * JT) {
            bool in[8], some = false;
#pragma unroll
            for (int k = 0; k < 8; k++) {
                const int t = t0 + k * JT + tid;
                float x = -__builtin_inff();
                if (t < a.vocab)
                    x = a.dtype == QMH_F32   ? ((const float *)a.logits)[row + t]
                        : a.dtype == QMH_F16 ? qmh_to_f(((const qmh_f16 *)a.logits)[row + t])
                                             : qmh_to_f(((const qmh_bf16 *)a.logits)[row + t]);
                in[k] = x > -__builtin_inff() && key_of_d(sc + ((double)x - L)) == last;
                some |= in[k];
            }
            __syncthreads(); // bf has been read
            const bool here = __any(some);
            if (lane == 0) bf[w] = here;
            __syncthreads();
            uint32_t any = 0;
            for (int k = 0; k < NW; k++) any |= bf[k];
            if (!any) continue;
#pragma unroll
            for (int k = 0; k < 8; k++)
                if (at < n_out) put(in[k], p0 + (uint32_t)(t0 + k * JT + tid));
        }
    }
}

// How a row is cut: into segments of whole pieces, one a wave, as many as give the chip SCAN_WAVES waves: three a SIMD, so
// that they run in one round. 192 rows of 128256 f32 measured 43 us so, 52 with two a SIMD and 47 with four (pieces then
// divide worse); pieces of 8 logits a lane where that many waves have no more.
struct scan_plan {
    int ept, iters, segs; // segs: of a row, a multiple of a workgroup's waves
};
scan_plan plan_scan(const qmh_beam_args *a) {
    constexpr int W = SEL_T / 64;
    const int64_t rows = (int64_t)a->n_groups * a->n_beams, len = (int64_t)a->vocab + 15; // 15: a row that starts inside a vector
    scan_plan p;
    p.ept = rows * len <= (int64_t)SCAN_WAVES * 64 * 8 ? 8 : SCAN_EPT;
    const int64_t piece = 64 * p.ept, pieces = (len + piece - 1) / piece;
    int64_t segs = SCAN_WAVES / rows / W * W;
    segs = segs < W ? W : segs;
    p.iters = (int)((pieces + segs - 1) / segs);
    p.segs = (int)((pieces + (int64_t)p.iters * W - 1) / ((int64_t)p.iters * W)) * W;
    return p;
}
// Which join: MANY where most of a row's candidates are not worth reading. One prompt, 12 rows of 57576, n_out 24 (116 segments a
// row): 15.2 us with it, 39 without; 4 rows of 151936, n_out 8 (300): 13.7 and 24; 64 rows of 32000, n_out 16 (32): 14.4 and 15.9;
// 128 rows of 50000, n_out 32 (20): 30.5 and 39.4; 192 of 128256, n_out 16 (16): 41.2 and 40.3; 16 rows of 3000, n_out 64 (8): 42 and 30.
bool many_segments(const qmh_beam_args *a, int segs) { return segs >= 16 && segs * a->n_out > 256; }

// --------------------------------------------------------------------------- reorder

// Thread: one unit of U (the widest that every row is aligned to) of one row, for all beams of a group. 12 MB take 6.2 us, 4 of
// them an empty launch's; 684 MB (32 sequences, rows of 2800 bytes) 4.1 TB/s. Every beam that
// takes another's state is read before any is written, so any parents move in place; a row's last bytes go in 4-byte
// pieces, read together too, and single bytes. parents: uniform, by scalar loads.
typedef const __attribute__((address_space(4))) int32_t *const_i32;
typedef uint32_t v4u __attribute__((ext_vector_type(4)));
template <typename U, int BM>
__global__ __launch_bounds__(256, BM > 16 ? 2 : 4) void k_beam_reorder(const qmh_beam_state s, uint8_t *dst, const uint8_t *src, const int32_t *parent,
                                                      uint32_t n_groups, int K, uint32_t row_units, uint32_t blocks_per, uint32_t first) {
    const uint32_t block = blockIdx.x + first, og = block / blocks_per, ub = block - og * blocks_per;
    const uint32_t o = og / n_groups, g = og - o * n_groups;
    const uint32_t u = ub * 256 + threadIdx.x, r = u / row_units, c = u - r * row_units;
    const_i32 par = (const_i32)(uintptr_t)(parent + g * K);
    if constexpr (BM > 16) { // U is 1 or 4 bytes: a row's last bytes singly
        __shared__ U keep[64 * 256];
        if (r >= s.n_rows) return;
        const int64_t at = (int64_t)c * sizeof(U), base = o * s.outer_stride + (int64_t)g * K * s.seq_stride + r * s.row_stride + at;
        auto source = [&](int j) { return par[j] >= 0 && par[j] < K ? par[j] : j; };
        auto move = [&](auto z, int64_t b) { // a byte has the thread's word to itself, too
            using V = decltype(z);
            qmh_move_many(
                keep + threadIdx.x, K,
                [&](int j, U &u) {
                    if (source(j) == j && dst == src) return false;
                    u = *(const V *)(src + b + source(j) * s.seq_stride);
                    return true;
                },
                [&](int j, U u) {
                    if (source(j) != j || dst != src) *(V *)(dst + b + j * s.seq_stride) = (V)u;
                });
        };
        if (at + (int64_t)sizeof(U) <= s.live) move(U{}, base);
        else
            for (int64_t k = 0; at + k < s.live; k++) move(uint8_t{}, base + k);
        return;
    }
    int from[BM]; // -1: nothing to do
#pragma unroll
    for (int j = 0; j < BM; j++) {
        const int p = par[j < K ? j : 0], f = p >= 0 && p < K ? p : j;
        from[j] = j >= K || (f == j && dst == src) ? -1 : f;
    }
    if (r >= s.n_rows) return;
    int64_t at = (int64_t)c * sizeof(U);
    const int64_t base = o * s.outer_stride + (int64_t)g * K * s.seq_stride + r * s.row_stride + at;
    const uint8_t *f = src + base;
    uint8_t *t = dst + base;
    const int64_t left = s.live - at;
    if (left >= (int64_t)sizeof(U)) {
        U v[BM];
#pragma unroll
        for (int j = 0; j < BM; j++)
            if (from[j] >= 0) v[j] = *(const U *)(f + from[j] * s.seq_stride);
#pragma unroll
        for (int j = 0; j < BM; j++)
            if (from[j] >= 0) *(U *)(t + j * s.seq_stride) = v[j];
        return;
    }
    int done = 0;
    if constexpr (sizeof(U) == 16) { // 1 to 3 words
        const int words = (int)(left >> 2);
        uint32_t v[BM][3];
#pragma unroll
        for (int j = 0; j < BM; j++)
            if (from[j] >= 0)
#pragma unroll
                for (int k = 0; k < 3; k++)
                    if (k < words) v[j][k] = *(const uint32_t *)(f + from[j] * s.seq_stride + 4 * k);
#pragma unroll
        for (int j = 0; j < BM; j++)
            if (from[j] >= 0)
#pragma unroll
                for (int k = 0; k < 3; k++)
                    if (k < words) *(uint32_t *)(t + j * s.seq_stride + 4 * k) = v[j][k];
        done = 4 * words;
    }
    for (; done < left; done++) {
        uint8_t v[BM];
#pragma unroll
        for (int j = 0; j < BM; j++)
            if (from[j] >= 0) v[j] = f[from[j] * s.seq_stride + done];
#pragma unroll
        for (int j = 0; j < BM; j++)
            if (from[j] >= 0) t[j * s.seq_stride + done] = v[j];
    }
}

// The step's choice becomes the sequences' next tokens and positions: thread j of group blockIdx.x. A place that no
// continuation took (token -1) goes on with token 0; its score of -inf keeps it out of later choices.
__global__ __launch_bounds__(64) void k_beam_advance(const int32_t *parent, const int32_t *token, int eos, int K, int32_t *done, int32_t *tok,
                                                     int32_t *pos, int32_t *hist, int hist_stride, int step) {
    const int j = threadIdx.x, i = blockIdx.x * K + j;
    int d = 0, t = -1;
    if (j < K) {
        const int p = parent[i];
        t = token[i];
        d = p >= 0 && p < K && (done[blockIdx.x * K + p] || t == eos);
    }
    __syncthreads(); // every parent's flag has been read
    if (j < K) {
        done[i] = d;
        tok[i] = t < 0 ? 0 : t;
        pos[i]++;
        hist[(int64_t)i * hist_stride + step] = t;
    }
}

} // namespace

extern "C" size_t qmh_beam_ws_bytes(const qmh_beam_args *a) {
    if (a->n_groups == 0) return 0; // no rows to divide the waves among
    const size_t lists = (size_t)a->n_groups * a->n_beams * plan_scan(a).segs;
    return lists * (sizeof(scan_head) + a->n_out * sizeof(uint2));
}

extern "C" int qmh_launch_beam_select(const qmh_beam_args *a, void *ws, void *stream) {
    hipStream_t st = (hipStream_t)stream;
    const scan_plan p = plan_scan(a);
    const int rows = a->n_groups * a->n_beams;
    scan_head *heads = (scan_head *)ws;
    uint2 *cands = (uint2 *)(heads + (size_t)rows * p.segs);
    qmh_for_type(a->dtype, [&](auto z) {
        using T = decltype(z);
        constexpr int VEC = 16 / sizeof(T);
        // rows over y in passes of at most 65535
        for (int r0 = 0; r0 < rows; r0 += 65535) {
            const dim3 g(p.segs / (SEL_T / 64), rows - r0 < 65535 ? rows - r0 : 65535);
            if (p.ept == 8) hipLaunchKernelGGL((k_beam_scan<T, 8, VEC>), g, dim3(SEL_T), 0, st, *a, heads, cands, r0, p.iters);
            else hipLaunchKernelGGL((k_beam_scan<T, SCAN_EPT, VEC>), g, dim3(SEL_T), 0, st, *a, heads, cands, r0, p.iters);
        }
    });
    const bool many = many_segments(a, p.segs);
    const dim3 g(a->n_groups);
    if (a->n_beams <= 8) {
        if (many) hipLaunchKernelGGL((k_beam_join<true, 512>), g, dim3(512), 0, st, *a, heads, cands, p.segs);
        else hipLaunchKernelGGL((k_beam_join<false, 512>), g, dim3(512), 0, st, *a, heads, cands, p.segs);
    } else {
        if (many) hipLaunchKernelGGL((k_beam_join<true, 1024>), g, dim3(1024), 0, st, *a, heads, cands, p.segs);
        else hipLaunchKernelGGL((k_beam_join<false, 1024>), g, dim3(1024), 0, st, *a, heads, cands, p.segs);
    }
    return (int)hipGetLastError();
}

template <typename U>
static int reorder_as(const qmh_beam_state *s, void *dst, const void *src, const int32_t *parent, int n_groups, int K,
                      hipStream_t st) {
    const int64_t row_units = (s->live + (int64_t)sizeof(U) - 1) / (int64_t)sizeof(U), units = row_units * s->n_rows;
    const int64_t per = (units + 255) / 256, blocks = per * n_groups * s->n_outer;
    if (row_units > 0x7fffffff || units > 0x7fffff00 || blocks > 0x7fffffff) return (int)hipErrorInvalidValue;
    const dim3 t(256);
    uint8_t *d = (uint8_t *)dst;
    const uint8_t *f = (const uint8_t *)src;
    const uint32_t ru = (uint32_t)row_units, p = (uint32_t)per;
    for (int64_t b0 = 0; b0 < blocks; b0 += QMH_MOST_BLOCKS) { // blocks move different bytes: any number of launches
        const dim3 g((uint32_t)(blocks - b0 < QMH_MOST_BLOCKS ? blocks - b0 : QMH_MOST_BLOCKS));
        const uint32_t b = (uint32_t)b0;
        if (K <= 4) hipLaunchKernelGGL((k_beam_reorder<U, 4>), g, t, 0, st, *s, d, f, parent, n_groups, K, ru, p, b);
        else if (K <= 8) hipLaunchKernelGGL((k_beam_reorder<U, 8>), g, t, 0, st, *s, d, f, parent, n_groups, K, ru, p, b);
        else if (K <= 16) hipLaunchKernelGGL((k_beam_reorder<U, 16>), g, t, 0, st, *s, d, f, parent, n_groups, K, ru, p, b);
        else if constexpr (sizeof(U) <= 4) hipLaunchKernelGGL((k_beam_reorder<U, 64>), g, t, 0, st, *s, d, f, parent, n_groups, K, ru, p, b);
    }
    return (int)hipGetLastError();
}

extern "C" int qmh_launch_beam_reorder(const qmh_beam_state *s, void *dst, const void *src, const int32_t *parent, int n_groups,
                                       int n_beams, void *stream) {
    hipStream_t st = (hipStream_t)stream;
    const uint64_t all = (uint64_t)(uintptr_t)dst | (uint64_t)(uintptr_t)src | (uint64_t)s->seq_stride |
                         (s->n_outer > 1 ? (uint64_t)s->outer_stride : 0) | (s->n_rows > 1 ? (uint64_t)s->row_stride : 0);
    // past 16 beams units are of 4 bytes, kept in LDS
    if (all % 16 == 0 && n_beams <= 16) return reorder_as<v4u>(s, dst, src, parent, n_groups, n_beams, st);
    if (all % 4 == 0) return reorder_as<uint32_t>(s, dst, src, parent, n_groups, n_beams, st);
    return reorder_as<uint8_t>(s, dst, src, parent, n_groups, n_beams, st);
}

extern "C" int qmh_launch_beam_advance(const int32_t *parent, const int32_t *token, int eos, int n_groups, int n_beams, int32_t *done,
                                       int32_t *tok, int32_t *pos, int32_t *hist, int hist_stride, int step, void *stream) {
    hipLaunchKernelGGL(k_beam_advance, dim3(n_groups), dim3(64), 0, (hipStream_t)stream, parent, token, eos, n_beams, done, tok, pos, hist,
                       hist_stride, step);
    return (int)hipGetLastError();
}
