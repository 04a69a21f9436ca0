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
constexpr int SEL_CAP = 512;  // candidates it ranks in LDS
constexpr int JOIN_T = 512;   // threads of the join
constexpr int JOIN_CAP = 1024;

// e^(x - ref) in 64 bits for x <= ref, both floats, ref finite: x log2 e - ref log2 e = k + f, |f| <= 1/2, and 2^k times the
// Taylor polynomial of 2^f to degree 10, whose remainder is below (ln 2 / 2)^11 / 11! = 2.2e-13 of the value: far
// inside the distance of scores that decide a choice. Adding 1.5 2^52 rounds to k and leaves it in the low word. Values
// below ref - 700 count as that.
__device__ __forceinline__ double exp_below(float x, float low, double ref2) {
    const double t = __builtin_fma((double)fmaxf(x, low), 1.4426950408889634074, -ref2);
    const double s = t + 0x1.8p52, f = t - (s - 0x1.8p52);
    double p = 7.0549116208011233299e-9;
    p = __builtin_fma(p, f, 1.0178086009239699728e-7);
    p = __builtin_fma(p, f, 1.3215486790144309488e-6);
    p = __builtin_fma(p, f, 1.5252733804059840280e-5);
    p = __builtin_fma(p, f, 1.5403530393381609954e-4);
    p = __builtin_fma(p, f, 1.3333558146428443423e-3);
    p = __builtin_fma(p, f, 9.6181291076284771619e-3);
    p = __builtin_fma(p, f, 5.5504108664821579953e-2);
    p = __builtin_fma(p, f, 2.4022650695910071233e-1);
    p = __builtin_fma(p, f, 6.9314718055994530942e-1);
    p = __builtin_fma(p, f, 1.0);
    return __hiloint2double(__double2hiint(p) + (__double2loint(s) << 20), __double2loint(p));
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

// the sum of n over the workgroup
__device__ __forceinline__ int block_total(int n, int *buf) {
    for (int s = 1; s < 64; s <<= 1) n += __shfl_xor(n, s);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) buf[threadIdx.x >> 6] = n;
    __syncthreads();
    return buf[0] + buf[1] + buf[2] + buf[3];
}

struct scan_head { // a wave's part of a chunk of a row: its maximum and the sum of exp(x - max); NaN: the row has none
    double sum;
    float max, pad;
};

// The largest t that at least n <= 64 of a wave's values reach, 0 if there is none above: bit by bit, by ballots.
__device__ __forceinline__ uint32_t wave_nth(uint32_t v, int n) {
    uint32_t t = 0;
#pragma unroll
    for (int b = 31; b >= 0; b--) {
        const uint32_t u = t | 1u << b;
        t = __popcll(__ballot(v >= u)) >= n ? u : t;
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
            for (int i = part; i < n; i += per) r += before(i, c);
        for (int x = 1; x < per; x *= 2) r += __shfl_xor(r, x);
        if (c < n && part == 0) done(c, r);
    }
}

// Chunk blockIdx.x (SEL_T * EPT logits) of a row: each wave's maximum and sum of exponentials below it, in 64 bits,
// and the chunk's n_out best logits in order. The logits stay in registers. Below the n_out-th largest of the lanes'
// own maxima in a wave nothing is among the best; what reaches the largest such bound of the four waves (a few times n_out,
// unless values repeat) is ranked by counting. Where more than SEL_CAP reach it, the exact bound is searched bit by bit.
template <typename T, int EPT, int VEC>
__global__ __launch_bounds__(SEL_T) void k_beam_scan(const qmh_beam_args a, scan_head *heads, uint2 *cands, int row0) {
    __shared__ uint2 cand[SEL_CAP];
    __shared__ int cnt[4], ncand;
    __shared__ uint32_t bounds[4];
    const int tid = threadIdx.x, w = tid >> 6, row = row0 + blockIdx.y, n_out = a.n_out;
    const int64_t slot = (int64_t)row * gridDim.x + blockIdx.x;
    if ((a.done && a.done[row]) || !(a.score[row] > -__builtin_inff())) return; // the join does not look at it
    const T *x = (const T *)a.logits + row * a.stride;
    // vectors from the row's start rounded down to a vector: the ones that hold some element of the row
    const int skew = VEC > 1 ? (int)(((uintptr_t)x / sizeof(T)) % VEC) : 0;
    const int base = (int)blockIdx.x * SEL_T * EPT - skew;
    float xs[EPT];
    {
        qmh_vec<T, VEC> v[EPT / VEC];
#pragma unroll
        for (int k = 0; k < EPT / VEC; k++) {
            const int i = base + (k * SEL_T + tid) * VEC;
            if (i + VEC > 0 && i < a.vocab) v[k] = *(const qmh_vec<T, VEC> *)(x + i);
        }
#pragma unroll
        for (int k = 0; k < EPT; k++) xs[k] = qmh_to_f(v[k / VEC].e[k % VEC]);
    }
    auto index = [&](int k) { return base + ((k / VEC) * SEL_T + tid) * VEC + k % VEC; };
    if (base < 0 || base + SEL_T * EPT > a.vocab) // the row's ends
#pragma unroll
        for (int k = 0; k < EPT; k++)
            if ((uint32_t)index(k) >= (uint32_t)a.vocab) xs[k] = -__builtin_inff();
    if (tid == 0) ncand = 0;
    float top = xs[0];
#pragma unroll
    for (int k = 1; k < EPT; k++) top = __builtin_elementwise_maximum(top, xs[k]); // NaN if one is
    const bool bad = __any(!(top < __builtin_inff()));
    const float m = qmh_wave_max(top), ref = m > -__builtin_inff() && m < __builtin_inff() ? m : 0.0f;
    // the bound first: it is short and the sums' latency hides in it
    uint32_t mine = key_of(top);
    if (bad) { // NaN hides the lane's maximum
        mine = 0;
#pragma unroll
        for (int k = 0; k < EPT; k++) {
            const uint32_t q = key_of(xs[k]);
            mine = q > mine ? q : mine;
        }
    }
    const uint32_t bw = wave_nth(mine, n_out);
    if ((tid & 63) == 0) bounds[w] = bw;
    const double ref2 = (double)ref * 1.4426950408889634074;
    const float low = ref - 700.0f;
    double sum = 0.0, sum2 = 0.0;
#pragma unroll
    for (int k = 0; k < EPT; k += 2) {
        sum += exp_below(xs[k], low, ref2);
        sum2 += exp_below(xs[k + 1], low, ref2);
    }
    sum = qmh_wave_sum_d(sum + sum2);
    __syncthreads();
    uint32_t from = bounds[0];
#pragma unroll
    for (int k = 1; k < 4; k++) from = bounds[k] > from ? bounds[k] : from;
    // as a float (at least the lowest finite one): -inf and NaN never reach it
    float at_least = of_key(from ? from : 0x00800000u);
    int reach = 0;
#pragma unroll
    for (int k = 0; k < EPT; k++) reach += xs[k] >= at_least;
    int at = reach ? atomicAdd(&ncand, reach) : 0;
    __syncthreads();
    int last = 0x7fffffff; // candidates equal to the bound: only up to this index
    if (ncand > SEL_CAP) {
        // the largest bound that n_out keys reach, then the lowest indexes among the keys equal to it
        from = 0;
        for (int b = 31; b >= 0; b--) {
            const uint32_t t = from | 1u << b;
            int n = 0;
#pragma unroll
            for (int k = 0; k < EPT; k++) n += key_of(xs[k]) >= t;
            if (block_total(n, cnt) >= n_out) from = t;
        }
        int above = 0;
#pragma unroll
        for (int k = 0; k < EPT; k++) above += key_of(xs[k]) > from;
        above = block_total(above, cnt);
        int lo = -1; // the largest index that leaves fewer than n_out
        for (int b = 24; b >= 0; b--) {
            const int t = lo + (1 << b);
            int n = 0;
#pragma unroll
            for (int k = 0; k < EPT; k++) n += key_of(xs[k]) == from && index(k) <= t;
            if (above + block_total(n, cnt) < n_out) lo = t;
        }
        last = lo + 1;
        at_least = of_key(from);
        if (tid == 0) ncand = 0;
        __syncthreads();
        reach = 0;
#pragma unroll
        for (int k = 0; k < EPT; k++) reach += key_of(xs[k]) > from || (key_of(xs[k]) == from && index(k) <= last);
        at = reach ? atomicAdd(&ncand, reach) : 0;
        __syncthreads();
    }
    if (reach)
#pragma unroll
        for (int k = 0; k < EPT; k++)
            if (xs[k] > at_least || (xs[k] == at_least && index(k) <= last)) cand[at++] = make_uint2(key_of(xs[k]), (uint32_t)index(k));
    __syncthreads();
    const int n = ncand;
    rank_all(
        n, SEL_T, [&](int i, int c) { return cand[i].x > cand[c].x || (cand[i].x == cand[c].x && cand[i].y < cand[c].y); },
        [&](int c, int r) {
            if (r < n_out) cands[slot * n_out + r] = cand[c];
        });
    if (tid >= n && tid < n_out) cands[slot * n_out + tid] = make_uint2(0, 0);
    if ((tid & 63) == 0) heads[slot * 4 + w] = scan_head{bad ? __builtin_nan("") : m > -__builtin_inff() ? sum : 0.0, m, 0.0f};
}

// A group's choice from its rows' chunks: each row's log sum (a wave a row), then the n_out best totals as in the scan:
// a bound from the lanes' best, what reaches it ranked in LDS. Where more than JOIN_CAP reach it, one after another.
__global__ __launch_bounds__(JOIN_T) void k_beam_join(const qmh_beam_args a, const scan_head *heads, const uint2 *cands, int chunks) {
    constexpr int NW = JOIN_T / 64;
    __shared__ double lse[64], score[64];
    __shared__ uint64_t ckey[JOIN_CAP], bk[NW];
    __shared__ uint32_t cplace[JOIN_CAP], bounds[NW], bf[NW];
    __shared__ int ncand;
    const int g = blockIdx.x, tid = threadIdx.x, w = tid >> 6, lane = tid & 63, K = a.n_beams, n_out = a.n_out;
    if (tid == 0) ncand = 0;
    for (int b = w; b < K; b += NW) {
        const int row = g * K + b;
        const float sc = a.score[row];
        const bool done = a.done && a.done[row];
        double s = __builtin_nan("");
        if (!done && sc > -__builtin_inff()) {
            const scan_head *h = heads + (int64_t)row * chunks * 4;
            float m = -__builtin_inff();
            for (int c = lane; c < chunks * 4; c += 64) m = fmaxf(m, h[c].max);
            m = qmh_wave_max(m);
            s = 0.0;
            const double ref2 = (double)m * 1.4426950408889634074;
            for (int c = lane; c < chunks * 4; c += 64) s = __builtin_fma(h[c].sum, exp_below(h[c].max, m - 700.0f, ref2), s);
            s = (double)m + log(qmh_wave_sum_d(s)); // a row without a logit: NaN or -inf, and no continuation
        }
        if (lane == 0) {
            lse[b] = s;
            score[b] = done ? -(double)sc : (double)sc;
            if (done) lse[b] = __builtin_inf(); // marks a finished row
        }
    }
    __syncthreads();
    // a wave's own rows: lane's j-th candidate of row b as an ordered key (0: none), its place beam * vocab + token
    const int per = chunks * n_out;
    auto key_at = [&](int b, int j, uint32_t &place) -> uint64_t {
        const double L = lse[b];
        if (L == __builtin_inf()) { // finished: one continuation
            place = (uint32_t)(b * a.vocab + a.eos);
            return j == 0 ? key_of_d(-score[b]) : 0ull;
        }
        const uint2 v = cands[(int64_t)(g * K + b) * per + j];
        place = (uint32_t)(b * a.vocab) + v.y;
        return v.x && L == L ? key_of_d(score[b] + ((double)of_key(v.x) - L)) : 0ull;
    };
    auto each = [&](auto body) {
        uint32_t place = 0;
        for (int b = w; b < K; b += NW) {
            for (int j = lane; j < per; j += 64) {
                const uint64_t q = key_at(b, j, place);
                if (q) body(q, place);
            }
        }
    };
    uint32_t mine = 0;
    each([&](uint64_t q, uint32_t) { mine = (uint32_t)(q >> 32) > mine ? (uint32_t)(q >> 32) : mine; });
    const uint32_t bw = wave_nth(mine, n_out);
    if (lane == 0) bounds[w] = bw;
    __syncthreads();
    uint32_t from = 1;
#pragma unroll
    for (int k = 0; k < NW; k++) from = bounds[k] > from ? bounds[k] : from;
    each([&](uint64_t q, uint32_t place) {
        if ((uint32_t)(q >> 32) < from) return;
        const int at = atomicAdd(&ncand, 1);
        if (at < JOIN_CAP) {
            ckey[at] = q;
            cplace[at] = place;
        }
    });
    __syncthreads();
    auto write = [&](int o, uint64_t k, uint32_t p) {
        const int64_t at = (int64_t)g * n_out + o;
        a.out_score[at] = k ? (float)of_key_d(k) : -__builtin_inff();
        a.out_parent[at] = k ? (int)(p / (uint32_t)a.vocab) : -1;
        a.out_token[at] = k ? (int)(p % (uint32_t)a.vocab) : -1;
    };
    const int n = ncand;
    if (n <= JOIN_CAP) { // every score has been read: out_score may be score
        rank_all(
            n, JOIN_T, [&](int i, int c) { return ckey[i] > ckey[c] || (ckey[i] == ckey[c] && cplace[i] < cplace[c]); },
            [&](int c, int r) {
                if (r < n_out) write(r, ckey[c], cplace[c]);
            });
        if (tid >= n && tid < n_out) write(tid, 0, 0);
        return;
    }
    uint64_t below = ~0ull; // what was chosen last: its total, then its place
    int64_t after = -1;
    for (int o = 0; o < n_out; o++) {
        uint64_t best = 0;
        uint32_t at = 0xffffffffu;
        each([&](uint64_t q, uint32_t place) {
            if (q > below || (q == below && (int64_t)place <= after)) return;
            if (q > best || (q == best && place < at)) {
                best = q;
                at = place;
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
            ckey[o] = best;
            cplace[o] = at;
        }
    }
    __syncthreads();
    if (tid < n_out) write(tid, ckey[tid], cplace[tid]);
}

int scan_chunks(const qmh_beam_args *a, int ept) { return (a->vocab + 15 + SEL_T * ept - 1) / (SEL_T * ept); }
// elements a thread holds: 8 spreads few rows over more workgroups, 32 leaves fewer candidates to the join
int scan_ept(const qmh_beam_args *a) { return (int64_t)a->n_groups * a->n_beams * scan_chunks(a, 8) <= 1024 ? 8 : 32; }

// --------------------------------------------------------------------------- reorder

// Thread: one unit of U (the widest that every row is aligned to) of one row, for all beams of a group. Every beam that
// takes another's state is read before any is written, so any parents move in place; a row's last bytes go in 4-byte
// pieces, read together too, and single bytes. parents: uniform, by scalar loads.
typedef const __attribute__((address_space(4))) int32_t *const_i32;
typedef uint32_t v4u __attribute__((ext_vector_type(4)));
template <typename U, int BM>
__global__ __launch_bounds__(256, BM > 16 ? 2 : 4) void k_beam_reorder(const qmh_beam_state s, uint8_t *dst, const uint8_t *src, const int32_t *parent,
                                                      uint32_t n_groups, int K, uint32_t row_units, uint32_t blocks_per) {
    const uint32_t og = blockIdx.x / blocks_per, ub = blockIdx.x - og * blocks_per;
    const uint32_t o = og / n_groups, g = og - o * n_groups;
    const uint32_t u = ub * 256 + threadIdx.x, r = u / row_units, c = u - r * row_units;
    const_i32 par = (const_i32)(uintptr_t)(parent + g * K);
    if constexpr (BM > 16) { // U is 1 or 4 bytes: a row's last bytes singly
        __shared__ U keep[64 * 256];
        if (r >= s.n_rows) return;
        const int64_t at = (int64_t)c * sizeof(U), base = o * s.outer_stride + (int64_t)g * K * s.seq_stride + r * s.row_stride + at;
        auto source = [&](int j) { return par[j] >= 0 && par[j] < K ? par[j] : j; };
        auto move = [&](auto z, U *slot, int64_t b) {
            using V = decltype(z);
            qmh_move_many(
                (V *)slot, K,
                [&](int j, V &u) {
                    if (source(j) == j && dst == src) return false;
                    u = *(const V *)(src + b + source(j) * s.seq_stride);
                    return true;
                },
                [&](int j, V u) {
                    if (source(j) != j || dst != src) *(V *)(dst + b + j * s.seq_stride) = u;
                });
        };
        if (at + (int64_t)sizeof(U) <= s.live) move(U{}, keep + threadIdx.x, base);
        else
            for (int64_t k = 0; at + k < s.live; k++) move(uint8_t{}, (U *)((uint8_t *)keep + threadIdx.x), base + k);
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

} // namespace

extern "C" size_t qmh_beam_ws_bytes(const qmh_beam_args *a) {
    const size_t slots = (size_t)a->n_groups * a->n_beams * scan_chunks(a, scan_ept(a));
    return slots * (4 * sizeof(scan_head) + a->n_out * sizeof(uint2));
}

extern "C" int qmh_launch_beam_select(const qmh_beam_args *a, void *ws, void *stream) {
    hipStream_t st = (hipStream_t)stream;
    const int rows = a->n_groups * a->n_beams, ept = scan_ept(a), chunks = scan_chunks(a, ept);
    scan_head *heads = (scan_head *)ws;
    uint2 *cands = (uint2 *)(heads + (size_t)rows * chunks * 4);
    qmh_for_type(a->dtype, [&](auto z) {
        using T = decltype(z);
        constexpr int VEC = 16 / sizeof(T);
        // rows over y in passes of at most 65535
        for (int r0 = 0; r0 < rows; r0 += 65535) {
            const dim3 g(chunks, rows - r0 < 65535 ? rows - r0 : 65535), t(SEL_T);
            if (ept == 8) hipLaunchKernelGGL((k_beam_scan<T, 8, VEC>), g, t, 0, st, *a, heads, cands, r0);
            else hipLaunchKernelGGL((k_beam_scan<T, 32, VEC>), g, t, 0, st, *a, heads, cands, r0);
        }
    });
    hipLaunchKernelGGL(k_beam_join, dim3(a->n_groups), dim3(JOIN_T), 0, st, *a, heads, cands, chunks);
    return (int)hipGetLastError();
}

template <typename U>
static int reorder_as(const qmh_beam_state *s, void *dst, const void *src, const int32_t *parent, int n_groups, int K,
                      hipStream_t st) {
    const int64_t row_units = (s->live + (int64_t)sizeof(U) - 1) / (int64_t)sizeof(U), units = row_units * s->n_rows;
    const int64_t per = (units + 255) / 256, blocks = per * n_groups * s->n_outer;
    if (row_units > 0x7fffffff || units > 0x7fffff00 || blocks > 0x7fffffff) return (int)hipErrorInvalidValue;
    const dim3 g((uint32_t)blocks), t(256);
    uint8_t *d = (uint8_t *)dst;
    const uint8_t *f = (const uint8_t *)src;
    const uint32_t ru = (uint32_t)row_units, p = (uint32_t)per;
    if (K <= 4) hipLaunchKernelGGL((k_beam_reorder<U, 4>), g, t, 0, st, *s, d, f, parent, n_groups, K, ru, p);
    else if (K <= 8) hipLaunchKernelGGL((k_beam_reorder<U, 8>), g, t, 0, st, *s, d, f, parent, n_groups, K, ru, p);
    else if (K <= 16) hipLaunchKernelGGL((k_beam_reorder<U, 16>), g, t, 0, st, *s, d, f, parent, n_groups, K, ru, p);
    else if constexpr (sizeof(U) <= 4) hipLaunchKernelGGL((k_beam_reorder<U, 64>), g, t, 0, st, *s, d, f, parent, n_groups, K, ru, p);
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
