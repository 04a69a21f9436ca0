// gfx950 kernels of a paged KV cache: qmh_paged_append (per-head norms, position rotation, rows into pages),
// qmh_paged_attention (a shared prefix and each sequence's own pages) and qmh_paged_reorder. No reference
// counterpart; accuracy as the declarations state, not bitwise.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "qmh_device.h"
#include "qmh_launch.h"
#include "qmh_paged_attn.h"
#include "qmh_types.h"

namespace {

// --------------------------------------------------------------------------- append

struct append_args {
    qmh_append_args a;
    qmh_pages p;
    qmh_rotary_tables r; // pairs 0: no rotation
    int split;           // waves per token
    int lanes;           // lanes per head, a power of two
};

// One wave takes one token's heads (or a share of them), 64 / lanes of them at a time, the next ones' loads under way.
// A lane holds a unit of a head: two vectors of VW elements, whose elements pair up in the rotated part (halves: VW elements
// of each half; PAIRS: 2 VW elements in a row) and follow one another behind it. So both layouts turn in
// registers and a head's sum of squares is one reduction over its lanes. The sines and cosines are made once for all
// heads of the token, a pair a lane, and handed round: position 1024 h + l is turned by the angle sum of two
// table rows, in 64 bits, rounded to 32 at the end. IT: units of a lane (2 only for one-element vectors of heads past 128).
// Bound by the rows' bytes: 4001 tokens of (32 + 2 x 32) x 128 f16 take 41 us (197 MB, 4.75 TB/s; a large copy reaches 5.1).
template <typename T, int VW, int IT, bool PAIRS>
__global__ __launch_bounds__(256) void k_paged_append(const append_args s) {
    const qmh_append_args &a = s.a;
    const int wave = __builtin_amdgcn_readfirstlane((int)(blockIdx.x * 4 + (threadIdx.x >> 6)));
    const int lane = threadIdx.x & 63, t = wave / s.split, part = wave - t * s.split;
    if (t >= a.n_tokens) return;
    const int hd = s.p.head_dim, KV = s.p.n_kv_heads, H = a.q ? a.n_heads : 0, NH = H + (a.k ? 2 * KV : 0);
    const int half = s.r.pairs, rot = 2 * half;
    const int pos = a.pos ? a.pos[t] : a.slot ? a.slot[t] : 0;
    if (pos < 0 || (half && pos >= s.r.max_pos)) return; // padding, rotated or not
    int64_t row0 = 0; // the token's row of its page, for kv head 0
    int ps = 0;
    if (a.k) {
        const int sq = a.seq[t], sl = a.slot[t];
        ps = s.p.page_size;
        if (sq < 0 || sq >= a.n_seq || sl < 0 || sl >= a.table_stride * ps) return;
        const int page = a.table[(int64_t)sq * a.table_stride + sl / ps];
        if (page < 0 || page >= s.p.n_pages) return;
        row0 = (int64_t)page * KV * ps + sl % ps;
    }
    const int l = lane & (s.lanes - 1), per = 64 / s.lanes, units = hd / (2 * VW);
    // the token's sines and cosines, pair p (and p + 64) by lane p; each lane then takes those of its unit
    float cp[2] = {1.0f, 1.0f}, wp[2] = {0.0f, 0.0f};
#pragma unroll
    for (int k = 0; k < 2; k++) {
        const int pr = lane + 64 * k;
        if (pr < half) {
            const double2 hi = ((const double2 *)s.r.hi)[(int64_t)(pos / QMH_ROTARY_LO) * half + pr];
            const double2 lo = ((const double2 *)s.r.lo)[(int64_t)(pos % QMH_ROTARY_LO) * half + pr];
            cp[k] = (float)__builtin_fma(hi.x, lo.x, -(hi.y * lo.y));
            wp[k] = (float)__builtin_fma(hi.y, lo.x, hi.x * lo.y);
        }
    }
    int at0[IT], at1[IT];
    float c[IT][VW], w[IT][VW];
    bool turns[IT]; // a unit that does not is left out of the products: an infinite element would reach its neighbour through a sine of 0
#pragma unroll
    for (int k = 0; k < IT; k++) {
        const int u = l + k * s.lanes;
        const bool turn = turns[k] = u * VW < half;
        at0[k] = !turn ? rot + 2 * (u * VW - half) : PAIRS ? 2 * u * VW : u * VW;
        at1[k] = turn && !PAIRS ? at0[k] + half : at0[k] + VW;
#pragma unroll
        for (int i = 0; i < VW; i++) {
            const int pr = u * VW + i;
            c[k][i] = __shfl(cp[0], pr & 63);
            w[k][i] = __shfl(wp[0], pr & 63);
            if (half > 64) {
                const float c1 = __shfl(cp[1], pr & 63), w1 = __shfl(wp[1], pr & 63);
                c[k][i] = pr < 64 ? c[k][i] : c1;
                w[k][i] = pr < 64 ? w[k][i] : w1;
            }
        }
    }
    // a head's row by its number: queries, keys, values
    auto source = [&](int h) {
        if (h < H) return (const T *)a.q + t * a.q_stride + h * hd;
        return h < H + KV ? (const T *)a.k + t * a.k_stride + (h - H) * hd : (const T *)a.v + t * a.v_stride + (h - H - KV) * hd;
    };
    qmh_vec<T, VW> v0[IT], v1[IT], n0[IT], n1[IT]; // this head's unit and the next one's, on its way
    auto fetch = [&](int h) {
        if (h >= NH) return;
        const T *src = source(h);
#pragma unroll
        for (int k = 0; k < IT; k++)
            if (l + k * s.lanes < units) {
                n0[k] = *(const qmh_vec<T, VW> *)(src + at0[k]);
                n1[k] = *(const qmh_vec<T, VW> *)(src + at1[k]);
            }
    };
    const int step = s.split * per;
    for (int h = part * per + lane / s.lanes, first = 1; h - lane / s.lanes < NH; h += step, first = 0) {
        if (first) fetch(h);
#pragma unroll
        for (int k = 0; k < IT; k++) {
            v0[k] = n0[k];
            v1[k] = n1[k];
        }
        fetch(h + step);
        if (h >= NH) continue;
        const int kind = h < H ? 0 : h < H + KV ? 1 : 2;
        const int g = kind == 0 ? h : kind == 1 ? h - H : h - H - KV;
        T *dst = kind == 0 ? (T *)a.q_out + t * a.q_out_stride + g * hd : (kind == 1 ? (T *)s.p.k : (T *)s.p.v) + (row0 + (int64_t)g * ps) * hd;
        const float *gain = kind == 0 ? a.q_gain : kind == 1 ? a.k_gain : nullptr;
        float inv = 1.0f;
        if (a.q_gain || a.k_gain) { // every lane takes part in the exchange
            float ss = 0.0f;
#pragma unroll
            for (int k = 0; k < IT; k++)
                if (l + k * s.lanes < units)
#pragma unroll
                    for (int i = 0; i < VW; i++) {
                        const float x = qmh_to_f(v0[k].e[i]), y = qmh_to_f(v1[k].e[i]);
                        ss = __builtin_fmaf(x, x, __builtin_fmaf(y, y, ss));
                    }
            for (int o = 1; o < s.lanes; o <<= 1) ss += __shfl_xor(ss, o);
            inv = 1.0f / sqrtf(ss / (float)hd + a.eps);
        }
#pragma unroll
        for (int k = 0; k < IT; k++)
            if (l + k * s.lanes < units) {
                if (kind != 2) { // values go as they are
#pragma unroll
                    for (int i = 0; i < VW; i++) {
                        // the i-th pair of the unit: two neighbours, or element i of both vectors
                        constexpr bool NB = PAIRS && VW > 1;
                        qmh_vec<T, VW> &vx = NB && 2 * i >= VW ? v1[k] : v0[k], &vy = NB && 2 * i < VW ? v0[k] : v1[k];
                        const int ix = NB ? (2 * i) % VW : i, iy = NB ? (2 * i + 1) % VW : i;
                        const int ex = NB ? at0[k] + 2 * i : at0[k] + i, ey = NB ? at0[k] + 2 * i + 1 : at1[k] + i;
                        float x = qmh_to_f(vx.e[ix]), y = qmh_to_f(vy.e[iy]);
                        if (gain) {
                            x = x * inv * gain[ex];
                            y = y * inv * gain[ey];
                        }
                        const float xt = __builtin_fmaf(x, c[k][i], -(y * w[k][i])), yt = __builtin_fmaf(x, w[k][i], y * c[k][i]);
                        vx.e[ix] = (T)(turns[k] ? xt : x);
                        vy.e[iy] = (T)(turns[k] ? yt : y);
                    }
                }
                *(qmh_vec<T, VW> *)(dst + at0[k]) = v0[k];
                *(qmh_vec<T, VW> *)(dst + at1[k]) = v1[k];
            }
    }
}

// --------------------------------------------------------------------------- reorder

// A block moves 256 units of one page index of k or v, all kv heads in a row, for all beams of a group. The beams that
// take another's state are listed first (by one wave, a beam a lane, so the chain parent -> length and pages ->
// data is walked once); then a thread reads its unit of all of them before it writes any, so any parents move in
// place. BM: most beams; past 16 in units of 4 bytes through LDS. Measured: 48 us for 8 groups of 6 beams, 3 of them moved,
// 451 positions of 32 x 128 f16 (236 MB, 4.9 TB/s; a large copy reaches 5.1); 52, 55 and 56 with 2, 4 and 8 units a thread.
template <typename U, int BM>
__global__ __launch_bounds__(256) void k_paged_reorder(const qmh_pages p, const int32_t *__restrict__ table, int table_stride,
                                                       const int32_t *__restrict__ len, int max_len,
                                                       const int32_t *__restrict__ parent, int K, uint32_t n_pi, uint32_t subs, uint32_t row_bytes, uint32_t first) {
    __shared__ int2 from_to[64];
    __shared__ int live[64], count, least;
    // block: ((group * page indexes + page index) * 2 + (k, v)) * subs + piece
    const uint32_t b = blockIdx.x + first;
    const uint32_t rest = b / subs, sub = b - rest * subs, gp = rest >> 1, g = gp / n_pi, pi = gp - g * n_pi;
    if (threadIdx.x < 64) {
        const int j = threadIdx.x, from = j < K ? parent[g * K + j] : -1;
        int n = 0;
        int2 ft = make_int2(-1, -1);
        if (from >= 0 && from < K && from != j) {
            n = len[g * K + from];
            n = n < 0 ? 0 : n < max_len ? n : max_len;
            n -= (int)(pi * p.page_size); // positions of this page
            n = n < p.page_size ? n : p.page_size;
            if (n > 0) ft = make_int2(table[(int64_t)(g * K + from) * table_stride + pi], table[(int64_t)(g * K + j) * table_stride + pi]);
        }
        const bool moves = n > 0 && ft.x >= 0 && ft.x < p.n_pages && ft.y >= 0 && ft.y < p.n_pages;
        const uint64_t all = __ballot(moves);
        if (moves) {
            const int at = __popcll(all & ((1ull << j) - 1));
            from_to[at] = ft;
            live[at] = n;
        }
        const uint64_t part = __ballot(moves && n < p.page_size);
        if (j == 0) {
            count = __popcll(all);
            least = part ? 0 : p.page_size;
        }
    }
    __syncthreads();
    const int nm = uniform(count);
    if (nm == 0) return;
    const bool whole = uniform(least) != 0;
    uint8_t *pool = (uint8_t *)((rest & 1) ? p.v : p.k);
    const uint32_t page_bytes = (uint32_t)p.n_kv_heads * p.page_size * row_bytes; // up to 2^30
    const uint32_t off = (sub * 256 + threadIdx.x) * (uint32_t)sizeof(U);
    if (off >= page_bytes) return;
    const int t = whole ? 0 : (int)((off / row_bytes) & (p.page_size - 1));
    if constexpr (BM > 16) {
        __shared__ U keep[64 * 256];
        qmh_move_many(
            keep + threadIdx.x, nm,
            [&](int m, U &u) {
                if (t >= live[m]) return false;
                u = *(const U *)(pool + (int64_t)uniform(from_to[m].x) * page_bytes + off);
                return true;
            },
            [&](int m, U u) {
                if (t < live[m]) *(U *)(pool + (int64_t)uniform(from_to[m].y) * page_bytes + off) = u;
            });
        return;
    }
    // M beams: exactly, or (EXACT false) at most
    auto move = [&](auto mm, auto exact) {
        constexpr int M = decltype(mm)::value;
        constexpr bool EXACT = decltype(exact)::value;
        U v[M];
#pragma unroll
        for (int m = 0; m < M; m++)
            if ((EXACT || m < nm) && t < live[m]) v[m] = *(const U *)(pool + (int64_t)uniform(from_to[m].x) * page_bytes + off);
#pragma unroll
        for (int m = 0; m < M; m++)
            if ((EXACT || m < nm) && t < live[m]) *(U *)(pool + (int64_t)uniform(from_to[m].y) * page_bytes + off) = v[m];
    };
    switch (nm) {
    case 1: move(std::integral_constant<int, 1>{}, std::true_type{}); break;
    case 2: move(std::integral_constant<int, 2>{}, std::true_type{}); break;
    case 3: move(std::integral_constant<int, 3>{}, std::true_type{}); break;
    case 4: move(std::integral_constant<int, 4>{}, std::true_type{}); break;
    default: move(std::integral_constant<int, BM <= 16 ? BM : 1>{}, std::false_type{}); break;
    }
}

} // namespace

extern "C" int qmh_launch_paged_append(const qmh_append_args *a, const qmh_rotary_tables *r, int vw, void *stream) {
    append_args s;
    s.a = *a;
    s.p = *a->pages;
    if (r) s.r = *r;
    else s.r = qmh_rotary_tables{nullptr, nullptr, 0, QMH_ROTARY_PAIRS, 0};
    const int units = s.p.head_dim / (2 * vw), nh = (a->q ? a->n_heads : 0) + (a->k ? 2 * s.p.n_kv_heads : 0);
    s.lanes = 1;
    while (s.lanes < units && s.lanes < 64) s.lanes <<= 1;
    const int passes = (nh * s.lanes + 63) / 64;
    // a token's heads over several waves, down to one pass each, while that still adds waves to the chip (8 on each of
    // its 1024 SIMDs, three rounds of them): 4001 tokens of 96 x 128 f16 take 44, 43, 42 and 41 us in 4001, 8002, 16004 and
    // 24006 waves
    s.split = 1;
    while (s.split < passes && (int64_t)s.split * a->n_tokens < 24576) s.split++;
    const int64_t blocks = ((int64_t)a->n_tokens * s.split + 3) / 4;
    qmh_for_type(s.p.dtype, [&](auto z) {
        using T = decltype(z);
        const dim3 g((uint32_t)blocks), t(256);
        hipStream_t st = (hipStream_t)stream;
        auto go = [&](auto layout) {
            constexpr bool P = decltype(layout)::value;
            if (units > 64) hipLaunchKernelGGL((k_paged_append<T, 1, 2, P>), g, t, 0, st, s);
            else if (vw == 1) hipLaunchKernelGGL((k_paged_append<T, 1, 1, P>), g, t, 0, st, s);
            else if (vw == 2) hipLaunchKernelGGL((k_paged_append<T, 2, 1, P>), g, t, 0, st, s);
            else if (vw == 4) hipLaunchKernelGGL((k_paged_append<T, 4, 1, P>), g, t, 0, st, s);
            else if constexpr (sizeof(T) == 2) hipLaunchKernelGGL((k_paged_append<T, 8, 1, P>), g, t, 0, st, s);
        };
        if (s.r.layout == QMH_ROTARY_PAIRS) go(std::true_type{});
        else go(std::false_type{});
    });
    return (int)hipGetLastError();
}

extern "C" size_t qmh_attention_ws_bytes(const qmh_attention_args *a, int cus) {
    return attention_ws<false>(a, (int64_t)a->n_seq * a->q_len, cus);
}

extern "C" int qmh_launch_paged_attention(const qmh_attention_args *a, int cus, void *ws, void *stream) {
    const attn_tree none = {a->n_seq * a->q_len, nullptr, nullptr, 0, 0};
    return run_attention<false>(a, none, cus, ws, (hipStream_t)stream);
}

extern "C" int qmh_launch_paged_reorder(const qmh_pages *p, const int32_t *table, int table_stride, const int32_t *len,
                                        int max_len, const int32_t *parent, int n_groups, int n_beams, void *stream) {
    const int row_bytes = p->head_dim * (p->dtype == QMH_F32 ? 4 : 2), unit = n_beams <= 16 ? 16 : 4;
    const int n_pi = (max_len + p->page_size - 1) / p->page_size;
    const int64_t page_bytes = (int64_t)p->n_kv_heads * p->page_size * row_bytes;
    const int64_t subs = (page_bytes + 256 * unit - 1) / (256 * unit), blocks = (int64_t)n_groups * n_pi * 2 * subs;
    if (blocks > 0x7fffffff) return (int)hipErrorInvalidValue;
    const dim3 t(256);
    hipStream_t st = (hipStream_t)stream;
    for (int64_t b0 = 0; b0 < blocks; b0 += QMH_MOST_BLOCKS) { // blocks move different bytes: any number of launches
        const dim3 g((uint32_t)(blocks - b0 < QMH_MOST_BLOCKS ? blocks - b0 : QMH_MOST_BLOCKS));
        const uint32_t b = (uint32_t)b0;
        if (n_beams <= 8)
            hipLaunchKernelGGL((k_paged_reorder<v4u, 8>), g, t, 0, st, *p, table, table_stride, len, max_len, parent, n_beams, n_pi, subs, row_bytes, b);
        else if (n_beams <= 16)
            hipLaunchKernelGGL((k_paged_reorder<v4u, 16>), g, t, 0, st, *p, table, table_stride, len, max_len, parent, n_beams, n_pi, subs, row_bytes, b);
        else
            hipLaunchKernelGGL((k_paged_reorder<uint32_t, 64>), g, t, 0, st, *p, table, table_stride, len, max_len, parent, n_beams, n_pi, subs, row_bytes, b);
    }
    return (int)hipGetLastError();
}
