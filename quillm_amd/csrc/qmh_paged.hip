// gfx950 kernels of a paged KV cache: qmh_paged_append (per-head norms, position rotation, rows into pages),
// qmh_paged_attention (a shared prefix and each sequence's own pages) and qmh_paged_reorder. No reference
// counterpart; accuracy as the declarations state, not bitwise.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "qmh_device.h"
#include "qmh_launch.h"
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

// One wave takes one token's heads, 64 / lanes of them at a time. A lane holds a unit of a head: two vectors of VW
// elements, whose elements pair up in the rotated part (HALVES: VW elements of each half; PAIRS: 2 VW elements in
// a row) and follow one another behind it. So both layouts turn in registers, a head's sum of squares is one
// reduction over its lanes, and the sines and cosines of a lane's pairs are made once for all heads of the token:
// position 1024 h + l is turned by the angle sum of two table rows, in 64 bits. IT: units of a lane (2 only for
// one-element vectors of heads past 128).
template <typename T, int VW, int IT>
__global__ __launch_bounds__(256) void k_paged_append(const append_args s) {
    const qmh_append_args &a = s.a;
    const int wave = __builtin_amdgcn_readfirstlane((int)(blockIdx.x * 4 + (threadIdx.x >> 6)));
    const int lane = threadIdx.x & 63, t = wave / s.split, part = wave - t * s.split;
    if (t >= a.n_tokens) return;
    const int hd = s.p.head_dim, KV = s.p.n_kv_heads, H = a.q ? a.n_heads : 0, NH = H + (a.k ? 2 * KV : 0);
    const int half = s.r.pairs, rot = 2 * half;
    const int pos = a.pos ? a.pos[t] : a.slot ? a.slot[t] : 0;
    if (half && (pos < 0 || pos >= s.r.max_pos)) return;
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
    int at0[IT], at1[IT];
    float c[IT][VW], w[IT][VW];
#pragma unroll
    for (int k = 0; k < IT; k++) {
        const int u = l + k * s.lanes;
        const bool turn = u * VW < half;
        at0[k] = !turn ? rot + 2 * (u * VW - half) : s.r.layout == QMH_ROTARY_HALVES ? u * VW : 2 * u * VW;
        at1[k] = turn && s.r.layout == QMH_ROTARY_HALVES ? at0[k] + half : at0[k] + VW;
#pragma unroll
        for (int i = 0; i < VW; i++) {
            c[k][i] = 1.0f;
            w[k][i] = 0.0f;
            if (turn) {
                const int pr = u * VW + i;
                const double2 hi = ((const double2 *)s.r.hi)[(int64_t)(pos / QMH_ROTARY_LO) * half + pr];
                const double2 lo = ((const double2 *)s.r.lo)[(int64_t)(pos % QMH_ROTARY_LO) * half + pr];
                c[k][i] = (float)__builtin_fma(hi.x, lo.x, -(hi.y * lo.y));
                w[k][i] = (float)__builtin_fma(hi.y, lo.x, hi.x * lo.y);
            }
        }
    }
    const bool pairs = s.r.layout == QMH_ROTARY_PAIRS;
    for (int h0 = part * per; h0 < NH; h0 += s.split * per) {
        const int h = h0 + lane / s.lanes;
        if (h >= NH) continue;
        const int kind = h < H ? 0 : h < H + KV ? 1 : 2;
        const int g = kind == 0 ? h : kind == 1 ? h - H : h - H - KV;
        const T *src;
        T *dst;
        if (kind == 0) {
            src = (const T *)a.q + t * a.q_stride + g * hd;
            dst = (T *)a.q_out + t * a.q_out_stride + g * hd;
        } else {
            src = kind == 1 ? (const T *)a.k + t * a.k_stride + g * hd : (const T *)a.v + t * a.v_stride + g * hd;
            dst = (kind == 1 ? (T *)s.p.k : (T *)s.p.v) + (row0 + (int64_t)g * ps) * hd;
        }
        qmh_vec<T, VW> v0[IT], v1[IT];
#pragma unroll
        for (int k = 0; k < IT; k++)
            if (l + k * s.lanes < units) {
                v0[k] = *(const qmh_vec<T, VW> *)(src + at0[k]);
                v1[k] = *(const qmh_vec<T, VW> *)(src + at1[k]);
            }
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
                        // the i-th pair of the unit: element i of both vectors, or two neighbours
                        T *px = &v0[k].e[i], *py = &v1[k].e[i];
                        int ex = at0[k] + i, ey = at1[k] + i;
                        if (pairs && VW > 1) {
                            px = 2 * i < VW ? &v0[k].e[(2 * i) % VW] : &v1[k].e[(2 * i) % VW];
                            py = 2 * i < VW ? &v0[k].e[(2 * i + 1) % VW] : &v1[k].e[(2 * i + 1) % VW];
                            ex = at0[k] + 2 * i;
                            ey = ex + 1;
                        }
                        float x = qmh_to_f(*px), y = qmh_to_f(*py);
                        if (gain) {
                            x = x * inv * gain[ex];
                            y = y * inv * gain[ey];
                        }
                        *px = (T)__builtin_fmaf(x, c[k][i], -(y * w[k][i]));
                        *py = (T)__builtin_fmaf(x, w[k][i], y * c[k][i]);
                    }
                }
                *(qmh_vec<T, VW> *)(dst + at0[k]) = v0[k];
                *(qmh_vec<T, VW> *)(dst + at1[k]) = v1[k];
            }
    }
}

// --------------------------------------------------------------------------- attention

// One wave per (row of queries, head): 64 positions at a time, a lane's score each, then the lanes over head_dim.
template <typename T>
__global__ __launch_bounds__(256) void k_paged_attention(const qmh_attention_args a, const qmh_pages p) {
    const int wave = __builtin_amdgcn_readfirstlane((int)(blockIdx.x * 4 + (threadIdx.x >> 6))), lane = threadIdx.x & 63;
    const int row = wave / a.n_heads, h = wave - row * a.n_heads;
    if (row >= a.n_seq * a.q_len) return;
    const int hd = p.head_dim, ps = p.page_size, KV = p.n_kv_heads, kvh = h / (a.n_heads / KV);
    const int sq = row / a.q_len, j = row - sq * a.q_len, g = sq / (a.n_seq / a.n_groups);
    const T *q = (const T *)a.q + row * a.q_stride + h * hd;
    float m = -__builtin_inff(), l = 0.0f, acc[4] = {0.f, 0.f, 0.f, 0.f};
    bool bad = false;
    for (int own = 0; own < 2; own++) {
        const int most = own ? a.max_len : a.max_prefix;
        if (!most) continue;
        const int all = own ? a.len[sq] : a.prefix_len[g];
        if (all < 0 || all > most) {
            bad = true;
            continue;
        }
        const int n = own ? all - a.q_len + 1 + j : all;
        const int32_t *tab = own ? a.table + (int64_t)sq * a.table_stride : a.prefix_table + (int64_t)g * a.prefix_stride;
        for (int t0 = 0; t0 < n; t0 += 64) {
            const int t = t0 + lane < n ? t0 + lane : n - 1;
            int page = tab[t / ps];
            if (page < 0 || page >= p.n_pages) {
                bad = true;
                page = 0;
            }
            const int64_t at = (((int64_t)page * KV + kvh) * ps + t % ps) * hd;
            const T *k = (const T *)p.k + at;
            float s = 0.0f;
            for (int d = 0; d < hd; d++) s = __builtin_fmaf(qmh_to_f(q[d]), qmh_to_f(k[d]), s);
            s = t0 + lane < n ? s * a.scale : -__builtin_inff();
            float mn = fmaxf(m, qmh_wave_max(s));
            const float ref = mn == -__builtin_inff() ? 0.0f : mn;
            const float e = expf(s - ref), f = expf(m - ref);
            m = mn;
            l *= f;
            for (int i = 0; i < 4; i++) acc[i] *= f;
            for (int i = 0; i < 64 && t0 + i < n; i++) {
                const float pi = __shfl(e, i);
                const int64_t ai = __shfl(at, i);
                l += pi;
                for (int c = 0; c < 4; c++)
                    if (lane + 64 * c < hd) acc[c] = __builtin_fmaf(pi, qmh_to_f(((const T *)p.v)[ai + lane + 64 * c]), acc[c]);
            }
        }
    }
    if (__any(bad)) l = __builtin_nanf("");
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    T *out = (T *)a.out + row * a.out_stride + h * hd;
    for (int c = 0; c < 4; c++)
        if (lane + 64 * c < hd) out[lane + 64 * c] = (T)(acc[c] * inv);
}

// --------------------------------------------------------------------------- reorder

// A block moves a 4 KiB piece (V16: 16-byte units, else 4-byte ones and 1 KiB) of one page and kv head of k or v for
// all beams of a group: a thread reads its unit of every beam that takes another's state, then writes them, so any
// parents are moved in place. BM: most beams.
template <typename U, int BM>
__global__ __launch_bounds__(256) void k_paged_reorder(const qmh_pages p, const int32_t *__restrict__ table, int table_stride,
                                                       const int32_t *__restrict__ len, int max_len,
                                                       const int32_t *__restrict__ parent, int K, int n_pi, int subs, int row_bytes) {
    // block: ((group * pages + page index) * kv heads + head) * 2 + (k, v)) * subs + piece
    uint32_t b = blockIdx.x;
    const int sub = b % subs;
    b /= subs;
    const int isv = b & 1;
    b >>= 1;
    const int head = b % p.n_kv_heads;
    b /= p.n_kv_heads;
    const int pi = b % n_pi, g = b / n_pi;
    const int64_t piece = (int64_t)p.page_size * row_bytes;
    const int64_t off = ((int64_t)sub * 256 + threadIdx.x) * (int64_t)sizeof(U);
    if (off >= piece) return;
    const int t = pi * p.page_size + (int)(off / row_bytes);
    uint8_t *base = (uint8_t *)(isv ? p.v : p.k) + head * piece + off;
    const int64_t page_bytes = piece * p.n_kv_heads;
    U v[BM];
    uint64_t moves = 0;
#pragma unroll
    for (int j = 0; j < BM; j++) {
        if (j >= K) break;
        const int i = g * K + j, from = parent[i];
        if (from < 0 || from >= K || from == j) continue;
        int n = len[g * K + from];
        n = n < max_len ? n : max_len;
        if (t >= n) continue;
        const int ps = table[(int64_t)(g * K + from) * table_stride + pi], pd = table[(int64_t)i * table_stride + pi];
        if (ps < 0 || ps >= p.n_pages || pd < 0 || pd >= p.n_pages) continue;
        v[j] = *(const U *)(base + ps * page_bytes);
        moves |= 1ull << j;
    }
#pragma unroll
    for (int j = 0; j < BM; j++) {
        if (j >= K) break;
        if (moves >> j & 1) *(U *)(base + table[(int64_t)(g * K + j) * table_stride + pi] * page_bytes) = v[j];
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
    // few tokens: their heads over several waves, as many as there are passes; many: one wave each
    s.split = 1;
    while (s.split < passes && (int64_t)s.split * a->n_tokens < 4096) s.split++;
    const int64_t blocks = ((int64_t)a->n_tokens * s.split + 3) / 4;
    qmh_for_type(s.p.dtype, [&](auto z) {
        using T = decltype(z);
        const dim3 g((uint32_t)blocks), t(256);
        hipStream_t st = (hipStream_t)stream;
        if (units > 64) hipLaunchKernelGGL((k_paged_append<T, 1, 2>), g, t, 0, st, s);
        else if (vw == 1) hipLaunchKernelGGL((k_paged_append<T, 1, 1>), g, t, 0, st, s);
        else if (vw == 2) hipLaunchKernelGGL((k_paged_append<T, 2, 1>), g, t, 0, st, s);
        else if (vw == 4) hipLaunchKernelGGL((k_paged_append<T, 4, 1>), g, t, 0, st, s);
        else if constexpr (sizeof(T) == 2) hipLaunchKernelGGL((k_paged_append<T, 8, 1>), g, t, 0, st, s);
    });
    return (int)hipGetLastError();
}

extern "C" size_t qmh_attention_ws_bytes(const qmh_attention_args *a, int cus) {
    (void)a;
    (void)cus;
    return 0;
}

extern "C" int qmh_launch_paged_attention(const qmh_attention_args *a, int cus, void *ws, void *stream) {
    (void)cus;
    (void)ws;
    const int64_t waves = (int64_t)a->n_seq * a->q_len * a->n_heads;
    if (waves > 0x7fffffff - 4) return (int)hipErrorInvalidValue;
    qmh_for_type(a->pages->dtype, [&](auto z) {
        hipLaunchKernelGGL((k_paged_attention<decltype(z)>), dim3((uint32_t)((waves + 3) / 4)), dim3(256), 0, (hipStream_t)stream,
                           *a, *a->pages);
    });
    return (int)hipGetLastError();
}

extern "C" int qmh_launch_paged_reorder(const qmh_pages *p, const int32_t *table, int table_stride, const int32_t *len,
                                        int max_len, const int32_t *parent, int n_groups, int n_beams, void *stream) {
    const int row_bytes = p->head_dim * (p->dtype == QMH_F32 ? 4 : 2), unit = n_beams <= 16 ? 16 : 4;
    const int n_pi = (max_len + p->page_size - 1) / p->page_size;
    const int subs = (int)(((int64_t)p->page_size * row_bytes / unit + 255) / 256);
    const int64_t blocks = (int64_t)n_groups * n_pi * p->n_kv_heads * 2 * subs;
    if (blocks > 0x7fffffff) return (int)hipErrorInvalidValue;
    const dim3 g((uint32_t)blocks), t(256);
    hipStream_t st = (hipStream_t)stream;
    if (n_beams <= 4)
        hipLaunchKernelGGL((k_paged_reorder<uint4, 4>), g, t, 0, st, *p, table, table_stride, len, max_len, parent, n_beams, n_pi, subs, row_bytes);
    else if (n_beams <= 8)
        hipLaunchKernelGGL((k_paged_reorder<uint4, 8>), g, t, 0, st, *p, table, table_stride, len, max_len, parent, n_beams, n_pi, subs, row_bytes);
    else if (n_beams <= 16)
        hipLaunchKernelGGL((k_paged_reorder<uint4, 16>), g, t, 0, st, *p, table, table_stride, len, max_len, parent, n_beams, n_pi, subs, row_bytes);
    else
        hipLaunchKernelGGL((k_paged_reorder<uint32_t, 64>), g, t, 0, st, *p, table, table_stride, len, max_len, parent, n_beams, n_pi, subs, row_bytes);
    return (int)hipGetLastError();
}
