// gfx950 kernels of a paged KV cache: qmh_paged_append (per-head norms, position rotation, rows into pages),
// qmh_paged_attention (a shared prefix and each sequence's own pages) and qmh_paged_reorder. No reference
// counterpart; accuracy as the declarations state, not bitwise.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

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

// --------------------------------------------------------------------------- attention
//
// A wave holds 16 NR rows of queries (a row: one query of one head; rows that share keys lie together: a group's
// sequences for the prefix, a sequence's queries and the heads of its kv head for its own pages) and walks positions, KS at a time,
// with the running maximum and sum of a softmax. Both products are MFMAs on registers alone, no LDS:
//   S^T = K Q^T   16x16 tiles: lane (i = lane & 15, g = lane >> 4) gives row i of K, 16 bytes of each 64; it gets the scores
//                 of query i at positions 4 g + e
//   O^T = V^T P^T the probabilities are where the product wants them: its k index is numbered so that lane group g
//                 holds positions 4 g + e (and 16 + 4 g + e). For V^T a lane loads HDP / 16 neighbouring values of
//                 the rows it holds, whole rows per 16 lanes, and takes the d-th tile's row i to be d = i HDP / 16 + tile;
//                 16-bit pairs are turned by byte permutes.
// Rows behind a list's end are out of the loads' range and read as zero, whatever lies there. The four waves
// of a workgroup take the steps of one chunk of positions in turn and are joined through LDS; chunks are joined by
// k_attention_join. Probabilities are rounded to the rows' 16-bit type for the product with V, which the matrix units then take
// at their full rate (their sum is taken of the rounded ones), everything else is f32; f32 rows stay f32 throughout, on the f32
// MFMAs. They are multiples of 2^7 there (ONE below): with the 2^8 that a score may pass its reference by, f16 holds them up to 2^15 of its 2^16,
// and down to 2^-32 of the row's largest, half of its smallest step.
// What bounds it: reading keys and values while a kv head has few rows (32 sequences of 350 to 700 own positions and
// two shared prefixes of up to 4096, 32 x 128 bf16: 78 us for 396 MB, 5.1 TB/s, the rate of a large copy); VALU
// issue where many rows share them (64 sequences x 8 heads on a prefix of 16380, 4 x 64 f16: a step of 64 rows and 32
// positions is 36 MFMAs (577 cycles) and 163 VALU instructions, 32 of them exponentials at a quarter of the rate; the
// prefix runs at 800 TFLOP/s between 32760 and 65520 positions, 27 us in all with starts, ends and the join of parts).
// Two waves a SIMD (at most 256 registers) measured 47 -> 35 us against one; eight waves a workgroup and the next
// scores between this step's exponentials gained nothing.

typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v2f __attribute__((ext_vector_type(2)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));
typedef qmh_f16 v8h __attribute__((ext_vector_type(8)));
typedef qmh_f16 v2h __attribute__((ext_vector_type(2)));
typedef qmh_bf16 v8b __attribute__((ext_vector_type(8)));
typedef qmh_bf16 v2b __attribute__((ext_vector_type(2)));

__device__ __forceinline__ v4f mma32(qmh_f16, v4u a, v4u b, v4f c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
}
__device__ __forceinline__ v4f mma32(qmh_bf16, v4u a, v4u b, v4f c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8b, a), __builtin_bit_cast(v8b, b), c, 0, 0, 0);
}
// two floats rounded to nearest into 16 bits each
__device__ __forceinline__ uint32_t pack2(qmh_f16, float x, float y) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((v2f){x, y}, v2h));
}
__device__ __forceinline__ uint32_t pack2(qmh_bf16, float x, float y) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((v2f){x, y}, v2b));
}

typedef const __attribute__((address_space(4))) int32_t *const_i32; // scalar loads
__device__ __forceinline__ const_i32 as_const(const int32_t *p) { return (const_i32)(uintptr_t)p; }

__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

// how the work is divided (the same for the workspace's size and the launch)
struct attn_plan {
    int joint;       // prefix and own pages in one pass of each sequence, no parts
    int G;           // heads per kv head
    int per;         // sequences per group
    int nrp, nro;    // 16-row tiles of a wave: prefix, own
    int pt, ps, pc;  // prefix: row tiles, splits, positions of a split
    int ot, os, oc;  // own
    uint32_t pre_blocks;
    int64_t blocks;  // below 2^31
    int64_t rows;    // all rows of queries (query x head)
};

struct attn_args {
    qmh_attention_args a;
    qmh_pages p;
    attn_plan n;
    int lg_ps;
    float *part; // [parts][rows][head_dim], unnormalised
    float2 *ml;  // [parts][rows]: maximum and sum
};

struct attn_list {
    const int32_t *tab;
    int own;      // a sequence's own pages: its queries see different numbers of positions
    int n;        // positions
    int from, to; // this chunk's; to <= n
    int cap;      // the table has pages (of whatever kind) up to this position
};

template <typename T, int HDP, int NR>
struct attn_wave {
    static constexpr bool F = sizeof(T) == 4;
    static constexpr int KS = F ? 16 : 32;            // positions a step
    static constexpr int RT = KS / 16;                // 16-row blocks of K a step
    static constexpr int KC = HDP * (int)sizeof(T) / 64; // 16-byte loads of a K row per lane
    static constexpr int VE = HDP / 16;               // values of a V row per lane
    static constexpr int VB = VE * (int)sizeof(T);    // their bytes
    static constexpr int VW = VB / 4;                 // and words
    static constexpr int LDS_COL = HDP + 4;
    static constexpr int LDS_FLOATS = 4 * 16 * NR * LDS_COL + 4 * 16 * NR * 2 + 16 * NR * 2;

    v4u Q[NR][KC];
    v4f O[NR][VE];
    // l: the sum of a row's probabilities: a lane's own positions in l[0], or (16 bit) all of them in every element, by a
    // product with ones
    v4f l[NR];
    static constexpr float ONE = 7.0f; // the exponent of a score at its row's reference
    // the reference, its negative in powers of two and ONE (ONE alone: it is far from 0, scores are taken less m first), the score
    // that raises it
    float m[NR], off[NR], pass[NR];
    bool far; // some row's is, or was
    int lim[NR];
    v4u k[RT][KC];
    uint32_t v[RT * 4][VW];

    // page numbers of a step, fetched one step before its loads go out (the first ones without waiting for the
    // list's length)
    struct pages {
        int page[RT];
    };
    __device__ __forceinline__ pages fetch(const attn_args &s, const attn_list &L, int base) const {
        pages x;
#pragma unroll
        for (int r = 0; r < RT; r++) x.page[r] = as_const(L.tab)[min(base + 16 * r, L.cap) >> s.lg_ps];
        return x;
    }

    // where a step's blocks of 16 positions lie in the pools, and their bytes in rows that are somebody's: rows from L.to
    // on are out of range
    struct blocks {
        int64_t off[RT];
        int bytes[RT];
    };
    __device__ __forceinline__ blocks locate(const attn_args &s, const attn_list &L, const pages &pg, int base, int kvh, bool &bad) const {
        blocks x;
        const int rb = s.p.head_dim * (int)sizeof(T);
#pragma unroll
        for (int r = 0; r < RT; r++) {
            const int at = base + 16 * r, left = L.to - at, page = pg.page[r];
            const int rows = uniform(left < 0 ? 0 : left > 16 ? 16 : left);
            const bool none = (uint32_t)page >= (uint32_t)s.p.n_pages;
            bad |= none && rows > 0;
            x.off[r] = (((int64_t)uniform(none ? 0 : page) * s.p.n_kv_heads + kvh) * s.p.page_size + (at & (s.p.page_size - 1))) * rb;
            x.bytes[r] = rows * rb;
        }
        return x;
    }
    __device__ __forceinline__ void load_k(const attn_args &s, const blocks &bl) {
        const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4, rb = s.p.head_dim * (int)sizeof(T);
#pragma unroll
        for (int r = 0; r < RT; r++) {
            const __amdgpu_buffer_rsrc_t rk = __builtin_amdgcn_make_buffer_rsrc((uint8_t *)s.p.k + bl.off[r], (short)0, bl.bytes[r], 0x00020000);
#pragma unroll
            for (int c = 0; c < KC; c++) {
                const int b = (4 * c + g) * 16;
                k[r][c] = __builtin_bit_cast(v4u, __builtin_amdgcn_raw_buffer_load_b128(rk, b < rb ? i * rb + b : 0x7ffffff0, 0, 0));
            }
        }
    }
    __device__ __forceinline__ void load_v(const attn_args &s, const blocks &bl) {
        const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4, rb = s.p.head_dim * (int)sizeof(T);
#pragma unroll
        for (int r = 0; r < RT; r++) {
            const __amdgpu_buffer_rsrc_t rv = __builtin_amdgcn_make_buffer_rsrc((uint8_t *)s.p.v + bl.off[r], (short)0, bl.bytes[r], 0x00020000);
#pragma unroll
            for (int e = 0; e < 4; e++)
#pragma unroll
                for (int c = 0; c < (VB + 15) / 16; c++) {
                    const int b = i * VB + 16 * c, o = b < rb ? (4 * g + e) * rb + b : 0x7ffffff0;
                    if constexpr (VB >= 16) {
                        const v4u w = __builtin_bit_cast(v4u, __builtin_amdgcn_raw_buffer_load_b128(rv, o, 0, 0));
#pragma unroll
                        for (int d = 0; d < 4; d++) v[4 * r + e][4 * c + d] = w[d];
                    } else {
                        const auto w = __builtin_amdgcn_raw_buffer_load_b64(rv, o, 0, 0);
                        v[4 * r + e][0] = w[0];
                        v[4 * r + e][1] = w[1];
                    }
                }
        }
    }

    __device__ __forceinline__ void scores(v4f (&S)[NR][RT]) const {
#pragma unroll
        for (int c = 0; c < NR; c++)
#pragma unroll
            for (int r = 0; r < RT; r++) {
                v4f acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int x = 0; x < KC; x++) {
                    if constexpr (F) {
#pragma unroll
                        for (int j = 0; j < 4; j++)
                            acc = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(k[r][x][j]), __uint_as_float(Q[c][x][j]), acc, 0, 0, 0);
                    } else {
                        acc = mma32(T{}, k[r][x], Q[c][x], acc);
                    }
                }
                S[c][r] = acc;
            }
    }

    // the probabilities of a step's scores, packed for the product with V; masked: some row does not see all of it
    __device__ __forceinline__ void weigh(v4f (&S)[NR][RT], v4u (&P)[NR], int base, float sc, bool masked) {
        const int g = (threadIdx.x & 63) >> 4;
        if (masked) {
#pragma unroll
            for (int c = 0; c < NR; c++)
#pragma unroll
                for (int r = 0; r < RT; r++)
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        if (base + 16 * r + 4 * g + e >= lim[c]) S[c][r][e] = -__builtin_inff();
        }
        // The reference value of a row's exponentials is raised only when a score passes it by 2^8: the sums stay exact
        // floats either way, and the rescaling of O is rare. (maximum: NaN wins, and needs no canonical operands.)
        // Exponents are one fused product while the reference is at most 1024 powers of two: rounding it moves them by 2^-15 then. Beyond, that
        // grows to whole powers and past the types' ranges, so the scores' own difference is taken first (an instruction more a
        // score in waves that have such a row), and every larger score raises the reference.
        bool up = false;
        float mx[NR];
#pragma unroll
        for (int c = 0; c < NR; c++) {
            float x = S[c][0][0];
#pragma unroll
            for (int r = 0; r < RT; r++)
#pragma unroll
                for (int e = 0; e < 4; e++) x = __builtin_elementwise_maximum(x, S[c][r][e]);
            mx[c] = x;
            up |= x > pass[c];
        }
        if (__any(up)) {
            bool out = far;
#pragma unroll
            for (int c = 0; c < NR; c++) {
                float x = mx[c];
                x = fmaxf(x, __uint_as_float(qmh_xor16_u(__float_as_uint(x))));
                x = fmaxf(x, __uint_as_float(qmh_xor32_u(__float_as_uint(x))));
                if (x > m[c]) {
                    const float f = m[c] == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f((m[c] - x) * sc);
                    m[c] = x;
                    const float o = __builtin_fmaf(-x, sc, ONE);
                    const bool distant = __builtin_fabsf(o) > 1024.0f;
                    off[c] = distant ? ONE : o;
                    pass[c] = distant ? x : x + 8.0f / sc;
                    out |= distant;
                    l[c] = l[c] * f;
#pragma unroll
                    for (int t = 0; t < VE; t++) O[c][t] = O[c][t] * f;
                }
            }
            far = __any(out);
        }
        if (far) {
#pragma unroll
            for (int c = 0; c < NR; c++) {
                const float from = off[c] == ONE ? m[c] : 0.0f;
#pragma unroll
                for (int r = 0; r < RT; r++)
#pragma unroll
                    for (int e = 0; e < 4; e++) S[c][r][e] -= from;
            }
        }
#pragma unroll
        for (int c = 0; c < NR; c++) {
#pragma unroll
            for (int r = 0; r < RT; r++)
#pragma unroll
                for (int e = 0; e < 4; e++) S[c][r][e] = __builtin_amdgcn_exp2f(__builtin_fmaf(S[c][r][e], sc, off[c]));
        }
        if (masked) { // also where the scale is 0
            asm volatile(""); // a branch: no selects in the other steps
#pragma unroll
            for (int c = 0; c < NR; c++)
#pragma unroll
                for (int r = 0; r < RT; r++)
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        if (base + 16 * r + 4 * g + e >= lim[c]) S[c][r][e] = 0.0f;
        }
#pragma unroll
        for (int c = 0; c < NR; c++) {
            if constexpr (F) {
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    l[c][0] += S[c][0][e];
                    P[c][e] = __float_as_uint(S[c][0][e]);
                }
            } else {
#pragma unroll
                for (int e = 0; e < 4; e++) P[c][e] = pack2(T{}, S[c][e / 2][(2 * e) % 4], S[c][e / 2][(2 * e + 1) % 4]);
                const uint32_t one = pack2(T{}, 1.0f, 1.0f);
                l[c] = mma32(T{}, (v4u){one, one, one, one}, P[c], l[c]);
            }
        }
    }

    __device__ __forceinline__ void add_values(const v4u (&P)[NR]) {
        if constexpr (F) {
#pragma unroll
            for (int t = 0; t < VE; t++)
#pragma unroll
                for (int c = 0; c < NR; c++)
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        O[c][t] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(v[e][t]), __uint_as_float(P[c][e]), O[c][t], 0, 0, 0);
        } else {
#pragma unroll
            for (int u = 0; u < VW; u++) {
                v4u lo, hi; // tiles 2 u and 2 u + 1
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const uint32_t a = v[(2 * j) % (4 * RT)][u], b = v[(2 * j + 1) % (4 * RT)][u];
                    lo[j] = __builtin_amdgcn_perm(b, a, 0x05040100);
                    hi[j] = __builtin_amdgcn_perm(b, a, 0x07060302);
                }
#pragma unroll
                for (int c = 0; c < NR; c++) {
                    O[c][(2 * u) % VE] = mma32(T{}, lo, P[c], O[c][(2 * u) % VE]);
                    O[c][(2 * u + 1) % VE] = mma32(T{}, hi, P[c], O[c][(2 * u + 1) % VE]);
                }
            }
        }
    }

    // This wave's steps of the list's chunk; full: positions that every row sees. The next step's keys are loaded as soon
    // as the scores are made, its values as soon as the step's are used: each has the other's work to arrive in.
    __device__ __forceinline__ void walk(const attn_args &s, const attn_list &L, int kvh, float sc, int full, bool &bad) {
        const int w = uniform((int)(threadIdx.x >> 6));
        int base = L.from + w * KS;
        if (base > L.cap) return; // no table entry to look at (a list that is none has no table)
        pages pg = fetch(s, L, base);
        if (base >= L.to) return;
        blocks bl = locate(s, L, pg, base, kvh, bad);
        load_k(s, bl);
        load_v(s, bl);
        pg = fetch(s, L, base + 4 * KS);
        for (;;) {
            v4f S[NR][RT];
            v4u P[NR];
            scores(S);
            bl = locate(s, L, pg, base + 4 * KS, kvh, bad);
            load_k(s, bl);
            weigh(S, P, base, sc, base + KS > full);
            add_values(P);
            load_v(s, bl);
            pg = fetch(s, L, base + 8 * KS);
            base += 4 * KS;
            if (base >= L.to) break;
        }
    }
};

// Rows [row0, row0 + 16 NR) of the R that share a kv head's keys: row r is token t0 + r / G, head r % G of it. They see
// the chunk of the shared prefix and then the chunk of own pages. part < 0: the result goes out, else it is part `part`.
template <typename T, int HDP, int NR>
__device__ __forceinline__ void attend(const attn_args &s, float *lds, int row0, int R, int t0, int kvh, const attn_list &shared,
                                       const attn_list &own, bool bad, int part) {
    using W = attn_wave<T, HDP, NR>;
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, i = lane & 15, g = lane >> 4, G = s.n.G, hd = s.p.head_dim;
    const int H = s.a.n_heads, h0 = kvh * G;
    const float sc = __builtin_fabsf(s.a.scale) * 1.44269504088896340736f; // exponentials are powers of two
    W x;
    x.far = false;
#pragma unroll
    for (int c = 0; c < NR; c++) {
        int r = row0 + 16 * c + i;
        r = r < R ? r : R - 1; // rows past the last are computed with its queries and not written
        const T *q = (const T *)s.a.q + (int64_t)(t0 + r / G) * s.a.q_stride + (int64_t)(h0 + r % G) * hd;
        const uint32_t flip = s.a.scale < 0.0f ? (W::F ? 0x80000000u : 0x80008000u) : 0u; // the scale's sign
#pragma unroll
        for (int k = 0; k < W::KC; k++) {
            const int e = (4 * k + g) * (16 / (int)sizeof(T));
            v4u v = {0, 0, 0, 0};
            if (e < hd) v = *(const v4u *)(q + e) ^ flip;
            x.Q[c][k] = v;
        }
        x.m[c] = x.pass[c] = -__builtin_inff();
        x.off[c] = 0.0f; // not ONE: no score yet
        x.l[c] = (v4f){0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int t = 0; t < W::VE; t++) x.O[c][t] = (v4f){0.f, 0.f, 0.f, 0.f};
    }
#pragma unroll 1
    for (int k = 0; k < 2; k++) {
        attn_list L = k ? own : shared;
        int full = L.to;
#pragma unroll
        for (int c = 0; c < NR; c++) x.lim[c] = L.n;
        if (L.own) {
            const int first = L.n - s.a.q_len + 1, last = row0 + 16 * NR < R ? row0 + 16 * NR - 1 : R - 1;
            L.to = min(L.to, first + last / G);
            full = min(L.to, first + row0 / G);
#pragma unroll
            for (int c = 0; c < NR; c++) {
                const int r = row0 + 16 * c + i;
                x.lim[c] = first + (r < R ? r : R - 1) / G;
            }
        }
        x.walk(s, L, kvh, sc, full, bad);
    }
    // join the waves
    float *ob = lds;                                           // [wave][16 NR][LDS_COL]
    float2 *mb = (float2 *)(lds + 4 * 16 * NR * W::LDS_COL);   // [wave][16 NR]
    int2 *where = (int2 *)(mb + 4 * 16 * NR);                  // [16 NR]: token, head
#pragma unroll
    for (int c = 0; c < NR; c++) {
        float l = x.l[c][0];
        if constexpr (W::F) {
            l += __uint_as_float(qmh_xor16_u(__float_as_uint(l)));
            l += __uint_as_float(qmh_xor32_u(__float_as_uint(l)));
        }
        if (bad) l = __builtin_nanf(""); // a page or length that is none
        if (g == 0) {
            mb[w * 16 * NR + 16 * c + i] = make_float2(x.m[c], l);
            const int r = row0 + 16 * c + i;
            if (w == 0) where[16 * c + i] = make_int2(t0 + r / G, h0 + r % G);
        }
        float *o = ob + (w * 16 * NR + 16 * c + i) * W::LDS_COL + 4 * g * W::VE;
#pragma unroll
        for (int e = 0; e < 4; e++)
#pragma unroll
            for (int t = 0; t < W::VE; t += 4)
                *(v4f *)(o + e * W::VE + t) = (v4f){x.O[c][t][e], x.O[c][t + 1][e], x.O[c][t + 2][e], x.O[c][t + 3][e]};
    }
    __syncthreads();
    constexpr int D4 = HDP / 4;
    const int d = 4 * (threadIdx.x % D4); // 256 is a multiple of D4
    if (d >= hd) return;
    for (int col = threadIdx.x / D4; col < 16 * NR && row0 + col < R; col += 256 / D4) {
        float m = -__builtin_inff(), l = 0.0f;
#pragma unroll
        for (int k = 0; k < 4; k++) m = fmaxf(m, mb[k * 16 * NR + col].x);
        v4f o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const float2 a = mb[k * 16 * NR + col];
            const float f = a.x == -__builtin_inff() ? 1.0f : __builtin_amdgcn_exp2f((a.x - m) * sc); // a wave without steps: sums of 0 (or NaN)
            l = __builtin_fmaf(a.y, f, l);
            o += *(const v4f *)(ob + (k * 16 * NR + col) * W::LDS_COL + d) * f;
        }
        const int2 th = where[col];
        if (part < 0) {
            const float inv = l == 0.0f ? 0.0f : 1.0f / l;
            qmh_vec<T, 4> y;
#pragma unroll
            for (int e = 0; e < 4; e++) y.e[e] = (T)(o[e] * inv);
            *(qmh_vec<T, 4> *)((T *)s.a.out + (int64_t)th.x * s.a.out_stride + (int64_t)th.y * hd + d) = y;
        } else {
            const int64_t at = (int64_t)part * s.n.rows + (int64_t)th.x * H + th.y;
            if (d == 0) s.ml[at] = make_float2(m, l);
            *(v4f *)(s.part + at * hd + d) = o;
        }
    }
}

template <typename T, int HDP, int NRP, int NRO>
__global__ __launch_bounds__(256, 2) void k_paged_attention(const attn_args s) {
    __shared__ __align__(16) float lds[attn_wave<T, HDP, (NRP > NRO ? NRP : NRO)>::LDS_FLOATS];
    const attn_plan &n = s.n;
    const int KV = s.p.n_kv_heads, Q = s.a.q_len;
    uint32_t b = blockIdx.x;
    const attn_list none = {nullptr, 0, 0, 0, 0, -1};
    if (b < n.pre_blocks) { // split, (group, kv head); row tile: tiles of the same keys 8 blocks apart, on one XCD's cache
        const uint32_t gks = (uint32_t)s.a.n_groups * KV, line = b / (8 * n.pt), in = b - line * 8 * n.pt, unit = line * 8 + (in & 7);
        const int tile = (int)(in >> 3), split = (int)(unit / gks);
        if (split >= n.ps) return;
        const uint32_t gk = unit - split * gks, g = gk / KV, kvh = gk - g * KV;
        int len = uniform(as_const(s.a.prefix_len)[g]);
        const bool bad = len < 0 || len > s.a.max_prefix;
        if (bad) len = 0;
        const attn_list L = {s.a.prefix_table + (int64_t)g * s.a.prefix_stride, 0, len, split * n.pc, min(len, (split + 1) * n.pc), s.a.max_prefix - 1};
        attend<T, HDP, NRP>(s, lds, tile * 16 * NRP, n.per * Q * n.G, g * n.per * Q, kvh, L, none, bad, split);
        return;
    }
    b -= n.pre_blocks;
    const uint32_t units = (uint32_t)s.a.n_seq * KV, st = b / units, unit = b - st * units;
    const uint32_t tile = st / n.os, split = st - tile * n.os, sq = unit / KV, kvh = unit - sq * KV, g = sq / n.per;
    int len = s.a.max_len ? uniform(as_const(s.a.len)[sq]) : 0, plen = 0;
    bool bad = len < 0 || len > s.a.max_len;
    if (bad) len = 0;
    if (n.joint && s.a.max_prefix) {
        plen = uniform(as_const(s.a.prefix_len)[g]);
        if (plen < 0 || plen > s.a.max_prefix) {
            bad = true;
            plen = 0;
        }
    }
    const attn_list S = {s.a.prefix_table + (int64_t)g * s.a.prefix_stride, 0, plen, 0, plen, s.a.max_prefix - 1};
    const attn_list L = {s.a.table + (int64_t)sq * s.a.table_stride, 1, len, (int)split * n.oc, min(len, ((int)split + 1) * n.oc), s.a.max_len - 1};
    attend<T, HDP, NRO>(s, lds, tile * 16 * NRO, Q * n.G, sq * Q, kvh, S, L, bad, n.ps + n.os > 1 ? n.ps + (int)split : -1);
}

// 4 to 5 us, most of it a launch. out = the parts of a row joined, a wave a row (parts at most 64: lane k weighs part k). 64 / D4 parts are read at
// once, 4 values a lane.
template <typename T, int D4>
__global__ __launch_bounds__(256) void k_attention_join(const attn_args s, int parts) {
    constexpr int PG = 64 / D4;
    const int lane = threadIdx.x & 63, hd = s.p.head_dim, d = 4 * (lane % D4);
    const uint32_t row = (uint32_t)uniform((int)(blockIdx.x * 4 + (threadIdx.x >> 6)));
    if (row >= s.n.rows) return;
    const float sc = __builtin_fabsf(s.a.scale) * 1.44269504088896340736f;
    float2 a = make_float2(-__builtin_inff(), 0.0f);
    if (lane < parts) a = s.ml[(int64_t)lane * s.n.rows + row];
    const float m = qmh_wave_max(a.x);
    const float f = a.x == -__builtin_inff() ? 1.0f : __builtin_amdgcn_exp2f((a.x - m) * sc); // without a score: sums of 0 (or NaN)
    float l = a.y * f;
#pragma unroll
    for (int k = 1; k < 64; k <<= 1) l += __shfl_xor(l, k);
    v4f o = {0.f, 0.f, 0.f, 0.f};
    const float *part = s.part + (int64_t)row * hd + (d < hd ? d : 0);
    const int64_t step = s.n.rows * hd;
    for (int r = 0; r < parts; r += 4 * PG) { // by all lanes together: each one's weight is asked for by others
        const int k0 = r + lane / D4;
        v4f v[4];
#pragma unroll
        for (int j = 0; j < 4; j++) v[j] = k0 + j * PG < parts ? *(const v4f *)(part + (k0 + j * PG) * step) : (v4f){0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < 4; j++) o += v[j] * __shfl(f, (k0 + j * PG) & 63);
    }
#pragma unroll
    for (int x = D4; x < 64; x <<= 1)
#pragma unroll
        for (int e = 0; e < 4; e++) o[e] += __shfl_xor(o[e], x);
    if (lane >= D4 || d >= hd) return;
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    const uint32_t token = row / s.a.n_heads, h = row - token * s.a.n_heads;
    qmh_vec<T, 4> y;
#pragma unroll
    for (int e = 0; e < 4; e++) y.e[e] = (T)(o[e] * inv);
    *(qmh_vec<T, 4> *)((T *)s.a.out + token * s.a.out_stride + (int64_t)h * hd + d) = y;
}

attn_plan plan_attention(const qmh_attention_args *a, int cus) {
    attn_plan n = {};
    const qmh_pages *p = a->pages;
    const int KV = p->n_kv_heads;
    const int most = p->head_dim > 128 ? 1 : p->head_dim > 64 ? 2 : 4; // what the registers hold
    n.G = a->n_heads / KV;
    n.per = a->n_seq / a->n_groups;
    n.rows = (int64_t)a->n_seq * a->q_len * a->n_heads;
    const int64_t ro = (int64_t)a->q_len * n.G, rp = a->max_prefix ? ro * n.per : ro;
    auto tiles = [&](int64_t r) { return r <= 16 || most == 1 ? 1 : r <= 32 || most == 2 ? 2 : 4; };
    n.nrp = tiles(rp);
    n.nro = ro <= 16 ? 1 : n.nrp;
    n.pt = (int)((rp + 16 * n.nrp - 1) / (16 * n.nrp));
    n.ot = (int)((ro + 16 * n.nro - 1) / (16 * n.nro));
    const int64_t up = (int64_t)a->n_groups * KV * n.pt, uo = (int64_t)a->n_seq * KV * n.ot;
    int64_t pre = 0;
    n.os = 1;
    n.oc = a->max_len ? a->max_len : 1;
    // Short sequences: a workgroup each that reads the prefix itself, which costs less than a launch that joins parts, while
    // its walk is short (counted in positions of 64 16-bit values) and the prefix is not read too often. Joint against parts:
    // 4 x 4 heads of 64 f16, 300 + 100 positions 6.6 us to 7.8; 32 of 128 bf16, 4 sequences, 180 + 60 7.3 to 8.7, but 2 x 16
    // sequences, 200 + 50 (98 MB more) 17.3 to 15.2; own pages alone: 192 walks of 500 7.5 to 11, 32 of 500 x 128 even, 2 of
    // 500 f32 8.7 to 7.9.
    const int64_t far = (int64_t)a->max_prefix + a->max_len, es = p->dtype == QMH_F32 ? 4 : 2;
    const int64_t walk = far * (p->head_dim <= 64 ? 1 : p->head_dim <= 128 ? 2 : 4) * (es / 2);
    const int64_t again = (uo - up) * a->max_prefix * p->head_dim * es * 2;
    n.joint = a->max_prefix ? walk <= 512 && again <= 32 << 20 : walk <= (uo >= 32 ? 1024 : 512);
    if (!n.joint) {
        // chunks of positions, about the same for both, that fill the chip's workgroups (two per CU) once
        const int64_t all = up * a->max_prefix + uo * a->max_len;
        const int unit = 4 * (p->dtype == QMH_F32 ? 16 : 32); // a step of every wave
        const double c = (double)all / (2 * cus);
        auto split = [&](int len, int most, int *chunk) {
            int k = (int)(len / c + 0.5);
            k = k < 1 ? 1 : k > most ? most : k;
            *chunk = ((len + k - 1) / k + unit - 1) / unit * unit;
            return (len + *chunk - 1) / *chunk;
        };
        if (a->max_prefix) {
            n.ps = split(a->max_prefix, 40, &n.pc);
            pre = ((int64_t)a->n_groups * KV * n.ps + 7) / 8 * 8 * n.pt;
        }
        if (a->max_len) n.os = split(a->max_len, 24, &n.oc);
    }
    n.pre_blocks = (uint32_t)(pre < 0x7fffffff ? pre : 0x7fffffff);
    n.blocks = pre + uo * n.os;
    return n;
}

template <typename T, int HDP>
void launch_attention(const attn_args &s, hipStream_t st) {
    const dim3 g((uint32_t)s.n.blocks), t(256);
    const int p = s.n.nrp, o = s.n.nro;
    if (p == 1) hipLaunchKernelGGL((k_paged_attention<T, HDP, 1, 1>), g, t, 0, st, s);
    else if constexpr (HDP <= 128) {
        if (p == 2 && o == 1) hipLaunchKernelGGL((k_paged_attention<T, HDP, 2, 1>), g, t, 0, st, s);
        else if (p == 2) hipLaunchKernelGGL((k_paged_attention<T, HDP, 2, 2>), g, t, 0, st, s);
    }
    if constexpr (HDP <= 64) {
        if (p == 4 && o == 1) hipLaunchKernelGGL((k_paged_attention<T, HDP, 4, 1>), g, t, 0, st, s);
        else if (p == 4) hipLaunchKernelGGL((k_paged_attention<T, HDP, 4, 4>), g, t, 0, st, s);
    }
    const int parts = s.n.ps + s.n.os;
    if (parts > 1) {
        hipLaunchKernelGGL((k_attention_join<T, HDP / 4>), dim3((uint32_t)((s.n.rows + 3) / 4)), t, 0, st, s, parts);
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
    if (a->n_seq == 0) return 0;
    const attn_plan n = plan_attention(a, cus);
    const size_t parts = n.ps + n.os;
    return parts > 1 ? parts * n.rows * (a->pages->head_dim * sizeof(float) + sizeof(float2)) : 0;
}

extern "C" int qmh_launch_paged_attention(const qmh_attention_args *a, int cus, void *ws, void *stream) {
    attn_args s;
    s.a = *a;
    s.p = *a->pages;
    s.n = plan_attention(a, cus);
    s.lg_ps = __builtin_ctz(s.p.page_size);
    s.part = (float *)ws;
    s.ml = (float2 *)(s.part + (size_t)(s.n.ps + s.n.os) * s.n.rows * s.p.head_dim);
    if (s.n.blocks > QMH_MOST_BLOCKS || (s.n.rows + 3) / 4 > QMH_MOST_BLOCKS) return (int)hipErrorInvalidValue;
    qmh_for_type(s.p.dtype, [&](auto z) {
        using T = decltype(z);
        if (s.p.head_dim <= 64) launch_attention<T, 64>(s, (hipStream_t)stream);
        else if (s.p.head_dim <= 128) launch_attention<T, 128>(s, (hipStream_t)stream);
        else launch_attention<T, 256>(s, (hipStream_t)stream);
    });
    return (int)hipGetLastError();
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
