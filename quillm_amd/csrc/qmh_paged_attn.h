// Attention over keys and values in pages: the kernel of qmh_paged_attention (consecutive queries) and of qmh_tree_attention (TREE:
// nodes of a drafted tree). No reference counterpart; accuracy as the declarations state, not bitwise.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "qmh_device.h"
#include "qmh_launch.h"
#include "qmh_types.h"

namespace {

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
//
// Trees: nodes in place of queries, each with the positions of a step that it sees as bits (look), which cost only the steps that some
// row does not see all of. Measured: 8 sequences of 4100, 16 to 32 nodes, 32 x 128 bf16 82 to 88 us by device (a copy of their keys and values: 82).
// Where many rows share the keys (64 nodes x 8 heads, 12 sequences of 6000, 64 f16: 69 us, 420 TFLOP/s) the first-level cache is the bound:
// 16 lanes next to each other ask for 16 rows' parts of a key, 256 of a step's 430 lookups, four waves a CU at once. Without its loads a
// step of 64 rows takes 1140 cycles, with them 1650. Copies straight into LDS, a buffer a wave, halve the lookups, but their own
// instructions (some 100 a step) cost more: 78 us two steps ahead, 71 one step ahead. One buffer for the four waves was not tried. Two waves
// a SIMD are 1.6 times one. Tree kernels spill, likely for what makes a tile again (attend_nodes): 46 to 73 scalar registers and 20 to 56
// bytes of scratch a lane up to heads of 128, 156 to 204 (16 bit) and 324 (f32) past that; without trees 0 to 10, none, 116 and 252.

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

// nodes of a drafted tree in place of consecutive queries
struct attn_tree {
    int n_rows;           // rows of q and out
    const int32_t *first; // rows of a sequence: first[i] to first[i + 1]; NULL: i * q_len to (i + 1) * q_len
    const uint32_t *mask; // NULL: node j sees nodes 0 to j
    int64_t stride;       // words from a sequence's mask to the next one's
    int words;            // words from a node's row to the next one's
};

struct attn_args {
    qmh_attention_args a;
    attn_tree tree;
    qmh_pages p;
    attn_plan n;
    int lg_ps;
    float *part; // [parts][rows][head_dim], unnormalised
    float2 *ml;  // [parts][rows]: maximum and sum
};

struct attn_list {
    const int32_t *tab;
    int own;      // a sequence's own pages: its queries see different positions
    int n;        // positions
    int from, to; // this chunk's; to <= n
    int cap;      // the table has pages (of whatever kind) up to this position
};

template <typename T, int HDP, int NR, bool TREE>
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

    int tid;
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
    int lim[NR];          // positions that a row sees; trees: its row of the mask, a word's number, or how many nodes of a chain it sees
    uint32_t vis[NR];     // trees: which positions of the step it sees, where that is not all of them
    const uint32_t *mask; // trees: the sequence's
    int ctx;              // trees: positions before the first node
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
        const int lane = tid & 63, i = lane & 15, g = lane >> 4, rb = s.p.head_dim * (int)sizeof(T);
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
        const int lane = tid & 63, i = lane & 15, g = lane >> 4, rb = s.p.head_dim * (int)sizeof(T);
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

    // whether row c of this lane does not see the step's position at (4 g + e in block r)
    __device__ __forceinline__ bool hidden(int c, int base, int at) const {
        if constexpr (TREE) return !((vis[c] >> at) & 1);
        else return base + at >= lim[c];
    }

    // Trees: the positions of a step that each row sees, as bits. A node's row of the mask starts at position ctx, what lies before is
    // seen by all; words are asked for a step ahead.
    __device__ __forceinline__ void look(const attn_list &L, int base) {
        const int left = L.n - base, k0 = base - ctx;
        const uint32_t in = left >= 32 ? ~0u : left <= 0 ? 0u : (1u << left) - 1;
#pragma unroll
        for (int c = 0; c < NR; c++) {
            vis[c] = in;
            if (!L.own || k0 <= -32) continue;
            if (mask) {
                const int w = k0 >> 5, most = (L.n - ctx + 31) >> 5; // k0 may be below 0: w is then -1
                const uint32_t lo = w < 0 ? ~0u : w < most ? mask[lim[c] + w] : 0u, hi = w + 1 < most ? mask[lim[c] + w + 1] : 0u;
                vis[c] &= __builtin_amdgcn_alignbit(hi, lo, (uint32_t)k0 & 31);
            } else {
                const int n = lim[c] - k0;
                vis[c] &= n >= 32 ? ~0u : n <= 0 ? 0u : (1u << n) - 1;
            }
        }
    }

    // the probabilities of a step's scores, packed for the product with V; masked: some row does not see all of it
    __device__ __forceinline__ void weigh(v4f (&S)[NR][RT], v4u (&P)[NR], int base, float sc, bool masked) {
        const int g = (tid & 63) >> 4;
        if (masked) {
#pragma unroll
            for (int c = 0; c < NR; c++)
#pragma unroll
                for (int r = 0; r < RT; r++)
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        if (hidden(c, base, 16 * r + 4 * g + e)) S[c][r][e] = -__builtin_inff();
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
            if constexpr (TREE) // bits looked at again: kept as truth values from above they would fill the scalar registers
#pragma unroll
                for (int c = 0; c < NR; c++) asm volatile("" : "+v"(vis[c]));
#pragma unroll
            for (int c = 0; c < NR; c++)
#pragma unroll
                for (int r = 0; r < RT; r++)
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        if (hidden(c, base, 16 * r + 4 * g + e)) S[c][r][e] = 0.0f;
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
        const int w = uniform(tid >> 6);
        int base = L.from + w * KS;
        if (base > L.cap) return; // no table entry to look at (a list that is none has no table)
        pages pg = fetch(s, L, base);
        if (base >= L.to) return;
        blocks bl = locate(s, L, pg, base, kvh, bad);
        load_k(s, bl);
        load_v(s, bl);
        pg = fetch(s, L, base + 4 * KS);
        if (TREE && base + KS > full) look(L, base);
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
            if (TREE && base + KS > full) look(L, base);
        }
    }
};

// Trees: a node that a row does not see must not reach it, whatever its values hold, but a product with 0 makes NaN of a value
// that is not finite, and a page that is none makes NaN of the sums of all rows. Where sums are not finite, and some node's values are not
// either or its page is none, a tile is made again: the positions before the nodes as ever, then each row's nodes here, by the
// whole workgroup, from what the row sees alone: 256 nodes at a time, their scores a thread
// each, then an output element a thread. That happens only there: looking at the values in the walk cost it registers, and 10 of 98 us of
// 8 sequences of 4100, 32 x 128.
constexpr int NODE_FLOATS = 256 + 256 + 512 + 4; // what it needs of LDS
template <typename T>
__device__ __forceinline__ void attend_nodes(const attn_args &s, float *lds, float m, float l, float o, int r, int R, int t0, int sq, int kvh,
                                             const attn_list &own, bool bad, int part) {
    const int tid = threadIdx.x, hd = s.p.head_dim, G = s.n.G, node = r / G, ctx = own.n - R / G;
    const int64_t token = t0 + node, head = kvh * G + r % G;
    const float sc = __builtin_fabsf(s.a.scale) * 1.44269504088896340736f;
    float *q = lds, *weight = lds + 256;  // [256] each; a weight of -1: not seen
    int64_t *at = (int64_t *)(lds + 512); // [256]: where the node's row lies in the pools
    float *top = (float *)(at + 256);     // [4]
    if (tid < hd) {
        const float x = qmh_to_f(((const T *)s.a.q)[token * s.a.q_stride + head * hd + tid]);
        q[tid] = s.a.scale < 0.0f ? -x : x;
    }
#pragma unroll 1
    for (int base = own.from > ctx ? own.from : ctx; base < own.to; base += 256) {
        __syncthreads(); // q is there, the last nodes are done with
        const int pos = base + tid, n = pos - ctx;
        bool sees = pos < own.to;
        if (sees) sees = s.tree.mask ? (s.tree.mask[sq * s.tree.stride + (int64_t)node * s.tree.words + (n >> 5)] >> (n & 31)) & 1 : n <= node;
        const int page = sees ? own.tab[pos >> s.lg_ps] : 0;
        float x = -__builtin_inff();
        if (page < 0 || page >= s.p.n_pages) {
            x = __builtin_nanf(""); // the row's result is
            at[tid] = 0;
        } else if (sees) {
            const int64_t row = (((int64_t)page * s.p.n_kv_heads + kvh) * s.p.page_size + (pos & (s.p.page_size - 1))) * hd;
            at[tid] = row;
            x = 0.0f;
#pragma unroll 1
            for (int d = 0; d < hd; d += 16 / (int)sizeof(T)) {
                const qmh_vec<T, 16 / sizeof(T)> kv = *(const qmh_vec<T, 16 / sizeof(T)> *)((const T *)s.p.k + row + d);
#pragma unroll
                for (int i = 0; i < 16 / (int)sizeof(T); i++) x = __builtin_fmaf(q[d + i], qmh_to_f(kv.e[i]), x);
            }
        }
        const float t = qmh_wave_max(x);
        if ((tid & 63) == 0) top[tid >> 6] = t;
        __syncthreads();
        const float up = fmaxf(fmaxf(m, fmaxf(top[0], top[1])), fmaxf(top[2], top[3])), ref = up == -__builtin_inff() ? 0.0f : up;
        const float f = m == -__builtin_inff() ? 1.0f : __builtin_amdgcn_exp2f((m - up) * sc); // without a score: sums of 0 (or NaN)
        m = up;
        weight[tid] = sees ? __builtin_amdgcn_exp2f(__builtin_fmaf(x - ref, sc, 7.0f)) : -1.0f; // times 2^7, as in the walk
        __syncthreads();
        l *= f;
        o *= f;
#pragma unroll 1
        for (int j = 0; j < 256 && base + j < own.to; j++) {
            const float p = weight[j];
            if (p < 0.0f) continue;
            l += p;
            if (tid < hd) o = __builtin_fmaf(p, qmh_to_f(((const T *)s.p.v)[at[j] + tid]), o);
        }
    }
    __syncthreads();
    if (tid >= hd) return;
    if (bad) l = __builtin_nanf("");
    if (part < 0) {
        ((T *)s.a.out)[token * s.a.out_stride + head * hd + tid] = (T)(l == 0.0f ? 0.0f : o / l);
    } else {
        const int64_t to = (int64_t)part * s.n.rows + token * s.a.n_heads + head;
        if (tid == 0) s.ml[to] = make_float2(m, l);
        s.part[to * hd + tid] = o;
    }
}
// whether the list's nodes, of those in its chunk, have a value that is not finite or a page that is none (for the whole workgroup)
template <typename T>
__device__ __forceinline__ bool odd_nodes(const attn_args &s, int ctx, int kvh, const attn_list &own) {
    constexpr int N = 16 / (int)sizeof(T);
    const int from = own.from > ctx ? own.from : ctx, per = s.p.head_dim / N;
    bool odd = false;
    for (int i = threadIdx.x; i < (own.to - from) * per; i += 256) {
        const int pos = from + i / per, page = own.tab[pos >> s.lg_ps];
        if (page < 0 || page >= s.p.n_pages) {
            odd = true;
            continue;
        }
        const int64_t row = (((int64_t)page * s.p.n_kv_heads + kvh) * s.p.page_size + (pos & (s.p.page_size - 1))) * s.p.head_dim;
        const qmh_vec<T, N> x = *(const qmh_vec<T, N> *)((const T *)s.p.v + row + i % per * N);
#pragma unroll
        for (int e = 0; e < N; e++) odd |= !__builtin_isfinite(qmh_to_f(x.e[e]));
    }
    return __syncthreads_or(odd);
}

// Rows [row0, row0 + 16 NR) of the R that share a kv head's keys: row r is token t0 + r / G, head r % G of it. They see
// the chunk of the shared prefix and then the chunk of own pages; sq: whose these are. part < 0: the result goes out, else it is part `part`.
// True (trees): the tile has to be made again, with `again`.
template <typename T, int HDP, int NR, bool TREE>
__device__ __forceinline__ bool attend_once(const attn_args &s, float *lds, int row0, int R, int t0, int sq, int kvh, const attn_list &shared,
                                            const attn_list &own, bool bad, int part, bool again) {
    using W = attn_wave<T, HDP, NR, TREE>;
    int tid = threadIdx.x;
    if constexpr (TREE) asm volatile("" : "+v"(tid)); // nothing made of it stays in registers from one time to the other
    const int lane = tid & 63, w = tid >> 6, i = lane & 15, g = lane >> 4, G = s.n.G, hd = s.p.head_dim;
    const int H = s.a.n_heads, h0 = kvh * G;
    const float sc = __builtin_fabsf(s.a.scale) * 1.44269504088896340736f; // exponentials are powers of two
    W x;
    x.tid = tid;
    __shared__ uint32_t odd[2]; // trees: which of the rows have sums that are not finite
    if (TREE && tid < 2) odd[tid] = 0;
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
        if (TREE && again && L.own) { // the positions before the nodes: all rows see them
            L.n = own.n - R / G;
            L.to = min(L.to, L.n);
            L.own = 0;
        }
        int full = L.to;
#pragma unroll
        for (int c = 0; c < NR; c++) x.lim[c] = L.n;
        if (TREE) {
            x.ctx = own.n - R / G; // of a bad length below 0, its steps none
            x.mask = s.tree.mask ? s.tree.mask + sq * s.tree.stride : nullptr;
            if (L.own) full = min(L.to, x.ctx);
#pragma unroll
            for (int c = 0; c < NR; c++) {
                int r = row0 + 16 * c + i;
                r = (r < R ? r : R - 1) / G;
                x.lim[c] = s.tree.mask ? r * s.tree.words : r + 1;
            }
        } else if (L.own) {
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
    const int d = 4 * (tid % D4); // 256 is a multiple of D4
    if (!TREE && d >= hd) return false;
    for (int col = tid / D4; d < hd && col < 16 * NR && row0 + col < R; col += 256 / D4) {
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
        if (TREE && again) { // for attend_nodes
            *(v4f *)(ob + col * W::LDS_COL + d) = o;
            if (d == 0) where[col] = make_int2(__float_as_int(m), __float_as_int(l));
            continue;
        }
        if constexpr (TREE)
            if (!__builtin_isfinite(o[0] + o[1] + (o[2] + o[3]) + l)) atomicOr(&odd[col >> 5], 1u << (col & 31));
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
    if constexpr (TREE) {
        __syncthreads();
        if (again) {
#pragma unroll 1
            for (int col = 0; col < 16 * NR && row0 + col < R; col++) {
                const int2 ml = where[col];
                const float o = ob[col * W::LDS_COL + ((int)threadIdx.x < hd ? threadIdx.x : 0)];
                attend_nodes<T>(s, lds + W::LDS_FLOATS, __int_as_float(ml.x), __int_as_float(ml.y), o, row0 + col, R, t0, sq, kvh, own, bad, part);
            }
            return false;
        }
        return own.own && own.to > own.n - R / G && (odd[0] | odd[1]) && odd_nodes<T>(s, own.n - R / G, kvh, own);
    }
    return false;
}
template <typename T, int HDP, int NR, bool TREE>
__device__ __forceinline__ void attend(const attn_args &s, float *lds, int row0, int R, int t0, int sq, int kvh, const attn_list &shared,
                                       const attn_list &own, bool bad, int part) {
    bool again = false;
#pragma unroll 1
    do again = attend_once<T, HDP, NR, TREE>(s, lds, row0, R, t0, sq, kvh, shared, own, bad, part, again);
    while (TREE && again);
}

// the rows of sequence sq: t0 to t0 + the result, 0 where they are none
template <bool TREE>
__device__ __forceinline__ int attn_rows(const attn_args &s, int sq, int &t0) {
    const int Q = s.a.q_len;
    if (!TREE || !s.tree.first) {
        t0 = sq * Q;
        return Q;
    }
    t0 = uniform(as_const(s.tree.first)[sq]);
    const int64_t t1 = uniform(as_const(s.tree.first)[sq + 1]), rows = t1 - t0;
    return t0 < 0 || rows < 0 || t1 > s.tree.n_rows || rows > Q ? 0 : (int)rows;
}
// the rows of a group from sequence sq on, those of sequences that are left out among them as far as q has them: the others' results
// must not depend on them. They may be more than the group's sequences may have.
template <bool TREE>
__device__ __forceinline__ int group_rows(const attn_args &s, int sq, int &t0) {
    if (!TREE || !s.tree.first) {
        t0 = sq * s.a.q_len;
        return s.n.per * s.a.q_len;
    }
    t0 = max(uniform(as_const(s.tree.first)[sq]), 0);
    const int t1 = max(min(uniform(as_const(s.tree.first)[sq + s.n.per]), s.tree.n_rows), 0);
    return max(t1 - t0, 0);
}

template <typename T, int HDP, int NRP, int NRO, bool TREE>
__global__ __launch_bounds__(256, 2) void k_paged_attention(const attn_args s) {
    __shared__ __align__(16) float lds[attn_wave<T, HDP, (NRP > NRO ? NRP : NRO), TREE>::LDS_FLOATS + (TREE ? NODE_FLOATS : 0)];
    const attn_plan &n = s.n;
    const int KV = s.p.n_kv_heads;
    uint32_t b = blockIdx.x;
    const attn_list none = {nullptr, 0, 0, 0, 0, -1};
    if (b < n.pre_blocks) { // split, (group, kv head); row tile: tiles of the same keys 8 blocks apart, on one XCD's cache
        const uint32_t gks = (uint32_t)s.a.n_groups * KV, line = b / (8 * n.pt), in = b - line * 8 * n.pt, unit = line * 8 + (in & 7);
        const int tile = (int)(in >> 3), split = (int)(unit / gks);
        if (split >= n.ps) return;
        const uint32_t gk = unit - split * gks, g = gk / KV, kvh = gk - g * KV;
        int t0;
        const int R = group_rows<TREE>(s, g * n.per, t0) * n.G;
        if (TREE && tile * 16 * NRP >= R) return;
        int len = uniform(as_const(s.a.prefix_len)[g]);
        const bool bad = len < 0 || len > s.a.max_prefix;
        if (bad) len = 0;
        const attn_list L = {s.a.prefix_table + (int64_t)g * s.a.prefix_stride, 0, len, split * n.pc, min(len, (split + 1) * n.pc), s.a.max_prefix - 1};
        // tiles behind the last workgroup's are there only with sequences that are left out; a time's reads of LDS end before its last barrier
        int row0 = tile * 16 * NRP;
#pragma unroll 1
        do attend_once<T, HDP, NRP, TREE>(s, lds, row0, R, t0, 0, kvh, L, none, bad, split, false);
        while (TREE && (row0 += n.pt * 16 * NRP) < R);
        return;
    }
    b -= n.pre_blocks;
    const uint32_t units = (uint32_t)s.a.n_seq * KV, st = b / units, unit = b - st * units;
    const uint32_t tile = st / n.os, split = st - tile * n.os, sq = unit / KV, kvh = unit - sq * KV, g = sq / n.per;
    int t0;
    const int R = attn_rows<TREE>(s, sq, t0) * n.G;
    if (TREE && (int)tile * 16 * NRO >= R) return;
    int len = s.a.max_len ? uniform(as_const(s.a.len)[sq]) : 0, plen = 0;
    bool bad = len < 0 || len > s.a.max_len || (TREE && len < R / n.G);
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
    attend<T, HDP, NRO, TREE>(s, lds, tile * 16 * NRO, R, t0, sq, kvh, S, L, bad, n.ps + n.os > 1 ? n.ps + (int)split : -1);
}

// 4 to 5 us, most of it a launch. out = the parts of a row joined, a wave a row (parts at most 64: lane k weighs part k). 64 / D4 parts are read at
// once, 4 values a lane.
template <typename T, int D4, bool TREE>
__global__ __launch_bounds__(256) void k_attention_join(const attn_args s, int parts) {
    constexpr int PG = 64 / D4;
    const int lane = threadIdx.x & 63, hd = s.p.head_dim, d = 4 * (lane % D4);
    const uint32_t row = (uint32_t)uniform((int)(blockIdx.x * 4 + (threadIdx.x >> 6)));
    if (row >= s.n.rows) return;
    if (TREE && s.tree.first) { // rows that are nobody's
        const int t = (int)(row / s.a.n_heads);
        if (t < as_const(s.tree.first)[0] || t >= as_const(s.tree.first)[s.a.n_seq]) return;
    }
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

// n_rows: rows of q (at most n_seq * q_len are used)
template <bool TREE>
attn_plan plan_attention(const qmh_attention_args *a, int64_t n_rows, int cus) {
    attn_plan n = {};
    const qmh_pages *p = a->pages;
    const int KV = p->n_kv_heads;
    const int most = p->head_dim > 128 ? 1 : p->head_dim > 64 ? 2 : 4; // what the registers hold
    n.G = a->n_heads / KV;
    n.per = a->n_seq / a->n_groups;
    n.rows = n_rows * a->n_heads;
    const int64_t ro = (int64_t)a->q_len * n.G, rp = a->max_prefix ? (ro * n.per < n_rows * n.G ? ro * n.per : n_rows * n.G) : ro;
    auto tiles = [&](int64_t r) { return r <= 16 || most == 1 ? 1 : r <= 32 || most == 2 ? 2 : 4; };
    n.nrp = tiles(rp);
    n.nro = ro <= 16 ? 1 : n.nrp;
    // f32 products take so long that rows which are none cost more than keys read again
    if (TREE && p->dtype == QMH_F32 && (ro + 15) / 16 * 2 <= (ro + 16 * n.nro - 1) / (16 * n.nro) * n.nro) n.nro = 1;
    n.pt = (int)((rp + 16 * n.nrp - 1) / (16 * n.nrp));
    n.ot = (int)((ro + 16 * n.nro - 1) / (16 * n.nro));
    const int64_t up = (int64_t)a->n_groups * KV * n.pt, uo = (int64_t)a->n_seq * KV * n.ot;
    n.blocks = up + uo;
    if (up > QMH_MOST_BLOCKS || uo > QMH_MOST_BLOCKS) return n; // too many, however they are split
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
        if (TREE && !a->max_prefix && a->max_len) {
            // Trees without a prefix: one workgroup a CU where few rows share the keys (reading them bounds it: 8 x 32 walks of 4100 x 128 take
            // 87 us whole, 95 in two chunks each; 4 x 32 52 in two, 57 in four), two a CU where many do and their products bound it (24 tiles
            // of 30011 x 64 35 us in 16 chunks, 31 in 21; but 256 of 6000 48 whole, 51 in two). The rule looks at tiles alone: each of these was
            // measured at one length, and many tiles of long sequences may want more parts than it gives them.
            const int64_t slots = uo * 4 >= cus * 3 ? uo : n.ot >= 4 ? 2 * cus : cus;
            const int64_t k = slots / uo < 48 ? slots / uo : 48;
            n.oc = (int)((a->max_len + k - 1) / k + unit - 1) / unit * unit;
            n.os = (a->max_len + n.oc - 1) / n.oc;
        } else if (a->max_len) {
            n.os = split(a->max_len, 24, &n.oc);
        }
    }
    n.pre_blocks = (uint32_t)(pre < 0x7fffffff ? pre : 0x7fffffff);
    n.blocks = pre + uo * n.os;
    return n;
}

template <typename T, int HDP, bool TREE>
void launch_attention(const attn_args &s, hipStream_t st) {
    const dim3 g((uint32_t)s.n.blocks), t(256);
    const int p = s.n.nrp, o = s.n.nro;
    if (p == 1) hipLaunchKernelGGL((k_paged_attention<T, HDP, 1, 1, TREE>), g, t, 0, st, s);
    else if constexpr (HDP <= 128) {
        if (p == 2 && o == 1) hipLaunchKernelGGL((k_paged_attention<T, HDP, 2, 1, TREE>), g, t, 0, st, s);
        else if (p == 2) hipLaunchKernelGGL((k_paged_attention<T, HDP, 2, 2, TREE>), g, t, 0, st, s);
    }
    if constexpr (HDP <= 64) {
        if (p == 4 && o == 1) hipLaunchKernelGGL((k_paged_attention<T, HDP, 4, 1, TREE>), g, t, 0, st, s);
        else if (p == 4) hipLaunchKernelGGL((k_paged_attention<T, HDP, 4, 4, TREE>), g, t, 0, st, s);
    }
    const int parts = s.n.ps + s.n.os;
    if (parts > 1) {
        hipLaunchKernelGGL((k_attention_join<T, HDP / 4, TREE>), dim3((uint32_t)((s.n.rows + 3) / 4)), t, 0, st, s, parts);
    }
}

template <bool TREE>
size_t attention_ws(const qmh_attention_args *a, int64_t n_rows, int cus) {
    if (a->n_seq == 0 || n_rows == 0) return 0;
    const attn_plan n = plan_attention<TREE>(a, n_rows, cus);
    const size_t parts = n.ps + n.os;
    return parts > 1 ? parts * n.rows * (a->pages->head_dim * sizeof(float) + sizeof(float2)) : 0;
}

template <bool TREE>
int run_attention(const qmh_attention_args *a, const attn_tree &tree, int cus, void *ws, hipStream_t st) {
    attn_args s;
    s.a = *a;
    s.tree = tree;
    s.p = *a->pages;
    s.n = plan_attention<TREE>(a, tree.n_rows, cus);
    s.lg_ps = __builtin_ctz(s.p.page_size);
    s.part = (float *)ws;
    s.ml = (float2 *)(s.part + (size_t)(s.n.ps + s.n.os) * s.n.rows * s.p.head_dim);
    if (s.n.blocks > QMH_MOST_BLOCKS || (s.n.rows + 3) / 4 > QMH_MOST_BLOCKS) return (int)hipErrorInvalidValue;
    qmh_for_type(s.p.dtype, [&](auto z) {
        using T = decltype(z);
        if (s.p.head_dim <= 64) launch_attention<T, 64, TREE>(s, st);
        else if (s.p.head_dim <= 128) launch_attention<T, 128, TREE>(s, st);
        else launch_attention<T, 256, TREE>(s, st);
    });
    return (int)hipGetLastError();
}

} // namespace
