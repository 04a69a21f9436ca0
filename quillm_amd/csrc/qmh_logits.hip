// gfx950 kernels of qmh_logits_edit: penalties for repeated tokens, biases and grammar masks on rows of logits, and each
// row's best token. No reference counterpart.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "qmh_device.h"
#include "qmh_launch.h"
#include "qmh_types.h"

namespace {

// A workgroup takes a segment of the vocabulary for some rows of one sequence. First it counts the history's tokens that fall into its
// segment, in LDS, and lists the tokens that any edit touches (the hot ones). A dense pass then goes over the rows: it copies
// them (where they go elsewhere), puts -inf where the grammar forbids a token, and finds the best of the tokens that are
// not hot; it is left out where there is nothing of it to do, and vectors that stay as they are, or are forbidden as a whole,
// are not read. A sparse pass edits the hot ones: they are few, so their divisions and gathers do not weigh.
constexpr int SEG = 4096;
constexpr int ROWS = 32; // of a workgroup, at most
constexpr uint32_t PROMPT = 1u << 31, NODE = 1u << 30; // beside a count of outputs: in the prompt; a node's token

typedef uint32_t v4u __attribute__((ext_vector_type(4)));
struct __attribute__((packed, aligned(2))) v4u_any { // rows start at any element
    v4u v;
};

// larger for larger values, above 0 for any above -inf; then the lower token
__device__ __forceinline__ uint64_t best_key(float x, int token) {
    const uint32_t u = __float_as_uint(x + 0.0f); // -0 is 0
    return (uint64_t)(u ^ (u >> 31 ? 0xffffffffu : 0x80000000u)) << 32 | (uint32_t)~token;
}

template <typename T>
__device__ __forceinline__ float element(v4u x, int e) {
    if constexpr (sizeof(T) == 4) return __uint_as_float(x[e]);
    else return qmh_to_f(__builtin_bit_cast(T, (uint16_t)(e & 1 ? x[e / 2] >> 16 : x[e / 2])));
}

// the rows of sequence sq: t0 to t0 + the result, 0 where they are none
__device__ __forceinline__ int logits_rows(const qmh_logits_args &a, int sq, int &t0) {
    if (!a.first) {
        t0 = sq * a.rows_per_seq;
        return a.rows_per_seq;
    }
    t0 = a.first[sq];
    const int64_t t1 = a.first[sq + 1], n = t1 - t0;
    return t0 < 0 || n < 0 || t1 > a.n_rows || n > a.rows_per_seq ? 0 : (int)n;
}

template <typename T>
__global__ __launch_bounds__(256) void k_logits_edit(const qmh_logits_args a, int segs, int chunks, int chunk, uint32_t first_block, uint64_t *keys) {
    constexpr int N = 16 / (int)sizeof(T); // tokens of a vector
    constexpr uint32_t ALL = (1u << N) - 1;
    __shared__ __align__(16) uint32_t count[SEG], bias_at[SEG];
    __shared__ uint16_t hot[SEG];
    __shared__ uint64_t hot_bits[SEG / 64], row_key[ROWS];
    __shared__ int node[1024];
    __shared__ int n_hot;
    const uint32_t b = blockIdx.x + first_block, unit = b / chunks, sq = unit / segs;
    const int seg = unit - sq * segs, tid = threadIdx.x, lane = tid & 63;
    int t0;
    const int n = logits_rows(a, sq, t0), r0 = (int)(b - unit * chunks) * chunk, r1 = min(r0 + chunk, n);
    if (r0 >= n) return;
    const int v0 = seg * SEG, vn = min(SEG, a.vocab - v0); // the segment's tokens
    const float rep = a.repetition ? a.repetition[sq] : 1.0f, by = rep > 0.0f ? rep : 1.0f;
    const float presence = a.presence ? a.presence[sq] : 0.0f, frequency = a.frequency ? a.frequency[sq] : 0.0f;
    const bool penal = by != 1.0f || presence != 0.0f || frequency != 0.0f;
    const int n_node = penal && a.node_token ? n : 0;

    // ---- what is touched
    for (int i = tid; i < SEG; i += 256) count[i] = bias_at[i] = 0;
    if (tid < ROWS) row_key[tid] = 0;
    if (tid == 0) n_hot = 0;
    __syncthreads();
    if (penal && a.history) {
        const int64_t len = max(0, a.history_len[sq]);
        const int h = (int)min(len, a.history_stride), prompt = a.prompt_len ? a.prompt_len[sq] : 0;
        const int32_t *hist = a.history + sq * a.history_stride;
        for (int i = tid; i < h; i += 256) {
            const uint32_t e = (uint32_t)(hist[i] - v0);
            if (hist[i] < 0 || e >= (uint32_t)vn) continue;
            if (i < prompt) atomicOr(&count[e], PROMPT);
            else atomicAdd(&count[e], 1u);
        }
    }
    for (int k = tid; k < n_node; k += 256) {
        const int t = a.node_token[(int64_t)sq * a.node_stride + k];
        const uint32_t e = (uint32_t)(t - v0);
        node[k] = t;
        if (t >= 0 && e < (uint32_t)vn) atomicOr(&count[e], NODE);
    }
    if (a.bias) {
        const int nb = min(max(0, a.bias_len[sq]), a.bias_stride);
        for (int i = tid; i < nb; i += 256) {
            const int t = a.bias_token[(int64_t)sq * a.bias_stride + i];
            const uint32_t e = (uint32_t)(t - v0);
            if (t >= 0 && e < (uint32_t)vn) atomicMax(&bias_at[e], (uint32_t)i + 1);
        }
    }
    __syncthreads();
    for (int e = tid; e < SEG; e += 256) {
        const bool is = count[e] || bias_at[e];
        const uint64_t all = __ballot(is);
        int at = 0;
        if (lane == 0) {
            hot_bits[e / 64] = all;
            if (all) at = atomicAdd(&n_hot, __popcll(all));
        }
        at = __shfl(at, 0);
        if (is) hot[at + __popcll(all & ((1ull << lane) - 1))] = (uint16_t)e;
    }
    __syncthreads();

    // ---- the rows
    const bool inplace = a.out == a.logits;
    auto grammar = [&](int r) -> const uint32_t * {
        if (!a.allow) return nullptr;
        const int row = a.allow_row ? a.allow_row[t0 + r] : t0 + r;
        return row < 0 || row >= a.n_allow ? nullptr : a.allow + row * a.allow_stride;
    };
    for (int r = r0; r < r1; r++) {
        const uint32_t *ok = grammar(r);
        if (!a.best && (!a.out || inplace) && !ok) continue;
        const T *x = (const T *)a.logits + (t0 + r) * a.stride + v0;
        T *y = a.out ? (T *)a.out + (t0 + r) * a.out_stride + v0 : nullptr;
        float best = -__builtin_inff();
        int best_at = 0;
        uint32_t best_may = 0;
        v4u best_v = {0, 0, 0, 0};
        for (int t = tid * N; t < vn; t += 256 * N) {
            const int left = vn - t;
            const uint32_t here = left >= N ? ALL : (1u << left) - 1;
            uint32_t may = here;
            if (ok) may &= ok[(v0 + t) >> 5] >> (t & 31);
            if (!a.best && inplace && may == here) continue;
            v4u v = {0, 0, 0, 0};
            if (left >= N) {
                if (a.best || may) v = ((const v4u_any *)(x + t))->v;
            } else {
                qmh_vec<T, N> e = {};
#pragma unroll
                for (int i = 0; i < N; i++)
                    if (i < left) e.e[i] = x[t + i];
                v = __builtin_bit_cast(v4u, e);
            }
            if (a.best) {
                const uint32_t eff = may & ~(uint32_t)(hot_bits[t / 64] >> (t & 63));
                float m = -__builtin_inff();
#pragma unroll
                for (int e = 0; e < N; e++) m = fmaxf(m, (eff >> e) & 1 ? element<T>(v, e) : -__builtin_inff());
                if (m > best) {
                    best = m;
                    best_at = t;
                    best_may = eff;
                    best_v = v;
                }
            }
            if (!y || (inplace && may == here)) continue;
            qmh_vec<T, N> e = __builtin_bit_cast(qmh_vec<T, N>, v);
#pragma unroll
            for (int i = 0; i < N; i++)
                if (!((may >> i) & 1)) e.e[i] = (T)-__builtin_inff();
            if (left >= N) ((v4u_any *)(y + t))->v = __builtin_bit_cast(v4u, e);
            else
#pragma unroll
                for (int i = 0; i < N; i++)
                    if (i < left) y[t + i] = e.e[i];
        }
        if (a.best) {
            const float top = qmh_wave_max(best);
            if (best == top && best > -__builtin_inff()) { // mostly one lane
                int at = 0;
#pragma unroll
                for (int e = N - 1; e >= 0; e--)
                    if ((best_may >> e) & 1 && element<T>(best_v, e) == best) at = e;
                atomicMax((unsigned long long *)&row_key[r - r0], (unsigned long long)best_key(best, v0 + best_at + at));
            }
        }
    }
    __syncthreads(); // the hot tokens' places are written again

    // ---- the hot tokens
    const int hots = n_hot;
    for (int i = tid; i < hots * (r1 - r0); i += 256) {
        const int r = r0 + i / hots, e = hot[i % hots], t = v0 + e;
        const uint32_t *ok = grammar(r);
        if (ok && !((ok[t >> 5] >> (t & 31)) & 1)) continue;
        uint32_t c = count[e], m = c & (NODE - 1);
        if (c & NODE) {
            const uint32_t *see = a.mask ? a.mask + sq * a.mask_stride + (int64_t)r * a.mask_words : nullptr;
            for (int k = 0; k < n_node; k++)
                if (node[k] == t && (see ? (see[k >> 5] >> (k & 31)) & 1 : k <= r)) m++;
        }
        float x = qmh_to_f(((const T *)a.logits)[(t0 + r) * a.stride + t]);
        if (m || c & PROMPT) x = x > 0.0f ? x / by : x * by;
        if (m) x -= frequency * (float)m + presence;
        if (bias_at[e]) x += a.bias[(int64_t)sq * a.bias_stride + bias_at[e] - 1];
        if (a.out) ((T *)a.out)[(t0 + r) * a.out_stride + t] = (T)x;
        if (a.best && x > -__builtin_inff()) atomicMax((unsigned long long *)&row_key[r - r0], (unsigned long long)best_key(x, t));
    }
    if (!a.best) return;
    __syncthreads();
    if (tid < r1 - r0) {
        const uint64_t key = row_key[tid];
        if (segs == 1) a.best[t0 + r0 + tid] = key ? (int)~(uint32_t)key : -1;
        else keys[(int64_t)(t0 + r0 + tid) * segs + seg] = key;
    }
}

// a row's best over its segments: a wave a row, a workgroup a sequence
__global__ __launch_bounds__(256) void k_logits_best(const qmh_logits_args a, int segs, const uint64_t *keys) {
    const int lane = threadIdx.x & 63;
    int t0;
    const int n = logits_rows(a, blockIdx.x, t0);
    for (int r = threadIdx.x >> 6; r < n; r += 4) {
        uint64_t key = 0;
        for (int s = lane; s < segs; s += 64) key = max(key, keys[(int64_t)(t0 + r) * segs + s]);
#pragma unroll
        for (int k = 1; k < 64; k <<= 1) key = max(key, (uint64_t)__shfl_xor((unsigned long long)key, k));
        if (lane == 0) a.best[t0 + r] = key ? (int)~(uint32_t)key : -1;
    }
}

int segments(const qmh_logits_args *a) { return (a->vocab + SEG - 1) / SEG; }

} // namespace

extern "C" size_t qmh_logits_ws_bytes(const qmh_logits_args *a, int) {
    const int segs = segments(a);
    return a->best && segs > 1 ? sizeof(uint64_t) * (size_t)a->n_rows * segs : 0;
}

extern "C" int qmh_launch_logits_edit(const qmh_logits_args *a, int cus, void *ws, void *stream) {
    hipStream_t st = (hipStream_t)stream;
    const int segs = segments(a);
    const int64_t units = (int64_t)a->n_seq * segs;
    // rows of a workgroup: as many as leave about four workgroups a CU, which count the history again each
    int most = a->rows_per_seq < a->n_rows ? a->rows_per_seq : a->n_rows;
    int chunks = (int)((4 * cus + units - 1) / units);
    chunks = chunks < most ? chunks : most;
    if (chunks < (most + ROWS - 1) / ROWS) chunks = (most + ROWS - 1) / ROWS;
    const int chunk = (most + chunks - 1) / chunks;
    chunks = (most + chunk - 1) / chunk;
    const int64_t blocks = units * chunks;
    if (blocks > 0xffffffffll) return (int)hipErrorInvalidValue;
    qmh_for_type(a->dtype, [&](auto z) {
        using T = decltype(z);
        for (int64_t b0 = 0; b0 < blocks; b0 += QMH_MOST_BLOCKS) { // workgroups write different places: any number of launches
            const dim3 g((uint32_t)(blocks - b0 < QMH_MOST_BLOCKS ? blocks - b0 : QMH_MOST_BLOCKS));
            hipLaunchKernelGGL((k_logits_edit<T>), g, dim3(256), 0, st, *a, segs, chunks, chunk, (uint32_t)b0, (uint64_t *)ws);
        }
    });
    if (a->best && segs > 1) hipLaunchKernelGGL(k_logits_best, dim3(a->n_seq), dim3(256), 0, st, *a, segs, (const uint64_t *)ws);
    return (int)hipGetLastError();
}
