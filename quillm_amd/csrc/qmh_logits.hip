// gfx950 kernels of qmh_logits_edit: penalties for repeated tokens, biases and grammar masks on rows of logits, and each
// row's best token. No reference counterpart.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "qmh_device.h"
#include "qmh_launch.h"
#include "qmh_types.h"

namespace {

// A workgroup takes a segment of the vocabulary for some rows of one sequence. First it counts the history's tokens that fall into its
// segment, in LDS, and lists the tokens that any edit touches (the hot ones). A dense pass then goes over pieces of the rows, a wave
// a piece: it copies them (where they go elsewhere), puts -inf where the grammar forbids a token, and finds the best of the
// tokens that are not hot; it is left out where there is nothing of it to do, and vectors that stay as they are, or are forbidden as a whole,
// are not read. A sparse pass edits the hot ones: they are few, so their divisions and gathers do not weigh (in the dense pass, each lane
// its own, they cost 24-row trees 25 us instead of 18).
// What bounds it, measured: one row of 32000 f32 edited in place 5 us, a launch and the chain numbers, history, count, list, gather; 384
// rows of 32003 bf16, best tokens alone, 18.7 us: two launches, and per workgroup 10 us of that chain and its 1000 VALU instructions a wave (the
// read itself is 5 us); 160 rows of 128256 f32 written elsewhere 49 us for 166 MB, 39 of it without a history of 4000. Twice the rows
// under way, eight waves a SIMD and a wave a whole row's segment gained nothing.
constexpr int SEG = 4096, NT = 512;
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

// x where the mask is all ones, -inf where it is 0
__device__ __forceinline__ float choose(int mask, float x) {
    return __uint_as_float((__float_as_uint(x) & (uint32_t)mask) | (0xff800000u & ~(uint32_t)mask));
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
__global__ __launch_bounds__(NT) __attribute__((amdgpu_waves_per_eu(6))) void k_logits_edit(const qmh_logits_args a, int segs, int chunks, int chunk, uint32_t first_block, uint64_t *keys) {
    constexpr int N = 16 / (int)sizeof(T);     // tokens of a vector
    constexpr int VB = 4, PIECE = VB * 64 * N; // vectors of a lane, tokens of a wave at a time
    constexpr uint32_t ALL = (1u << N) - 1;
    __shared__ __align__(16) uint32_t count[SEG], bias_at[SEG];
    __shared__ uint16_t hot[SEG];
    __shared__ __align__(16) uint8_t hot_bits[SEG / 4]; // four tokens a byte
    __shared__ uint64_t row_key[ROWS];
    __shared__ int row_allow[ROWS], node[1024];
    __shared__ int n_hot;
    const uint32_t b = blockIdx.x + first_block, unit = b / chunks, sq = unit / segs;
    const int seg = unit - sq * segs, tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    int t0;
    const int n = logits_rows(a, sq, t0), r0 = (int)(b - unit * chunks) * chunk, r1 = min(r0 + chunk, n);
    if (r0 >= n) return;
    const int v0 = seg * SEG, vn = min(SEG, a.vocab - v0); // the segment's tokens
    const float rep = a.repetition ? a.repetition[sq] : 1.0f, by = rep > 0.0f ? rep : 1.0f;
    const float presence = a.presence ? a.presence[sq] : 0.0f, frequency = a.frequency ? a.frequency[sq] : 0.0f;
    const int said = a.history ? a.history_len[sq] : 0, prompt = a.prompt_len ? a.prompt_len[sq] : 0, biased = a.bias ? a.bias_len[sq] : 0;
    const bool penal = by != 1.0f || presence != 0.0f || frequency != 0.0f;
    const int n_node = penal && a.node_token ? n : 0;
    const bool inplace = a.out == a.logits, all_read = a.best || (a.out && !inplace);

    // Pieces of rows, dealt out to the waves. A wave's first one is loaded while the history is counted.
    const bool whole = vn == SEG;
    const int pieces = whole ? SEG / PIECE : (vn + PIECE - 1) / PIECE, tasks = (r1 - r0) * pieces;
    v4u x[VB];
    const uint32_t *ok;
    uint32_t words[VB];
    auto fetch = [&](int task) {
        const int row = task / pieces, p0 = (task - row * pieces) * PIECE + lane * N;
        ok = nullptr;
        if (a.allow) {
            const int ar = a.allow_row ? a.allow_row[t0 + r0 + row] : t0 + r0 + row;
            if (ar >= 0 && ar < a.n_allow) ok = a.allow + ar * a.allow_stride + (v0 >> 5);
        }
        if (ok)
#pragma unroll
            for (int k = 0; k < VB; k++)
                if (p0 + k * 64 * N < vn) words[k] = ok[(p0 + k * 64 * N) >> 5];
        if (!all_read) return;
        const T *from = (const T *)a.logits + (t0 + r0 + row) * a.stride + v0 + p0;
        if (whole) {
#pragma unroll
            for (int k = 0; k < VB; k++) x[k] = ((const v4u_any *)(from + k * 64 * N))->v;
            return;
        }
#pragma unroll
        for (int k = 0; k < VB; k++)
            if (p0 + k * 64 * N + N <= vn) x[k] = ((const v4u_any *)(from + k * 64 * N))->v;
        const int k = (vn - p0) / (64 * N), left = (vn - p0) % (64 * N); // the vocabulary's last tokens, where they fill no vector
        if (vn > p0 && k < VB && left < N) {
            qmh_vec<T, N> e = {};
#pragma unroll
            for (int i = 0; i < N - 1; i++)
                if (i < left) e.e[i] = from[k * 64 * N + i];
#pragma unroll
            for (int q = 0; q < VB; q++)
                if (q == k) x[q] = __builtin_bit_cast(v4u, e);
        }
    };
    if (w < tasks) fetch(w);
    // so are the lists' first tokens
    constexpr int HB = sizeof(T) == 4 ? 8 : 4;
    const int h = penal && said > 0 ? (int)min((int64_t)said, a.history_stride) : 0, nb = min(biased, a.bias_stride);
    const int32_t *hist = a.history + sq * a.history_stride, *biases = a.bias_token + (int64_t)sq * a.bias_stride;
    int early[HB];
#pragma unroll
    for (int k = 0; k < HB; k++) early[k] = tid + k * NT < h ? hist[tid + k * NT] : -1;
    const int early_bias = tid < nb ? biases[tid] : -1, early_node = tid < n_node ? a.node_token[(int64_t)sq * a.node_stride + tid] : -1;

    // ---- what is touched
    for (int i = tid; i < SEG / 4; i += NT) ((v4u *)count)[i] = ((v4u *)bias_at)[i] = (v4u){0, 0, 0, 0};
    if (tid < ROWS) {
        row_key[tid] = 0;
        const int r = r0 + tid;
        int row = -1;
        if (a.allow && r < r1) row = a.allow_row ? a.allow_row[t0 + r] : t0 + r;
        row_allow[tid] = row < a.n_allow ? row : -1;
    }
    if (tid == 0) n_hot = 0;
    __syncthreads();
    auto told = [&](int t, int i) { // token t, the history's i-th
        const uint32_t e = (uint32_t)(t - v0);
        if (t < 0 || e >= (uint32_t)vn) return;
        if (i < prompt) atomicOr(&count[e], PROMPT);
        else atomicAdd(&count[e], 1u);
    };
#pragma unroll
    for (int k = 0; k < HB; k++) told(early[k], tid + k * NT);
    for (int i0 = tid + HB * NT; i0 < h; i0 += HB * NT) {
        int t[HB];
#pragma unroll
        for (int k = 0; k < HB; k++) t[k] = i0 + k * NT < h ? hist[i0 + k * NT] : -1;
#pragma unroll
        for (int k = 0; k < HB; k++) told(t[k], i0 + k * NT);
    }
    for (int k = tid; k < n_node; k += NT) {
        const int t = k == tid ? early_node : a.node_token[(int64_t)sq * a.node_stride + k];
        const uint32_t e = (uint32_t)(t - v0);
        node[k] = t;
        if (t >= 0 && e < (uint32_t)vn) atomicOr(&count[e], NODE);
    }
    for (int i = tid; i < nb; i += NT) {
        const int t = i == tid ? early_bias : biases[i];
        const uint32_t e = (uint32_t)(t - v0);
        if (t >= 0 && e < (uint32_t)vn) atomicMax(&bias_at[e], (uint32_t)i + 1);
    }
    __syncthreads();
    { // a thread looks at four tokens at a time, a wave lists the hot ones of its share with one atomic
        constexpr int Q = SEG / (4 * NT);
        uint64_t is[Q][4];
        int mine = 0;
#pragma unroll
        for (int q = 0; q < Q; q++) {
            v4u c = ((v4u *)count)[q * NT + tid];
            if (biased > 0) c |= ((v4u *)bias_at)[q * NT + tid];
            uint32_t byte = 0;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                is[q][j] = __ballot(c[j] != 0);
                mine += __popcll(is[q][j]);
                byte |= c[j] ? 1u << j : 0u;
            }
            hot_bits[q * NT + tid] = (uint8_t)byte;
        }
        int at = 0;
        if (lane == 0 && mine) at = atomicAdd(&n_hot, mine);
        at = __builtin_amdgcn_readfirstlane(at);
        if (mine)
#pragma unroll
            for (int q = 0; q < Q; q++)
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    if ((is[q][j] >> lane) & 1)
                        hot[at + __builtin_amdgcn_mbcnt_hi((uint32_t)(is[q][j] >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)is[q][j], 0))] =
                            (uint16_t)(4 * (q * NT + tid) + j);
                    at += __popcll(is[q][j]);
                }
    }
    __syncthreads();

    // ---- the rows
    for (int task = w; task < tasks; task += NT / 64) {
        const int row = task / pieces, r = r0 + row, p0 = (task - row * pieces) * PIECE + lane * N;
        if (task != w) fetch(task);
        if (!all_read && !ok) continue;
        uint32_t may[VB];
#pragma unroll
        for (int k = 0; k < VB; k++) {
            const int t = p0 + k * 64 * N;
            may[k] = ALL;
            if (!whole) may[k] = vn - t >= N ? ALL : vn > t ? (1u << (vn - t)) - 1 : 0u;
            if (ok && t < vn) may[k] &= words[k] >> (t & 31);
        }
        if (a.best) {
            float best = -__builtin_inff();
            int at = 0;
            uint32_t eff[VB];
#pragma unroll
            for (int k = 0; k < VB; k++) {
                const int t = p0 + k * 64 * N;
                uint32_t hots = hot_bits[t / 4];
                if constexpr (N == 8) hots |= (uint32_t)hot_bits[t / 4 + 1] << 4;
                eff[k] = may[k] & ~hots;
                float m = -__builtin_inff();
#pragma unroll
                for (int e = 0; e < N; e++) // a bit as a mask chooses the element or -inf
                    m = fmaxf(m, choose((int)(eff[k] << (31 - e)) >> 31, element<T>(x[k], e)));
                if (m > best) {
                    best = m;
                    at = k;
                }
            }
            const float top = qmh_wave_max(best); // every lane takes part
            if (best == top && best > -__builtin_inff()) { // mostly one lane
                uint32_t same = 0;
#pragma unroll
                for (int k = 0; k < VB; k++)
                    if (at == k)
#pragma unroll
                        for (int e = 0; e < N; e++) same |= element<T>(x[k], e) == best ? eff[k] & 1u << e : 0u;
                const int t = v0 + p0 + at * 64 * N + __builtin_ctz(same);
                atomicMax((unsigned long long *)&row_key[row], (unsigned long long)best_key(best, t));
            }
        }
        if (!a.out) continue;
        const T *from = (const T *)a.logits + (t0 + r) * a.stride + v0 + p0;
        T *to = (T *)a.out + (t0 + r) * a.out_stride + v0 + p0;
#pragma unroll
        for (int k = 0; k < VB; k++) {
            const int left = vn - p0 - k * 64 * N;
            if (inplace && may[k] == ALL) continue;
            if (whole || left >= N) {
                v4u v = {0, 0, 0, 0};
                if (all_read) v = x[k];
                else if (may[k]) v = ((const v4u_any *)(from + k * 64 * N))->v; // of what is forbidden as a whole nothing is read
                qmh_vec<T, N> e = __builtin_bit_cast(qmh_vec<T, N>, v);
#pragma unroll
                for (int i = 0; i < N; i++)
                    if (!((may[k] >> i) & 1)) e.e[i] = (T)-__builtin_inff();
                ((v4u_any *)(to + k * 64 * N))->v = __builtin_bit_cast(v4u, e);
            } else {
                for (int i = 0; i < left; i++)
                    if (!(inplace && (may[k] >> i) & 1)) to[k * 64 * N + i] = (may[k] >> i) & 1 ? from[k * 64 * N + i] : (T)-__builtin_inff();
            }
        }
    }
    __syncthreads(); // the hot tokens' places are written again, and what the rows hold is known

    // ---- the hot tokens: one a thread, four rows at a time
    const int hots = n_hot;
    for (int i = tid; i < hots; i += NT) {
        const int e = hot[i], t = v0 + e;
        const uint32_t c = count[e], ba = bias_at[e];
        const float bias = ba ? a.bias[(int64_t)sq * a.bias_stride + ba - 1] : 0.0f;
        for (int ra = r0; ra < r1; ra += 4) {
            T v[4];
            uint32_t may[4], path[4] = {0, 0, 0, 0}; // how often the rows' own paths have the token
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const int r = min(ra + k, r1 - 1), ar = row_allow[r - r0];
                v[k] = ((const T *)a.logits)[(t0 + r) * a.stride + t];
                may[k] = ar < 0 ? ~0u : a.allow[ar * a.allow_stride + (t >> 5)];
            }
            if (c & NODE)
                for (int q0 = 0; q0 < n_node; q0 += 32) {
                    uint32_t at = 0; // which of 32 nodes have it
                    for (int q = 0; q < 32 && q0 + q < n_node; q++) at |= (uint32_t)(node[q0 + q] == t) << q;
                    if (!at) continue;
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        const int r = min(ra + k, r1 - 1), chain = r + 1 - q0;
                        const uint32_t see = a.mask ? a.mask[sq * a.mask_stride + (int64_t)r * a.mask_words + (q0 >> 5)]
                                                    : chain >= 32 ? ~0u : chain <= 0 ? 0u : (1u << chain) - 1;
                        path[k] += __popc(at & see);
                    }
                }
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const int r = ra + k;
                if (r >= r1 || !((may[k] >> (t & 31)) & 1)) continue;
                const uint32_t m = (c & (NODE - 1)) + path[k];
                float y = qmh_to_f(v[k]);
                if (m || c & PROMPT) y = y > 0.0f ? y / by : y * by;
                if (m) y -= frequency * (float)m + presence;
                if (ba) y += bias;
                if (a.out) ((T *)a.out)[(t0 + r) * a.out_stride + t] = (T)y;
                if (!a.best) continue;
                const uint64_t key = y > -__builtin_inff() ? best_key(y, t) : 0;
                if (key > row_key[r - r0]) atomicMax((unsigned long long *)&row_key[r - r0], (unsigned long long)key); // few are
            }
        }
    }
    if (!a.best) return;
    __syncthreads();
    if (tid < r1 - r0) {
        const uint64_t key = row_key[tid];
        if (segs == 1) a.best[t0 + r0 + tid] = key ? (int)~(uint32_t)key : -1;
        else keys[(int64_t)(t0 + r0 + tid) * segs + seg] = key;
    }
}

// a row's best over its segments: a wave a row
__global__ __launch_bounds__(256) void k_logits_best(const qmh_logits_args a, int segs, const uint64_t *keys) {
    const int lane = threadIdx.x & 63;
    int t0;
    const int n = logits_rows(a, blockIdx.x, t0);
    for (int r = blockIdx.y * 4 + (threadIdx.x >> 6); r < n; r += gridDim.y * 4) {
        uint64_t key = 0;
        for (int s = lane; s < segs; s += 64) key = max(key, keys[(int64_t)(t0 + r) * segs + s]);
#pragma unroll
        for (int k = 1; k < 64; k <<= 1) key = max(key, (uint64_t)__shfl_xor((unsigned long long)key, k));
        if (lane == 0) a.best[t0 + r] = key ? (int)~(uint32_t)key : -1;
    }
}

int segments(const qmh_logits_args *a) { return (a->vocab + SEG - 1) / SEG; }
// rows of a sequence, at most
int most_rows(const qmh_logits_args *a) { return a->rows_per_seq < a->n_rows ? a->rows_per_seq : a->n_rows; }

} // namespace

extern "C" size_t qmh_logits_ws_bytes(const qmh_logits_args *a, int) {
    const int segs = segments(a);
    return a->best && segs > 1 ? sizeof(uint64_t) * (size_t)a->n_rows * segs : 0;
}

extern "C" int64_t qmh_logits_blocks(const qmh_logits_args *a) { return (int64_t)a->n_seq * segments(a) * ((most_rows(a) + ROWS - 1) / ROWS); }

extern "C" int qmh_launch_logits_edit(const qmh_logits_args *a, int cus, void *ws, void *stream) {
    hipStream_t st = (hipStream_t)stream;
    const int segs = segments(a);
    const int64_t units = (int64_t)a->n_seq * segs;
    // rows of a workgroup: as few as fill the chip's workgroups once (three a CU); each counts the history again
    const int most = most_rows(a);
    int chunks = units < 3 * cus ? (int)(3 * cus / units) : 1;
    chunks = chunks < most ? chunks : most;
    if (chunks < (most + ROWS - 1) / ROWS) chunks = (most + ROWS - 1) / ROWS;
    const int chunk = (most + chunks - 1) / chunks;
    chunks = (most + chunk - 1) / chunk;
    const int64_t blocks = units * chunks; // below 2^32: the host code checks it
    qmh_for_type(a->dtype, [&](auto z) {
        using T = decltype(z);
        constexpr int64_t most_blocks = qmh_most_blocks(NT);
        for (int64_t b0 = 0; b0 < blocks; b0 += most_blocks) { // workgroups write different places: any number of launches
            const dim3 g((uint32_t)(blocks - b0 < most_blocks ? blocks - b0 : most_blocks));
            hipLaunchKernelGGL((k_logits_edit<T>), g, dim3(NT), 0, st, *a, segs, chunks, chunk, (uint32_t)b0, (uint64_t *)ws);
        }
    });
    const int failed = (int)hipGetLastError();
    if (failed) return failed; // what the next one reads is not there
    if (a->best && segs > 1) hipLaunchKernelGGL(k_logits_best, dim3(a->n_seq, most < 4 * 60 ? (most + 3) / 4 : 60), dim3(256), 0, st, *a, segs, (const uint64_t *)ws);
    return (int)hipGetLastError();
}
