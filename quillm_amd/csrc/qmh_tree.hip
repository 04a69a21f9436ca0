// gfx950 kernels for drafted trees over a paged cache: qmh_paged_plan (pages, rows, slots, positions, masks), qmh_tree_attention
// (its kernel is the one of qmh_paged_attn.h) and qmh_tree_accept. No reference counterpart.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "qmh_device.h"
#include "qmh_launch.h"
#include "qmh_paged_attn.h"
#include "qmh_types.h"

namespace {

// --------------------------------------------------------------------------- plan

constexpr int PLAN_SEQS = 1024;    // sequences and
constexpr int PLAN_TOKENS = 4096;  // tokens of a call that one workgroup does alone
constexpr int PLAN_CHUNK = 1024;   // tokens of a workgroup otherwise
constexpr int TREE_MOST = 1024;    // nodes of a tree

// Nothing here computes: a call is a chain of loads (lengths, sums, pages or parents, stores), so the work goes into as few launches and
// dependent steps as can be. A node's thread walks to its root, a read of LDS a step. Measured: trees of 48 sequences, 870 nodes, 4.2 us, an empty launch's time; prompts of 201 sequences, 181000 rows
// in two launches 10 us (3.4 of scan, 6 of rows, 2.2 MB).
// What the scan finds: exclusive sums over the sequences (n + 1 of each) of tokens, pages taken and pages given, a sequence's pages
// before and after, and the positions it keeps. For a call of one workgroup they lie in LDS, else in the workspace.
struct plan_arrays {
    int *tok, *take, *give, *have, *need, *keep, *ring; // ring: its first free page and how many there are
};

__device__ __forceinline__ bool plan_ring(const qmh_plan_args &a, int first, int count) {
    return first >= 0 && first < a.free_size && count >= 0 && count <= a.free_size;
}

struct __attribute__((packed, aligned(4))) plan_four {
    int x[4];
};

// the sequence that number k of the ones counted in start[0..n] belongs to (k < start[n])
__device__ __forceinline__ int plan_find(const int *start, int n, int k) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (start[mid] <= k) lo = mid;
        else hi = mid;
    }
    return lo;
}

// inclusive sum over the wave's lanes
__device__ __forceinline__ int wave_sums(int x) {
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, true); // row_shr:1 and on, 16 lanes a row
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false); // row_bcast:15 to rows 1 and 3
    x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false); // row_bcast:31 to rows 2 and 3
    return x;
}

// inclusive sums of N values over the workgroup's WAVES waves; total: of all of them. part: of this call alone
template <int N, int WAVES>
__device__ __forceinline__ void plan_sums(int (&x)[N], int (&total)[N], int *part) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
#pragma unroll
    for (int i = 0; i < N; i++) x[i] = wave_sums(x[i]);
    if constexpr (WAVES == 1) {
#pragma unroll
        for (int i = 0; i < N; i++) total[i] = __builtin_amdgcn_readlane(x[i], 63);
        return;
    }
    if (lane == 63)
#pragma unroll
        for (int i = 0; i < N; i++) part[i * WAVES + w] = x[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; i++) {
        const int sum = wave_sums(lane < WAVES ? part[i * WAVES + lane] : 0);
        total[i] = __builtin_amdgcn_readlane(sum, WAVES - 1);
        const int before = __shfl(sum, w - 1);
        x[i] += w ? before : 0;
    }
}

// WAVES waves go over the sequences and say what becomes of each. Sums of what is asked for decide who is served; sums over
// the served ones say where their pages and rows are. Pages add up to less than 2^31 (the tables have no more places); rows
// that are asked for are counted up to what there is and one more.
template <int WAVES>
__device__ __forceinline__ void plan_scan(const qmh_plan_args &a, const plan_arrays &p) {
    __shared__ int part[2][7 * WAVES]; // of every other round
    const int ring_first = a.free_state[0], ring_count = a.free_state[1];
    const bool ring_ok = plan_ring(a, ring_first, ring_count);
    const int pages_left = ring_ok ? ring_count : 0, room = ring_ok ? a.free_size - ring_count : 0;
    const int64_t cap = (int64_t)a.table_stride * a.page_size;
    const int lg = __builtin_ctz(a.page_size);
    int asked_take = 0, asked_give = 0, at_tok = 0, at_take = 0, at_give = 0;
    int64_t asked_tok = 0;
    for (int s0 = 0; s0 < a.n_seq; s0 += 64 * WAVES) {
        int *mine = part[(s0 / (64 * WAVES)) & 1];
        const int s = s0 + threadIdx.x;
        int why = 3, take = 0, give = 0, have = 0, need = 0, add = 0, keep = 0;
        if (s < a.n_seq) {
            const int len = a.len[s];
            keep = a.keep ? a.keep[s] : len;
            add = a.add ? a.add[s] : 0;
            const bool fine = len >= 0 && len <= cap && keep >= 0 && keep <= len && add >= 0 && (int64_t)keep + add <= cap && (!a.parent || add <= a.tree_size);
            if (fine) {
                why = 0;
                have = (int)(((int64_t)len + a.page_size - 1) >> lg);
                need = (int)(((int64_t)keep + add + a.page_size - 1) >> lg);
                take = need > have ? need - have : 0;
                give = have > need ? have - need : 0;
            }
        }
        int pages[2] = {take, give}, all[2];
        plan_sums<2, WAVES>(pages, all, mine);
        if (!why && ((take && (int64_t)asked_take + pages[0] > pages_left) || (give && (int64_t)asked_give + pages[1] > room))) why = 1;
        asked_take += all[0];
        asked_give += all[1];
        // 1024 rows of up to 2^24 + 1 pass 32 bits: their upper and lower halves do not
        const int want = why ? 0 : min(add, a.n_tokens + 1);
        int rows[2] = {want >> 12, want & 4095}, rows_all[2];
        plan_sums<2, WAVES>(rows, rows_all, mine + 2 * WAVES);
        if (!why && add && asked_tok + ((int64_t)rows[0] << 12) + rows[1] > a.n_tokens) why = 2;
        asked_tok += ((int64_t)rows_all[0] << 12) + rows_all[1];
        if (why) take = give = add = 0;
        int got[3] = {add, take, give}, sum[3];
        plan_sums<3, WAVES>(got, sum, mine + 4 * WAVES);
        if (s < a.n_seq) {
            p.tok[s] = at_tok + got[0] - add;
            p.take[s] = at_take + got[1] - take;
            p.give[s] = at_give + got[2] - give;
            p.have[s] = have;
            p.need[s] = need;
            p.keep[s] = keep;
            if (!why) a.len[s] = keep + add;
            if (a.refused) a.refused[s] = why;
            if (a.n_tokens) a.first[s] = at_tok + got[0] - add;
        }
        at_tok += sum[0];
        at_take += sum[1];
        at_give += sum[2];
    }
    if (threadIdx.x == 0) {
        p.tok[a.n_seq] = at_tok;
        p.take[a.n_seq] = at_take;
        p.give[a.n_seq] = at_give;
        p.ring[0] = ring_ok ? ring_first : 0;
        p.ring[1] = pages_left;
        if (a.n_tokens) a.first[a.n_seq] = at_tok;
        if (ring_ok) {
            const uint32_t f = (uint32_t)ring_first + at_take;
            a.free_state[0] = (int)(f >= (uint32_t)a.free_size ? f - a.free_size : f);
            a.free_state[1] = ring_count - at_take + at_give;
        }
    }
}

// Pages k0, k0 + step, ... of those that move, each found by its number: any split of them over sequences costs the same.
__device__ __forceinline__ void plan_pages(const qmh_plan_args &a, const plan_arrays &p, int k0, int step) {
    const int n = a.n_seq, takes = p.take[n], gives = p.give[n], first = p.ring[0], count = p.ring[1];
    auto ring = [&](uint32_t k) { // below 3 times its size
        const uint32_t z = a.free_size;
        k = k >= z ? k - z : k;
        return a.free_pages + (k >= z ? k - z : k);
    };
    for (int k = k0; k < takes; k += step) {
        const int page = *ring((uint32_t)first + k), s = plan_find(p.take, n, k);
        a.table[(int64_t)s * a.table_stride + p.have[s] + (k - p.take[s])] = page;
    }
    for (int k = k0; k < gives; k += step) {
        const int s = plan_find(p.give, n, k);
        int32_t *at = a.table + (int64_t)s * a.table_stride + p.need[s] + (k - p.give[s]);
        *ring((uint32_t)first + count + k) = *at;
        *at = -1;
    }
}

// Tokens [t0, t1) of all sequences' rows. par: room for t1 - t0 + TREE_MOST parents (trees).
__device__ __forceinline__ void plan_tokens(const qmh_plan_args &a, const plan_arrays &p, int t0, int t1, int16_t *par) {
    const int n = a.n_seq, total = p.tok[n], end = t1 < total ? t1 : total;
    if (!a.parent) { // four a thread: mostly of one sequence
        for (int t = t0 + 4 * threadIdx.x; t < t1; t += 4 * blockDim.x) {
            int x[3][4], s = t < total ? plan_find(p.tok, n, t) : n;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                if (t + i >= total) s = n;
                else if (t + i >= p.tok[s + 1] && t + i >= p.tok[++s + 1]) s = plan_find(p.tok, n, t + i); // past sequences without rows
                const int slot = s < n ? p.keep[s] + (t + i - p.tok[s]) : -1;
                x[0][i] = s < n ? s : -1;
                x[1][i] = slot;
                x[2][i] = s < n ? (int)((uint32_t)(a.base ? a.base[s] : 0) + slot) : -1;
            }
            int32_t *out[3] = {a.seq + t, a.slot + t, a.pos + t};
#pragma unroll
            for (int k = 0; k < 3; k++)
                if (t + 4 <= t1) *(plan_four *)out[k] = *(const plan_four *)x[k];
                else
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        if (t + i < t1) out[k][i] = x[k][i];
        }
        return;
    }
    int from = t0;
    if (t0 < end) {
        from = p.tok[plan_find(p.tok, n, t0)]; // the first token's tree from its root on
        for (int t = from + threadIdx.x; t < end; t += blockDim.x) {
            const int s = plan_find(p.tok, n, t), j = t - p.tok[s], x = a.parent[(int64_t)s * a.parent_stride + j];
            par[t - from] = (int16_t)(x < 0 || x >= j ? -1 : x);
        }
        __syncthreads();
    }
    const int words = (a.tree_size + 31) >> 5;
    for (int t = t0 + threadIdx.x; t < t1; t += blockDim.x) {
        if (t >= total) {
            a.seq[t] = a.slot[t] = a.pos[t] = -1;
            continue;
        }
        const int s = plan_find(p.tok, n, t), j = t - p.tok[s], keep = p.keep[s], base = a.base ? a.base[s] : 0;
        const int16_t *up = par + (p.tok[s] - from);
        uint32_t *out = a.mask ? a.mask + ((int64_t)s * a.tree_size + j) * words : nullptr;
        // one walk: ancestors come in falling order, so the mask's words are done with from the last one down
        int depth = -1, x = j;
        for (int w = (words - 1) & ~1; w >= 0; w -= 2) {
            uint64_t bits = 0;
            for (; x >= 32 * w; x = up[x]) bits |= 1ull << (x & 63);
            depth += __popcll(bits);
            if (out) {
                out[w] = (uint32_t)bits;
                if (w + 1 < words) out[w + 1] = (uint32_t)(bits >> 32);
            }
        }
        a.seq[t] = s;
        a.slot[t] = keep + j;
        a.pos[t] = (int)((uint32_t)base + keep + depth);
    }
}

// NS: sequences whose numbers LDS has room for
template <int NS>
struct plan_room {
    int tok[NS + 1], take[NS + 1], give[NS + 1], have[NS], need[NS], keep[NS], ring[2];
    __device__ __forceinline__ plan_arrays in() { return plan_arrays{tok, take, give, have, need, keep, ring}; }
};

__global__ __launch_bounds__(1024) void k_plan_one(const qmh_plan_args a) {
    __shared__ plan_room<PLAN_SEQS> room;
    __shared__ int16_t par[PLAN_TOKENS];
    const plan_arrays p = room.in();
    if (a.n_seq > 64) plan_scan<16>(a, p);
    else if (threadIdx.x < 64) plan_scan<1>(a, p);
    __syncthreads();
    plan_pages(a, p, threadIdx.x, 1024);
    if (a.n_tokens) plan_tokens(a, p, 0, a.n_tokens, par);
}

__device__ __forceinline__ plan_arrays plan_in(int *ws, int n) {
    int *x = ws + 4;
    return plan_arrays{x, x + n + 1, x + 2 * (n + 1), x + 3 * (n + 1), x + 3 * (n + 1) + n, x + 3 * (n + 1) + 2 * n, ws};
}

__global__ __launch_bounds__(1024) void k_plan_scan(const qmh_plan_args a, int *ws) { plan_scan<16>(a, plan_in(ws, a.n_seq)); }

__global__ __launch_bounds__(256) void k_plan_write(const qmh_plan_args a, int *ws) {
    __shared__ plan_room<PLAN_SEQS> room;
    __shared__ int16_t par[PLAN_CHUNK + TREE_MOST];
    plan_arrays p = plan_in(ws, a.n_seq);
    if (a.n_seq <= PLAN_SEQS) { // the searches go through LDS
        const int n = a.n_seq;
        for (int s = threadIdx.x; s <= n; s += 256) {
            room.tok[s] = p.tok[s];
            room.take[s] = p.take[s];
            room.give[s] = p.give[s];
            if (s < n) {
                room.have[s] = p.have[s];
                room.need[s] = p.need[s];
                room.keep[s] = p.keep[s];
            }
        }
        if (threadIdx.x < 2) room.ring[threadIdx.x] = p.ring[threadIdx.x];
        __syncthreads();
        p = room.in();
    }
    plan_pages(a, p, blockIdx.x * 256 + threadIdx.x, gridDim.x * 256);
    const int t0 = (int)blockIdx.x * PLAN_CHUNK; // at most 2^24 / PLAN_CHUNK blocks
    if (t0 < a.n_tokens) plan_tokens(a, p, t0, min(t0 + PLAN_CHUNK, a.n_tokens), par);
}

// One workgroup does a call whose sums fit its LDS and whose rows it writes as fast as two launches would: a call of 200 sequences and
// 3600 tree nodes takes 6 us less there, of 3000 plain rows 2 us less, of 7500 as long.
bool plan_alone(const qmh_plan_args *a) { return a->n_seq <= PLAN_SEQS && a->n_tokens <= PLAN_TOKENS; }

// --------------------------------------------------------------------------- accept

// A workgroup (x: piece, y: sequence) follows the path and moves its piece of what the accepted positions hold. For each node the
// lowest of its children that the model chose is found by all threads at once, then the path is a chain of LDS reads. Positions
// only move down and in order, so a thread that loads eight of its unit before it stores them needs no second buffer. Every
// workgroup of a sequence follows the path for itself: a launch of its own would take longer. Measured: 4 trees of 16 nodes in 6 layers of 2 x 48
// f32 4.9 us, a launch and its chain (rows, nodes, path, pages, data); 64 trees of 61 in 4 layers of 32 x 128 f16, 27 MB, 8.9 us.
__global__ __launch_bounds__(256) void k_tree_accept(const qmh_accept_args a, const qmh_pages pg, int row_bytes, uint32_t units) {
    __shared__ int follow[TREE_MOST], path[TREE_MOST];
    __shared__ int64_t from[TREE_MOST], to[TREE_MOST];
    __shared__ int found[2];
    const int sq = blockIdx.y, tid = threadIdx.x;
    int t0 = sq * a.tree_size, n = a.tree_size; // below n_rows, which the host checks
    bool fine = true;
    if (a.first) {
        t0 = a.first[sq];
        const int64_t t1 = a.first[sq + 1];
        fine = t0 >= 0 && t1 >= t0 && t1 - t0 <= a.tree_size && t1 <= a.n_rows;
        n = fine ? (int)(t1 - t0) : 0;
    }
    const int len = a.len[sq];
    fine = fine && len >= n && (!a.pages || len <= (int64_t)a.table_stride * pg.page_size);
    if (!fine) n = 0;
    const int32_t *parent = a.parent + (int64_t)sq * a.parent_stride, *token = a.token + (int64_t)sq * a.token_stride, *choice = a.choice + t0;
    for (int c = tid; c < n; c += 256) follow[c] = n;
    __syncthreads();
    for (int c = tid; c < n; c += 256) {
        const int p = parent[c], t = token[c];
        if (p >= 0 && p < c && t >= 0 && choice[p] == t) atomicMin(&follow[p], c);
    }
    __syncthreads();
    if (tid == 0) {
        int k = 0, same = 0;
        for (int x = 0; x < n; x = follow[x]) {
            path[k] = x;
            same += x == k;
            k++;
        }
        found[0] = k;
        found[1] = same; // positions that stay where they are: the path's first ones
    }
    __syncthreads();
    const int count = found[0], stay = found[1], begin = len - n;
    if (blockIdx.x == 0) {
        if (tid == 0) {
            a.count[sq] = count;
            a.next[sq] = count ? choice[path[count - 1]] : -1;
            a.keep[sq] = fine ? begin + count : -1;
        }
        if (a.path)
            for (int k = tid; k < a.tree_size; k += 256) a.path[(int64_t)sq * a.tree_size + k] = k < count ? path[k] : -1;
        if (a.history && count) {
            const int h = a.history_len[sq];
            if (h >= 0 && h < a.history_stride) {
                for (int k = tid; k < count && h + k < a.history_stride; k += 256) a.history[sq * a.history_stride + h + k] = token[path[k]];
                __syncthreads(); // every thread has the length
                if (tid == 0) a.history_len[sq] = (int)min((int64_t)h + count, a.history_stride);
            }
        }
    }
    if (!a.pages || count == stay) return;
    const int ps = pg.page_size, lg = __builtin_ctz(ps);
    const int64_t page_bytes = (int64_t)pg.n_kv_heads * ps * row_bytes;
    for (int k = stay + tid; k < count; k += 256) {
        const int x = begin + path[k], y = begin + k;
        const int px = a.table[(int64_t)sq * a.table_stride + (x >> lg)], py = a.table[(int64_t)sq * a.table_stride + (y >> lg)];
        const bool ok = px >= 0 && px < pg.n_pages && py >= 0 && py < pg.n_pages;
        from[k] = ok ? px * page_bytes + (int64_t)(x & (ps - 1)) * row_bytes : -1;
        to[k] = py * page_bytes + (int64_t)(y & (ps - 1)) * row_bytes;
    }
    __syncthreads();
    const uint32_t per_row = row_bytes / 16, per_layer = pg.n_kv_heads * per_row;
    const int64_t layer_bytes = a.layer_stride * (pg.dtype == QMH_F32 ? 4 : 2);
    for (uint32_t u = blockIdx.x * 256 + tid; u < units; u += gridDim.x * 256) {
        const uint32_t layer = u / (2 * per_layer), in = u - layer * 2 * per_layer, kv = in >= per_layer, x = in - kv * per_layer;
        const uint32_t h = x / per_row, o = x - h * per_row;
        uint8_t *pool = (uint8_t *)(kv ? pg.v : pg.k) + (layer ? layer * layer_bytes : 0) + (int64_t)h * ps * row_bytes + o * 16;
        for (int k = stay; k < count; k += 8) {
            v4u v[8];
            const int m = count - k;
#pragma unroll
            for (int i = 0; i < 8; i++)
                if (i < m && from[k + i] >= 0) v[i] = *(const v4u *)(pool + from[k + i]);
#pragma unroll
            for (int i = 0; i < 8; i++)
                if (i < m && from[k + i] >= 0) *(v4u *)(pool + to[k + i]) = v[i];
        }
    }
}

} // namespace

extern "C" size_t qmh_plan_ws_bytes(const qmh_plan_args *a) {
    return plan_alone(a) ? 0 : sizeof(int) * (4 + 6 * ((size_t)a->n_seq + 1));
}

extern "C" int qmh_launch_paged_plan(const qmh_plan_args *a, void *ws, void *stream) {
    hipStream_t st = (hipStream_t)stream;
    if (plan_alone(a)) {
        hipLaunchKernelGGL(k_plan_one, dim3(1), dim3(1024), 0, st, *a);
        return (int)hipGetLastError();
    }
    const int rows = (a->n_tokens + PLAN_CHUNK - 1) / PLAN_CHUNK, pages = (a->n_seq + 255) / 256;
    hipLaunchKernelGGL(k_plan_scan, dim3(1), dim3(1024), 0, st, *a, (int *)ws);
    hipLaunchKernelGGL(k_plan_write, dim3(rows > pages ? rows : pages), dim3(256), 0, st, *a, (int *)ws);
    return (int)hipGetLastError();
}

// the rows that sequences may have
static int tree_rows(const qmh_tree_args *a) { return a->first ? a->n_rows : a->base.n_seq * a->base.q_len; }

extern "C" size_t qmh_tree_ws_bytes(const qmh_tree_args *a, int cus) {
    return attention_ws<true>(&a->base, tree_rows(a), cus);
}

extern "C" int qmh_launch_tree_attention(const qmh_tree_args *a, int cus, void *ws, void *stream) {
    const attn_tree t = {tree_rows(a), a->first, a->mask, a->mask_stride, a->mask_words};
    return run_attention<true>(&a->base, t, cus, ws, (hipStream_t)stream);
}

extern "C" int qmh_launch_tree_accept(const qmh_accept_args *a, void *stream) {
    qmh_pages pg = {};
    int row_bytes = 16, pieces = 1;
    uint32_t units = 0;
    if (a->pages) {
        pg = *a->pages;
        row_bytes = pg.head_dim * (pg.dtype == QMH_F32 ? 4 : 2);
        units = (uint32_t)a->n_layers * 2 * pg.n_kv_heads * (row_bytes / 16); // at most 2^10 * 2 * 2^10 * 2^6
        const int64_t most = QMH_MOST_BLOCKS / a->n_seq; // at least 256
        pieces = (int)(units / 256 + 1 < most ? (units + 255) / 256 : most);
    }
    hipLaunchKernelGGL(k_tree_accept, dim3(pieces, a->n_seq), dim3(256), 0, (hipStream_t)stream, *a, pg, row_bytes, units);
    return (int)hipGetLastError();
}
