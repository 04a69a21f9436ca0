// Element types of rows, pages and logits (f32, f16, bf16) for the kernels that are templates over them.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

typedef _Float16 qmh_f16;
typedef __bf16 qmh_bf16;

__device__ __forceinline__ float qmh_to_f(float x) { return x; }
__device__ __forceinline__ float qmh_to_f(qmh_f16 x) { return (float)x; }
__device__ __forceinline__ float qmh_to_f(qmh_bf16 x) { return (float)x; }

// blocks of so many threads in a launch: a grid holds fewer than 2^32 threads
constexpr int64_t qmh_most_blocks(int threads) { return 0xffffffffll / threads; }
constexpr int64_t QMH_MOST_BLOCKS = qmh_most_blocks(256);
static_assert(QMH_MOST_BLOCKS == (1 << 24) - 1 && qmh_most_blocks(512) * 512 < 1ll << 32 && qmh_most_blocks(512) == (1 << 23) - 1);

// N elements of T that are loaded and stored at once (N * sizeof(T) up to 16 bytes, aligned to it)
template <typename T, int N>
struct alignas(sizeof(T) * N) qmh_vec {
    T e[N];
};

// body(T{}) for the element type of a dtype code
template <typename F>
static inline void qmh_for_type(int dtype, F body) {
    if (dtype == QMH_F32) body(float{});
    else if (dtype == QMH_F16) body(qmh_f16{});
    else body(qmh_bf16{});
}

// Past 16 beams a thread's unit of every beam goes through LDS (slot m * blockDim.x of keep, the thread's own: no barrier),
// eight loads under way at a time: get(m, u) loads beam m's unit, or says that it does not move, put(m, u) stores it.
template <typename U, typename G, typename P>
__device__ __forceinline__ void qmh_move_many(U *keep, int n, G get, P put) {
    for (int m0 = 0; m0 < n; m0 += 8) {
        U v[8];
        bool moves[8];
#pragma unroll
        for (int k = 0; k < 8; k++) moves[k] = m0 + k < n && get(m0 + k, v[k]);
#pragma unroll
        for (int k = 0; k < 8; k++)
            if (moves[k]) keep[(m0 + k) * 256] = v[k];
    }
    for (int m = 0; m < n; m++) put(m, keep[m * 256]);
}
