// Element types of rows, pages and logits (f32, f16, bf16) for the kernels that are templates over them.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

typedef _Float16 qmh_f16;
typedef __bf16 qmh_bf16;

__device__ __forceinline__ float qmh_to_f(float x) { return x; }
__device__ __forceinline__ float qmh_to_f(qmh_f16 x) { return (float)x; }
__device__ __forceinline__ float qmh_to_f(qmh_bf16 x) { return (float)x; }

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
