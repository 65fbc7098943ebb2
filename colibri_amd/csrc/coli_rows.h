// coli_rows.h -- rows of f32, fp16 or bf16 that start at any address their type
// allows (shared by sorted.hip and fp4.hip).
#pragma once

#include "coli_device.h"

typedef uint32_t u32x4a1 __attribute__((ext_vector_type(4), aligned(1)));   // 16 bytes at any address
typedef uint32_t u32a1 __attribute__((aligned(1)));
typedef uint16_t u16a1 __attribute__((aligned(1)));

// N elements from p on as f32, and back, rounded to nearest even: 16 bytes a load. NT: past
// the caches.
template <typename T, int N, bool NT = false> __device__ __forceinline__ void el_load(const T *p, float (&f)[N]) {
    constexpr int V = 16 / sizeof(T);
    if constexpr (N % V) {
#pragma unroll
        for (int i = 0; i < N; i++) f[i] = (float)*GPTR(T, p + i);
    } else {
        struct Raw { T e[V]; };
#pragma unroll
        for (int k = 0; k < N; k += V) {
            const Raw r = __builtin_bit_cast(Raw, NT ? (u32x4)__builtin_nontemporal_load(GPTR(u32x4a1, p + k))
                                                     : (u32x4)*GPTR(u32x4a1, p + k));
#pragma unroll
            for (int i = 0; i < V; i++) f[k + i] = (float)r.e[i];
        }
    }
}
// One value as T. fp16 of a finished f32: left to itself the compiler folds a product into
// v_fma_mixlo_f16 with +0 as its addend, which makes +0 of -0.
template <typename T> __device__ __forceinline__ T el_of(float f) {
    if constexpr (__is_same(T, _Float16)) asm("" : "+v"(f));
    return (T)f;
}
template <typename T, int N, bool NT = false> __device__ __forceinline__ void el_store(T *p, const float (&f)[N]) {
    constexpr int V = 16 / sizeof(T);
    if constexpr (N % V) {
#pragma unroll
        for (int i = 0; i < N; i++) p[i] = el_of<T>(f[i]);
    } else {
        struct Raw { T e[V]; };
#pragma unroll
        for (int k = 0; k < N; k += V) {
            Raw r;
#pragma unroll
            for (int i = 0; i < V; i++) r.e[i] = el_of<T>(f[k + i]);
            if constexpr (NT) __builtin_nontemporal_store((u32x4a1)__builtin_bit_cast(u32x4, r), (u32x4a1 *)(p + k));
            else *(u32x4a1 *)(p + k) = __builtin_bit_cast(u32x4, r);
        }
    }
}
