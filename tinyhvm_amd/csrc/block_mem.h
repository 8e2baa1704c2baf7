// block_mem.h - global memory as the residual block's kernels take it:
// addresses arrive as 64-bit words, and loads and stores through them are
// global ones of up to 16 bytes. A vector may start at any element (a row of
// an odd length is aligned to its elements only), which the card allows.
#ifndef BLOCK_MEM_H
#define BLOCK_MEM_H

#include <hip/hip_runtime.h>
#include "thvm_abi.h"

typedef _Float16 f16;

template <typename T> using glob = __attribute__((address_space(1))) T;
template <typename T, u32 N> struct Any { typedef T vec __attribute__((ext_vector_type(N), aligned(sizeof(T)))); };
template <typename T, u32 N> using any_vec = typename Any<T, N>::vec;

// elements e .. e + N - 1 of a row of n, zeros past its end
template <typename T, u32 N>
__device__ __forceinline__ void load_n(const glob<T> *row, u32 e, u32 n, float *out) {
    if (e + N <= n) {
        const any_vec<T, N> p = *(const glob<any_vec<T, N>> *)(row + e);
#pragma unroll
        for (u32 j = 0; j < N; j++) out[j] = (float)p[j];
    } else {
#pragma unroll
        for (u32 j = 0; j < N; j++) out[j] = e + j < n ? (float)row[e + j] : 0.0f;
    }
}

// the same, as they are
template <typename T, u32 N>
__device__ __forceinline__ any_vec<T, N> load_raw(const glob<T> *row, u32 e, u32 n) {
    any_vec<T, N> p;
    if (e + N <= n) p = *(const glob<any_vec<T, N>> *)(row + e);
    else
#pragma unroll
        for (u32 j = 0; j < N; j++) p[j] = e + j < n ? row[e + j] : (T)0.0f;
    return p;
}

template <typename T, u32 N>
__device__ __forceinline__ void store_n(glob<T> *row, u32 e, u32 n, const float *in) {
    if (e + N <= n) {
        any_vec<T, N> p;
#pragma unroll
        for (u32 j = 0; j < N; j++) p[j] = (T)in[j];
        *(glob<any_vec<T, N>> *)(row + e) = p;
    } else {
#pragma unroll
        for (u32 j = 0; j < N; j++)
            if (e + j < n) row[e + j] = (T)in[j];
    }
}

#endif
