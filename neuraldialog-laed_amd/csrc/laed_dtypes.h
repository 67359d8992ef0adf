// Element types of the operators that take 32-bit and 16-bit tensors: loads convert to fp32, every sum, state and
// statistic is held in fp32 or wider, results are rounded once, on the store (to nearest even).
#pragma once
#include "laed_common.h"

typedef __bf16 laed_bf16;
typedef _Float16 laed_f16;

template <typename T> __device__ __forceinline__ float laed_to_float(T v) { return (float)v; }
template <typename T> __device__ __forceinline__ T laed_from_float(float v) { return (T)v; }

// N elements of T as one aligned access (N * sizeof(T) <= 16)
template <typename T, int N> struct alignas(sizeof(T) * N) laed_vec { T v[N]; };

#define LAED_BY_DTYPE(dtype, DO)            \
    do {                                    \
        if ((dtype) == LAED_BF16) { DO(laed_bf16); } \
        else if ((dtype) == LAED_F16) { DO(laed_f16); } \
        else { DO(float); }                 \
    } while (0)
