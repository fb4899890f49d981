// seq_common.hpp -- what the sequence kernels share: vector types, and rows of any length and alignment in 16-byte pieces.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "pvder_sequence.h"

namespace pvder_seq {

constexpr int kEinval = -10001;            // PVDER_EINVAL (pvder_hip.h)

typedef float f4 __attribute__((ext_vector_type(4)));
typedef float f8 __attribute__((ext_vector_type(8)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef __bf16 b4 __attribute__((ext_vector_type(4)));
typedef short s4 __attribute__((ext_vector_type(4)));
typedef unsigned int u4 __attribute__((ext_vector_type(4)));

template <typename T> struct Vec;
template <> struct Vec<float> { typedef f4 type; static constexpr int N = 4; };
template <> struct Vec<__bf16> { typedef b8 type; static constexpr int N = 8; };

// 16 bytes of a row from element d on; elements at and behind `dim` are zeros and not read.  No alignment is asked of the row.
template <typename T> __device__ __forceinline__ typename Vec<T>::type load_row(const T *row, int d, int dim) {
    constexpr int V = Vec<T>::N;
    typename Vec<T>::type f;
    if (d + V <= dim) {
        __builtin_memcpy(&f, row + d, 16);
    } else {
#pragma unroll
        for (int e = 0; e < V; ++e) f[e] = d + e < dim ? row[d + e] : (T)0.f;
    }
    return f;
}
template <typename T> __device__ __forceinline__ void store_row(T *row, int d, int dim, typename Vec<T>::type f) {
    constexpr int V = Vec<T>::N;
    if (d + V <= dim) {
        __builtin_memcpy(row + d, &f, 16);
    } else {
#pragma unroll
        for (int e = 0; e < V; ++e)
            if (d + e < dim) row[d + e] = f[e];
    }
}

// g^n of a decay given as its base-2 logarithm lg <= 0; g^0 = 1 also where lg is -infinity
__device__ __forceinline__ float power(float lg, int n) { return n == 0 ? 1.f : exp2f(lg * (float)n); }
// log_decay as the kernels take it: growth and NaN count as no decay
__device__ __forceinline__ float log2_decay(float log_decay) { return (log_decay < 0.f ? log_decay : 0.f) * 1.44269504088896340736f; }

}  // namespace pvder_seq
