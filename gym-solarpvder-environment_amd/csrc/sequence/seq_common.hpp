// seq_common.hpp -- what the sequence kernels share: vector types, and rows of any length and alignment in 16-byte pieces.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "pvder_sequence.h"

namespace pvder_seq {

constexpr int kEinval = -10001;            // PVDER_EINVAL (pvder_hip.h)
constexpr long long kMostThreads = 0xffffffffll;           // of a launch: HIP counts them in 32 bits

typedef float f4 __attribute__((ext_vector_type(4)));
typedef float f8 __attribute__((ext_vector_type(8)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef __bf16 b4 __attribute__((ext_vector_type(4)));
typedef short s4 __attribute__((ext_vector_type(4)));
typedef unsigned int u4 __attribute__((ext_vector_type(4)));

// Global memory as a base that a wave shares (held in scalar registers, and hidden from the compiler's address arithmetic, which would
// carry an address of 64 bits for every load round a loop) and an offset of each lane, 32 bits.
typedef const __attribute__((address_space(1))) char *gbytes;
typedef __attribute__((address_space(1))) char *gbytes_out;
__device__ __forceinline__ gbytes shared_base(const void *p) {
    gbytes b = (gbytes)p;
    asm volatile("" : "+s"(b));
    return b;
}
__device__ __forceinline__ gbytes_out shared_base_out(void *p) {
    gbytes_out b = (gbytes_out)p;
    asm volatile("" : "+s"(b));
    return b;
}

// Memory of a wave with its end: what lies behind `bytes` reads as zero and is not written, without a branch.
typedef __amdgpu_buffer_rsrc_t window;
__device__ __forceinline__ window window_of(const void *p, unsigned bytes) {
    return __builtin_amdgcn_make_buffer_rsrc((void *)p, 0, (int)bytes, 0x00027000);
}

template <typename T> struct Vec;
template <> struct Vec<float> { typedef f4 type; static constexpr int N = 4; };
template <> struct Vec<__bf16> { typedef b8 type; static constexpr int N = 8; };

// f's elements from `n` on, in the first places; zeros behind them (n >= 0)
__device__ __forceinline__ f4 behind(f4 f, int n) {
    u4 u = __builtin_bit_cast(u4, f);
    if (n & 2) u = u4{u.z, u.w, 0u, 0u};
    if (n & 1) u = u4{u.y, u.z, u.w, 0u};
    if (n >= 4) u = u4{0u, 0u, 0u, 0u};
    return __builtin_bit_cast(f4, u);
}
__device__ __forceinline__ b8 behind(b8 f, int n) {
    u4 u = __builtin_bit_cast(u4, f);
    if (n & 4) u = u4{u.z, u.w, 0u, 0u};
    if (n & 2) u = u4{u.y, u.z, u.w, 0u};
    if (n & 1) u = u4{(u.x >> 16) | (u.y << 16), (u.y >> 16) | (u.z << 16), (u.z >> 16) | (u.w << 16), u.w >> 16};
    if (n >= 8) u = u4{0u, 0u, 0u, 0u};
    return __builtin_bit_cast(b8, u);
}

// 16 bytes of a row from element d on; elements at and behind `dim` are zeros and not read.  No alignment is asked of the row.
// Rows of 16 bytes and more take one load whatever d is (the piece that the row's end cuts is read from 16 bytes before that end and
// shifted), so that loads of many rows are in flight together; a row behind the last (`ok` false) has to be readable all the same.
template <typename T> __device__ __forceinline__ typename Vec<T>::type load_row(const T *row, int d, int dim, bool ok = true) {
    constexpr int V = Vec<T>::N;
    typename Vec<T>::type f;
    if (dim >= V) {
        const int last = dim - V, at = d < last ? d : last;
        __builtin_memcpy(&f, row + at, 16);
        f = behind(f, ok ? d - at : V);
    } else {
#pragma unroll
        for (int e = 0; e < V; ++e) f[e] = ok && d + e < dim ? row[d + e] : (T)0.f;
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

// a * b, and 0 where b is 0 whatever a is (NaN and infinities too)
extern "C" __device__ float pvder_seq_mul_legacy(float, float) __asm("llvm.amdgcn.fmul.legacy");
__device__ __forceinline__ float mul_or_zero(float a, float b) { return pvder_seq_mul_legacy(a, b); }

// g^n of a decay given as its base-2 logarithm lg <= 0, zero where it would be no normal number; g^0 = 1 also where lg is -infinity
__device__ __forceinline__ float power(float lg, int n) { return __builtin_amdgcn_exp2f(n == 0 ? 0.f : lg * (float)n); }
// log_decay as the kernels take it: growth and NaN count as no decay
__device__ __forceinline__ float log2_decay(float log_decay) { return (log_decay < 0.f ? log_decay : 0.f) * 1.44269504088896340736f; }

}  // namespace pvder_seq
