// What the token-level operators (layer_norm.hip, linear_ce.hip, muon.hip) share: element types, their conversions and the
// reductions of a wave.  Element types of the C ABI: 0 = fp32, 1 = bf16, 2 = fp16.
#pragma once
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

namespace ssecg_lm {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

enum { kF32 = 0, kB16 = 1, kF16 = 2 };
inline bool dtype_ok(int t) { return t == kF32 || t == kB16 || t == kF16; }

// 16 bytes of elements, at any alignment that the element itself has (the hardware takes unaligned global accesses)
template <typename T> struct Vec;
template <> struct Vec<float> { static constexpr int N = 4; typedef float type __attribute__((ext_vector_type(4), aligned(4))); };
template <> struct Vec<__bf16> { static constexpr int N = 8; typedef __bf16 type __attribute__((ext_vector_type(8), aligned(2))); };
template <> struct Vec<_Float16> { static constexpr int N = 8; typedef _Float16 type __attribute__((ext_vector_type(8), aligned(2))); };

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}

// elements [c0, c0 + 16 bytes) of a row of C; beyond C: zeros, and nothing is written there
template <typename T>
__device__ __forceinline__ typename Vec<T>::type load_vec(const T* __restrict__ p, int c0, int C) {
    constexpr int V = Vec<T>::N;
    typename Vec<T>::type v;
    if (c0 + V <= C) {
        v = *reinterpret_cast<const typename Vec<T>::type*>(p + c0);
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = c0 + i < C ? p[c0 + i] : (T)0.f;
    }
    return v;
}

template <typename T>
__device__ __forceinline__ void store_vec(T* __restrict__ p, int c0, int C, typename Vec<T>::type v) {
    constexpr int V = Vec<T>::N;
    if (c0 + V <= C) {
        *reinterpret_cast<typename Vec<T>::type*>(p + c0) = v;
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (c0 + i < C) p[c0 + i] = v[i];
    }
}

// runs the statements with T = the element type of the ABI code
#define SSECG_LM_DTYPE(code, T, ...)                                   \
    do {                                                               \
        if ((code) == ssecg_lm::kF32) { using T = float; __VA_ARGS__; }      \
        else if ((code) == ssecg_lm::kB16) { using T = __bf16; __VA_ARGS__; } \
        else { using T = _Float16; __VA_ARGS__; }                      \
    } while (0)

}  // namespace ssecg_lm
