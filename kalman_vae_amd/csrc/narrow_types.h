// Element types of the sequence-network and optimiser kernels: float, bfloat16 and half in memory,
// float in registers, and e4m3 bytes (OCP: 4 exponent bits, 3 mantissa bits, largest value 448).
#pragma once

#include <hip/hip_runtime.h>

#include <stdint.h>

#include <type_traits>

#include "../../include/kvae_kalman.h"

namespace kvae {

using bf16_t = __bf16;
using f16_t = _Float16;

__device__ __forceinline__ float widen(float x) { return x; }
__device__ __forceinline__ float widen(bf16_t x) { return (float)x; }
__device__ __forceinline__ float widen(f16_t x) { return (float)x; }

// nearest, ties to even (the conversion instructions' default mode)
template <typename T>
__device__ __forceinline__ T narrow(float x) {
    return (T)x;
}

// V consecutive elements.  The address needs the element's own alignment only: gfx950 takes
// wide global accesses at any address, so a view that starts at an odd element, or rows of an
// odd length, go through the same wide instructions as aligned ones.
template <typename T, int V>
struct Pack {
    T v[V];
};
template <int BYTES>
struct RawVec;
template <>
struct RawVec<2> { using type = uint16_t; };
template <>
struct RawVec<4> { typedef uint32_t type __attribute__((aligned(2))); };
template <>
struct RawVec<8> { typedef uint32_t type __attribute__((ext_vector_type(2), aligned(2))); };
template <>
struct RawVec<16> { typedef uint32_t type __attribute__((ext_vector_type(4), aligned(2))); };

// (more than 16 bytes: consecutive accesses of 16)
template <typename T, int V>
__device__ __forceinline__ Pack<T, V> load_pack(const T* p) {
    constexpr int BYTES = sizeof(T) * V, PIECE = BYTES < 16 ? BYTES : 16;
    using R = typename RawVec<PIECE>::type;
    Pack<T, V> out;
#pragma unroll
    for (int i = 0; i < BYTES / PIECE; ++i) {
        const R r = *reinterpret_cast<const R*>(p + i * (PIECE / sizeof(T)));
        __builtin_memcpy(&out.v[i * (PIECE / sizeof(T))], &r, PIECE);
    }
    return out;
}
template <typename T, int V>
__device__ __forceinline__ void store_pack(T* p, const Pack<T, V>& x) {
    constexpr int BYTES = sizeof(T) * V, PIECE = BYTES < 16 ? BYTES : 16;
    using R = typename RawVec<PIECE>::type;
#pragma unroll
    for (int i = 0; i < BYTES / PIECE; ++i) {
        R r;
        __builtin_memcpy(&r, &x.v[i * (PIECE / sizeof(T))], PIECE);
        *reinterpret_cast<R*>(p + i * (PIECE / sizeof(T))) = r;
    }
}

// f(T{}) for the element type T of a dtype code; KVAE_E_UNSUPPORTED for another code
template <typename F>
int for_element_type(int dtype, F&& f) {
    switch (dtype) {
        case KVAE_F32: return f(float{});
        case KVAE_BF16: return f(bf16_t{});
        case KVAE_F16: return f(f16_t{});
        default: return KVAE_E_UNSUPPORTED;
    }
}

}  // namespace kvae
