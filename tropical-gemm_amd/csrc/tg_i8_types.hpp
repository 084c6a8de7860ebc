// tg_i8_types.hpp -- element types, vector loads and wave reductions of the
// 8-bit layer's kernels.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace tg {

using bf16_t = __bf16;
using f16_t = _Float16;

// 16- and 8-byte words that may start at any address: global memory is read
// and written unaligned by one instruction on gfx950, so rows need no
// alignment of their own.
typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(1)));
typedef uint32_t u32x4_word __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u32x2_word __attribute__((ext_vector_type(2), aligned(4)));
typedef uint32_t u32x2_any __attribute__((ext_vector_type(2), aligned(1)));
typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(1)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

template <typename T>
__device__ __forceinline__ float to_f32(T x) {
    return static_cast<float>(x);
}

// Eight elements from p as f32: one 16-byte load (two for f32).
template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&v)[8]) {
    if constexpr (sizeof(T) == 4) {
        const f32x4 a = *reinterpret_cast<const f32x4_any*>(p);
        const f32x4 b = *reinterpret_cast<const f32x4_any*>(p + 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[i] = a[i];
            v[4 + i] = b[i];
        }
    } else {
        typedef T t8 __attribute__((ext_vector_type(8)));
        const u32x4 a = *reinterpret_cast<const u32x4_any*>(p);
        const t8 t = __builtin_bit_cast(t8, a);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = to_f32(t[i]);
    }
}

// The first n (below 8) of eight elements, zeros after them.
template <typename T>
__device__ __forceinline__ void load_part(const T* p, int n, float (&v)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < n ? to_f32(p[i]) : 0.0f;
}

template <typename T>
__device__ __forceinline__ void load_upto8(const T* p, int n, float (&v)[8]) {
    if (n >= 8) load8(p, v);
    else load_part(p, n, v);
}

template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&v)[8]) {
    if constexpr (sizeof(T) == 4) {
        *reinterpret_cast<f32x4_any*>(p) = f32x4{v[0], v[1], v[2], v[3]};
        *reinterpret_cast<f32x4_any*>(p + 4) = f32x4{v[4], v[5], v[6], v[7]};
    } else {
        typedef T t8 __attribute__((ext_vector_type(8)));
        t8 t;
#pragma unroll
        for (int i = 0; i < 8; ++i) t[i] = static_cast<T>(v[i]);
        *reinterpret_cast<u32x4_any*>(p) = __builtin_bit_cast(u32x4, t);
    }
}

template <typename T>
__device__ __forceinline__ void store_upto8(T* p, int n, const float (&v)[8]) {
    if (n >= 8) {
        store8(p, v);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < n) p[i] = static_cast<T>(v[i]);
    }
}

__device__ __forceinline__ void store_i8_upto8(int8_t* p, int n, const int (&q)[8]) {
    u32x2 w;
#pragma unroll
    for (int h = 0; h < 2; ++h)
        w[h] = (uint32_t(q[4 * h]) & 255u) | (uint32_t(q[4 * h + 1]) & 255u) << 8 |
               (uint32_t(q[4 * h + 2]) & 255u) << 16 | uint32_t(q[4 * h + 3]) << 24;
    if (n >= 8) {
        *reinterpret_cast<u32x2_any*>(p) = w;
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < n) p[i] = int8_t(q[i]);
    }
}

__device__ __forceinline__ void load_i8_upto8(const int8_t* p, int n, float (&v)[8]) {
    if (n >= 8) {
        const u32x2 w = *reinterpret_cast<const u32x2_any*>(p);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = float(int32_t(w[i / 4] << (24 - 8 * (i % 4))) >> 24);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = i < n ? float(p[i]) : 0.0f;
    }
}

// Larger of two, NaN where either is NaN.
__device__ __forceinline__ float max_nan(float a, float b) { return __builtin_elementwise_maximum(a, b); }

// Sum / maximum over the 64 lanes, the same bits in every lane.
__device__ __forceinline__ float wave_sum(float x) {
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) x += __shfl_xor(x, d);
    return x;
}
__device__ __forceinline__ float wave_max(float x) {
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) x = max_nan(x, __shfl_xor(x, d));
    return x;
}

// Workgroup `id` of `count`, renumbered so that each of the 8 XCDs, round which
// consecutive workgroups go, takes a run of neighbours.
__device__ __forceinline__ int xcd_run(int id, int count) {
    const int per = count / 8, rest = count % 8, x = id % 8;
    return x * per + (x < rest ? x : rest) + id / 8;
}

}  // namespace tg
