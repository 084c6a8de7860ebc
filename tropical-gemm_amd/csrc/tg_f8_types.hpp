// tg_f8_types.hpp -- e4m3 numbers and e8m0 scales.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "tg_i8_types.hpp"

namespace tg {

typedef float f32x2 __attribute__((ext_vector_type(2)));

// 2^(s - 127), NaN for 255.
__device__ __forceinline__ float e8m0_to_f32(uint32_t s) {
    const uint32_t bits = s == 0 ? 0x00400000u : s == 255 ? 0x7fc00000u : s << 23;
    return __builtin_bit_cast(float, bits);
}

// Four e4m3 numbers from f32 (nearest, ties to even), and back (exact).
__device__ __forceinline__ uint32_t e4m3_pack(float a, float b, float c, float d) {
    const int low = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return uint32_t(__builtin_amdgcn_cvt_pk_fp8_f32(c, d, low, true));
}
__device__ __forceinline__ void e4m3_unpack(uint32_t w, float* v) {
    const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8(int(w), false), b = __builtin_amdgcn_cvt_pk_f32_fp8(int(w), true);
    v[0] = a[0], v[1] = a[1], v[2] = b[0], v[3] = b[1];
}

// v without its first n (0 ... 7) elements, zeros behind.
__device__ __forceinline__ void shift8(int n, float (&v)[8]) {
#pragma unroll
    for (int d = 4; d > 0; d >>= 1) {
        const bool by = (n & d) != 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = by ? (i + d < 8 ? v[i + d] : 0.0f) : v[i];
    }
}

// Eight of them from p, at any address: the first n, zeros behind.
__device__ __forceinline__ u32x2 load_f8_upto8(const uint8_t* p, int n) {
    u32x2 w = {0, 0};
    if (n >= 8) {
        w = *reinterpret_cast<const u32x2_any*>(p);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < n) w[i / 4] |= uint32_t(p[i]) << (8 * (i % 4));
    }
    return w;
}
__device__ __forceinline__ void store_f8_upto8(uint8_t* p, int n, u32x2 w) {
    if (n >= 8) {
        *reinterpret_cast<u32x2_any*>(p) = w;
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < n) p[i] = uint8_t(w[i / 4] >> (8 * (i % 4)));
    }
}

}  // namespace tg
