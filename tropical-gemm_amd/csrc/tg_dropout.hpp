// tg_dropout.hpp -- which elements dropout keeps, from a counter-based
// generator: nothing of it is stored, every kernel that needs it makes it again.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "tg_layers.hpp"

namespace tg {

// Philox4x32-10 (Salmon, Moraes, Dror, Shaw: "Parallel random numbers: as easy
// as 1, 2, 3", SC 2011).
__device__ __forceinline__ void philox(uint32_t (&c)[4], uint32_t k0, uint32_t k1) {
#pragma unroll
    for (int i = 0; i < 10; ++i) {
        const uint64_t p = uint64_t(c[0]) * 0xD2511F53u, q = uint64_t(c[2]) * 0xCD9E8D57u;
        c[0] = uint32_t(q >> 32) ^ c[1] ^ k0;
        c[1] = uint32_t(q);
        c[2] = uint32_t(p >> 32) ^ c[3] ^ k1;
        c[3] = uint32_t(p);
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
}

// 16 bits for each element: eight neighbours in a row share one counter, (column
// / 8, row, offset).  Ten rounds are 20 wide multiplications; with 32 bits an
// element the generator's work would be twice as much.  A probability is then a
// multiple of 2^-16.
struct Keep {
    uint32_t below, k0, k1, o0, o1;
    float factor;
    __device__ __forceinline__ explicit Keep(const Dropout& d)
        : below(d.below), o0(uint32_t(d.offset)), o1(uint32_t(d.offset >> 32)), factor(d.factor) {
        const uint64_t seed = d.seed_at != nullptr ? *d.seed_at : d.seed;
        k0 = __builtin_amdgcn_readfirstlane(uint32_t(seed));
        k1 = __builtin_amdgcn_readfirstlane(uint32_t(seed >> 32));
    }
    // Bit i: element 8 * group + i of the row is kept.
    __device__ __forceinline__ uint32_t group(int64_t row, uint32_t group) const {
        uint32_t c[4] = {group, uint32_t(row), o0, o1}, a = k0, b = k1;
        asm volatile("" : "+s"(a), "+s"(b));  // or a loop keeps the keys of all rounds in registers
        philox(c, a, b);
        uint32_t bits = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            bits |= uint32_t((c[i] & 0xffffu) >= below) << (2 * i);
            bits |= uint32_t((c[i] >> 16) >= below) << (2 * i + 1);
        }
        return bits;
    }
    // Bit i: element `at` + i is kept, for any `at`.
    __device__ __forceinline__ uint32_t from(int64_t row, int64_t at) const {
        const uint32_t g = uint32_t(at / 8);
        const int shift = int(at % 8);
        uint32_t bits = group(row, g);
        if (shift != 0) bits = (bits | group(row, g + 1) << 8) >> shift;
        return bits;
    }
    __device__ __forceinline__ void apply(uint32_t bits, float (&v)[8]) const {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = (bits >> i & 1u) != 0 ? v[i] * factor : 0.0f;
    }
    __device__ __forceinline__ void apply(int64_t row, int64_t at, float (&v)[8]) const { apply(from(row, at), v); }
};

}  // namespace tg
