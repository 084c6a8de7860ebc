// tg_i8_pack.hpp -- operands laid out for tg_i8_tiles: rows along the sum, of
// whole 128-byte steps, 16-byte aligned, zeros past the sum's end.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "tg_i8_stream.hpp"
#include "tg_i8_types.hpp"

namespace tg {

inline int64_t pack_ceil(int64_t a, int64_t b) { return (a + b - 1) / b; }

// A job is run by `count` workgroups of 256 threads, each with its number.

struct PackNothing {
    static constexpr int kLdsWords = 1;
    int64_t blocks() const { return 0; }
    __device__ __forceinline__ void run(int, int, uint32_t*) const {}
};

// Rows of `bytes` bytes at any address to rows of `ld` bytes (a multiple of
// 128): 16 bytes a thread.
struct PackBytes {
    static constexpr int kLdsWords = 1;
    const int8_t* src;
    int64_t ld_src, rows;
    int bytes;
    int8_t* dst;
    int64_t ld;
    int64_t blocks() const {
        const int64_t n = pack_ceil(rows * (ld / 16), 256);
        return n < 65536 ? n : 65536;
    }
    __device__ __forceinline__ void run(int block, int count, uint32_t*) const {
        const int64_t chunks = ld / 16, total = rows * chunks;
        for (int64_t i = int64_t(block) * 256 + threadIdx.x; i < total; i += int64_t(count) * 256) {
            const int64_t row = i / chunks, c = i - row * chunks;
            StreamTail x;
            x.load(src + row * ld_src, int(c) * 16, bytes);
            *reinterpret_cast<u32x4*>(dst + row * ld + c * 16) = x.get();
        }
    }
};

// |s|, or 0 where it is not finite.
__device__ __forceinline__ float finite_size(float s) {
    s = fabsf(s);
    return s < __builtin_huge_valf() ? s : 0.0f;
}

// e such that top * 2^e lies in [64, 128) (0 for top 0; |e| at most 120), for
// products q * scale * 2^e in f16 with top the largest scale: at most 128 *
// 128, and with all of f16's bits down to 2^-20 of the largest scale.
__device__ __forceinline__ int range_exponent(float top) {
    if (!(top > 0.0f)) return 0;
    int e = 0;
    (void)frexpf(top, &e);  // top in [2^(e-1), 2^e)
    e = 7 - e;
    return e > 120 ? 120 : e < -120 ? -120 : e;
}

// What f16 gradients take of their scales: q * scale * 2^e in f16 where no scale
// that matters lies further than 2^20 below the largest.  Otherwise, `wide`, q
// stays an integer (exact in bf16) and the gradient times its scales becomes two
// bf16 planes, 16 bits of any size, for twice the products (8192 x 4096 x 4096:
// 403 us instead of 223, 407 instead of 249).  Only the GPU knows which: every
// kernel behind this one looks.
//
// Scales below 2^-70 do not matter: |g| < 2^16, |q| <= 2^7, and 2^20 such terms
// stay below 2^-27, an eighth of f16's least number.
struct ScaleRange {
    float factor, back;  // 2^e and its inverse (1 for `wide`)
    int wide;
};
constexpr float kLeastScale = 0x1p-70f;
__device__ __forceinline__ void add_scale(float s, float& top, float& low) {
    s = finite_size(s);
    top = fmaxf(top, s);
    if (s >= kLeastScale) low = fminf(low, s);
}
__device__ __forceinline__ ScaleRange scale_range(float top, float low) {
    const int e = range_exponent(top);
    const bool wide = low < top * 0x1p-20f;
    return {ldexpf(1.0f, e), wide ? 1.0f : ldexpf(1.0f, -e), wide};
}

// The range of all the scales.
static __global__ __launch_bounds__(1024) void tg_i8_scale_range(const float* __restrict__ scale, int64_t n,
                                                          ScaleRange* __restrict__ out) {
    __shared__ float part[2][16];
    float top = 0.0f, low = __builtin_huge_valf();
    for (int64_t i = threadIdx.x; i < n; i += 1024) add_scale(scale[i], top, low);
    top = wave_max(top);
    low = -wave_max(-low);
    if (threadIdx.x % 64 == 0) {
        part[0][threadIdx.x / 64] = top;
        part[1][threadIdx.x / 64] = low;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int i = 1; i < 16; ++i) {
            top = fmaxf(top, part[0][i]);
            low = fminf(low, part[1][i]);
        }
        *out = scale_range(top, low);
    }
}

// v as 1 to 3 numbers of type D that add up to it: one rounding, an f32's first
// 16 bits as two bf16 numbers, or its 24 bits as three (cut, not rounded, but for
// the second of two: the largest numbers stay finite, and it is less work).
template <typename D, int PLANES>
__device__ __forceinline__ void split_value(float v, D (&d)[PLANES]) {
    if constexpr (PLANES == 1) {
        d[0] = static_cast<D>(v);
    } else {
        float r = v;
#pragma unroll
        for (int i = 0; i < PLANES; ++i) {
            const uint32_t bits = __builtin_bit_cast(uint32_t, r);
            d[i] = PLANES == 2 && i == 1 ? static_cast<D>(r) : __builtin_bit_cast(D, uint16_t(bits >> 16));
            r -= __builtin_bit_cast(float, bits & 0xffff0000u);
            if (i == 0) r = fabsf(v) < __builtin_huge_valf() ? r : v != v ? v : 0.0f;  // an infinity stays in the first
        }
    }
}

// Transposes: dst[c][r] = src[r][c] * scale[r] * factor in type D (scale and
// factor may be null), rows of dst of PLANES planes of `depth` (a multiple of
// 64, at least rows) elements, zeros from r = rows on.  A workgroup takes 64
// rows by 128 bytes of them (at least 64 columns), whole lines both ways,
// through LDS: pairs of rows are written there as words of two, 33 words a
// column, so that the words of 8 x 8 lanes meet 64 banks.  Bound by memory:
// 8192 x 4096 bf16 and as many 8-bit integers in one launch 42.9 us (235 MB,
// 5.5 TB/s); 4096 x 4096 8-bit integers 13.5 us (50 MB, 3.7 TB/s).
template <typename S, typename D, int PLANES>
struct PackTurned {
    static_assert(sizeof(D) == 2, "pairs are words");
    static constexpr int COLS = sizeof(S) == 1 ? 128 : 64, GROUPS = COLS / 8, PASSES = GROUPS * 32 / 256;
    const S* src;
    int64_t ld_src, rows, cols;
    const float *scale, *factor;
    D* dst;
    int64_t depth;
    static constexpr int kLdsWords = PLANES * COLS * 33;
    int64_t blocks() const { return depth / 64 * pack_ceil(cols, COLS); }
    __device__ __forceinline__ void run(int block, int count, uint32_t* lds) const {
        uint32_t(*tile)[COLS][33] = reinterpret_cast<uint32_t(*)[COLS][33]>(lds);
        const int t = threadIdx.x, tiles_r = int(depth / 64);
        block = xcd_run(block, count);
        const int64_t r0 = int64_t(block % tiles_r) * 64, c0 = int64_t(block / tiles_r) * COLS;
        float v[PASSES][2][8] = {};
        const int cg = t % GROUPS;
        const int64_t c = c0 + cg * 8;
        const int left = cols - c < 8 ? int(cols - c) : 8;
#pragma unroll
        for (int pass = 0; pass < PASSES; ++pass)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int64_t r = r0 + (pass * (256 / GROUPS) + t / GROUPS) * 2 + h;
                if (r >= rows || left <= 0) continue;
                if constexpr (sizeof(S) == 1) load_i8_upto8(src + r * ld_src + c, left, v[pass][h]);
                else load_upto8(src + r * ld_src + c, left, v[pass][h]);
                if (scale != nullptr) {
                    const float s = factor != nullptr ? scale[r] * factor[0] : scale[r];
#pragma unroll
                    for (int i = 0; i < 8; ++i) v[pass][h][i] *= s;
                }
            }
#pragma unroll
        for (int pass = 0; pass < PASSES; ++pass)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                D lo[PLANES], hi[PLANES];
                split_value<D, PLANES>(v[pass][0][i], lo);
                split_value<D, PLANES>(v[pass][1][i], hi);
#pragma unroll
                for (int p = 0; p < PLANES; ++p)
                    tile[p][cg * 8 + i][pass * (256 / GROUPS) + t / GROUPS] =
                        uint32_t(__builtin_bit_cast(uint16_t, lo[p])) |
                        uint32_t(__builtin_bit_cast(uint16_t, hi[p])) << 16;
            }
        __syncthreads();
#pragma unroll
        for (int p = 0; p < PLANES; ++p)
#pragma unroll
            for (int pass = 0; pass < COLS / 32; ++pass) {
                const int k = pass * 32 + t / 8, w = t % 8 * 4;
                if (c0 + k >= cols) continue;
                const u32x4 x = {tile[p][k][w], tile[p][k][w + 1], tile[p][k][w + 2], tile[p][k][w + 3]};
                *reinterpret_cast<u32x4*>(dst + ((c0 + k) * PLANES + p) * depth + r0 + w * 2) = x;
            }
    }
};

// Rows as PLANES bf16 planes each: dst[i][p][r] from src[i][r] * scale[r].
template <typename S, int PLANES>
struct PackSplit {
    static constexpr int kLdsWords = 1;
    const S* src;
    int64_t ld_src, rows, cols;
    const float* scale;
    bf16_t* dst;
    int64_t depth;
    int64_t blocks() const {
        const int64_t n = pack_ceil(rows * (depth / 8), 256);
        return n < 65536 ? n : 65536;
    }
    __device__ __forceinline__ void run(int block, int count, uint32_t*) const {
        const int64_t groups = depth / 8, total = rows * groups;
        for (int64_t i = int64_t(block) * 256 + threadIdx.x; i < total; i += int64_t(count) * 256) {
            const int64_t row = i / groups, at = (i - row * groups) * 8;
            const int left = cols - at < 8 ? int(cols - at) : 8;
            float v[8] = {}, s[8] = {};
            if (left > 0) {
                load_upto8(src + row * ld_src + at, left, v);
                load_upto8(scale + at, left, s);
            }
            bf16_t d[8][PLANES];
#pragma unroll
            for (int e = 0; e < 8; ++e) split_value<bf16_t, PLANES>(v[e] * s[e], d[e]);
#pragma unroll
            for (int p = 0; p < PLANES; ++p) {
                u32x4 w;
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    w[e] = uint32_t(__builtin_bit_cast(uint16_t, d[2 * e][p])) |
                           uint32_t(__builtin_bit_cast(uint16_t, d[2 * e + 1][p])) << 16;
                *reinterpret_cast<u32x4*>(dst + (row * PLANES + p) * depth + at) = w;
            }
        }
    }
};

// Job n, or w where the scales' range is wide: both of as many workgroups, or
// each fit for any number of them.  Where n is nothing, few workgroups look.
template <typename N, typename W>
struct PackEither {
    static constexpr int kLdsWords = N::kLdsWords > W::kLdsWords ? N::kLdsWords : W::kLdsWords;
    N n;
    W w;
    const ScaleRange* range;
    int64_t blocks() const {
        const int64_t a = n.blocks(), b = w.blocks();
        return a > 0 ? a : b < 2048 ? b : 2048;
    }
    __device__ __forceinline__ void run(int block, int count, uint32_t* lds) const {
        if (range->wide != 0) w.run(block, count, lds);
        else n.run(block, count, lds);
    }
};

// Job a on the first `na` workgroups, job b on the `nb` behind them.
template <typename A, typename B>
__global__ __launch_bounds__(256) void tg_i8_pack(A a, B b, int na, int nb) {
    constexpr int WA = A::kLdsWords, WB = B::kLdsWords;
    __shared__ uint32_t lds[WA > WB ? WA : WB];
    if (int(blockIdx.x) < na) a.run(int(blockIdx.x), na, lds);
    else b.run(int(blockIdx.x) - na, nb, lds);
}

}  // namespace tg
