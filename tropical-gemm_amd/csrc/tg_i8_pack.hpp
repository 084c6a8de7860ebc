// tg_i8_pack.hpp -- operands laid out for tg_i8_tiles: rows along the sum, of
// whole 128-byte steps, 16-byte aligned, zeros past the sum's end.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "tg_i8_stream.hpp"
#include "tg_i8_types.hpp"

namespace tg {

// Rows of `bytes` bytes at any address to rows of `ld` bytes (a multiple of
// 128): 16 bytes a thread.
__global__ __launch_bounds__(256) void tg_i8_pack_bytes(const int8_t* __restrict__ src, int64_t ld_src, int64_t rows,
                                                        int bytes, int8_t* __restrict__ dst, int64_t ld) {
    const int64_t chunks = ld / 16, total = rows * chunks;
    for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < total; i += int64_t(gridDim.x) * 256) {
        const int64_t row = i / chunks, c = i - row * chunks;
        *reinterpret_cast<u32x4*>(dst + row * ld + c * 16) = stream_tail(src + row * ld_src, int(c) * 16, bytes);
    }
}

// The factor 2^e that puts the largest finite scale into [64, 128), and its
// inverse, for products q * scale * 2^e in f16: at most 127 * 128, and with
// all of f16's bits down to 2^-21 of the largest scale.
__global__ __launch_bounds__(1024) void tg_i8_scale_range(const float* __restrict__ scale, int64_t n,
                                                          float* __restrict__ out) {
    __shared__ float part[16];
    float top = 0.0f;
    for (int64_t i = threadIdx.x; i < n; i += 1024) {
        const float s = fabsf(scale[i]);
        if (s < __builtin_huge_valf()) top = fmaxf(top, s);
    }
    top = wave_max(top);
    if (threadIdx.x % 64 == 0) part[threadIdx.x / 64] = top;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int i = 1; i < 16; ++i) top = fmaxf(top, part[i]);
        int e = 0;
        if (top > 0.0f) {
            (void)frexpf(top, &e);  // top in [2^(e-1), 2^e)
            e = 7 - e;
            e = e > 120 ? 120 : e < -120 ? -120 : e;
        }
        out[0] = ldexpf(1.0f, e);
        out[1] = ldexpf(1.0f, -e);
    }
}

// v as 1 or 3 numbers of type D that add up to it: one rounding, or all of an
// f32's 24 bits in three bf16 numbers.
template <typename D, int PLANES>
__device__ __forceinline__ void split_value(float v, D (&d)[PLANES]) {
    d[0] = static_cast<D>(v);
    if constexpr (PLANES == 3) {
        // An infinity or NaN stays in the first.
        const float r = fabsf(v) < __builtin_huge_valf() ? v - static_cast<float>(d[0]) : 0.0f;
        d[1] = static_cast<D>(r);
        d[2] = static_cast<D>(r - static_cast<float>(d[1]));
    }
}

// Transposes: dst[c][r] = src[r][c] * scale[r] * factor in type D (scale and
// factor may be null), rows of dst of PLANES planes of `depth` (a multiple of
// 64, at least rows) elements, zeros from r = rows on.  A workgroup takes 64
// rows by 64 columns through LDS: pairs of rows are written there as words of
// two, 33 words a column, so that a wave's 8 x 8 words meet 64 banks.
template <typename S, typename D, int PLANES>
__global__ __launch_bounds__(256) void tg_i8_pack_turned(const S* __restrict__ src, int64_t ld_src, int64_t rows,
                                                         int64_t cols, const float* __restrict__ scale,
                                                         const float* __restrict__ factor, D* __restrict__ dst,
                                                         int64_t depth, int64_t tiles_r) {
    static_assert(sizeof(D) == 2, "pairs are words");
    __shared__ uint32_t tile[PLANES][64][33];
    const int t = threadIdx.x;
    const int64_t r0 = int64_t(blockIdx.x) % tiles_r * 64, c0 = int64_t(blockIdx.x) / tiles_r * 64;
    {
        const int cg = t % 8, rp = t / 8;
        const int64_t c = c0 + cg * 8;
        const int left = cols - c < 8 ? int(cols - c) : 8;
        float v[2][8] = {};
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int64_t r = r0 + rp * 2 + h;
            if (r >= rows || left <= 0) continue;
            if constexpr (sizeof(S) == 1) load_i8_upto8(src + r * ld_src + c, left, v[h]);
            else load_upto8(src + r * ld_src + c, left, v[h]);
            if (scale != nullptr) {
                const float s = factor != nullptr ? scale[r] * factor[0] : scale[r];
#pragma unroll
                for (int i = 0; i < 8; ++i) v[h][i] *= s;
            }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            D lo[PLANES], hi[PLANES];
            split_value<D, PLANES>(v[0][i], lo);
            split_value<D, PLANES>(v[1][i], hi);
#pragma unroll
            for (int p = 0; p < PLANES; ++p)
                tile[p][cg * 8 + i][rp] = uint32_t(__builtin_bit_cast(uint16_t, lo[p])) |
                                          uint32_t(__builtin_bit_cast(uint16_t, hi[p])) << 16;
        }
    }
    __syncthreads();
#pragma unroll
    for (int p = 0; p < PLANES; ++p)
#pragma unroll
        for (int pass = 0; pass < 2; ++pass) {
            const int c = pass * 32 + t / 8, w = t % 8 * 4;
            if (c0 + c >= cols) continue;
            const u32x4 v = {tile[p][c][w], tile[p][c][w + 1], tile[p][c][w + 2], tile[p][c][w + 3]};
            *reinterpret_cast<u32x4*>(dst + ((c0 + c) * PLANES + p) * depth + r0 + w * 2) = v;
        }
}

// f32 rows as three bf16 planes each: dst[i][p][r] from src[i][r] * scale[r].
__global__ __launch_bounds__(256) void tg_i8_pack_split(const float* __restrict__ src, int64_t ld_src, int64_t rows,
                                                        int64_t cols, const float* __restrict__ scale,
                                                        bf16_t* __restrict__ dst, int64_t depth) {
    const int64_t groups = depth / 8, total = rows * groups;
    for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < total; i += int64_t(gridDim.x) * 256) {
        const int64_t row = i / groups, at = (i - row * groups) * 8;
        const int left = cols - at < 8 ? int(cols - at) : 8;
        float v[8] = {}, s[8] = {};
        if (left > 0) {
            load_upto8(src + row * ld_src + at, left, v);
            load_upto8(scale + at, left, s);
        }
        bf16_t d[8][3];
#pragma unroll
        for (int e = 0; e < 8; ++e) split_value<bf16_t, 3>(v[e] * s[e], d[e]);
#pragma unroll
        for (int p = 0; p < 3; ++p) {
            u32x4 w;
#pragma unroll
            for (int e = 0; e < 4; ++e)
                w[e] = uint32_t(__builtin_bit_cast(uint16_t, d[2 * e][p])) |
                       uint32_t(__builtin_bit_cast(uint16_t, d[2 * e + 1][p])) << 16;
            *reinterpret_cast<u32x4*>(dst + (row * 3 + p) * depth + at) = w;
        }
    }
}

}  // namespace tg
