// tg_f8_pack.hpp -- gradients' operands laid out for tg_i8_tiles in bf16: rows
// along the sum, of whole 128-byte steps, zeros past the sum's end.
#pragma once

#include "tg_f8.hpp"
#include "tg_f8_types.hpp"
#include "tg_i8_pack.hpp"

namespace tg {

// dst[c][r] = src[r][c] times its scale, exact in bf16: four significant bits and
// a power of two.  Rows of dst have `depth` (a multiple of 64, at least rows)
// elements, zeros from r = rows on.  A workgroup takes 64 rows of one block of
// columns; LDS as in PackTurned.  4096 x 4096: 14 us (50 MB).
struct PackF8Turned {
    static constexpr int COLS = kF8Block, GROUPS = COLS / 8, PASSES = GROUPS * 32 / 256;
    static constexpr int kLdsWords = COLS * 33;
    const uint8_t* src;
    int64_t ld_src, rows, cols;
    F8Scale scale;
    int shift;  // rows of a scale: 2^shift
    bf16_t* dst;
    int64_t depth;
    int64_t blocks() const { return depth / 64 * pack_ceil(cols, COLS); }
    __device__ __forceinline__ void run(int block, int count, uint32_t* lds) const {
        uint32_t(*tile)[33] = reinterpret_cast<uint32_t(*)[33]>(lds);
        const int t = threadIdx.x, tiles_r = int(depth / 64), cg = t % GROUPS;
        block = xcd_run(block, count);
        const int64_t r0 = int64_t(block % tiles_r) * 64, cb = block / tiles_r, c0 = cb * COLS, c = c0 + cg * 8;
        const int left = cols - c < 8 ? int(cols - c) : 8;
        u32x2 w[PASSES][2] = {};
        float s[PASSES][2] = {};
#pragma unroll
        for (int pass = 0; pass < PASSES; ++pass)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int64_t r = r0 + (pass * (256 / GROUPS) + t / GROUPS) * 2 + h;
                if (r >= rows || left <= 0) continue;
                w[pass][h] = load_f8_upto8(src + r * ld_src + c, left);
                s[pass][h] = e8m0_to_f32(scale.p[(r >> shift) * scale.row + cb * scale.col]);
            }
#pragma unroll
        for (int pass = 0; pass < PASSES; ++pass) {
            float v[2][8];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                e4m3_unpack(w[pass][h][0], v[h]);
                e4m3_unpack(w[pass][h][1], v[h] + 4);
            }
#pragma unroll
            for (int i = 0; i < 8; ++i)
                tile[cg * 8 + i][pass * (256 / GROUPS) + t / GROUPS] =
                    uint32_t(__builtin_bit_cast(uint16_t, static_cast<bf16_t>(v[0][i] * s[pass][0]))) |
                    uint32_t(__builtin_bit_cast(uint16_t, static_cast<bf16_t>(v[1][i] * s[pass][1]))) << 16;
        }
        __syncthreads();
#pragma unroll
        for (int pass = 0; pass < COLS / 32; ++pass) {
            const int k = pass * 32 + t / 8, at = t % 8 * 4;
            if (c0 + k >= cols) continue;
            *reinterpret_cast<u32x4*>(dst + (c0 + k) * depth + r0 + at * 2) =
                u32x4{tile[k][at], tile[k][at + 1], tile[k][at + 2], tile[k][at + 3]};
        }
    }
};

// dst[r][c] = src[r][c] times its scale, exact in bf16, in rows of `depth`
// elements (a multiple of 64), zeros behind; eight elements a thread.
struct PackF8Rows {
    static constexpr int kLdsWords = 1;
    const uint8_t* src;
    int64_t ld_src, rows, cols;
    F8Scale scale;
    int shift;  // rows of a scale: 2^shift
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
            float v[8] = {};
            if (at < cols) {
                const float s = e8m0_to_f32(scale.p[(row >> shift) * scale.row + at / kF8Block * scale.col]);
                const u32x2 w = load_f8_upto8(src + row * ld_src + at, cols - at < 8 ? int(cols - at) : 8);
                e4m3_unpack(w[0], v);
                e4m3_unpack(w[1], v + 4);
                if (cols - at >= 8) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[e] *= s;
                } else {  // what lies behind the row stays zero beside a NaN
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[e] = at + e < cols ? v[e] * s : 0.0f;
                }
            }
            store8(dst + row * depth + at, v);
        }
    }
};

// Rows as PLANES bf16 planes each that add up to them: dst[i][p][r] from src[i][r].
template <typename S, int PLANES>
struct PackPlanes {
    static constexpr int kLdsWords = 1;
    const S* src;
    int64_t ld_src, rows, cols;
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
            float v[8] = {};
            if (left > 0) load_upto8(src + row * ld_src + at, left, v);
            bf16_t d[8][PLANES];
#pragma unroll
            for (int e = 0; e < 8; ++e) split_value<bf16_t, PLANES>(v[e], d[e]);
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

}  // namespace tg
