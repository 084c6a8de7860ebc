// tg_f8_rows.hip -- blocks of 1 x 128 or 128 x 128 elements to e4m3 numbers with
// one power of two as their scale, and back.  Bound by memory.
#include "../../include/tropical_gemm_hip.h"
#include "tg_f8.hpp"
#include "tg_f8_types.hpp"

namespace tg {
namespace {

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

template <typename F>
hipError_t by_type(int type, F&& f) {
    switch (type) {
        case TG_BF16: return f(bf16_t());
        case TG_F16: return f(f16_t());
        default: return f(float());
    }
}

// The least e with top <= 448 * 2^e = 1.75 * 2^(8 + e), at least kF8LeastExponent:
// a power of two costs no bits of a floating-point number, the product's matrix
// instructions apply it themselves, and what a number stands for is exact in
// bf16.
__device__ __forceinline__ int block_exponent(float top) {
    const uint32_t bits = __builtin_bit_cast(uint32_t, top);
    const int e = int(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
    return e > kF8LeastExponent ? e : kF8LeastExponent;
}

// A workgroup takes ROWS rows of COLS columns (whole blocks), a thread eight
// neighbours of eight rows; all loads are issued before the first is used.  SHORT:
// rows below eight elements.  A block
// that holds a NaN or an infinity becomes NaNs with scale 1, so that products of it
// are NaN.  bf16, 8192 x 8192 in blocks of a row: 41 to 43 us (201 MB, 4.7 to 4.9
// TB/s); f32, 5003 x 4099 in square blocks: 22 to 25 us (103 MB).
template <typename T, int BR, int COLS, bool SHORT>
__global__ __launch_bounds__(256) void tg_f8_blocks(const T* __restrict__ x, int64_t ldx, uint8_t* __restrict__ q,
                                                    uint8_t* __restrict__ scale, int64_t ld_scale, int64_t rows,
                                                    int64_t cols, int64_t strips) {
    constexpr int P = 8, LANES = COLS / 8, STEP = 256 / LANES, ROWS = P * STEP, BLOCKS = COLS / kF8Block;
    static_assert(BR == 1 || ROWS == BR, "whole blocks");
    __shared__ uint8_t exps[BLOCKS][ROWS];
    __shared__ float tops[4];
    const int t = threadIdx.x, r = t / LANES, b = t % LANES / 16;
    const int64_t strip = blockIdx.x % strips, r0 = blockIdx.x / strips * ROWS;
    const int64_t at = strip * COLS + t % LANES * 8;
    const int left = cols - at < 8 ? int(cols - at) : 8;  // none where not positive
    // A row's last group is loaded with the elements before it, which are shifted
    // out, so that it is one load as any other; and stored as one with the bytes of
    // the lane before it, where that is in the same wave.
    const int64_t from = left < 8 ? cols - 8 : at;
    const bool joined = t % (LANES < 64 ? LANES : 64) != 0, edge = (strip + 1) * COLS > cols;
    float v[P][8];
#pragma unroll
    for (int i = 0; i < P; ++i) {
        const int64_t row = r0 + r + STEP * i;
        if (row < rows && left > 0) {
            if constexpr (SHORT) load_part(x + row * ldx + at, left, v[i]);
            else load8(x + row * ldx + from, v[i]);
        } else
#pragma unroll
            for (int e = 0; e < 8; ++e) v[i][e] = 0.0f;
    }
    if (!SHORT && left < 8 && left > 0) {
#pragma unroll
        for (int i = 0; i < P; ++i) shift8(8 - left, v[i]);
    }
    float top[P];
#pragma unroll
    for (int i = 0; i < P; ++i) {
        top[i] = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) top[i] = max_nan(top[i], fabsf(v[i][e]));
    }
    if constexpr (BR == 1) {
#pragma unroll
        for (int i = 0; i < P; ++i)
#pragma unroll
            for (int d = 8; d > 0; d >>= 1) top[i] = max_nan(top[i], __shfl_xor(top[i], d));
    } else {
#pragma unroll
        for (int i = 1; i < P; ++i) top[0] = max_nan(top[0], top[i]);
        top[0] = wave_max(top[0]);
        if (t % 64 == 0) tops[t / 64] = top[0];
        __syncthreads();
        top[0] = max_nan(max_nan(tops[0], tops[1]), max_nan(tops[2], tops[3]));
#pragma unroll
        for (int i = 1; i < P; ++i) top[i] = top[0];
    }
#pragma unroll
    for (int i = 0; i < P; ++i) {
        const int64_t row = r0 + r + STEP * i;
        const bool finite = top[i] < __builtin_huge_valf();
        const int e = finite ? block_exponent(top[i]) : 0;
        const float f = __builtin_bit_cast(float, uint32_t(127 - e) << 23);
        if (BR == 1 && t % 16 == 0) exps[b][r + STEP * i] = uint8_t(e + 127);
        if (BR != 1 && i == 0 && t == 0) scale[strip * ld_scale + blockIdx.x / strips] = uint8_t(e + 127);
        u32x2 w;
#pragma unroll
        for (int h = 0; h < 2; ++h)
            w[h] = e4m3_pack(v[i][4 * h] * f, v[i][4 * h + 1] * f, v[i][4 * h + 2] * f, v[i][4 * h + 3] * f);
        if (!finite) w = u32x2{0x7f7f7f7fu, 0x7f7f7f7fu};
        if (row >= rows) continue;  // the same in the row's lanes
        if (SHORT || edge) {
            const u32x2 before = {uint32_t(__shfl_up(w[0], 1)), uint32_t(__shfl_up(w[1], 1))};
            if (!SHORT && left < 8 && joined) {
                if (left > 0) {
                    const int bits = left * 8;
                    const uint64_t a = __builtin_bit_cast(uint64_t, before), b8 = __builtin_bit_cast(uint64_t, w);
                    *reinterpret_cast<u32x2_any*>(q + row * cols + from) = __builtin_bit_cast(u32x2, a >> bits | b8 << (64 - bits));
                }
            } else {
                store_f8_upto8(q + row * cols + at, left, w);
            }
        } else {
            *reinterpret_cast<u32x2_any*>(q + row * cols + at) = w;
        }
    }
    if constexpr (BR == 1) {  // the scales of a column of blocks are neighbours
        __syncthreads();
        const int64_t row = r0 + t % ROWS, cb = strip * BLOCKS + t / ROWS;
        if (t < BLOCKS * ROWS && row < rows && cb * kF8Block < cols) scale[cb * ld_scale + row] = exps[t / ROWS][t % ROWS];
    }
}

// Columns of a workgroup: one block, or eight where 8-bit rows do not start at whole
// words of eight bytes, so that fewer lines are written in two parts (bf16, 8192 x
// 8192: 43 us as one, 45 as eight; 8192 x 4095: 34 and 26).
bool wide_strips(int64_t cols) { return cols >= 512 && cols % 8 != 0; }

template <typename T, int BR, int COLS, bool SHORT = false>
hipError_t launch_blocks(const F8Quantize& p, hipStream_t st) {
    constexpr int ROWS = 8 * 256 / (COLS / 8);
    // A launch's thread count stays below 2^32.
    const int64_t strips = ceil_div(p.cols, COLS), most = (int64_t(1) << 23) / strips * ROWS;
    for (int64_t r0 = 0; r0 < p.rows; r0 += most) {
        const int64_t n = p.rows - r0 < most ? p.rows - r0 : most;
        hipLaunchKernelGGL((tg_f8_blocks<T, BR, COLS, SHORT>), dim3(unsigned(ceil_div(n, ROWS) * strips)), dim3(256), 0, st,
                           static_cast<const T*>(p.x) + r0 * p.ldx, p.ldx, p.q + r0 * p.cols, p.scale + r0 / BR,
                           ceil_div(p.rows, BR), n, p.cols, strips);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

// y = round(q * scale), eight elements a thread.  bf16, 8192 x 8192: 33 us (201 MB, q
// still in the last cache).
template <typename T>
__global__ __launch_bounds__(256) void tg_f8_restore(const uint8_t* __restrict__ q, int64_t ldq, F8Scale scale,
                                                     int shift, T* __restrict__ y, int64_t rows, int64_t cols,
                                                     int64_t groups) {
    const int64_t stride = int64_t(gridDim.x) * 256;
    for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < rows * groups; i += stride) {
        const int64_t row = i / groups, at = (i - row * groups) * 8;
        const int n = cols - at < 8 ? int(cols - at) : 8;
        const float s = e8m0_to_f32(scale.p[(row >> shift) * scale.row + at / kF8Block * scale.col]);
        const u32x2 w = load_f8_upto8(q + row * ldq + at, n);
        float v[8];
        e4m3_unpack(w[0], v);
        e4m3_unpack(w[1], v + 4);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] *= s;
        store_upto8(y + row * cols + at, n, v);
    }
}

}  // namespace

hipError_t f8_quantize(const F8Quantize& p, hipStream_t st) {
    if (p.rows == 0 || p.cols == 0) return hipSuccess;
    return by_type(p.type, [&](auto tag) {
        using T = decltype(tag);
        if (p.cols < 8)
            return p.block_rows != 1 ? launch_blocks<T, kF8Block, kF8Block, true>(p, st) : launch_blocks<T, 1, kF8Block, true>(p, st);
        if (p.block_rows != 1) return launch_blocks<T, kF8Block, kF8Block>(p, st);
        return wide_strips(p.cols) ? launch_blocks<T, 1, 1024>(p, st) : launch_blocks<T, 1, kF8Block>(p, st);
    });
}

hipError_t f8_dequantize(int type, const F8Matrix& q, void* y, int64_t rows, int64_t cols, hipStream_t st) {
    if (rows == 0 || cols == 0) return hipSuccess;
    const int64_t groups = ceil_div(cols, 8), blocks = ceil_div(rows * groups, 256);
    return by_type(type, [&](auto tag) {
        using T = decltype(tag);
        hipLaunchKernelGGL((tg_f8_restore<T>), dim3(unsigned(blocks < 65536 ? blocks : 65536)), dim3(256), 0, st, q.q,
                           q.ld, q.scale, q.block_rows == 1 ? 0 : 7, static_cast<T*>(y), rows, cols, groups);
        return hipGetLastError();
    });
}

}  // namespace tg
