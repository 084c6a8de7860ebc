// tg_f8_stream.hpp -- the product of a few rows of A (up to 64) with a weight
// matrix: every row of B is read once, straight into registers.
#pragma once

#include "tg_f8_tiles.hpp"
#include "tg_i8_stream.hpp"

namespace tg {

struct F8StreamArgs {
    const uint8_t *a, *b;
    int64_t lda, ldb;
    const uint8_t *sa, *sb;
    int64_t sa_row, sa_col, sb_row, sb_col;
    int m, n, k;
};

// Sixteen e4m3 numbers as two operands of eight bf16 (exact).
__device__ __forceinline__ void f8_widen(u32x4 x, u32x4 (&y)[2]) {
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const bf16x2 lo = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x[i], 1.0f, false);
        const bf16x2 hi = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x[i], 1.0f, true);
        y[i / 2][i % 2 * 2] = __builtin_bit_cast(uint32_t, lo);
        y[i / 2][i % 2 * 2 + 1] = __builtin_bit_cast(uint32_t, hi);
    }
}

// v * 2^(sa + sb - 254), NaN where either scale is.
__device__ __forceinline__ f32x4 f8_scaled(f32x4 v, int sa, int sb) {
    if (sa == 255 || sb == 255) v[0] = v[1] = v[2] = v[3] = __builtin_nanf("");
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = __builtin_amdgcn_ldexpf(v[i], sa + sb - 254);
    return v;
}

// acc += a block's sum times its scales.  For f32 outputs in bf16, with every
// product exact and sums of f32; the other types need less (tg_f8_tiles.hpp).
template <bool EXACT>
__device__ __forceinline__ void f8_block(const u32x4 (&fb)[2], const u32x4 (&fa)[2], int sb, int sa, f32x4& acc) {
    if constexpr (!EXACT) {
        acc = f8_mma16(f8_operand(fb[0], fb[1]), f8_operand(fa[0], fa[1]), acc, sb, sa);
    } else {
        f32x4 sum = {0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            u32x4 wb[2], wa[2];
            f8_widen(fb[i], wb);
            f8_widen(fa[i], wa);
            sum = mma<Mma::BF16>(wb[0], wa[0], sum);
            sum = mma<Mma::BF16>(wb[1], wa[1], sum);
        }
        acc += f8_scaled(sum, sa, sb);
    }
}

// A workgroup takes 16 rows of B (columns of C) and up to 16 * R rows of A; its
// W waves take the sum's blocks of 128 in turn and add their sums in LDS.  Bound
// by reading B: a wave has 2 KiB of B on their way, and the waves of a CU
// together cover HBM's latency.  Rows need no alignment: they go through
// registers.  WORDS: rows start at multiples of four bytes.  M = 1, 8192 x 8192: 13
// us (67 MB, 5.2 TB/s; weights partly in the last cache).
template <int R, int W, bool WORDS, typename T>
__global__ __launch_bounds__(W * 64) void tg_f8_stream(F8StreamArgs p, TileStore<T> out) {
    typedef StreamUnit<WORDS> Unit;
    constexpr bool EXACT = std::is_same<T, float>::value;
    __shared__ f32x4 part[R][W][64];
    const int t = threadIdx.x, lane = t % 64, wave = t / 64;
    const int n0 = int(blockIdx.x) * 16;
    // The lane's rows as it loads; those past the matrices repeat the last one
    // (their sums are not stored).
    const int lr = lane / 4, lc = lane % 4;
    const int8_t* pa[R];
    const int8_t* pb = reinterpret_cast<const int8_t*>(p.b) + int64_t(n0 + lr < p.n ? n0 + lr : p.n - 1) * p.ldb;
    const uint8_t* psa[R];  // of row lane % 16, as the matrix instruction has it
    const uint8_t* psb = p.sb + int64_t(n0 / kF8Block) * p.sb_row;
    int at_a[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        pa[r] = reinterpret_cast<const int8_t*>(p.a) + int64_t(r * 16 + lr < p.m ? r * 16 + lr : p.m - 1) * p.lda;
        at_a[r] = int(reinterpret_cast<uintptr_t>(pa[r]) & 3);
        psa[r] = p.sa + int64_t(r * 16 + lane % 16 < p.m ? r * 16 + lane % 16 : p.m - 1) * p.sa_row;
    }
    const int at_b = int(reinterpret_cast<uintptr_t>(pb) & 3);
    f32x4 acc[R] = {};
    const int units = p.k / 128;
    // What does not need the sum is loaded before it, so that its latency is
    // not added to the end.
    const bool last = wave == units % W && p.k % 128 != 0;
    StreamTail ta[R][2], tb[2];
    if (last) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int k = units * 128 + i * 64 + lc * 16;
            tb[i].load(pb, k, p.k);
#pragma unroll
            for (int r = 0; r < R; ++r) ta[r][i].load(pa[r], k, p.k);
        }
    }
    // Wave r < R stores rows r * 16 ...: a lane four columns of one.
    const int li = wave * 16 + lane % 16, lg = lane / 16;
    const bool stores = wave < R && li < p.m;
    float bias[4] = {};
    if (stores && out.bias != nullptr) {
#pragma unroll
        for (int e = 0; e < 4; ++e) bias[e] = to_f32(out.bias[n0 + lg * 4 + e < p.n ? n0 + lg * 4 + e : p.n - 1]);
    }
    for (int u = wave; u < units; u += W) {
        Unit xa[R], xb;
        int sa[R];
        const int sb = psb[int64_t(u) * p.sb_col];
        xb.load(pb + int64_t(u) * 128, at_b);
#pragma unroll
        for (int r = 0; r < R; ++r) {
            xa[r].load(pa[r] + int64_t(u) * 128, at_a[r]);
            sa[r] = psa[r][int64_t(u) * p.sa_col];
        }
        u32x4 fa[2], fb[2];
        xb.get(at_b, fb);
#pragma unroll
        for (int r = 0; r < R; ++r) {
            xa[r].get(at_a[r], fa);
            f8_block<EXACT>(fb, fa, sb, sa[r], acc[r]);
        }
    }
    if (last) {
        const int sb = psb[int64_t(units) * p.sb_col];
        const u32x4 fb[2] = {Unit::turn(tb[0].get()), Unit::turn(tb[1].get())};
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int sa = psa[r][int64_t(units) * p.sa_col];
            const u32x4 fa[2] = {Unit::turn(ta[r][0].get()), Unit::turn(ta[r][1].get())};
            f8_block<EXACT>(fb, fa, sb, sa, acc[r]);
        }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) part[r][wave][lane] = acc[r];
    __syncthreads();
    if (!stores) return;
    f32x4 sum = part[wave][0][lane];
#pragma unroll
    for (int w = 1; w < W; ++w) sum += part[wave][w][lane];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const int n = n0 + lg * 4 + e;
        if (n < p.n) out.c[int64_t(li) * p.n + n] = static_cast<T>(out.bias != nullptr ? sum[e] + bias[e] : sum[e]);
    }
}

}  // namespace tg
