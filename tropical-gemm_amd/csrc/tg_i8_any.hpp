// tg_i8_any.hpp -- the 8-bit product of rows at any address, in one launch:
// for products so small that laying the rows out first (tg_i8_pack.hpp) costs
// more than it brings.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "tg_i8_stream.hpp"
#include "tg_i8_tiles.hpp"

namespace tg {

// At least 16 bytes of the sum (k).
struct AnyArgs {
    const int8_t* a;
    int64_t lda;
    const int8_t* b;
    int64_t ldb;
    int m, n, k, tiles_m, tiles_n;
};

// 64 x 64 outputs a workgroup of 2 x 2 waves, 128 bytes of the sum a step, on
// Tile's LDS rows and fragments.  Rows come through registers (a load straight
// into LDS needs aligned addresses), two steps ahead of their use, and LDS
// holds two steps.  A row's chunk that would end past it is its last 16 bytes,
// shifted on their way into LDS, zeros from the sum's end on.
// Bound by the loads' latency (as aligned words and the next lane's first, one
// more load a row: a third slower).  GPU time of M x N x K here and in two
// launches, us: 1001 x 1001 x 515: 6.4 and 7.8; 257 x 1031 x 1031: 7.6 and 8.0;
// 128 x 4096 x 4095: 16.1 and 19.7; 2049 x 1031 x 1031: 16.2 and 14.4.
template <typename T>
__global__ __launch_bounds__(256) void tg_i8_any(AnyArgs p, TileStore<T> out) {
    using Cfg = Tile<Mma::I8, 2, 2, 2, 2, 2>;
    constexpr int STAGE = Cfg::STAGE_A + Cfg::STAGE_B;
    __shared__ __attribute__((aligned(16))) char smem[2 * STAGE];
    lds_t* lds = (lds_t*)(smem);
    typedef __attribute__((address_space(3))) u32x4* put_t;
    typedef const __attribute__((address_space(3))) u32x4* frag_t;
    TileArgs tile{};
    tile.m = p.m;
    tile.n = p.n;
    tile.tiles_m = p.tiles_m;
    tile.tiles_n = p.tiles_n;
    int tm, tn;
    Cfg::place(tile, tm, tn);
    typename Cfg::template Beside<TileStore<T>> x;
    Cfg::beside(tile, tm, tn, out, x);

    // Thread t brings chunk t % 8 of rows t / 8 and t / 8 + 32 of A and of B;
    // rows past the matrix repeat its last one (their outputs are not stored).
    const int t = threadIdx.x, chunk = t % 8;
    const int8_t* row[4];
    int to[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int r = t / 8 + i % 2 * 32;
        if (i < 2) {
            row[i] = p.a + int64_t(tm * 64 + r < p.m ? tm * 64 + r : p.m - 1) * p.lda;
            to[i] = r * 128 + ((chunk ^ Cfg::key_a(r)) << 4);
        } else {
            row[i] = p.b + int64_t(tn * 64 + r < p.n ? tn * 64 + r : p.n - 1) * p.ldb;
            to[i] = Cfg::STAGE_A + r * 128 + ((chunk ^ Cfg::key_b(r)) << 4);
        }
    }
    u32x4 raw[2][4];
    auto load = [&](int s, u32x4(&v)[4]) {
        if (s * 128 >= p.k) return;
        const int k = s * 128 + chunk * 16;
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = *reinterpret_cast<const u32x4_any*>(row[i] + (k < p.k - 16 ? k : p.k - 16));
    };
    auto put = [&](int s, u32x4(&v)[4]) {
        if (s * 128 + 128 > p.k) {
            const int k = s * 128 + chunk * 16;
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = shift_out(v[i], k < p.k - 16 ? 0 : k - (p.k - 16));
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) *reinterpret_cast<put_t>(lds + s % 2 * STAGE + to[i]) = v[i];
    };
    const int lane = t % 64, wave = t / 64, li = lane % 16, lg = lane / 16;
    const int row_a = wave / 2 * 32 + li, row_b = wave % 2 * 32 + li / 4 * 8 + li % 4;
    const int at_a = row_a * 128 + ((lg ^ Cfg::key_a(row_a)) << 4);
    const int at_b = Cfg::STAGE_A + row_b * 128 + ((lg ^ Cfg::key_b(row_b)) << 4);
    typename Cfg::Acc acc[2][2] = {};
    auto products = [&](int stage) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            u32x4 xa[2], xb[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                xa[i] = *reinterpret_cast<frag_t>(lds + stage * STAGE + (at_a ^ (h * 64)) + i * 16 * 128);
                xb[i] = *reinterpret_cast<frag_t>(lds + stage * STAGE + (at_b ^ (h * 64)) + i * 4 * 128);
            }
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j) acc[i][j] = mma<Mma::I8>(xb[j], xa[i], acc[i][j]);
        }
    };

    // Steps past the last one are zeros.
    const int steps = (p.k + 127) / 128;
    load(0, raw[0]);
    load(1, raw[1]);
    put(0, raw[0]);
    load(2, raw[0]);
    __syncthreads();
    for (int s = 0; s < steps; s += 2) {
        products(0);
        put(s + 1, raw[1]);
        load(s + 3, raw[1]);
        __syncthreads();
        if (s + 1 < steps) products(1);
        put(s + 2, raw[0]);
        load(s + 4, raw[0]);
        __syncthreads();
    }
    Cfg::outputs(tile, tm, tn, acc, out, x);
}

}  // namespace tg
