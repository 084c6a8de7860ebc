// tg_f8_tiles.hpp -- C = A B^T of e4m3 numbers with a power of two for each 128
// of them along the sum, on matrix instructions that apply the scales.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "tg_f8_types.hpp"
#include "tg_i8_tiles.hpp"

namespace tg {

typedef int32_t i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

__device__ __forceinline__ i32x8 f8_operand(u32x4 lo, u32x4 hi) {
    return __builtin_bit_cast(i32x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
}

// D += 2^(sx + sy - 254) X Y^T, X and Y 32 rows of 64 bytes: lane l holds 32
// bytes of row l % 32 of both, and the row's scale (a byte) for them; of D it has
// column l % 32 of rows 8 * (i / 4) + 4 * (l / 32) + i % 4.  Which of the 64 bytes
// a lane holds does not matter as long as X and Y agree, for all 128 bytes of a
// block have one scale.
__device__ __forceinline__ f32x16 f8_mma32(i32x8 x, i32x8 y, f32x16 d, int sx, int sy) {
    return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(x, y, d, 0, 0, 0, sx, 0, sy);
}
//
// These instructions add products in groups of a few neighbours along the sum,
// where terms 2^-13 below a group's largest product and less are dropped, and the
// groups' sums in f32 (found with sums of two terms at all distances).  Of sums
// of normal values this costs 1.5e-5 of the result in the mean, nothing beside
// the rounding of 16-bit outputs (2e-4, 1.7e-3); f32 outputs are made from bf16
// instead, with exact products and sums of f32.
//
// The same for 16 rows of 128 bytes: lane l holds 32 bytes of row l % 16, and of D
// rows 4 * (l / 16) ... + 3 of column l % 16.
__device__ __forceinline__ f32x4 f8_mma16(i32x8 x, i32x8 y, f32x4 d, int sx, int sy) {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(x, y, d, 0, 0, 0, sx, 0, sy);
}

// One byte per lane straight into a word of LDS, as tile_load has 16.
__device__ __forceinline__ void tile_load_byte(const uint8_t* base, uint32_t off, uint32_t lds) {
    asm volatile(
        "s_mov_b32 m0, %0\n\t"
        "s_nop 0\n\t"
        "global_load_lds_ubyte %1, %2" ::"s"(lds), "v"(off), "s"(base));
}

struct F8TileArgs {
    const uint8_t *a, *b;  // 16-byte aligned; row strides are multiples of 16 below 2^23
    int64_t lda, ldb;
    const uint8_t *sa, *sb;        // scales: row r (of sb: 128 rows), block c at r * row + c * col
    int64_t sa_row, sa_col, sb_row, sb_col;  // sa_row below 2^23
    int m, n;
    int steps;             // 128-byte blocks of the sum
    int tail;              // bytes of the last one that count: a multiple of 16
    int tiles_m, tiles_n;
    int slice;             // steps of one blockIdx.y
};

// WM x WN waves, each FM x FN fragments of 32 x 32; LDS holds a ring of NB
// stages of one step: A's rows, B's rows, A's scales (a word each) and B's (a
// word a lane, for each wave).  A step is two halves of 64 bytes: while the
// matrix unit works on one half's fragments, the other half's are read from LDS
// into registers.  The step's barrier stands between the halves, where the next
// step's loads have landed and this step's stage is free; the loads of the step
// NB later go between the second half's products.
//
// Fragment i of A in a wave holds rows li * FM + i (li = lane % 32), so that a
// lane's scales are neighbours; B's rows are taken so that a lane has 16 * FN
// neighbouring columns of C.  In LDS a fragment's rows are neighbours, and chunk c
// of LDS row L lies at place c ^ (L / 2 % 8): LDS serves lanes {0-3, 12-15, 20-27}
// and {4-11, 16-19, 28-31} of each 32 at a time, and so they meet 16 different
// places of the 256 bytes that two rows take.
template <int WM, int WN, int FM, int FN, int NB>
struct F8Tile {
    static constexpr int BM = WM * FM * 32, BN = WN * FN * 32, WAVES = WM * WN, NT = WAVES * 64;
    static constexpr int LOADS_A = BM * 8 / NT, LOADS_B = BN * 8 / NT, LOADS = LOADS_A + LOADS_B + 2;
    static constexpr int AT_B = BM * 128, AT_SA = AT_B + BN * 128, AT_SB = AT_SA + BM * 4;
    static constexpr int STAGE = AT_SB + WAVES * 256, LDS = NB * STAGE;
    static_assert(BM * 8 % NT == 0 && BN * 8 % NT == 0 && BM % 64 == 0, "whole loads");
    static_assert(NB >= 2 && NB <= 4, "wait_for's cases");
    static_assert(128 % (FN * 32) == 0, "one scale of B for a wave");

    static __device__ __forceinline__ int key(int L) { return L >> 1 & 7; }
    // Matrix rows (from the tile's first) of LDS rows.
    static __device__ __forceinline__ int row_a(int L) {
        return L / (FM * 32) * (FM * 32) + L % 32 * FM + L % (FM * 32) / 32;
    }
    static __device__ __forceinline__ int row_b(int L) {
        const int r = L % 32;
        return L / (FN * 32) * (FN * 32) + (r / 4 % 2) * 16 * FN + L % (FN * 32) / 32 * 16 + r / 8 * 4 + r % 4;
    }

    // The workgroup's tile: each XCD takes a run of tiles in bands of 8 tile
    // rows, whose panels its L2 then holds.
    static __device__ __forceinline__ void place(const F8TileArgs& p, int& tm, int& tn) {
        int id = xcd_run(int(blockIdx.x), p.tiles_m * p.tiles_n);
        const int band = id / (8 * p.tiles_n);
        const int height = p.tiles_m - band * 8 < 8 ? p.tiles_m - band * 8 : 8;
        id -= band * 8 * p.tiles_n;
        tm = band * 8 + id % height;
        tn = id / height;
    }

    // Sums steps [s0, s1), at least one, of tile (tm, tn) into acc.
    static __device__ __forceinline__ void run(const F8TileArgs& p, int tm, int tn, int s0, int s1, lds_t* lds,
                                               f32x16 (&acc)[FM][FN]) {
        const int t = threadIdx.x, lane = t % 64, wave = __builtin_amdgcn_readfirstlane(t / 64);
        const uint32_t lds0 = __builtin_amdgcn_readfirstlane(uint32_t(reinterpret_cast<uintptr_t>(lds)));
        const int wm = wave / WN, wn = wave % WN, li = lane % 32, hh = lane / 32;
        const char* a0 = reinterpret_cast<const char*>(p.a) + int64_t(tm) * BM * p.lda;
        const char* b0 = reinterpret_cast<const char*>(p.b) + int64_t(tn) * BN * p.ldb;
        const bool cut = s1 == p.steps && p.tail < 128;  // the last step is a partial one

        // Thread t loads place t % 8 of LDS rows t / 8, t / 8 + NT / 8, ...; rows
        // past the matrix repeat its last one (their outputs are not stored),
        // chunks past a partial last step repeat the last that counts (they are
        // cleared in registers).
        uint32_t off_a[LOADS_A], off_b[LOADS_B];
        auto chunk = [&](int i) { return (t % 8) ^ key(t / 8 + i * (NT / 8)); };
#pragma unroll
        for (int i = 0; i < LOADS_A; ++i) {
            const int r = row_a(t / 8 + i * (NT / 8)), last = p.m - 1 - tm * BM;
            off_a[i] = uint32_t(r < last ? r : last) * uint32_t(p.lda) + chunk(i) * 16;
        }
#pragma unroll
        for (int i = 0; i < LOADS_B; ++i) {
            const int r = row_b(t / 8 + i * (NT / 8)), last = p.n - 1 - tn * BN;
            off_b[i] = uint32_t(r < last ? r : last) * uint32_t(p.ldb) + chunk(i) * 16;
        }
        // Scales: a wave loads those of 64 rows of A, and its own one of B.
        const int part = wave % (BM / 64) * 64;
        uint32_t off_sa;
        {
            const int r = part + lane, last = p.m - 1 - tm * BM;
            off_sa = uint32_t(r < last ? r : last) * uint32_t(p.sa_row);
        }
        const uint8_t* sa0 = p.sa + int64_t(tm) * BM * p.sa_row;
        const int block_b = (tn * BN + wn * FN * 32) / 128, last_b = (p.n - 1) / 128;
        const uint8_t* sb0 = p.sb + int64_t(block_b < last_b ? block_b : last_b) * p.sb_row;

        // Load i of the step that comes next.
        int next = s0;
        uint32_t to = lds0;
        auto load = [&](int i) {
            auto over = [&](int c) {
                const int past = c * 16 + 16 - p.tail;
                return uint32_t(cut && next == s1 - 1 && past > 0 ? past : 0);
            };
            if (i < LOADS_A) {
                tile_load(a0 + int64_t(next) * 128, off_a[i] - over(chunk(i)), to + wave * 1024 + i * (NT * 16));
            } else if (i < LOADS_A + LOADS_B) {
                i -= LOADS_A;
                tile_load(b0 + int64_t(next) * 128, off_b[i] - over(chunk(i)), to + AT_B + wave * 1024 + i * (NT * 16));
            } else if (i == LOADS_A + LOADS_B) {
                tile_load_byte(sa0 + int64_t(next) * p.sa_col, off_sa, to + AT_SA + part * 4);
            } else {
                tile_load_byte(sb0 + int64_t(next) * p.sb_col, 0, to + AT_SB + wave * 256);
            }
        };
        auto loaded = [&] {
            ++next;
            to = to == lds0 + (NB - 1) * STAGE ? lds0 : to + STAGE;
        };
        // Waits until all but the newest `steps` steps' loads have landed.
        auto wait_for = [&](int steps) {
            if (NB > 3 && steps >= 2) tile_wait<(NB > 3 ? 2 : 0) * LOADS>();
            else if (NB > 2 && steps >= 1) tile_wait<(NB > 2 ? 1 : 0) * LOADS>();
            else tile_wait<0>();
        };

        const int first_a = wm * FM * 32 + li, first_b = wn * FN * 32 + li;
        const int at_a = first_a * 128 + (((hh * 2) ^ key(first_a)) << 4);
        const int at_b = AT_B + first_b * 128 + (((hh * 2) ^ key(first_b)) << 4);
        const int at_sa = AT_SA + (wm * FM * 32 + li * FM) * 4, at_sb = AT_SB + wave * 256 + lane * 4;
        typedef const __attribute__((address_space(3))) u32x4* frag_t;
        typedef const __attribute__((address_space(3))) int32_t* word_t;
        u32x4 xa[2][FM][2], xb[2][FN][2];
        int sa[2][FM], sb[2];  // of this step and of the next
        // Part i of READS of what half `half` of the stage at `from` needs.
        constexpr int READS = 2 * (FM + FN);
        auto read = [&](int i, int half, int from) {
            const int f = i / 2, q = i % 2, flip = half * 64 ^ q * 16;
            if (f < FN) xb[half][f][q] = *reinterpret_cast<frag_t>(lds + from + (at_b ^ flip) + f * 4096);
            else xa[half][f - FN][q] = *reinterpret_cast<frag_t>(lds + from + (at_a ^ flip) + (f - FN) * 4096);
        };
        auto read_scales = [&](int from) {
            sb[1] = *reinterpret_cast<word_t>(lds + from + at_sb);
#pragma unroll
            for (int i = 0; i < FM; ++i) sa[1][i] = *reinterpret_cast<word_t>(lds + from + at_sa + i * 4);
        };
        auto next_scales = [&] {
            sb[0] = sb[1];
#pragma unroll
            for (int i = 0; i < FM; ++i) sa[0][i] = sa[1][i];
        };
        // Multiplies the fragments of half h.  Between the products go the next
        // half's reads (from the stage at `from`) and a later step's loads.
        auto products = [&](int h, auto reads, auto scales, auto loads, int from) {
            constexpr int SLOTS = FM * FN, FOR_READS = SLOTS > 4 ? SLOTS - 2 : SLOTS;
#pragma unroll
            for (int s = 0; s < SLOTS; ++s) {
                const int i = s / FN, j = s % FN;
                acc[i][j] = f8_mma32(f8_operand(xb[h][j][0], xb[h][j][1]), f8_operand(xa[h][i][0], xa[h][i][1]), acc[i][j],
                                     sb[0], sa[0][i]);
                if (SLOTS > 1) __builtin_amdgcn_sched_barrier(0);
                if constexpr (decltype(scales)::value)
                    if (s == 0) read_scales(from);
                if constexpr (decltype(reads)::value) {
#pragma unroll
                    for (int r = 0; r < READS; ++r)
                        if (r * FOR_READS / READS == s) read(r, h ^ 1, from);
                }
                if constexpr (decltype(loads)::value) {
#pragma unroll
                    for (int l = 0; l < LOADS; ++l)
                        if (l * SLOTS / LOADS == s) load(l);
                }
                if (SLOTS > 1) __builtin_amdgcn_sched_barrier(0);
            }
        };
        // Clears the chunks that lie past the sum's end.
        auto clear = [&](int h) {
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                if ((h * 4 + hh * 2 + q) * 16 < p.tail) continue;
#pragma unroll
                for (int i = 0; i < FM; ++i) xa[h][i][q] = u32x4{0, 0, 0, 0};
#pragma unroll
                for (int j = 0; j < FN; ++j) xb[h][j][q] = u32x4{0, 0, 0, 0};
            }
        };
        const std::true_type yes;
        const std::false_type no;

        for (int s = s0; s < s1 && s < s0 + NB; ++s) {
#pragma unroll
            for (int l = 0; l < LOADS; ++l) load(l);
            loaded();
        }
        if (s1 - s0 >= NB) tile_wait<(NB - 1) * LOADS>();
        else tile_wait<0>();
        read_scales(0);
        next_scales();
#pragma unroll
        for (int r = 0; r < READS; ++r) read(r, 0, 0);
        int s = s0, at = 0, then = STAGE;  // this step's stage and the next one's
        auto step_done = [&] {
            next_scales();
            at = then;
            then = then == (NB - 1) * STAGE ? 0 : then + STAGE;
        };
        for (; s < s1 - NB; ++s) {
            products(0, yes, no, no, at);
            tile_wait<(NB - 2) * LOADS>();
            products(1, yes, yes, yes, then);
            loaded();
            step_done();
        }
        for (; s < s1 - 1; ++s) {  // nothing is left to load
            products(0, yes, no, no, at);
            wait_for(s1 - 2 - s);
            products(1, yes, yes, no, then);
            step_done();
        }
        if (cut) clear(0);
        products(0, yes, no, no, at);
        if (cut) clear(1);
        products(1, no, no, no, 0);
    }

    // Hands the lane's outputs to `out` in groups of eight neighbours in a row.
    template <typename Out>
    static __device__ __forceinline__ void outputs(const F8TileArgs& p, int tm, int tn, const f32x16 (&acc)[FM][FN],
                                                   const Out& out) {
        const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
        const int m0 = tm * BM + wave / WN * FM * 32 + lane % 32 * FM;
        const int n0 = tn * BN + wave % WN * FN * 32 + lane / 32 * 16 * FN;
#pragma unroll
        for (int g = 0; g < 2 * FN; ++g) {
            const int n = n0 + g * 8;
            if (n >= p.n) continue;
            const typename Out::Cols cols = out.cols(n, p.n - n);
#pragma unroll
            for (int i = 0; i < FM; ++i) {
                if (m0 + i >= p.m) continue;
                float v[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = acc[i][g / 2][g % 2 * 8 + e];
                out.store(m0 + i, n, p.n - n, v, out.row(m0 + i), cols);
            }
        }
    }

    // The workgroup's tile over slice `y` of the sum, from there to `out`.
    template <typename Out>
    static __device__ __forceinline__ void whole(const F8TileArgs& p, int y, char* smem, const Out& out) {
        const int s0 = y * p.slice, s1 = s0 + p.slice < p.steps ? s0 + p.slice : p.steps;
        f32x16 acc[FM][FN] = {};
        int tm, tn;
        place(p, tm, tn);
        run(p, tm, tn, s0, s1, (lds_t*)(smem), acc);
        outputs(p, tm, tn, acc, out);
    }
};

template <int WM, int WN, int FM, int FN, int NB, int PER_CU, typename T>
__global__ __launch_bounds__(WM* WN * 64, PER_CU) void tg_f8_tiles(F8TileArgs p, TileStore<T> out) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    F8Tile<WM, WN, FM, FN, NB>::whole(p, 0, smem, out);
}

// Slice blockIdx.y of the sum: its sums to part + blockIdx.y * M * ld.
template <int WM, int WN, int FM, int FN, int NB, int PER_CU>
__global__ __launch_bounds__(WM* WN * 64, PER_CU) void tg_f8_tiles_slice(F8TileArgs p, TilePartial<float> out) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    out.c += int64_t(blockIdx.y) * p.m * out.ld;
    F8Tile<WM, WN, FM, FN, NB>::whole(p, int(blockIdx.y), smem, out);
}

}  // namespace tg
