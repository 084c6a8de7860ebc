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
// These instructions add products in groups of eight neighbours along the sum,
// where terms 2^-13 below a group's largest product and less are dropped, and the
// groups' sums in f32 (found with sums of two terms at all distances).  Largest goes
// by the operands' exponents, in which e4m3's numbers below 2^-6 count as 2^-6 and
// zeros not at all: at most 2^-10 of the sum of the products' magnitudes so counted
// are lost, which may be 2^3 times as much for each small operand (256 * 2^-9 hides
// what lies 2^-10 below it).  Of sums of normal values this
// costs 1.5e-5 of the result in the mean, little beside the rounding of 16-bit
// outputs (2e-4, 1.7e-3); of sums that cancel it may cost all of it.  f32 outputs
// are made from bf16 instead, with exact products and sums of f32.
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
template <int WM, int WN, int FM, int FN, int NB, int KS = 1>
struct F8Tile {
    static constexpr int BM = WM * FM * 32, BN = WN * FN * 32, WAVES = WM * WN, NT = WAVES * 64;
    static constexpr int LOADS_A = BM * 8 / NT, LOADS_B = BN * 8 / NT, LOADS = LOADS_A + LOADS_B + 2;
    static constexpr int AT_B = BM * 128, AT_SA = AT_B + BN * 128, AT_SB = AT_SA + BM * 4;
    static constexpr int STAGE = AT_SB + WAVES * 256, LDS = KS * NB * STAGE;
    static constexpr int THREADS = KS * NT, MERGE = KS > 1 ? WAVES * FM * FN * 4096 : 0;
    static_assert(BM * 8 % NT == 0 && BN * 8 % NT == 0 && BM % 64 == 0, "whole loads");
    static_assert(128 % (FN * 32) == 0, "one scale of B for a wave");
    static constexpr bool PAIRS = FM % 2 == 0 && FN % 2 == 0 && NB == 2;
    static_assert(PAIRS || (NB == 3 && FM * FN == 1), "run's forms");

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

    // Sums steps [s0, s1), at least one, of tile (tm, tn) into acc, of one fragment
    // each of A and B a wave.
    static __device__ __forceinline__ void run(const F8TileArgs& p, int tm, int tn, int s0, int s1, lds_t* lds,
                                               f32x16 (&acc)[FM][FN]) {
        const int t = threadIdx.x % NT, lane = t % 64, wave = __builtin_amdgcn_readfirstlane(t / 64);
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
            if (steps >= 1) tile_wait<LOADS>();
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
        // Multiplies the fragments of half h.  Behind the product go the next half's
        // reads (from the stage at `from`) and a later step's loads.
        auto products = [&](int h, auto reads, auto scales, auto loads, int from) {
            acc[0][0] = f8_mma32(f8_operand(xb[h][0][0], xb[h][0][1]), f8_operand(xa[h][0][0], xa[h][0][1]), acc[0][0], sb[0],
                                 sa[0][0]);
            if constexpr (decltype(scales)::value) read_scales(from);
            if constexpr (decltype(reads)::value) {
#pragma unroll
                for (int r = 0; r < READS; ++r) read(r, h ^ 1, from);
            }
            if constexpr (decltype(loads)::value) {
#pragma unroll
                for (int l = 0; l < LOADS; ++l) load(l);
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

    // The same for FM and FN even and NB = 2, with one wave on each SIMD: loads and
    // reads are spread evenly, and a load has more than a step's time to land.
    //
    // A step is two parts: the first multiplies the first half of A's fragments,
    // the second the second half, both with all of B's, for the whole 128 bytes.
    // Group 0 of a stage is A's first half, B's first half and the scales, group 1
    // the rest.  Group 0 of step s is read into registers during part 1 of step s
    // - 1, its place in LDS is free after the barrier that follows, filled for step
    // s + 2 during part 0 of s, and read again after the barrier in the middle of s +
    // 1.  Group 1 goes the same way half a step later.  B's fragments have registers
    // for one step: the second half's of a new step are read where the old ones have
    // been used for the last time.
    //
    // 8192^3 in 256 x 256 tiles, bf16: 395 to 419 us (2.6 to 2.8 P/s) with the
    // matrix unit busy 71% of the cycles and the clock at 1.88 GHz under the load; of
    // zeros 290 us, and the instructions alone, on random registers, 3.7 P/s: power is
    // the bound, and where in a step loads and reads go makes no difference any more.
    // With all of a step's loads and reads at its start, and outputs stored by the
    // lanes that hold them: 534 us.
    static __device__ __forceinline__ void run_pairs(const F8TileArgs& p, int tm, int tn, int s0, int s1, lds_t* lds,
                                                     f32x16 (&acc)[FM][FN]) {
        static_assert(NB == 2 && FM % 2 == 0 && FN % 2 == 0, "halves");
        const int t = threadIdx.x % NT, lane = t % 64, wave = __builtin_amdgcn_readfirstlane(t / 64);
        const uint32_t lds0 = __builtin_amdgcn_readfirstlane(uint32_t(reinterpret_cast<uintptr_t>(lds)));
        const int wm = wave / WN, wn = wave % WN, li = lane % 32, hh = lane / 32;
        const char* a0 = reinterpret_cast<const char*>(p.a) + int64_t(tm) * BM * p.lda;
        const char* b0 = reinterpret_cast<const char*>(p.b) + int64_t(tn) * BN * p.ldb;
        const bool cut = s1 == p.steps && p.tail < 128;  // the last step is a partial one

        // Load i of A in group g covers the LDS rows of fragments (of 32 rows each)
        // g * FM / 2 ... of every FM, NT / 8 rows a load; B likewise.
        constexpr int ROWS = NT / 8, GA = LOADS_A / 2, GB = LOADS_B / 2;
        static_assert(LOADS_A % 2 == 0 && LOADS_B % 2 == 0 && FM * 16 % ROWS == 0 && FN * 16 % ROWS == 0, "whole loads");
        auto lds_row = [](int i, int g, int frags) {  // first LDS row of load i
            const int at = i * ROWS, half = frags * 16;
            return at / half * frags * 32 + g * half + at % half;
        };
        auto chunk = [&](int row) { return (t % 8) ^ key(row + t / 8); };
        uint32_t off_a[2][GA], off_b[2][GB];
#pragma unroll
        for (int g = 0; g < 2; ++g) {
#pragma unroll
            for (int i = 0; i < GA; ++i) {
                const int L = lds_row(i, g, FM), r = row_a(L + t / 8), last = p.m - 1 - tm * BM;
                off_a[g][i] = uint32_t(r < last ? r : last) * uint32_t(p.lda) + chunk(L) * 16;
            }
#pragma unroll
            for (int i = 0; i < GB; ++i) {
                const int L = lds_row(i, g, FN), r = row_b(L + t / 8), last = p.n - 1 - tn * BN;
                off_b[g][i] = uint32_t(r < last ? r : last) * uint32_t(p.ldb) + chunk(L) * 16;
            }
        }
        const int part = wave % (BM / 64) * 64;
        const int row_sa = part + lane, last_sa = p.m - 1 - tm * BM;
        const uint32_t off_sa = uint32_t(row_sa < last_sa ? row_sa : last_sa) * uint32_t(p.sa_row);
        const uint8_t* sa0 = p.sa + int64_t(tm) * BM * p.sa_row;
        const int block_b = (tn * BN + wn * FN * 32) / 128, last_b = (p.n - 1) / 128;
        const uint8_t* sb0 = p.sb + int64_t(block_b < last_b ? block_b : last_b) * p.sb_row;

        // Load i of group g of step `step` into the stage at `to`.
        constexpr int LOADS0 = GA + GB + 2, LOADS1 = GA + GB;
        auto load = [&](int g, int i, int step, uint32_t to) {
            auto over = [&](int c) {
                const int past = c * 16 + 16 - p.tail;
                return uint32_t(cut && step == s1 - 1 && past > 0 ? past : 0);
            };
            if (i < GA) {
                const int L = lds_row(i, g, FM);
                tile_load(a0 + int64_t(step) * 128, off_a[g][i] - over(chunk(L)), to + L * 128 + wave * 1024);
            } else if (i < GA + GB) {
                const int L = lds_row(i - GA, g, FN);
                tile_load(b0 + int64_t(step) * 128, off_b[g][i - GA] - over(chunk(L)), to + AT_B + L * 128 + wave * 1024);
            } else if (i == GA + GB) {
                tile_load_byte(sa0 + int64_t(step) * p.sa_col, off_sa, to + AT_SA + part * 4);
            } else {
                tile_load_byte(sb0 + int64_t(step) * p.sb_col, 0, to + AT_SB + wave * 256);
            }
        };

        const int first_a = wm * FM * 32 + li, first_b = wn * FN * 32 + li;
        const int at_a = first_a * 128 + (((hh * 2) ^ key(first_a)) << 4);
        const int at_b = AT_B + first_b * 128 + (((hh * 2) ^ key(first_b)) << 4);
        const int at_sa = AT_SA + (wm * FM * 32 + li * FM) * 4, at_sb = AT_SB + wave * 256 + lane * 4;
        typedef const __attribute__((address_space(3))) u32x4* frag_t;
        typedef const __attribute__((address_space(3))) int32_t* word_t;
        constexpr int HM = FM / 2, HN = FN / 2;
        u32x4 xa[FM][4], xb[FN][4];  // quarter q of 128 bytes: half q / 2
        int sa[2][FM], sb[2];
        auto read_a = [&](int i, int q, int from) {
            xa[i][q] = *reinterpret_cast<frag_t>(lds + from + (at_a ^ (q / 2 * 64) ^ (q % 2 * 16)) + i * 4096);
        };
        auto read_b = [&](int j, int q, int from) {
            xb[j][q] = *reinterpret_cast<frag_t>(lds + from + (at_b ^ (q / 2 * 64) ^ (q % 2 * 16)) + j * 4096);
        };
        // Read r of group g, in the order of use.
        constexpr int READS = (HM + HN) * 4;
        auto read = [&](int g, int r, int from) {
            const int f = r / 4, q = r % 4;
            if (g == 0) {  // B's first, then A's
                if (f < 1) read_b(0, q, from);
                else if (f < 1 + HM) read_a(f - 1, q, from);
                else read_b(f - HM, q, from);
            } else {
                if (f < HN) read_b(HN + f, q, from);
                else read_a(HM + f - HN, q, from);
            }
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
        // Part `half` of a step: between the products go the reads of group 1 of
        // this step (part 0) or group 0 of the next (part 1) from the stage at
        // `from`, and the loads of group `half` of step `step` to `to`.
        constexpr int SLOTS = HM * FN * 2;
        auto products = [&](int half, auto reads, auto loads, int from, int step, uint32_t to) {
#pragma unroll
            for (int s = 0; s < SLOTS; ++s) {
                const int j = s / (2 * HM), h = s / HM % 2, i = half * HM + s % HM;
                acc[i][j] = f8_mma32(f8_operand(xb[j][2 * h], xb[j][2 * h + 1]), f8_operand(xa[i][2 * h], xa[i][2 * h + 1]),
                                     acc[i][j], sb[0], sa[0][i]);
                __builtin_amdgcn_sched_barrier(0);
                if constexpr (decltype(reads)::value) {
                    // B's fragment j of the next step takes the place of this one's
                    // behind its last product.
#pragma unroll
                    for (int r = 0; r < READS; ++r)
                        if (slot_of(half, r) == s) read(half ^ 1, r, from);
                    if (half == 1 && s == SLOTS / 2) read_scales(from);
                }
                if constexpr (decltype(loads)::value) {
                    const int count = half == 0 ? LOADS0 : LOADS1;
#pragma unroll
                    for (int l = 0; l < count; ++l)
                        if (l * SLOTS / count == s) load(half, l, step, to);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        };
        const std::true_type yes;
        const std::false_type no;

        for (int s = s0; s < s1 && s < s0 + 2; ++s) {
#pragma unroll
            for (int l = 0; l < LOADS0; ++l) load(0, l, s, lds0 + (s - s0) * STAGE);
#pragma unroll
            for (int l = 0; l < LOADS1; ++l) load(1, l, s, lds0 + (s - s0) * STAGE);
        }
        const bool one = s1 - s0 == 1;
        if (one) tile_wait<LOADS1>();
        else tile_wait<LOADS1 + LOADS0 + LOADS1>();
        read_scales(0);
        next_scales();
#pragma unroll
        for (int r = 0; r < READS; ++r) read(0, r, 0);
        int at = 0;  // this step's stage
        for (int s = s0; s < s1 - 2; ++s) {
            tile_wait<LOADS0 + LOADS1>();
            products(0, yes, yes, at, s + 2, lds0 + at);
            tile_wait<LOADS1 + LOADS0>();
            products(1, yes, yes, STAGE - at, s + 2, lds0 + at);
            next_scales();
            at = STAGE - at;
        }
        if (!one) {  // the step before the last: nothing is left to load
            tile_wait<LOADS0 + LOADS1>();
            products(0, yes, no, at, 0, 0);
            tile_wait<LOADS1>();
            products(1, yes, no, STAGE - at, 0, 0);
            next_scales();
            at = STAGE - at;
        }
        tile_wait<0>();
#pragma unroll
        for (int r = 0; r < READS; ++r) read(1, r, at);
        if (cut) {  // what lies past the sum's end counts as zero
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                if ((q / 2 * 4 + hh * 2 + q % 2) * 16 < p.tail) continue;
#pragma unroll
                for (int i = 0; i < FM; ++i) xa[i][q] = u32x4{0, 0, 0, 0};
#pragma unroll
                for (int j = 0; j < FN; ++j) xb[j][q] = u32x4{0, 0, 0, 0};
            }
        }
        products(0, no, no, 0, 0, 0);
        products(1, no, no, 0, 0, 0);
    }
    // The slot behind which read r goes: in part 0 at once, in part 1 not before
    // the last product of B's fragment that it replaces.
    static constexpr __device__ __forceinline__ int slot_of(int half, int r) {
        constexpr int HM = FM / 2, HN = FN / 2, SLOTS = HM * FN * 2, READS = (HM + HN) * 4, LAST = SLOTS - SLOTS / 4;
        const int even = r * LAST / READS;
        if (half == 0) return even;
        const int f = r / 4;
        if (f >= 1 && f < 1 + HM) return even;  // A's
        const int j = f < 1 ? 0 : f - HM, free = (j + 1) * 2 * HM - 1;
        return even > free ? even : free;
    }

    // Hands the wave's outputs to `out` in 16-byte chunks, those of a row by lanes
    // side by side: they go through LDS, where a row's chunk c lies at c ^ key, with
    // another key for each of the lanes that write at a time.  Stored from the
    // lanes as the matrix instructions leave them, a chunk of 32 rows at a time, a
    // 256 x 256 tile took 30 us.
    template <typename Out>
    static __device__ __forceinline__ void outputs(const F8TileArgs& p, int tm, int tn, char* smem,
                                                   const f32x16 (&acc)[FM][FN], const Out& out) {
        constexpr int SIZE = Out::SIZE, PER = 16 / SIZE;  // bytes of an output, outputs of a chunk
        constexpr int J = FN * 32 * SIZE > 256 ? FN / 2 : FN, COLS = J * 32, CH = COLS / PER;
        constexpr int ROWS = FM * 32, AT_ONCE = 64 / CH;  // rows that a wave stores at a time
        static_assert(MERGE + WAVES * ROWS * CH * 16 <= LDS, "the tile's outputs fit");
        const int lane = threadIdx.x % 64, wave = threadIdx.x / 64, li = lane % 32, hh = lane / 32;
        const int m0 = tm * BM + wave / WN * ROWS, n0 = tn * BN + wave % WN * FN * 32;
        u32x4* mine = reinterpret_cast<u32x4*>(smem + MERGE) + wave * ROWS * CH;
        auto place = [](int r, int c) { return r * CH + (c ^ (r / FM & (CH - 1))); };
#pragma unroll
        for (int j0 = 0; j0 < FN; j0 += J) {
            // A lane has 16 * FN columns, of which J * 16 belong to this pass: the
            // pass's columns are those of both halves of the lanes, one behind the other.
#pragma unroll
            for (int j = 0; j < J; ++j)
#pragma unroll
                for (int g = 0; g < 16 / PER; ++g) {
                    const int in_lane = (j0 + j) * 16 + g * PER, n = n0 + hh * 16 * FN + in_lane;
                    const auto beside = out.beside(n, p.n);
#pragma unroll
                    for (int i = 0; i < FM; ++i) {
                        float v[PER];
#pragma unroll
                        for (int e = 0; e < PER; ++e) v[e] = acc[i][j0 + j][g * PER + e];
                        mine[place(li * FM + i, hh * (CH / 2) + (j * 16 + g * PER) / PER)] = out.pack(v, beside);
                    }
                }
            const int c = lane % CH, n = n0 + c / (CH / 2) * 16 * FN + j0 * 16 + c % (CH / 2) * PER;
#pragma unroll 8
            for (int r0 = 0; r0 < ROWS; r0 += AT_ONCE) {
                const int r = r0 + lane / CH;
                out.template store<CH / 2>(m0 + r, n, p.m, p.n, mine[place(r, c)]);
            }
        }
    }

    // The workgroup's tile over slice `y` of the sum, from there to `out`.  KS 2:
    // the second half of the waves takes the second half of the slice's steps, at
    // least two, from stages of its own, and hands its sums over in LDS: where there
    // is a workgroup for each CU at most, waves that wait leave the matrix unit to
    // the others.
    template <typename Out>
    static __device__ __forceinline__ void whole(const F8TileArgs& p, int y, char* smem, const Out& out) {
        int s0 = y * p.slice, s1 = s0 + p.slice < p.steps ? s0 + p.slice : p.steps;
        f32x16 acc[FM][FN] = {};
        int tm, tn;
        place(p, tm, tn);
        const int part = KS > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x / NT) : 0;
        bool fewer = false;  // steps than the other half
        if constexpr (KS > 1) {
            static_assert(KS == 2, "halves");
            const int half = (s1 - s0 + 1) / 2;
            fewer = part != 0 && (s1 - s0) % 2 != 0;
            if (part == 0) s1 = s0 + half;
            else s0 += half;
        }
        lds_t* stages = (lds_t*)(smem) + part * NB * STAGE;
        if constexpr (PAIRS) run_pairs(p, tm, tn, s0, s1, stages, acc);
        else run(p, tm, tn, s0, s1, stages, acc);
        if (fewer) {  // the barriers of the step that it lacks
            __builtin_amdgcn_s_barrier();
            if (PAIRS) __builtin_amdgcn_s_barrier();
        }
        __syncthreads();  // all have read their last fragments
        if constexpr (KS > 1) {
            f32x4* sums = reinterpret_cast<f32x4*>(smem) + threadIdx.x % NT / 64 * (FM * FN * 256) + threadIdx.x % 64;
            if (part != 0) {
#pragma unroll
                for (int f = 0; f < FM * FN * 4; ++f) {
                    const f32x16& a = acc[f / 4 / FN][f / 4 % FN];
                    sums[f * 64] = f32x4{a[f % 4 * 4], a[f % 4 * 4 + 1], a[f % 4 * 4 + 2], a[f % 4 * 4 + 3]};
                }
            }
            __syncthreads();
            if (part != 0) return;
#pragma unroll
            for (int f = 0; f < FM * FN * 4; ++f) {
                const f32x4 v = sums[f * 64];
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[f / 4 / FN][f / 4 % FN][f % 4 * 4 + e] += v[e];
            }
        }
        outputs(p, tm, tn, smem, acc, out);
    }
};

// C = sum + bias[n] (null: none), rounded to T, of 16 bits.
template <typename T>
struct F8Store {
    static constexpr int SIZE = 2;
    const T* bias;
    T* c;
    int64_t n;

    struct Beside {
        float bias[8];
    };
    __device__ __forceinline__ Beside beside(int col, int cols) const {
        Beside b = {};
        if (bias != nullptr && col < cols) load_upto8(bias + col, cols - col, b.bias);
        return b;
    }
    __device__ __forceinline__ u32x4 pack(const float (&v)[8], const Beside& b) const {
        typedef T t8 __attribute__((ext_vector_type(8)));
        t8 t;
#pragma unroll
        for (int i = 0; i < 8; ++i) t[i] = static_cast<T>(bias != nullptr ? v[i] + b.bias[i] : v[i]);
        return __builtin_bit_cast(u32x4, t);
    }
    // Eight columns from `col` on; the RUN lanes of a row hold neighbours.  A store
    // of 16 bytes at an odd half of a word takes several times as long as one at
    // a word, so where rows may start there a lane stores whole words, the last with
    // the next lane's first column.
    template <int RUN>
    __device__ __forceinline__ void store(int row, int col, int rows, int cols, u32x4 w) const {
        const int lane = threadIdx.x % 64;
        const uint32_t next = __shfl_down(w[0], 1);
        T* to = c + int64_t(row) * n + col;
        const bool odd = (reinterpret_cast<uintptr_t>(to) & 2) != 0;
        if (row >= rows || col >= cols) return;
        typedef T t8 __attribute__((ext_vector_type(8)));
        const t8 t = __builtin_bit_cast(t8, w);
        if (cols - col < 8 || (odd && cols - col < 16 && lane % RUN != RUN - 1)) {
            // The row's end, or the lane before it, whose last word would reach there.
            const int left = cols - col < 8 ? cols - col : 8;
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (i < left) to[i] = t[i];
        } else if (!odd) {
            *reinterpret_cast<u32x4_word*>(to) = w;
        } else {
            const u32x4 s = {__builtin_amdgcn_alignbyte(w[1], w[0], 2), __builtin_amdgcn_alignbyte(w[2], w[1], 2),
                             __builtin_amdgcn_alignbyte(w[3], w[2], 2), __builtin_amdgcn_alignbyte(next, w[3], 2)};
            if (lane % RUN == 0) to[0] = t[0];
            if (lane % RUN != RUN - 1) {
                *reinterpret_cast<u32x4_word*>(to + 1) = s;
            } else {
                *reinterpret_cast<u32x2_word*>(to + 1) = u32x2{s[0], s[1]};
                *reinterpret_cast<uint32_t*>(to + 5) = s[2];
                to[7] = t[7];
            }
        }
    }
};

// Sums of a slice as they are, in rows of `ld` (a multiple of 8) f32 values.
struct F8Partial {
    static constexpr int SIZE = 4;
    float* c;
    int64_t ld;
    struct Beside {};
    __device__ __forceinline__ Beside beside(int, int) const { return {}; }
    __device__ __forceinline__ u32x4 pack(const float (&v)[4], const Beside&) const {
        return __builtin_bit_cast(u32x4, f32x4{v[0], v[1], v[2], v[3]});
    }
    template <int RUN>
    __device__ __forceinline__ void store(int row, int col, int rows, int, u32x4 w) const {
        if (row < rows && col < ld) *reinterpret_cast<u32x4*>(c + int64_t(row) * ld + col) = w;
    }
};

template <int WM, int WN, int FM, int FN, int NB, int KS, int PER_CU, typename T>
__global__ __launch_bounds__(WM* WN * 64 * KS, PER_CU) void tg_f8_tiles(F8TileArgs p, F8Store<T> out) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    F8Tile<WM, WN, FM, FN, NB, KS>::whole(p, 0, smem, out);
}

// Slice blockIdx.y of the sum: its sums to part + blockIdx.y * M * ld.
template <int WM, int WN, int FM, int FN, int NB, int KS, int PER_CU>
__global__ __launch_bounds__(WM* WN * 64 * KS, PER_CU) void tg_f8_tiles_slice(F8TileArgs p, F8Partial out) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    out.c += int64_t(blockIdx.y) * p.m * out.ld;
    F8Tile<WM, WN, FM, FN, NB, KS>::whole(p, int(blockIdx.y), smem, out);
}

}  // namespace tg
