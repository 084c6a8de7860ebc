// tg_i8_tiles.hpp -- C = A B^T on matrix instructions, for operands whose
// rows run along the sum: A is M rows and B is N rows of `bytes` bytes each,
// of 8-bit integers, bf16 or f16.  One kernel for the 8-bit product and (after
// tg_i8_pack.hpp) for the gradients.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "tg_i8_types.hpp"

namespace tg {

enum class Mma { I8, BF16, F16 };

// Matrix instructions of 16 x 16 outputs, 64 bytes of the sum.
//
// D += X Y^T: lane l holds bytes (l / 16) * 16 ... + 15 of row l % 16 of both,
// and of D rows 4 * (l / 16) ... + 3 of column l % 16.  (32 x 32 outputs read
// less from LDS and were not faster: the multiplier is the bound either way.)
template <Mma KIND>
struct MmaAcc {
    typedef float type __attribute__((ext_vector_type(4)));
};
template <>
struct MmaAcc<Mma::I8> {
    typedef int32_t type __attribute__((ext_vector_type(4)));
};

template <Mma KIND>
__device__ __forceinline__ typename MmaAcc<KIND>::type mma(u32x4 x, u32x4 y, typename MmaAcc<KIND>::type d) {
    if constexpr (KIND == Mma::I8) {
        typedef int32_t V __attribute__((ext_vector_type(4)));
        return __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(V, x), __builtin_bit_cast(V, y), d, 0, 0, 0);
    } else if constexpr (KIND == Mma::BF16) {
        typedef __bf16 V __attribute__((ext_vector_type(8)));
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(V, x), __builtin_bit_cast(V, y), d, 0, 0, 0);
    } else {
        typedef _Float16 V __attribute__((ext_vector_type(8)));
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(V, x), __builtin_bit_cast(V, y), d, 0, 0, 0);
    }
}

// Bytes of LDS.
typedef __attribute__((address_space(3))) char lds_t;

// One 16-byte load per lane straight into LDS: from base + off (off differs by
// lane) to lds + lane * 16.  base and lds are the same in all lanes.  Written
// as an instruction so that the compiler does not wait for it before every
// later LDS read (tile_wait() is the wait); it has no output registers, and
// m0 has no other use here.
__device__ __forceinline__ void tile_load(const char* base, uint32_t off, uint32_t lds) {
    asm volatile(
        "s_mov_b32 m0, %0\n\t"
        "s_nop 0\n\t"
        "global_load_lds_dwordx4 %1, %2" ::"s"(lds), "v"(off), "s"(base));
}

// At most N of this wave's loads into LDS are outstanding and every LDS read
// of it is done; then all waves of the workgroup meet.
template <int N>
__device__ __forceinline__ void tile_wait() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"i"(N) : "memory");
}

struct TileArgs {
    const char *a, *b;  // 16-byte aligned; row strides lda, ldb in bytes: multiples of 16 below 2^23
    int64_t lda, ldb;
    int m, n;           // rows of A and B
    int steps;          // 128-byte steps of the whole sum
    int tail;           // bytes of the last step that count: a multiple of 16, 16 ... 128
    int b_steps;        // A's step s meets B's step s % b_steps
    int64_t plane;      // bytes between the planes of a row of A
    int tiles_m, tiles_n;
    int slice;          // steps of one blockIdx.y (tg_i8_tiles_slice)
    const int* wide;    // f16: where it is not 0, A is two bf16 planes in a row of wide_a, B is bf16
    const char* wide_a;
    int64_t wide_lda;
};

// Tile of a workgroup: WM x WN waves, each FM x FN fragments of 16 x 16.
//
// LDS holds a ring of NB + 1 stages of A's BM rows of 128 bytes and one of NB
// stages of B's BN rows.  One step is two halves of 64 bytes.  While the matrix
// unit works on one half's fragments, the other half's are read from LDS into
// registers; the step's barrier stands between the halves, where the next
// step's loads have landed and this step's LDS is free.  A's loads of the step
// NB later go in the half before it (A's ring has a stage more), B's in the
// half behind it: a CU takes one 1 KiB load in 16 clocks at most, and waves
// that issue them faster stand still (8192^3 in 8 bits: 396 us; with A's and
// B's behind the barrier 421, all behind its first four rows 440; one build of
// each in turn, kept ones measure 396 to 426 from GPU to GPU, 2.6 to 2.8 P
// operations/s).  There the matrix unit is busy 67% of the cycles (79% in bf16:
// 8192 x 4096 x 4096 in 190 us once the clock has settled, 196 to 207 in the
// median of a run, 1.3 to 1.45 PFLOP/s) and the clock falls to 1.8 GHz under the
// load.  In products of few tiles a step takes longer than the issue of its
// loads: M = 512, N = K = 4096 in 12.4 to 12.9 us, 0.24 us a step on each CU for
// 24 KiB, which is 0.16 us at the rate above and 2.4 GHz (the rest, latency and
// the barrier, was not measured apart).
//
// The 16-byte chunk c of a row lies at place c ^ key(row).  LDS serves 16
// lanes of a 16-byte read at a time, lanes {0-3, 12-15, 20-27} and {4-11,
// 16-19, 28-31} of each 32, and key makes those 16 meet 16 different places of
// the 256 bytes that two rows take (no bank conflict is counted).  B's rows
// are taken so that a lane's FN fragments hold VPF FN neighbouring columns of C
// (whole 16-byte stores); B is the first operand, so that a fragment's values
// of a lane are neighbours in a row of C.
//
// P planes: a row of A is the sum of P rows, each multiplied with B's.
template <Mma KIND, int WM, int WN, int FM, int FN, int NB, int P = 1>
struct Tile {
    static constexpr int FS = 16, VPF = 4;  // a fragment's rows, and its values in a lane
    static constexpr int BM = WM * FM * FS, BN = WN * FN * FS, NT = WM * WN * 64;
    static constexpr int LOADS_A = P * BM * 8 / NT, LOADS_B = BN * 8 / NT, LOADS = LOADS_A + LOADS_B;
    static constexpr int NA = NB + 1, STAGE_A = P * BM * 128, STAGE_B = BN * 128, LDS = NA * STAGE_A + NB * STAGE_B;
    static_assert(BM * 8 * P % NT == 0 && BN * 8 % NT == 0 && NT % 64 == 0, "whole loads");
    static_assert(NB >= 2 && NB <= 4, "wait_for's cases");
    static_assert(FN >= 2, "work between two products");
    using Acc = typename MmaAcc<KIND>::type;
    using Value = std::conditional_t<KIND == Mma::I8, int32_t, float>;

    static __device__ __forceinline__ int key_a(int r) { return r & 7; }
    static __device__ __forceinline__ int key_b(int r) { return (r & 3) | (r / (VPF * FN) & 1) << 2; }

    // The workgroup's tile: each XCD takes a run of tiles in bands of 8 tile
    // rows, whose panels its L2 then holds.
    static __device__ __forceinline__ void place(const TileArgs& p, int& tm, int& tn) {
        int id = xcd_run(int(blockIdx.x), p.tiles_m * p.tiles_n);
        const int band = id / (8 * p.tiles_n);
        const int height = p.tiles_m - band * 8 < 8 ? p.tiles_m - band * 8 : 8;
        id -= band * 8 * p.tiles_n;
        tm = band * 8 + id % height;
        tn = id / height;
    }

    // Sums steps [s0, s1), at least one, of tile (tm, tn) into acc.
    static __device__ __forceinline__ void run(const TileArgs& p, int tm, int tn, int s0, int s1, lds_t* lds,
                                               Acc (&acc)[FM][FN]) {
        const int t = threadIdx.x, lane = t % 64, wave = __builtin_amdgcn_readfirstlane(t / 64);
        const uint32_t lds0 = __builtin_amdgcn_readfirstlane(uint32_t(reinterpret_cast<uintptr_t>(lds))) + wave * 1024;
        const char* a0 = p.a + int64_t(tm) * BM * p.lda;
        const char* b0 = p.b + int64_t(tn) * BN * p.ldb;
        const bool cut = s1 == p.steps && p.tail < 128;  // the last step is a partial one

        // Thread t loads place t % 8 of rows t / 8, t / 8 + NT / 8, ...; rows
        // past the matrix repeat its last one (their outputs are not stored),
        // chunks past a partial last step repeat the last that counts (they
        // are cleared in registers before they are used).
        uint32_t off_a[LOADS_A], off_b[LOADS_B];
        auto chunk_a = [&](int i) { return (t % 8) ^ key_a(t / 8 + i * (NT / 8)); };
        auto chunk_b = [&](int i) { return (t % 8) ^ key_b(t / 8 + i * (NT / 8)); };
#pragma unroll
        for (int i = 0; i < LOADS_A; ++i) {
            const int r = (t / 8 + i * (NT / 8)) % BM, k = (t / 8 + i * (NT / 8)) / BM, last = p.m - 1 - tm * BM;
            off_a[i] = uint32_t(r < last ? r : last) * uint32_t(p.lda) + uint32_t(k) * uint32_t(p.plane) + chunk_a(i) * 16;
        }
#pragma unroll
        for (int i = 0; i < LOADS_B; ++i) {
            const int r = t / 8 + i * (NT / 8), last = p.n - 1 - tn * BN;
            off_b[i] = uint32_t(r < last ? r : last) * uint32_t(p.ldb) + chunk_b(i) * 16;
        }
        // `count` loads from load `first` on of the step that comes next, A's
        // before B's; `over` is at most a chunk's own offset in its row, so
        // off - over stays inside the row.
        int next_a = s0, next_b = s0, turn_b = s0 % p.b_steps;
        uint32_t to_a = lds0, to_b = lds0 + NA * STAGE_A;
        auto over = [&](int step, int chunk) {
            const int past = chunk * 16 + 16 - p.tail;
            return uint32_t(cut && step == s1 - 1 && past > 0 ? past : 0);
        };
        auto load_a = [&](int first, int count) {
            const char* from = a0 + int64_t(next_a) * 128;
#pragma unroll
            for (int i = first; i < first + count; ++i)
                tile_load(from, off_a[i] - over(next_a, chunk_a(i)), to_a + i * (NT * 16));
        };
        auto load_b = [&](int first, int count) {
            const char* from = b0 + int64_t(turn_b) * 128;
#pragma unroll
            for (int i = first; i < first + count; ++i)
                tile_load(from, off_b[i] - over(next_b, chunk_b(i)), to_b + i * (NT * 16));
        };
        auto loaded_a = [&] {
            ++next_a;
            to_a = to_a == lds0 + (NA - 1) * STAGE_A ? lds0 : to_a + STAGE_A;
        };
        auto loaded_b = [&] {
            ++next_b;
            turn_b = turn_b + 1 == p.b_steps ? 0 : turn_b + 1;
            to_b = to_b == lds0 + NA * STAGE_A + (NB - 1) * STAGE_B ? lds0 + NA * STAGE_A : to_b + STAGE_B;
        };
        // Waits until all but the newest `steps` steps' loads have landed.
        auto wait_for = [&](int steps) {
            if (NB > 3 && steps >= 2) tile_wait<(NB > 3 ? 2 : 0) * LOADS>();
            else if (NB > 2 && steps >= 1) tile_wait<(NB > 2 ? 1 : 0) * LOADS>();
            else tile_wait<0>();
        };

        const int wm = wave / WN, wn = wave % WN, li = lane % FS, lg = lane / FS;
        const int row_a = wm * FM * FS + li, row_b = wn * FN * FS + li / 4 * (VPF * FN) + li % 4;
        // Fragment j's row, row_b + VPF j, has row_b's key, as fragment i's of
        // A, row_a + FS i, has row_a's.
        const int at_a = row_a * 128 + ((lg ^ key_a(row_a)) << 4);
        const int at_b = NA * STAGE_A + row_b * 128 + ((lg ^ key_b(row_b)) << 4);
        typedef const __attribute__((address_space(3))) u32x4* frag_t;
        // Row f of A's fragments: plane f % P of fragment f / P.
        constexpr int ROWS = FM * P;
        u32x4 xa[2][ROWS], xb[2][FN];
        // Part i of ROWS of a half's fragments, from the stages at (pa, pb).
        auto read_part = [&](int i, int half, int pa, int pb) {
            const lds_t *from_a = lds + pa, *from_b = lds + pb;
            xa[half][i] = *reinterpret_cast<frag_t>(from_a + (at_a ^ (half * 64)) + (i % P * BM + i / P * FS) * 128);
#pragma unroll
            for (int j = i * FN / ROWS; j < (i + 1) * FN / ROWS; ++j)
                xb[half][j] = *reinterpret_cast<frag_t>(from_b + (at_b ^ (half * 64)) + j * VPF * 128);
        };
        // Multiplies the fragments of half h, row by row.  Between each row's
        // products go its parts of a later step's loads and of the next
        // half's reads (done one row before the end, to be there in time).
        auto products = [&](int h, auto reads, auto loads_a, auto loads_b, int pa, int pb) {
#pragma unroll
            for (int i = 0; i < ROWS; ++i) {
                auto product = [&](int j) { acc[i / P][j] = mma<KIND>(xb[h][j], xa[h][i], acc[i / P][j]); };
                product(0);
                __builtin_amdgcn_sched_barrier(0);
                if constexpr (decltype(loads_a)::value)
                    load_a(i * LOADS_A / ROWS, (i + 1) * LOADS_A / ROWS - i * LOADS_A / ROWS);
                if constexpr (decltype(loads_b)::value)
                    load_b(i * LOADS_B / ROWS, (i + 1) * LOADS_B / ROWS - i * LOADS_B / ROWS);
                product(1);
                __builtin_amdgcn_sched_barrier(0);
                if constexpr (decltype(reads)::value) {
                    if (i == 0) read_part(0, h ^ 1, pa, pb);
                    if (i + 1 < ROWS) read_part(i + 1, h ^ 1, pa, pb);
                }
#pragma unroll
                for (int j = 2; j < FN; ++j) product(j);
                __builtin_amdgcn_sched_barrier(0);
            }
        };
        // Clears the fragments' chunks that lie past the sum's end: B's too but
        // for integers, as an infinity there would make NaN of A's zeros.
        auto clear = [&](int h) {
            if ((lg + 4 * h) * 16 < p.tail) return;
#pragma unroll
            for (int i = 0; i < ROWS; ++i) xa[h][i] = u32x4{0, 0, 0, 0};
            if constexpr (KIND != Mma::I8) {
#pragma unroll
                for (int j = 0; j < FN; ++j) xb[h][j] = u32x4{0, 0, 0, 0};
            }
        };
        const std::true_type yes;
        const std::false_type no;

        for (int s = s0; s < s1 && s < s0 + NB; ++s) {
            load_a(0, LOADS_A);
            load_b(0, LOADS_B);
            loaded_a();
            loaded_b();
        }
        if (s1 - s0 >= NB) tile_wait<(NB - 1) * LOADS>();
        else tile_wait<0>();
#pragma unroll
        for (int i = 0; i < ROWS; ++i) read_part(i, 0, 0, 0);
        // Places of this step's and the next one's stages.
        int s = s0, pa = 0, pb = 0, then_a = STAGE_A, then_b = STAGE_B;
        auto step_done = [&] {
            pa = then_a;
            pb = then_b;
            then_a = then_a == (NA - 1) * STAGE_A ? 0 : then_a + STAGE_A;
            then_b = then_b == (NB - 1) * STAGE_B ? 0 : then_b + STAGE_B;
        };
        for (; s < s1 - NB; ++s) {
            products(0, yes, yes, no, pa, pb);
            loaded_a();
            tile_wait<(NB - 2) * LOADS + LOADS_A>();
            products(1, yes, no, yes, then_a, then_b);
            loaded_b();
            step_done();
        }
        for (; s < s1 - 1; ++s) {  // nothing is left to load
            products(0, yes, no, no, pa, pb);
            wait_for(s1 - 2 - s);
            products(1, yes, no, no, then_a, then_b);
            step_done();
        }
        if (cut) clear(0);
        products(0, yes, no, no, pa, pb);
        if (cut) clear(1);
        products(1, no, no, no, 0, 0);
    }

    // What `Out` needs beside the sums, for the lane's rows and groups of eight
    // columns.
    template <typename Out>
    struct Beside {
        typename Out::Row rows[FM];
        typename Out::Cols cols[FN * VPF / 8];
    };
    static constexpr int GROUPS = FN * VPF / 8;
    static_assert(FN * VPF % 8 == 0, "groups of eight");
    // Loaded before the sum where registers allow it, so that its latency is
    // not added to the end.
    static constexpr bool EARLY_BESIDE = FM * FN <= 8;

    static __device__ __forceinline__ int first_row(int tm) {
        const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
        return tm * BM + wave / WN * FM * FS + lane % FS;
    }
    static __device__ __forceinline__ int first_col(int tn) {
        const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
        return tn * BN + wave % WN * FN * FS + lane / FS * VPF * FN;
    }

    template <typename Out>
    static __device__ __forceinline__ void beside(const TileArgs& p, int tm, int tn, const Out& out, Beside<Out>& x) {
        const int m0 = first_row(tm), n0 = first_col(tn);
#pragma unroll
        for (int i = 0; i < FM; ++i)
            if (m0 + i * FS < p.m) x.rows[i] = out.row(m0 + i * FS);
#pragma unroll
        for (int g = 0; g < GROUPS; ++g)
            if (n0 + g * 8 < p.n) x.cols[g] = out.cols(n0 + g * 8, p.n - n0 - g * 8);
    }

    // Hands the lane's outputs to `out` in groups of eight neighbours in a row.
    template <typename Out>
    static __device__ __forceinline__ void outputs(const TileArgs& p, int tm, int tn, const Acc (&acc)[FM][FN],
                                                   const Out& out, const Beside<Out>& x) {
        const int m0 = first_row(tm), n0 = first_col(tn);
        auto each = [&](auto inside) {
            constexpr bool IN = decltype(inside)::value;
#pragma unroll
            for (int i = 0; i < FM; ++i) {
                if (!IN && m0 + i * FS >= p.m) continue;
#pragma unroll
                for (int g = 0; g < GROUPS; ++g) {
                    if (!IN && n0 + g * 8 >= p.n) continue;
                    Value v[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[e] = acc[i][(g * 8 + e) / VPF][(g * 8 + e) % VPF];
                    out.store(m0 + i * FS, n0 + g * 8, IN ? 8 : p.n - n0 - g * 8, v, x.rows[i], x.cols[g]);
                }
            }
        };
        const bool in = int64_t(tm + 1) * BM <= p.m && int64_t(tn + 1) * BN <= p.n;
        if constexpr (Out::HALVES) {
            if (in && out.odd_rows()) return halves(m0, n0, acc, out, x);
        }
        if (in) each(std::true_type());
        else each(std::false_type());
    }

    // The same for 16-bit outputs inside the matrix, where rows start at any
    // half of a word: a store of 16 bytes at an odd half takes several times as
    // long as one at a word, so a lane stores the whole words of its columns, the
    // last with the next lane's first column (8-bit product of 8192 x 4097 x
    // 1024: 64 us with the stores at halves, 54 so; with 4094 columns 48).
    template <typename Out>
    static __device__ __forceinline__ void halves(int m0, int n0, const Acc (&acc)[FM][FN], const Out& out,
                                                  const Beside<Out>& x) {
        constexpr int W = GROUPS * 4;
        const int lg = threadIdx.x % 64 / FS;
#pragma unroll
        for (int i = 0; i < FM; ++i) {
            uint32_t w[W + 1];
#pragma unroll
            for (int g = 0; g < GROUPS; ++g) {
                Value v[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = acc[i][(g * 8 + e) / VPF][(g * 8 + e) % VPF];
                const u32x4 q = out.pack(v, x.rows[i], x.cols[g]);
#pragma unroll
                for (int e = 0; e < 4; ++e) w[g * 4 + e] = q[e];
            }
            w[W] = __shfl_down(w[0], FS);
            char* to = out.at(m0 + i * FS, n0);
            const int odd = int(reinterpret_cast<uintptr_t>(to) & 2);
            if (odd != 0 && lg == 0) *reinterpret_cast<uint16_t*>(to) = uint16_t(w[0]);
            uint32_t s[W];
#pragma unroll
            for (int e = 0; e < W; ++e) s[e] = __builtin_amdgcn_alignbyte(w[e + 1], w[e], odd);
            to += odd;
#pragma unroll
            for (int g = 0; g + 1 < GROUPS; ++g)
                *reinterpret_cast<u32x4_word*>(to + g * 16) = u32x4{s[g * 4], s[g * 4 + 1], s[g * 4 + 2], s[g * 4 + 3]};
            to += (GROUPS - 1) * 16;
            if (odd != 0 && lg == 3) {  // the next lane's columns are another wave's
                *reinterpret_cast<u32x2_word*>(to) = u32x2{s[W - 4], s[W - 3]};
                *reinterpret_cast<uint32_t*>(to + 8) = s[W - 2];
                *reinterpret_cast<uint16_t*>(to + 12) = uint16_t(s[W - 1]);
            } else {
                *reinterpret_cast<u32x4_word*>(to) = u32x4{s[W - 4], s[W - 3], s[W - 2], s[W - 1]};
            }
        }
    }

    // The workgroup's tile over slice `y` of the sum, from there to `out`.
    template <typename Out>
    static __device__ __forceinline__ void whole(const TileArgs& p, int y, char* smem, const Out& out) {
        const int s0 = y * p.slice, s1 = s0 + p.slice < p.steps ? s0 + p.slice : p.steps;
        Acc acc[FM][FN] = {};
        Beside<Out> x;
        int tm, tn;
        place(p, tm, tn);
        if (EARLY_BESIDE) beside(p, tm, tn, out, x);
        run(p, tm, tn, s0, s1, (lds_t*)(smem), acc);
        if (!EARLY_BESIDE) beside(p, tm, tn, out, x);
        outputs(p, tm, tn, acc, out, x);
    }
};

// C = sum * a_scale[m] * b_scale[n] + bias[n], rounded to T; a_scale, b_scale
// and bias may be null, `all` is one more factor where it is not.
template <typename T>
struct TileStore {
    const float *a_scale, *b_scale, *all;
    const T* bias;
    T* c;
    int64_t n;

    struct Row {
        float scale;
    };
    struct Cols {
        float scale[8], bias[8];
    };
    static constexpr bool HALVES = sizeof(T) == 2;
    // Not all rows start at a word.
    __device__ __forceinline__ bool odd_rows() const { return n % 2 != 0 || reinterpret_cast<uintptr_t>(c) % 4 != 0; }
    __device__ __forceinline__ char* at(int m, int col) const {
        return reinterpret_cast<char*>(c + int64_t(m) * n + col);
    }
    // Eight 16-bit outputs.
    template <typename V>
    __device__ __forceinline__ u32x4 pack(const V (&x)[8], const Row& r, const Cols& c8) const {
        typedef T t8 __attribute__((ext_vector_type(8)));
        float v[8];
        scaled(x, r, c8, v);
        t8 t;
#pragma unroll
        for (int i = 0; i < 8; ++i) t[i] = static_cast<T>(v[i]);
        return __builtin_bit_cast(u32x4, t);
    }
    __device__ __forceinline__ Row row(int m) const { return {a_scale != nullptr ? a_scale[m] : 1.0f}; }
    __device__ __forceinline__ Cols cols(int col, int left) const {
        Cols c;
        const float f = all != nullptr ? *all : 1.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) c.scale[i] = f, c.bias[i] = 0.0f;
        if (b_scale != nullptr) load_upto8(b_scale + col, left, c.scale);
        if (bias != nullptr) load_upto8(bias + col, left, c.bias);
        return c;
    }
    template <typename V>
    __device__ __forceinline__ void scaled(const V (&x)[8], const Row& r, const Cols& c8, float (&v)[8]) const {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = float(x[i]) * r.scale * c8.scale[i];
        if (bias != nullptr) {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] += c8.bias[i];
        }
    }
    template <typename V>
    __device__ __forceinline__ void store(int m, int col, int left, const V (&x)[8], const Row& r,
                                          const Cols& c8) const {
        float v[8];
        scaled(x, r, c8, v);
        store_upto8(c + int64_t(m) * n + col, left, v);
    }
};

// Sums of a slice as they are, in rows of `ld` (a multiple of 8) 32-bit values.
template <typename V>
struct TilePartial {
    static constexpr bool HALVES = false;
    V* c;
    int64_t ld;
    struct Row {};
    struct Cols {};
    __device__ __forceinline__ Row row(int) const { return {}; }
    __device__ __forceinline__ Cols cols(int, int) const { return {}; }
    __device__ __forceinline__ void store(int m, int col, int, const V (&x)[8], const Row&, const Cols&) const {
        typedef V V4 __attribute__((ext_vector_type(4)));
        V4* to = reinterpret_cast<V4*>(c + int64_t(m) * ld + col);
        to[0] = V4{x[0], x[1], x[2], x[3]};
        to[1] = V4{x[4], x[5], x[6], x[7]};
    }
};

// Slice `y` of the sum on KIND's instructions, or on bf16's where f16 operands
// have been laid out as such.
template <Mma KIND, int WM, int WN, int FM, int FN, int NB, int P, typename Out>
__device__ __forceinline__ void tiles_slice(TileArgs p, int y, char* smem, const Out& out) {
    if constexpr (KIND == Mma::F16) {
        if (*p.wide != 0) {
            p.a = p.wide_a;
            p.lda = p.wide_lda;
            p.steps *= 2;
            p.slice *= 2;
            p.tail = 128;
            Tile<Mma::BF16, WM, WN, FM, FN, NB, P>::whole(p, y, smem, out);
            return;
        }
    }
    Tile<KIND, WM, WN, FM, FN, NB, P>::whole(p, y, smem, out);
}

template <Mma KIND, int WM, int WN, int FM, int FN, int NB, int P, int PER_CU, typename T>
__global__ __launch_bounds__(WM* WN * 64, PER_CU) void tg_i8_tiles(TileArgs p, TileStore<T> out) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    tiles_slice<KIND, WM, WN, FM, FN, NB, P>(p, 0, smem, out);
}

// Slice blockIdx.y of the sum: its sums to part + blockIdx.y * M * ld.
template <Mma KIND, int WM, int WN, int FM, int FN, int NB, int P, int PER_CU>
__global__ __launch_bounds__(WM* WN * 64, PER_CU) void tg_i8_tiles_slice(
    TileArgs p, TilePartial<typename Tile<KIND, WM, WN, FM, FN, NB, P>::Value> out) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    out.c += int64_t(blockIdx.y) * p.m * out.ld;
    tiles_slice<KIND, WM, WN, FM, FN, NB, P>(p, int(blockIdx.y), smem, out);
}

// C from the slices' sums, added in their order (none: an empty sum).
template <typename V, typename T>
__global__ __launch_bounds__(256) void tg_i8_tiles_join(const V* __restrict__ part, int64_t ld, int slices, int64_t m,
                                                        int64_t n, TileStore<T> out) {
    typedef V V4 __attribute__((ext_vector_type(4)));
    const int64_t groups = ld / 8, total = m * groups;
    for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < total; i += int64_t(gridDim.x) * 256) {
        const int64_t row = i / groups, col = (i - row * groups) * 8;
        const V4* from = reinterpret_cast<const V4*>(part + row * ld + col);
        V4 a = {0, 0, 0, 0}, b = {0, 0, 0, 0};
        for (int s = 0; s < slices; ++s, from += m * ld / 4) {
            a += from[0];
            b += from[1];
        }
        const V v[8] = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
        const int left = int(n - col < 8 ? n - col : 8);
        out.store(int(row), int(col), left, v, out.row(int(row)), out.cols(int(col), left));
    }
}

}  // namespace tg
