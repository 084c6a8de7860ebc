// tg_i8_turn.hpp -- gradients of the 8-bit product in one launch: operands that
// lie across the sum are turned as they are read from LDS.  For sums and outputs
// so small that laying the operands out first (tg_i8_pack.hpp) costs more than
// it brings.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "tg_i8_pack.hpp"
#include "tg_i8_tiles.hpp"

namespace tg {

struct TurnArgs {
    const void* g;  // G(i, r) = g[i * ldg + r], or g[r * ldg + i] (TRANS)
    int64_t ldg;
    const int8_t* q;  // depth x n
    int64_t ldq;
    const float* scale;  // depth
    int m, n, depth, tiles_m, tiles_n;
};

// Every line holds the neighbours that are loaded together.
inline bool turn_fits(bool transposed, int64_t m, int64_t n, int64_t depth) {
    return n >= 8 && (transposed ? m : depth) >= 8;
}

// Four 16-bit values of one column each: lane i of 16 names with `at` four
// neighbours in row i / 4 of a block of 4 rows and 16 columns (four groups of
// four), and gets the block's column i.
__device__ __forceinline__ u32x2 turn_read(const lds_t* at) {
    typedef short V __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) V* p_t;
    return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((p_t)(at)));
}

// 64 x 64 outputs a workgroup of 4 x 2 waves, 64 terms of the sum a step.  q,
// and G where it lies across the sum, are scaled and rounded as PackTurned does
// it and go to LDS as they lie in memory, a term's 64 values in a row of 160
// bytes, so that the four rows that turn_read() reads at once meet 32 different
// banks.  G along the sum lies there as in Tile.  Loads run two steps ahead in
// registers (four are no faster), LDS holds two steps.  Bound by the vector
// unit, which scales, splits and rounds each workgroup's operands anew: 0.5 us a
// step in 16 bits, 1.0 in f32.  GPU time of rows x columns x sum here and with
// operands laid out first, us: bf16 1024 x 1024 x 256 5.0 and 7.9, x 513 7.8 and
// 9.9, x 2049 20.9 and 20.5; f32 1024 x 1024 x 64 4.7 and 8.0, x 513 13.4 and
// 14.9; bf16 4096 x 4096 x 513, which takes the other way, 56 and 31.
//
// Values past the matrices' edges are not stored and may be anything; a line's
// 16 bytes that would end past it are its last ones, shifted into place.  Terms
// past the sum's end are zeros of both operands.
//
// WIDE: f16 of a wide range of scales (ScaleRange), G as two bf16 planes: up to
// 2.6 times as long (1024 x 1024 x 1024: 29 us and 20 for 11.6 and 12.0).
template <typename T, bool TRANS, bool WIDE = false>
struct Turn {
    static constexpr bool F32 = std::is_same<T, float>::value, F16 = std::is_same<T, f16_t>::value;
    using D = std::conditional_t<F16 && !WIDE, f16_t, bf16_t>;
    // Planes of G; more than one: G takes the scales, q stays an integer.
    static constexpr int P = F32 ? 3 : WIDE ? 2 : 1, SIZE = sizeof(T);
    static constexpr bool SPLIT = P > 1;
    static constexpr Mma KIND = std::is_same<D, f16_t>::value ? Mma::F16 : Mma::BF16;
    using Shape = Tile<KIND, 4, 2, 1, 2, 2>;  // places and stores of the outputs
    using Acc = typename Shape::Acc;
    static constexpr int NT = 512, ROW = 160, PLANE = TRANS ? 64 * ROW : 64 * 128, STAGE = P * PLANE + 64 * ROW;
    static constexpr int LDS = 2 * STAGE, AHEAD = 2;

    // G's lines of a step: 64 of 64 values, 16 bytes a load.
    static constexpr int PER = 16 / SIZE, CHUNKS = 64 / PER, LINES = NT / CHUNKS, LOADS = 64 / LINES;

    struct Raw {
        u32x2 q;
        u32x4 g[LOADS];
        float s;                                     // of q's term
        float sg[SPLIT ? (TRANS ? LOADS : PER) : 1];  // of G's terms
    };

    typedef __attribute__((address_space(3))) u32x4* put16_t;

    // 16 bytes of a line of `count` elements from element `at` on, or its last.
    template <typename E>
    static __device__ __forceinline__ u32x4 get(const E* line, int at, int count) {
        constexpr int N = 16 / int(sizeof(E));
        return *reinterpret_cast<const u32x4_any*>(line + (at + N <= count ? at : count - N));
    }
    // Bytes by which they came too early.
    template <typename E>
    static __device__ __forceinline__ int late(int at, int count) {
        constexpr int N = 16 / int(sizeof(E));
        return at + N <= count ? 0 : (at + N - count) * int(sizeof(E));
    }

    // True where nothing of step r0 lies past an edge; the same in the whole
    // workgroup.  Those steps leave out the shifts and bounds, which are half of
    // the vector unit's work.
    static __device__ __forceinline__ bool inside(const TurnArgs& p, int m0, int n0, int r0) {
        return r0 + 64 <= p.depth && n0 + 64 <= p.n && (!TRANS || m0 + 64 <= p.m);
    }

    // The thread's lines of G and q in the first step, bounded to the matrix's
    // rows where they are rows of the output.
    struct Lines {
        int64_t g[LOADS], q;
    };
    static __device__ __forceinline__ Lines lines(const TurnArgs& p, int m0, int n0) {
        const int t = threadIdx.x;
        Lines l;
        l.q = int64_t(t / 8) * p.ldq + n0 + t % 8 * 8;
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            const int line = t / CHUNKS + i * LINES, at = t % CHUNKS * PER;
            if constexpr (TRANS) l.g[i] = int64_t(line) * p.ldg + m0 + at;
            else l.g[i] = int64_t(m0 + line < p.m ? m0 + line : p.m - 1) * p.ldg + at;
        }
        return l;
    }

    static __device__ __forceinline__ void load(const TurnArgs& p, int m0, int n0, int r0, const Lines& l, Raw& x) {
        if (r0 >= p.depth) return;  // the step is past the sum
        const int t = threadIdx.x, last = p.depth - 1;
        const T* g = static_cast<const T*>(p.g);
        const int at = t % CHUNKS * PER;
        if (inside(p, m0, n0, r0)) {
            x.q = *reinterpret_cast<const u32x2_any*>(p.q + int64_t(r0) * p.ldq + l.q);
            const T* from = g + (TRANS ? int64_t(r0) * p.ldg : r0);
#pragma unroll
            for (int i = 0; i < LOADS; ++i) x.g[i] = *reinterpret_cast<const u32x4_any*>(from + l.g[i]);
        } else {
            const int rq = r0 + t / 8 < last ? r0 + t / 8 : last, cq = n0 + t % 8 * 8;
            x.q = *reinterpret_cast<const u32x2_any*>(p.q + int64_t(rq) * p.ldq + (cq + 8 <= p.n ? cq : p.n - 8));
#pragma unroll
            for (int i = 0; i < LOADS; ++i) {
                const int line = t / CHUNKS + i * LINES;
                if constexpr (TRANS) {
                    x.g[i] = get(g + int64_t(r0 + line < last ? r0 + line : last) * p.ldg, m0 + at, p.m);
                } else {
                    x.g[i] = get(g + (l.g[i] - at), r0 + at, p.depth);
                }
            }
        }
        x.s = p.scale[r0 + t / 8 < last ? r0 + t / 8 : last];
        if constexpr (SPLIT && TRANS) {
#pragma unroll
            for (int i = 0; i < LOADS; ++i) {
                const int r = r0 + t / CHUNKS + i * LINES;
                x.sg[i] = p.scale[r < last ? r : last];
            }
        } else if constexpr (SPLIT) {
#pragma unroll
            for (int i = 0; i < PER; ++i) x.sg[i] = p.scale[r0 + at + i < last ? r0 + at + i : last];
        }
    }

    // Writes step r0's operands to LDS.
    static __device__ __forceinline__ void put(const TurnArgs& p, int m0, int n0, int r0, lds_t* stage, float factor,
                                               const Raw& x) {
        if (r0 >= p.depth) return;
        if (inside(p, m0, n0, r0)) put_step<true>(p, m0, n0, r0, stage, factor, x);
        else put_step<false>(p, m0, n0, r0, stage, factor, x);
    }
    template <bool INSIDE>
    static __device__ __forceinline__ void put_step(const TurnArgs& p, int m0, int n0, int r0, lds_t* stage,
                                                    float factor, const Raw& x) {
        typedef D d8 __attribute__((ext_vector_type(8)));
        typedef D d_per __attribute__((ext_vector_type(PER)));
        typedef T t_per __attribute__((ext_vector_type(PER)));
        typedef std::conditional_t<PER == 8, u32x4, u32x2> words;
        typedef __attribute__((address_space(3))) words* put_t;
        const int t = threadIdx.x;
        {
            u32x2 w = x.q;
            float s = SPLIT ? 1.0f : x.s * factor;
            if constexpr (!INSIDE) {
                const int past = n0 + t % 8 * 8 + 8 - p.n;
                const uint64_t all = __builtin_bit_cast(uint64_t, w);
                w = __builtin_bit_cast(u32x2, past <= 0 ? all : past < 8 ? all >> past * 8 : 0);
                if (r0 + t / 8 >= p.depth) {
                    w = u32x2{0, 0};
                    s = 0.0f;
                }
            }
            d8 d;
#pragma unroll
            for (int i = 0; i < 8; ++i) d[i] = static_cast<D>(float(int32_t(w[i / 4] << (24 - i % 4 * 8)) >> 24) * s);
            *reinterpret_cast<put16_t>(stage + P * PLANE + t / 8 * ROW + t % 8 * 16) = __builtin_bit_cast(u32x4, d);
        }
        const int at = t % CHUNKS * PER;
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            const int line = t / CHUNKS + i * LINES;
            u32x4 w = x.g[i];
            if constexpr (!INSIDE) {
                w = shift_out(w, TRANS ? late<T>(m0 + at, p.m) : late<T>(r0 + at, p.depth));
                if (TRANS && r0 + line >= p.depth) w = u32x4{0, 0, 0, 0};
            }
            const int chunk = at / 8;
            lds_t* to = stage + (TRANS ? line * ROW + chunk * 16 : line * 128 + ((chunk ^ (line & 7)) << 4));
            if constexpr (SPLIT) {
                const t_per f = __builtin_bit_cast(t_per, w);
                d_per d[P];
#pragma unroll
                for (int e = 0; e < PER; ++e) {
                    // A term past the end is zero whatever its scale.
                    const bool live = INSIDE || (TRANS ? r0 + line < p.depth : r0 + at + e < p.depth);
                    D part[P];
                    split_value<D, P>(live ? to_f32(f[e]) * x.sg[TRANS ? i : e] : 0.0f, part);
#pragma unroll
                    for (int k = 0; k < P; ++k) d[k][e] = part[k];
                }
#pragma unroll
                for (int k = 0; k < P; ++k)
                    *reinterpret_cast<put_t>(to + k * PLANE + at % 8 * 2) = __builtin_bit_cast(words, d[k]);
            } else {
                *reinterpret_cast<put16_t>(to) = w;
            }
        }
    }

    // Fragment of 16 columns (four groups of four, `apart` columns from each
    // other) and the 32 terms of half h: lane l has terms l / 16 * 8 ... + 7.
    static __device__ __forceinline__ u32x4 turned(const lds_t* rows, int col, int apart, int h) {
        const int lane = threadIdx.x % 64;
        const lds_t* at = rows + (h * 32 + lane / 16 * 8 + lane % 16 / 4) * ROW + (col + lane % 4 * apart) * 2;
        const u32x2 a = turn_read(at), b = turn_read(at + 4 * ROW);
        return u32x4{a[0], a[1], b[0], b[1]};
    }

    static __device__ __forceinline__ void products(const lds_t* stage, Acc (&acc)[1][2]) {
        typedef const __attribute__((address_space(3))) u32x4* frag_t;
        const int lane = threadIdx.x % 64, wave = threadIdx.x / 64, li = lane % 16, lg = lane / 16;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            u32x4 xb[2];
#pragma unroll
            for (int j = 0; j < 2; ++j) xb[j] = turned(stage + P * PLANE, wave % 2 * 32 + 4 * j, 8, h);
#pragma unroll
            for (int k = 0; k < P; ++k) {
                const int row = wave / 2 * 16;
                u32x4 xa;
                if constexpr (TRANS) {
                    xa = turned(stage + k * PLANE, row, 4, h);
                } else {
                    xa = *reinterpret_cast<frag_t>(stage + k * PLANE + (row + li) * 128 + (((lg + 4 * h) ^ (li & 7)) << 4));
                }
#pragma unroll
                for (int j = 0; j < 2; ++j) acc[0][j] = mma<KIND>(xb[j], xa, acc[0][j]);
            }
        }
    }
};

// The range of a sum's scales, as tg_i8_scale_range finds it, in every workgroup.
__device__ __forceinline__ ScaleRange turn_range(const TurnArgs& p) {
    __shared__ float part[2][8];
    float top = 0.0f, low = __builtin_huge_valf();
    for (int i = threadIdx.x; i < p.depth; i += 512) add_scale(p.scale[i], top, low);
    top = wave_max(top);
    low = -wave_max(-low);
    if (threadIdx.x % 64 == 0) {
        part[0][threadIdx.x / 64] = top;
        part[1][threadIdx.x / 64] = low;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        top = fmaxf(top, part[0][i]);
        low = fminf(low, part[1][i]);
    }
    return scale_range(top, low);
}

// The sum of a wide range, without haste: one step's operands at a time in the
// LDS that the other way's two take.
template <bool TRANS>
__device__ __forceinline__ void turn_wide(const TurnArgs& p, int m0, int n0, lds_t* lds,
                                          typename Turn<f16_t, TRANS, true>::Acc (&acc)[1][2]) {
    using Cfg = Turn<f16_t, TRANS, true>;
    static_assert(Cfg::STAGE <= Turn<f16_t, TRANS>::LDS, "one stage");
    const typename Cfg::Lines l = Cfg::lines(p, m0, n0);
    for (int r0 = 0; r0 < p.depth; r0 += 64) {
        typename Cfg::Raw x;
        Cfg::load(p, m0, n0, r0, l, x);
        Cfg::put(p, m0, n0, r0, lds, 1.0f, x);
        __syncthreads();
        Cfg::products(lds, acc);
        __syncthreads();
    }
}

template <typename T, bool TRANS>
__global__ __launch_bounds__(512) void tg_i8_turn(TurnArgs p, TileStore<T> out) {
    using Cfg = Turn<T, TRANS>;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    lds_t* lds = (lds_t*)(smem);
    TileArgs tile{};
    tile.m = p.m;
    tile.n = p.n;
    tile.tiles_m = p.tiles_m;
    tile.tiles_n = p.tiles_n;
    int tm, tn;
    Cfg::Shape::place(tile, tm, tn);
    const int m0 = tm * 64, n0 = tn * 64, steps = (p.depth + 63) / 64;
    constexpr int AHEAD = Cfg::AHEAD;
    const typename Cfg::Lines l = Cfg::lines(p, m0, n0);
    typename Cfg::Raw x[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) Cfg::load(p, m0, n0, i * 64, l, x[i]);
    ScaleRange range{1.0f, 1.0f, 0};
    if constexpr (Cfg::F16) range = turn_range(p);
    typename Cfg::Acc acc[1][2] = {};
    if (range.wide != 0) {
        if constexpr (Cfg::F16) turn_wide<TRANS>(p, m0, n0, lds, acc);
    } else {
        Cfg::put(p, m0, n0, 0, lds, range.factor, x[0]);
        Cfg::load(p, m0, n0, AHEAD * 64, l, x[0]);
        __syncthreads();
        for (int s0 = 0; s0 < steps; s0 += AHEAD) {
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) {
                const int s = s0 + i;
                if (s >= steps) break;
                Cfg::products(lds + i % 2 * Cfg::STAGE, acc);
                Cfg::put(p, m0, n0, (s + 1) * 64, lds + (i + 1) % 2 * Cfg::STAGE, range.factor, x[(i + 1) % AHEAD]);
                Cfg::load(p, m0, n0, (s + 1 + AHEAD) * 64, l, x[(i + 1) % AHEAD]);
                __syncthreads();
            }
        }
    }
    if constexpr (Cfg::F16) {
        acc[0][0] *= range.back;
        acc[0][1] *= range.back;
    }
    typename Cfg::Shape::template Beside<TileStore<T>> beside;
    Cfg::Shape::beside(tile, tm, tn, out, beside);
    Cfg::Shape::outputs(tile, tm, tn, acc, out, beside);
}

}  // namespace tg
