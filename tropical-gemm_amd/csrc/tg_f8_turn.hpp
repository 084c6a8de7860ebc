// tg_f8_turn.hpp -- gradients of the product in 8-bit floating point in one
// launch: operands that lie across the sum are turned as they are read from LDS.
// For sums and outputs so small that laying the operands out first
// (tg_f8_pack.hpp) costs more than it brings.
#pragma once

#include "tg_f8.hpp"
#include "tg_f8_types.hpp"
#include "tg_i8_turn.hpp"

namespace tg {

struct F8TurnArgs {
    const void* g;  // G(i, r) = g[i * ldg + r], or g[r * ldg + i] (TRANS)
    int64_t ldg;
    const uint8_t* q;  // depth x n
    int64_t ldq;
    F8Scale scale;
    int shift;  // rows of a scale: 2^shift
    int m, n, depth, tiles_m, tiles_n;
};

// 64 x 64 outputs a workgroup of 4 x 2 waves, 64 terms of the sum a step, as in
// Turn (tg_i8_turn.hpp): q in bf16 with its scales, and G where it lies across the
// sum, go to LDS as they lie in memory, a term's 64 values in a row of 160 bytes, so
// that the four rows that turn_read() reads at once meet 32 different banks.  G
// along the sum lies there in rows of 128 bytes, chunk c of row r at c ^ (r % 8).
// G in f16 or f32 becomes two or three bf16 planes that add up to it.  Loads run
// two steps ahead in registers, LDS holds two steps.  Bound by the vector unit,
// which makes each workgroup's operands anew: 0.5 us for every 64 of the sum in bf16,
// 0.8 in f16, 0.9 in f32.  GPU time of 300 x 512 (rows x columns of the gradient) here
// and with operands laid out first, us: a sum of 64 bf16 3.5 and 6.1, f32 4.2 and 6.4;
// of 513 7.8 and 8.2, 11.4 and 9.5; of 2049 20.1 and 14.8, 32.9 and 19.7.
//
// Values past the matrices' edges are not stored and may be anything; a line's
// 16 bytes that would end past it are its last ones, shifted into place.  Terms
// past the sum's end are zeros of both operands.
template <typename T, bool TRANS>
struct F8Turn {
    static constexpr int P = sizeof(T) == 4 ? 3 : std::is_same<T, f16_t>::value ? 2 : 1;
    using Shape = Tile<Mma::BF16, 4, 2, 1, 2, 2>;  // places and stores of the outputs
    using Acc = typename Shape::Acc;
    static constexpr int NT = 512, ROW = 160, PLANE = TRANS ? 64 * ROW : 64 * 128, STAGE = P * PLANE + 64 * ROW;
    static constexpr int LDS = 2 * STAGE, AHEAD = 2;
    // G's lines of a step: 64 of 64 values, 16 bytes a load.
    static constexpr int PER = 16 / int(sizeof(T)), CHUNKS = 64 / PER, LINES = NT / CHUNKS, LOADS = 64 / LINES;

    struct Raw {
        u32x2 q;
        u32x4 g[LOADS];
        int s;  // the scale of q's term
    };
    typedef __attribute__((address_space(3))) u32x4* put16_t;

    // 16 bytes of a line of `count` elements from element `at` on, or its last, and
    // the bytes by which those came too early.
    static __device__ __forceinline__ u32x4 get(const T* line, int at, int count) {
        return *reinterpret_cast<const u32x4_any*>(line + (at + PER <= count ? at : count - PER));
    }
    static __device__ __forceinline__ int late(int at, int count) {
        return at + PER <= count ? 0 : (at + PER - count) * int(sizeof(T));
    }
    // True where nothing of step r0 lies past an edge; the same in the whole
    // workgroup.  Those steps leave out the shifts and bounds.
    static __device__ __forceinline__ bool inside(const F8TurnArgs& p, int m0, int n0, int r0) {
        return r0 + 64 <= p.depth && n0 + 64 <= p.n && (!TRANS || m0 + 64 <= p.m);
    }

    // The thread's lines of G and q in the first step, bounded to the matrix's
    // rows where they are rows of the output.
    struct Lines {
        int64_t g[LOADS], q;
    };
    static __device__ __forceinline__ Lines lines(const F8TurnArgs& p, int m0, int n0) {
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

    static __device__ __forceinline__ void load(const F8TurnArgs& p, int m0, int n0, int r0, const Lines& l, Raw& x) {
        if (r0 >= p.depth) return;  // the step is past the sum
        const int t = threadIdx.x, last = p.depth - 1;
        const T* g = static_cast<const T*>(p.g);
        const int at = t % CHUNKS * PER, rq = r0 + t / 8 < last ? r0 + t / 8 : last;
        if (inside(p, m0, n0, r0)) {
            x.q = *reinterpret_cast<const u32x2_any*>(p.q + int64_t(r0) * p.ldq + l.q);
            const T* from = g + (TRANS ? int64_t(r0) * p.ldg : r0);
#pragma unroll
            for (int i = 0; i < LOADS; ++i) x.g[i] = *reinterpret_cast<const u32x4_any*>(from + l.g[i]);
        } else {
            const int cq = n0 + t % 8 * 8;
            x.q = *reinterpret_cast<const u32x2_any*>(p.q + int64_t(rq) * p.ldq + (cq + 8 <= p.n ? cq : p.n - 8));
#pragma unroll
            for (int i = 0; i < LOADS; ++i) {
                const int line = t / CHUNKS + i * LINES;
                if constexpr (TRANS) x.g[i] = get(g + int64_t(r0 + line < last ? r0 + line : last) * p.ldg, m0 + at, p.m);
                else x.g[i] = get(g + (l.g[i] - at), r0 + at, p.depth);
            }
        }
        // A tile's 64 columns lie in one block of 128.
        x.s = p.scale.p[int64_t(rq >> p.shift) * p.scale.row + int64_t(n0 / kF8Block) * p.scale.col];
    }

    // Writes step r0's operands to LDS.
    static __device__ __forceinline__ void put(const F8TurnArgs& p, int m0, int n0, int r0, lds_t* stage, const Raw& x) {
        if (r0 >= p.depth) return;
        if (inside(p, m0, n0, r0)) put_step<true>(p, m0, n0, r0, stage, x);
        else put_step<false>(p, m0, n0, r0, stage, x);
    }
    template <bool INSIDE>
    static __device__ __forceinline__ void put_step(const F8TurnArgs& p, int m0, int n0, int r0, lds_t* stage, const Raw& x) {
        typedef bf16_t d8 __attribute__((ext_vector_type(8)));
        typedef bf16_t d_per __attribute__((ext_vector_type(PER)));
        typedef T t_per __attribute__((ext_vector_type(PER)));
        typedef std::conditional_t<PER == 8, u32x4, u32x2> words;
        typedef __attribute__((address_space(3))) words* put_t;
        const int t = threadIdx.x;
        {
            u32x2 w = x.q;
            float s = e8m0_to_f32(uint32_t(x.s));
            if constexpr (!INSIDE) {
                const int past = n0 + t % 8 * 8 + 8 - p.n;
                const uint64_t all = __builtin_bit_cast(uint64_t, w);
                w = __builtin_bit_cast(u32x2, past <= 0 ? all : past < 8 ? all >> past * 8 : 0);
                if (r0 + t / 8 >= p.depth) {
                    w = u32x2{0, 0};
                    s = 0.0f;
                }
            }
            float v[8];
            e4m3_unpack(w[0], v);
            e4m3_unpack(w[1], v + 4);
            d8 d;
#pragma unroll
            for (int i = 0; i < 8; ++i) d[i] = static_cast<bf16_t>(v[i] * s);
            *reinterpret_cast<put16_t>(stage + P * PLANE + t / 8 * ROW + t % 8 * 16) = __builtin_bit_cast(u32x4, d);
        }
        const int at = t % CHUNKS * PER;
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            const int line = t / CHUNKS + i * LINES;
            u32x4 w = x.g[i];
            if constexpr (!INSIDE) {
                w = shift_out(w, TRANS ? late(m0 + at, p.m) : late(r0 + at, p.depth));
                if (TRANS && r0 + line >= p.depth) w = u32x4{0, 0, 0, 0};
            }
            const int chunk = at / 8;
            lds_t* to = stage + (TRANS ? line * ROW + chunk * 16 : line * 128 + ((chunk ^ (line & 7)) << 4));
            if constexpr (P > 1) {
                const t_per f = __builtin_bit_cast(t_per, w);
                d_per d[P];
#pragma unroll
                for (int e = 0; e < PER; ++e) {
                    bf16_t part[P];
                    split_value<bf16_t, P>(to_f32(f[e]), part);
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
                if constexpr (TRANS) xa = turned(stage + k * PLANE, row, 4, h);
                else xa = *reinterpret_cast<frag_t>(stage + k * PLANE + (row + li) * 128 + (((lg + 4 * h) ^ (li & 7)) << 4));
#pragma unroll
                for (int j = 0; j < 2; ++j) acc[0][j] = mma<Mma::BF16>(xb[j], xa, acc[0][j]);
            }
        }
    }
};

template <typename T, bool TRANS>
__global__ __launch_bounds__(512) void tg_f8_turn(F8TurnArgs p, TileStore<T> out) {
    using Cfg = F8Turn<T, TRANS>;
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
    typename Cfg::Acc acc[1][2] = {};
    Cfg::put(p, m0, n0, 0, lds, x[0]);
    Cfg::load(p, m0, n0, AHEAD * 64, l, x[0]);
    __syncthreads();
    for (int s0 = 0; s0 < steps; s0 += AHEAD) {
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            const int s = s0 + i;
            if (s >= steps) break;
            Cfg::products(lds + i % 2 * Cfg::STAGE, acc);
            Cfg::put(p, m0, n0, (s + 1) * 64, lds + (i + 1) % 2 * Cfg::STAGE, x[(i + 1) % AHEAD]);
            Cfg::load(p, m0, n0, (s + 1 + AHEAD) * 64, l, x[(i + 1) % AHEAD]);
            __syncthreads();
        }
    }
    typename Cfg::Shape::template Beside<TileStore<T>> beside;
    Cfg::Shape::beside(tile, tm, tn, out, beside);
    Cfg::Shape::outputs(tile, tm, tn, acc, out, beside);
}

}  // namespace tg
