// tg_f8_gemm.hip -- launches of the products in 8-bit floating point: rows times
// rows with a power of two for each block, and the two gradients, which read one
// 8-bit operand.
#include <atomic>

#include "../../include/tropical_gemm_hip.h"
#include "tg_f8.hpp"
#include "tg_f8_pack.hpp"
#include "tg_f8_stream.hpp"
#include "tg_f8_tiles.hpp"
#include "tg_f8_turn.hpp"
#include "tg_i8.hpp"

namespace tg {
namespace {

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
int64_t round_up(int64_t a, int64_t b) { return ceil_div(a, b) * b; }

template <typename F>
hipError_t by_type(int type, F&& f) {
    switch (type) {
        case TG_BF16: return f(bf16_t());
        case TG_F16: return f(f16_t());
        default: return f(float());
    }
}

// ---- choice of a tile ----------------------------------------------------

// A tile's sizes, workgroups per CU, halves of its waves that share the sum, and
// its time in us: `start` + step for each block of the sum while every workgroup
// has a CU of its own (`crowd` more as the last CUs fill), otherwise rounds of
// `round` + full for each block.  Fitted to 132 products on MI355X (M 64 ... 8192,
// N 1024 ... 8192, K 256 ... 8192): the tile with the least time so reckoned is 0.6%
// slower than the best of them in the mean, 16% at most.  A last round that only
// some CUs have with several workgroups takes most of a whole one's time.
//
// A block costs a CU 64 bytes a clock at most on their way into LDS: 0.23 us for
// 128 x 128 outputs, 0.47 for 256 x 256, four times as many, where the matrix
// instructions take 0.95; so the tiles are as large as they can be with all CUs at
// work.
struct TileTime {
    int bm, bn, per_cu, halves;
    double start, step, crowd, round, full;
};
constexpr TileTime kTiles[] = {
    {256, 256, 1, 1, 11.93, 0.946, 0.558, 10.31, 1.322}, {128, 256, 1, 1, 8.13, 0.491, 0.308, 6.00, 0.728},
    {128, 128, 2, 1, 5.96, 0.345, 0.089, 3.72, 0.820},   {128, 64, 1, 2, 5.82, 0.205, 0.073, 3.63, 0.272},
    {64, 64, 3, 1, 3.74, 0.248, 0.023, 1.51, 0.513},     {64, 64, 1, 2, 3.99, 0.197, 0.025, 2.03, 0.207},
};
constexpr int kTileForms = sizeof(kTiles) / sizeof(kTiles[0]);

struct TilePlan {
    int form, slices;
    int64_t tiles_m, tiles_n, slice, steps;
};

double tile_time(const TileTime& c, int64_t tiles, int64_t steps) {
    const double alone = c.step + (tiles > 128 ? c.crowd * double((tiles < 256 ? tiles : 256) - 128) / 128 : 0);
    if (tiles <= 256) return c.start + double(steps) * alone;
    const int64_t slots = 256 * int64_t(c.per_cu), whole = tiles / slots;
    const double last = double(tiles - whole * slots) / double(slots), depth = last * c.per_cu;
    double t = 3 + double(whole) * (c.round + double(steps) * c.full);
    if (last > 0 && c.per_cu > 1)
        t += c.round + double(steps) * (depth <= 1 ? alone : alone + (c.full - alone) * (0.6 + 0.4 * (depth - 1) / (c.per_cu - 1)));
    else if (last > 0)
        t += c.round + double(steps) * c.full * (0.75 + 0.25 * last);
    return t;
}

TilePlan plan_tiles(int64_t m, int64_t n, int64_t steps) {
    if (m <= 0 || n <= 0 || steps <= 0) return {0, 1, 0, 0, 1, 0};  // no tile, no slice of the sum
    TilePlan best = {0, 1, ceil_div(m, 256), ceil_div(n, 256), steps, steps};
    double least = 1e30;
    for (int f = 0; f < kTileForms; ++f) {
        const TileTime& c = kTiles[f];
        const int64_t tm = ceil_div(m, c.bm), tn = ceil_div(n, c.bn);
        if (tm * tn >= int64_t(1) << 23) continue;  // a launch's thread count stays below 2^32
        for (int s = 1; s <= 32; s *= 2) {
            const int64_t slice = ceil_div(steps, s), slices = ceil_div(steps, slice);
            if (s > 1 && (tm * tn * s > 512 || slice < 4)) break;
            if (steps - (slices - 1) * slice < c.halves) continue;  // a step for each half
            double t = tile_time(c, tm * tn * s, slice);
            // Partial sums' way through memory and the launch that joins them.
            if (s > 1) t += 4.5 + double(s + 1) * double(m) * double(n) * 4 / 4e6;
            if (t < least) {
                least = t;
                best = {f, int(slices), tm, tn, slice, steps};
            }
        }
    }
    return best;
}

std::string tiles_name(const TilePlan& pl) {
    const TileTime& c = kTiles[pl.form];
    std::string name = "tiles " + std::to_string(c.bm) + "x" + std::to_string(c.bn);
    if (c.halves > 1) name += " halves";
    if (pl.slices > 1) name += " slices " + std::to_string(pl.slices);
    return name;
}

size_t part_bytes(const TilePlan& pl, int64_t m, int64_t n) {
    return pl.slices > 1 ? size_t(pl.slices) * size_t(m) * size_t(round_up(n, 8)) * 4 : 0;
}

// Lets a kernel have `bytes` of LDS on the current device; `done` keeps for which it
// was asked before.
template <typename K>
hipError_t allow_lds(K* kernel, int bytes, std::atomic<uint64_t>& done) {
    int device = 0;
    const hipError_t found = hipGetDevice(&device);
    if (found != hipSuccess) return found;
    const uint64_t bit = device < 64 ? uint64_t(1) << device : 0;
    if ((done.load(std::memory_order_relaxed) & bit) != 0) return hipSuccess;
    const hipError_t e =
        hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == hipSuccess) done.fetch_or(bit, std::memory_order_relaxed);
    return e;
}

unsigned stride_grid(int64_t items) {
    const int64_t blocks = ceil_div(items, 256);
    return unsigned(blocks < 65536 ? blocks : 65536);
}

template <typename A, typename B>
hipError_t launch_pack(const A& a, const B& b, hipStream_t st) {
    const int64_t na = a.blocks(), nb = b.blocks();
    if (na + nb >= int64_t(1) << 24) return hipErrorInvalidConfiguration;
    hipLaunchKernelGGL((tg_i8_pack<A, B>), dim3(unsigned(na + nb)), dim3(256), 0, st, a, b, int(na), int(nb));
    return hipGetLastError();
}

template <typename T>
hipError_t launch_join(const float* part, int slices, int64_t m, int64_t n, const TileStore<T>& out, hipStream_t st) {
    const int64_t ld = round_up(n, 8);
    hipLaunchKernelGGL((tg_i8_tiles_join<float, T>), dim3(stride_grid(m * ld / 8)), dim3(256), 0, st, part, ld, slices, m,
                       n, out);
    return hipGetLastError();
}

template <int WM, int WN, int FM, int FN, int NB, int KS, int PER_CU, typename T>
hipError_t launch_form(F8TileArgs p, const TilePlan& pl, const TileStore<T>& out, void* part, hipStream_t st) {
    using Cfg = F8Tile<WM, WN, FM, FN, NB, KS>;
    const dim3 grid(unsigned(pl.tiles_m * pl.tiles_n), unsigned(pl.slices));
    if (pl.slices == 1) {
        const auto kernel = &tg_f8_tiles<WM, WN, FM, FN, NB, KS, PER_CU, T>;
        static std::atomic<uint64_t> allowed{0};
        const hipError_t attr = allow_lds(kernel, Cfg::LDS, allowed);
        if (attr != hipSuccess) return attr;
        hipLaunchKernelGGL(kernel, grid, dim3(Cfg::THREADS), Cfg::LDS, st, p, F8Store<T>{out.bias, out.c, out.n});
        return hipGetLastError();
    }
    const auto kernel = &tg_f8_tiles_slice<WM, WN, FM, FN, NB, KS, PER_CU>;
    static std::atomic<uint64_t> allowed{0};
    const hipError_t attr = allow_lds(kernel, Cfg::LDS, allowed);
    if (attr != hipSuccess) return attr;
    float* sums = static_cast<float*>(part);
    hipLaunchKernelGGL(kernel, grid, dim3(Cfg::THREADS), Cfg::LDS, st, p, F8Partial{sums, round_up(p.n, 8)});
    const hipError_t e = hipGetLastError();
    return e != hipSuccess ? e : launch_join(sums, pl.slices, p.m, p.n, out, st);
}

template <typename T>
hipError_t launch_tiles(F8TileArgs p, const TilePlan& pl, const TileStore<T>& out, void* part, hipStream_t st) {
    p.tiles_m = int(pl.tiles_m);
    p.tiles_n = int(pl.tiles_n);
    p.slice = int(pl.slice);
    p.steps = int(pl.steps);
    switch (pl.form) {
        case 0: return launch_form<2, 2, 4, 4, 2, 1, 1>(p, pl, out, part, st);
        case 1: return launch_form<2, 2, 2, 4, 2, 1, 1>(p, pl, out, part, st);
        case 2: return launch_form<2, 2, 2, 2, 2, 1, 2>(p, pl, out, part, st);
        case 3: return launch_form<2, 1, 2, 2, 2, 2, 1>(p, pl, out, part, st);
        case 4: return launch_form<2, 2, 1, 1, 3, 1, 3>(p, pl, out, part, st);
        default: return launch_form<2, 2, 1, 1, 3, 2, 1>(p, pl, out, part, st);
    }
}

// True when the tiles can read rows of `bytes` bytes in place.
bool in_place(const void* p, int64_t ld_bytes, int64_t bytes) {
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld_bytes % 16 == 0 && ld_bytes < (int64_t(1) << 23) && bytes % 16 == 0;
}

// Carves 256-byte aligned parts out of a workspace.
struct Carver {
    char* at;
    size_t used = 0;
    void* take(size_t bytes) {
        void* p = at == nullptr ? nullptr : at + used;
        used += (bytes + 255) / 256 * 256;
        return p;
    }
};

// ---- the product ---------------------------------------------------------

// Rows of A that tg_f8_stream takes (in sixteens; 0: the tiles take the
// product): B is read once and needs no layout, but every 16 rows of B read all
// of A, so more rows than 16 only where B is small or would have to be laid out
// first, which for f32 outputs it always has.  Up to 16 rows always, though for many
// columns the tiles take a tenth less.  us, cold weights, tg_f8_stream and the tiles,
// M x N x K:
//     bf16   16 x  4096 x 4096    6.7  11.3     16 x 16384 x 4096   17.9  16.3
//            32 x  4096 x 8192   12.8  14.1     32 x  8192 x 8192   23.3  20.4
//            48 x  8192 x 4096   14.9  15.0     48 x  8192 x 8192   25.8  26.8
//            64 x  4096 x 4096   10.3  13.2     64 x  4096 x 8192   16.6  15.0
// unaligned  48 x 16384 x 8191   68.7  75.1     64 x 16384 x 8191   80.9  75.8
//     f32    64 x  1024 x 4096    8.7  17.0     64 x 16384 x 8192   58.8   131
int stream_rows(const F8Gemm& p) {
    // A launch's thread count stays below 2^32: 1024 threads for 16 columns.
    if (p.m > 64 || p.n > (int64_t(1) << 26) - 16) return 0;
    const int rows = int(round_up(p.m, 16));
    if (rows <= 16 || p.type == TG_FLOAT32) return rows;
    if (!in_place(p.a, p.lda, p.k) || !in_place(p.b, p.ldb, p.k)) return rows <= 48 || p.n <= 8192 ? rows : 0;
    return double(p.n) * double(p.k) <= (rows <= 48 ? 1 << 25 : 1 << 24) ? rows : 0;
}

struct GemmPlan {
    int stream;  // rows of A of tg_f8_stream
    bool wide;   // f32: both operands laid out in bf16
    bool pack_a, pack_b;
    int64_t ld;  // of packed rows, in bytes
    TilePlan tiles;
};

GemmPlan plan_gemm(const F8Gemm& p) {
    GemmPlan pl{};
    pl.stream = stream_rows(p);
    if (pl.stream != 0) return pl;
    pl.wide = p.type == TG_FLOAT32;
    if (pl.wide) {
        pl.pack_a = pl.pack_b = true;
        pl.ld = round_up(p.k, 64) * 2;
        return pl;
    }
    pl.pack_a = !in_place(p.a, p.lda, p.k);
    pl.pack_b = !in_place(p.b, p.ldb, p.k);
    pl.ld = round_up(p.k, 128);
    pl.tiles = plan_tiles(p.m, p.n, ceil_div(p.k, 128));
    return pl;
}

struct GemmWs {
    uint8_t *a, *b;
    void* part;
    size_t bytes;
};

GemmWs carve_gemm(const F8Gemm& p, const GemmPlan& pl, void* ws) {
    Carver c{static_cast<char*>(ws)};
    GemmWs w{};
    if (p.m == 0 || p.n == 0 || p.k == 0 || pl.stream != 0) return w;
    if (pl.pack_a) w.a = static_cast<uint8_t*>(c.take(size_t(p.m) * size_t(pl.ld)));
    if (pl.pack_b) w.b = static_cast<uint8_t*>(c.take(size_t(p.n) * size_t(pl.ld)));
    w.part = c.take(pl.wide ? plane_gemm_ws(p.m, p.n, pl.ld / 128, 1) : part_bytes(pl.tiles, p.m, p.n));
    w.bytes = c.used;
    return w;
}

PackBytes bytes_job(const void* src, int64_t ld_src, int64_t rows, int64_t bytes, void* dst, int64_t ld) {
    return {static_cast<const int8_t*>(src), ld_src, rows, int(bytes), static_cast<int8_t*>(dst), ld};
}

// 32-bit aligned rows.
bool in_words(const F8Gemm& p) {
    auto words = [](const void* q, int64_t ld) { return reinterpret_cast<uintptr_t>(q) % 4 == 0 && ld % 4 == 0; };
    return words(p.a, p.lda) && words(p.b, p.ldb);
}

template <int R, int W, bool WORDS, typename T>
hipError_t launch_stream(const F8Gemm& p, const TileStore<T>& out, hipStream_t st) {
    const F8StreamArgs args{p.a, p.b, p.lda, p.ldb, p.a_scale.p, p.b_scale.p, p.a_scale.row, p.a_scale.col,
                            p.b_scale.row, p.b_scale.col, int(p.m), int(p.n), int(p.k)};
    hipLaunchKernelGGL((tg_f8_stream<R, W, WORDS, T>), dim3(unsigned(ceil_div(p.n, 16))), dim3(W * 64), 0, st, args, out);
    return hipGetLastError();
}

template <typename T>
hipError_t stream_typed(const F8Gemm& p, int rows, const TileStore<T>& out, hipStream_t st) {
    const bool words = in_words(p);
    switch (rows) {
        case 16: return words ? launch_stream<1, 16, true>(p, out, st) : launch_stream<1, 8, false>(p, out, st);
        case 32: return words ? launch_stream<2, 8, true>(p, out, st) : launch_stream<2, 8, false>(p, out, st);
        case 48: return words ? launch_stream<3, 8, true>(p, out, st) : launch_stream<3, 8, false>(p, out, st);
        default: return words ? launch_stream<4, 8, true>(p, out, st) : launch_stream<4, 8, false>(p, out, st);
    }
}

template <typename T>
hipError_t gemm_typed(const F8Gemm& p, void* ws, hipStream_t st) {
    const TileStore<T> out{nullptr, nullptr, nullptr, static_cast<const T*>(p.bias), static_cast<T*>(p.c), p.n};
    if (p.k == 0) return launch_join(nullptr, 0, p.m, p.n, out, st);
    const GemmPlan pl = plan_gemm(p);
    if (pl.stream != 0) return stream_typed(p, pl.stream, out, st);
    const GemmWs w = carve_gemm(p, pl, ws);
    if (pl.wide) {
        const hipError_t e = launch_pack(
            PackF8Rows{p.a, p.lda, p.m, p.k, p.a_scale, 0, reinterpret_cast<bf16_t*>(w.a), pl.ld / 2},
            PackF8Rows{p.b, p.ldb, p.n, p.k, p.b_scale, 7, reinterpret_cast<bf16_t*>(w.b), pl.ld / 2}, st);
        if (e != hipSuccess) return e;
        return plane_gemm(PlaneGemm{p.type, 1, w.a, w.b, pl.ld, pl.ld, pl.ld / 128, 128, p.bias, p.c, p.m, p.n}, w.part, st);
    }
    F8TileArgs t{};
    t.a = pl.pack_a ? w.a : p.a;
    t.b = pl.pack_b ? w.b : p.b;
    t.lda = pl.pack_a ? pl.ld : p.lda;
    t.ldb = pl.pack_b ? pl.ld : p.ldb;
    t.sa = p.a_scale.p, t.sa_row = p.a_scale.row, t.sa_col = p.a_scale.col;
    t.sb = p.b_scale.p, t.sb_row = p.b_scale.row, t.sb_col = p.b_scale.col;
    t.m = int(p.m);
    t.n = int(p.n);
    // A packed row is whole; beside one that is not, it only has to reach as far.
    t.tail = (pl.pack_a && pl.pack_b) || p.k % 128 == 0 ? 128 : int(round_up(p.k % 128, 16));
    if (pl.pack_a || pl.pack_b) {
        const PackBytes a = bytes_job(p.a, p.lda, pl.pack_a ? p.m : 0, p.k, w.a, pl.ld);
        const PackBytes b = bytes_job(p.b, p.ldb, pl.pack_b ? p.n : 0, p.k, w.b, pl.ld);
        const hipError_t e = launch_pack(a, b, st);
        if (e != hipSuccess) return e;
    }
    if constexpr (std::is_same<T, float>::value) return hipErrorInvalidValue;  // wide, above
    else return launch_tiles(t, pl.tiles, out, w.part, st);
}

// ---- gradients -----------------------------------------------------------
//
// Both are a product of G with the 8-bit operand q, whose rows run across the
// sum; q is turned so that they run along it, in bf16 with its scales multiplied
// in, which is exact.  G in bf16 is taken as it is, in f16 as two bf16 planes that
// add up to it (8 + 3 bits), in f32 as three (8 + 8 + 8): every product is exact,
// and the sums are f32.

// Time of tg_f8_turn in us, as plane_gemm_time gives it for the other way: a step
// takes the vector unit as long for each of a CU's tiles, and a wait of its own.
// Fitted to 232 gradients of each type (rows 64 ... 4096, columns 128 ... 2048, sums
// 64 ... 2049; 6% off in the root mean square).  Chosen with it, about half of them
// take one launch; the choices lose 0.1 us on the GPU in the mean (f32: 0.4).
double turn_time(const F8Grad& p) {
    const int64_t tiles = ceil_div(p.rows, 64) * ceil_div(p.cols, 64);
    if (tiles >= int64_t(1) << 23 || !turn_fits(p.transposed, p.rows, p.cols, p.depth)) return 1e30;
    // A CU holds `slots` tiles at a time; a last round takes at least one tile's time.
    const int64_t slots = p.type == TG_BF16 ? 4 : 2, rest = tiles % (256 * slots);
    const double last = rest > 256 ? double(rest) / 256 : rest > 0 ? 1 : 0;
    const double per_cu = double(tiles / (256 * slots) * slots) + last, steps = double(ceil_div(p.depth, 64));
    // Tiles at an edge take longer, and a round as long as they.
    const double edge = p.cols % 64 != 0 || (p.transposed && p.rows % 64 != 0) ? 1 : 0;
    if (p.type == TG_FLOAT32) return 1.9 + 1.46 * per_cu + steps * (0.33 + 0.61 * per_cu + 0.21 * edge);
    if (p.type == TG_F16) return 2.1 + 0.86 * per_cu + steps * (0.32 + 0.50 * per_cu + 0.15 * edge);
    return 2.4 + 0.66 * per_cu + steps * (0.21 + 0.32 * per_cu + 0.16 * edge);
}

// A launch that lays out rows: what it takes beside the bytes' way through memory,
// in us; and what one launch may take more than two where the GPU waits for the
// caller's thread.
constexpr double kPackTime = 2.5;
bool one_launch(double one, double two) { return one < two + (one < 12 ? 2 : 0); }

struct GradPlan {
    bool turn;  // one launch of tg_f8_turn
    bool pack_g;
    int planes, tail;
    int64_t depth, steps;  // of packed rows, in elements and in 128 bytes
};

GradPlan plan_grad(const F8Grad& p) {
    GradPlan pl{};
    pl.planes = p.type == TG_FLOAT32 ? 3 : p.type == TG_F16 ? 2 : 1;
    pl.pack_g = pl.planes > 1 || p.transposed || !in_place(p.g, p.ldg * 2, p.depth * 2);
    pl.depth = round_up(p.depth, 64);
    pl.steps = pl.depth / 64;
    pl.tail = pl.pack_g || p.depth % 64 == 0 ? 128 : int(p.depth % 64 * 2);
    const int64_t size = p.type == TG_FLOAT32 ? 4 : 2;
    const double bytes = double(pl.depth) * (3 * double(p.cols) + (pl.pack_g ? double(size + 2 * pl.planes) * double(p.rows) : 0));
    pl.turn = one_launch(turn_time(p), plane_gemm_time(p.rows, p.cols, pl.steps, pl.planes) + kPackTime + bytes / 4e6);
    return pl;
}

struct GradWs {
    void *g, *q, *part;
    size_t bytes;
};

GradWs carve_grad(const F8Grad& p, const GradPlan& pl, void* ws) {
    Carver c{static_cast<char*>(ws)};
    GradWs w{};
    if (p.rows == 0 || p.cols == 0 || p.depth == 0 || pl.turn) return w;
    if (pl.pack_g) w.g = c.take(size_t(p.rows) * size_t(pl.depth) * size_t(pl.planes) * 2);
    w.q = c.take(size_t(p.cols) * size_t(pl.depth) * 2);
    w.part = c.take(plane_gemm_ws(p.rows, p.cols, pl.steps, pl.planes));
    w.bytes = c.used;
    return w;
}

// Lays out q and, where it has to be, G in PLANES planes.
template <typename T, int PLANES>
hipError_t pack_grad(const F8Grad& p, const GradPlan& pl, const GradWs& w, hipStream_t st) {
    const T* g = static_cast<const T*>(p.g);
    bf16_t* to = static_cast<bf16_t*>(w.g);
    const PackF8Turned q{p.q.q, p.q.ld, p.depth, p.cols, p.q.scale, p.q.block_rows == 1 ? 0 : 7,
                         static_cast<bf16_t*>(w.q), pl.depth};
    if (!pl.pack_g) return launch_pack(q, PackNothing(), st);
    if (p.transposed)
        return launch_pack(q, PackTurned<T, bf16_t, PLANES>{g, p.ldg, p.depth, p.rows, nullptr, nullptr, to, pl.depth}, st);
    if constexpr (PLANES > 1)
        return launch_pack(q, PackPlanes<T, PLANES>{g, p.ldg, p.rows, p.depth, to, pl.depth}, st);
    else
        return launch_pack(q, bytes_job(p.g, p.ldg * 2, p.rows, p.depth * 2, w.g, pl.depth * 2), st);
}

template <typename T, bool TRANS>
hipError_t launch_turn(const F8Grad& p, hipStream_t st) {
    using Cfg = F8Turn<T, TRANS>;
    const auto kernel = &tg_f8_turn<T, TRANS>;
    static std::atomic<uint64_t> allowed{0};
    const hipError_t attr = allow_lds(kernel, Cfg::LDS, allowed);
    if (attr != hipSuccess) return attr;
    const F8TurnArgs args{p.g, p.ldg, p.q.q, p.q.ld, p.q.scale, p.q.block_rows == 1 ? 0 : 7, int(p.rows), int(p.cols),
                          int(p.depth), int(ceil_div(p.rows, 64)), int(ceil_div(p.cols, 64))};
    const TileStore<T> out{nullptr, nullptr, nullptr, nullptr, static_cast<T*>(p.out), p.cols};
    hipLaunchKernelGGL(kernel, dim3(unsigned(args.tiles_m * args.tiles_n)), dim3(Cfg::NT), Cfg::LDS, st, args, out);
    return hipGetLastError();
}

}  // namespace

std::string f8_gemm_plan(const F8Gemm& p) {
    if (p.m == 0 || p.n == 0) return "none";
    if (p.k == 0) return "bias";
    const GemmPlan pl = plan_gemm(p);
    if (pl.stream != 0) return "stream rows " + std::to_string(pl.stream) + (in_words(p) ? " words" : "");
    if (pl.wide) return "wide " + plane_gemm_plan(p.m, p.n, pl.ld / 128, 1);
    return tiles_name(pl.tiles) + (pl.pack_a ? " pack a" : "") + (pl.pack_b ? " pack b" : "");
}

std::string f8_grad_plan(const F8Grad& p) {
    if (p.rows == 0 || p.cols == 0) return "none";
    if (p.depth == 0) return "zero";
    const GradPlan pl = plan_grad(p);
    if (pl.turn) return "turn";
    return plane_gemm_plan(p.rows, p.cols, pl.steps, pl.planes) + (pl.pack_g ? " pack grad_c" : "");
}

size_t f8_gemm_ws(const F8Gemm& p) { return carve_gemm(p, plan_gemm(p), nullptr).bytes; }

hipError_t f8_gemm(const F8Gemm& p, void* ws, hipStream_t st) {
    if (p.m == 0 || p.n == 0) return hipSuccess;
    return by_type(p.type, [&](auto tag) { return gemm_typed<decltype(tag)>(p, ws, st); });
}

size_t f8_grad_ws(const F8Grad& p) { return carve_grad(p, plan_grad(p), nullptr).bytes; }

hipError_t f8_grad(const F8Grad& p, void* ws, hipStream_t st) {
    if (p.rows == 0 || p.cols == 0) return hipSuccess;
    if (p.depth == 0) return plane_gemm_zero(p.type, p.out, p.rows, p.cols, st);
    const GradPlan pl = plan_grad(p);
    if (pl.turn)
        return by_type(p.type, [&](auto tag) {
            using T = decltype(tag);
            return p.transposed ? launch_turn<T, true>(p, st) : launch_turn<T, false>(p, st);
        });
    const GradWs w = carve_grad(p, pl, ws);
    hipError_t e;
    switch (p.type) {
        case TG_BF16: e = pack_grad<bf16_t, 1>(p, pl, w, st); break;
        case TG_F16: e = pack_grad<f16_t, 2>(p, pl, w, st); break;
        default: e = pack_grad<float, 3>(p, pl, w, st);
    }
    if (e != hipSuccess) return e;
    const PlaneGemm t{p.type, pl.planes, pl.pack_g ? w.g : p.g, w.q, pl.pack_g ? pl.depth * pl.planes * 2 : p.ldg * 2,
                      pl.depth * 2, pl.steps, pl.tail, nullptr, p.out, p.rows, p.cols};
    return plane_gemm(t, w.part, st);
}

}  // namespace tg
