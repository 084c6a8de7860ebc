// tg_i8_gemm.hip -- launches of the 8-bit layer's products: rows times rows in
// 8-bit integers with scales, and the two gradients, which read one 8-bit
// operand.
#include <cstdio>

#include "../../include/tropical_gemm_hip.h"
#include "tg_i8.hpp"
#include "tg_i8_any.hpp"
#include "tg_i8_pack.hpp"
#include "tg_i8_stream.hpp"
#include "tg_i8_tiles.hpp"
#include "tg_i8_turn.hpp"

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

// A tile's sizes, workgroups per CU, and its time in us: `start` + step for
// each 128 bytes of the sum while every workgroup has a CU of its own (`crowd`
// more as the last CUs fill and share the way to memory), otherwise rounds of
// `round` + full for each 128 bytes.  Fitted to 275 products on MI355X (M 32
// ... 8192, N 512 ... 8192, K 512 ... 8192 bytes; 8-bit and bf16 alike, the time
// goes by bytes): the tile with the least time so reckoned is 0.25% slower
// than the best one in the mean, 18% at most.
//
// `planes`: a step takes that many planes of A (f32 gradients; fitted to 80
// products, outputs of four bytes among the time).
struct TileTime {
    int bm, bn, threads, per_cu, planes;
    double start, step, crowd, round, full;
};
constexpr TileTime kTiles[] = {
    {256, 256, 512, 1, 1, 7.67, 0.987, 0.659, 9.24, 1.359}, {128, 128, 512, 1, 1, 4.00, 0.336, 0.145, 2.31, 0.447},
    {128, 128, 256, 2, 1, 3.79, 0.417, 0.137, 3.10, 0.848}, {64, 128, 512, 2, 1, 3.16, 0.235, 0.065, 1.53, 0.547},
    {64, 64, 256, 2, 1, 2.78, 0.197, 0.022, 1.01, 0.336},   {32, 64, 256, 3, 1, 2.67, 0.176, 0.001, 0.74, 0.362},
    {64, 128, 512, 1, 3, 3.40, 0.396, 0.220, 3.00, 0.620},  {32, 64, 256, 2, 3, 2.90, 0.220, 0.010, 1.75, 0.458},
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
        t += c.round + double(steps) * (depth <= 1 ? alone : alone + (c.full - alone) * (depth - 1) / (c.per_cu - 1));
    else if (last > 0)
        t += c.round + double(steps) * c.full * (0.75 + 0.25 * last);
    return t;
}

// Tile and slices of the sum: slices where tiles are few, as long as the time
// they save outweighs their partial sums' way through memory and the launch
// that joins them (4.5 us and 4 TB/s; N = 256, K = 8192, M = 16: 9.8 us in
// slices, 13.9 without).
//
// A sum of `planes` planes is `steps` steps of a form that takes all planes in
// a step, or planes * steps of the largest form, one plane after another.
TilePlan plan_tiles(int64_t m, int64_t n, int64_t steps, int planes, double* time = nullptr) {
    if (m <= 0 || n <= 0 || steps <= 0) return {0, 1, 0, 0, 1, 0};
    TilePlan best = {0, 1, ceil_div(m, 256), ceil_div(n, 256), steps * planes, steps * planes};
    double least = 1e30;
    for (int f = 0; f < kTileForms; ++f) {
        const TileTime& c = kTiles[f];
        if (c.planes != planes && f != 0) continue;
        const int64_t tm = ceil_div(m, c.bm), tn = ceil_div(n, c.bn), all = c.planes == planes ? steps : steps * planes;
        // A launch's thread count stays below 2^32.
        if (tm * tn >= (int64_t(1) << 32) / c.threads) continue;
        for (int s = 1; s <= 32; s *= 2) {
            const int64_t slice = ceil_div(all, s);
            if (s > 1 && (tm * tn * s > 512 || slice < 4)) break;
            double t = tile_time(c, tm * tn * s, slice);
            if (s > 1) t += 4.5 + double(s + 1) * double(m) * double(n) * 4 / 4e6;
            if (t < least) {
                least = t;
                best = {f, int(ceil_div(all, slice)), tm, tn, slice, all};
            }
        }
    }
    if (time != nullptr) *time = least;
    return best;
}

size_t part_bytes(const TilePlan& pl, int64_t m, int64_t n) {
    return pl.slices > 1 ? size_t(pl.slices) * size_t(m) * size_t(round_up(n, 8)) * 4 : 0;
}

template <typename K>
hipError_t allow_lds(K* kernel, int bytes) {
    return hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
}

unsigned stride_grid(int64_t items) {
    const int64_t blocks = ceil_div(items, 256);
    return unsigned(blocks < 65536 ? blocks : 65536);
}

// Both jobs in one launch: what the second one's own launch would cost (2.5 us)
// is more than most small operands take.
template <typename A, typename B>
hipError_t launch_pack(const A& a, const B& b, hipStream_t st) {
    const int64_t na = a.blocks(), nb = b.blocks();
    if (na + nb >= int64_t(1) << 24) return hipErrorInvalidConfiguration;
    hipLaunchKernelGGL((tg_i8_pack<A, B>), dim3(unsigned(na + nb)), dim3(256), 0, st, a, b, int(na), int(nb));
    return hipGetLastError();
}

template <typename V, typename T>
hipError_t launch_join(const V* part, int slices, int64_t m, int64_t n, const TileStore<T>& out, hipStream_t st) {
    const int64_t ld = round_up(n, 8);
    hipLaunchKernelGGL((tg_i8_tiles_join<V, T>), dim3(stride_grid(m * ld / 8)), dim3(256), 0, st, part, ld, slices, m,
                       n, out);
    return hipGetLastError();
}

template <Mma KIND, int WM, int WN, int FM, int FN, int NB, int PER_CU, int P = 1, typename T>
hipError_t launch_form(TileArgs p, const TilePlan& pl, const TileStore<T>& out, void* part, hipStream_t st) {
    using Cfg = Tile<KIND, WM, WN, FM, FN, NB, P>;
    const dim3 grid(unsigned(pl.tiles_m * pl.tiles_n), unsigned(pl.slices));
    if (pl.slices == 1) {
        const auto kernel = &tg_i8_tiles<KIND, WM, WN, FM, FN, NB, P, PER_CU, T>;
        static const hipError_t attr = allow_lds(kernel, Cfg::LDS);
        if (attr != hipSuccess) return attr;
        hipLaunchKernelGGL(kernel, grid, dim3(Cfg::NT), Cfg::LDS, st, p, out);
        return hipGetLastError();
    }
    const auto kernel = &tg_i8_tiles_slice<KIND, WM, WN, FM, FN, NB, P, PER_CU>;
    static const hipError_t attr = allow_lds(kernel, Cfg::LDS);
    if (attr != hipSuccess) return attr;
    auto* sums = static_cast<typename Cfg::Value*>(part);
    hipLaunchKernelGGL(kernel, grid, dim3(Cfg::NT), Cfg::LDS, st, p, TilePartial<typename Cfg::Value>{sums, round_up(p.n, 8)});
    const hipError_t e = hipGetLastError();
    return e != hipSuccess ? e : launch_join(sums, pl.slices, p.m, p.n, out, st);
}

template <Mma KIND, typename T>
hipError_t launch_tiles(TileArgs p, const TilePlan& pl, const TileStore<T>& out, void* part, hipStream_t st) {
    p.tiles_m = int(pl.tiles_m);
    p.tiles_n = int(pl.tiles_n);
    p.slice = int(pl.slice);
    p.steps = int(pl.steps);
    if constexpr (KIND == Mma::BF16 && std::is_same<T, float>::value) {
        if (pl.form == 6) return launch_form<KIND, 2, 4, 2, 2, 2, 1, 3>(p, pl, out, part, st);
        if (pl.form == 7) return launch_form<KIND, 2, 2, 1, 2, 3, 2, 3>(p, pl, out, part, st);
    }
    switch (pl.form) {
        case 0: return launch_form<KIND, 2, 4, 8, 4, 2, 1>(p, pl, out, part, st);
        case 1: return launch_form<KIND, 2, 4, 4, 2, 4, 1>(p, pl, out, part, st);
        case 2: return launch_form<KIND, 2, 2, 4, 4, 2, 2>(p, pl, out, part, st);
        case 3: return launch_form<KIND, 2, 4, 2, 2, 3, 2>(p, pl, out, part, st);
        case 4: return launch_form<KIND, 2, 2, 2, 2, 3, 2>(p, pl, out, part, st);
        default: return launch_form<KIND, 2, 2, 1, 2, 4, 3>(p, pl, out, part, st);
    }
}

// True when tg_i8_tiles can read rows of `bytes` bytes in place.
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

// ---- the 8-bit product ---------------------------------------------------

// Rows of A that tg_i8_stream takes (in sixteens; 0: others take the product):
// B is read once and needs no layout, but every 16 rows of B read all of A, so
// more rows than 16 only where B is narrow or would have to be laid out first.
// us, cold weights, tg_i8_stream and the best other way, M x N x K:
//     16 x 4096 x 4096    6.6   10.7     16 x 28672 x 8192  47.2   44.7
//     32 x 4096 x 4096    7.2   10.9     32 x  8192 x 8192  19.8   19.5
//                                        32 x 16384 x 4096  19.9   16.3
// and unaligned
//     32 x 1024 x 8191    9.7   35.7     32 x 16384 x 4095  27.7   26.9
//     64 x 1024 x 8191   15.2   35.2     64 x  8192 x 8191  39.4   45.6
//     64 x 4096 x 4095   12.8   24.6     64 x 16384 x 4095  40.9   26.8
int stream_rows(const I8Gemm& p) {
    // A launch's thread count stays below 2^32: 1024 threads for 16 columns.
    if (p.m > 64 || p.n > (int64_t(1) << 26) - 16) return 0;
    if (p.m <= 16) return 16;
    const bool ready = in_place(p.a, p.lda, p.k) && in_place(p.b, p.ldb, p.k);
    if (p.m <= 32) return p.n <= 8192 || !ready ? 32 : 0;
    return p.n <= 8192 && !ready ? int(round_up(p.m, 16)) : 0;
}

struct GemmPlan {
    int stream;  // rows of A of tg_i8_stream
    bool any, pack_a, pack_b;
    int64_t ld;  // of packed rows
    TilePlan tiles;
};

// A launch that lays out rows: what it takes beside the bytes' way through
// memory, in us.
constexpr double kPackTime = 2.5;
// One launch of `one` us instead of two of `two`: it may take 2 us more where the
// GPU waits for the caller's thread, which spends 13 us on two launches and a
// workspace, 9 on one.
bool one_launch(double one, double two) { return one < two + (one < 12 ? 2 : 0); }

// Time of tg_i8_any in us, as tile_time gives it for the others.  Measured on
// 96 products of odd sizes (M 32 ... 8192, N 65 ... 4097, K 129 ... 8191): the
// way taken with it is at most 3 us slower than the other one but for more
// than 1000 tiles of one or two steps (19 us, or 26 as it is chosen).  Longer
// sums than 4096 are always laid out first (M = 64, N = 4097, K = 8191: 25 us
// against 35).
double any_time(const I8Gemm& p) {
    const int64_t tiles = ceil_div(p.m, 64) * ceil_div(p.n, 64);
    if (tiles >= int64_t(1) << 24 || p.k < 16 || p.k > 4096) return 1e30;
    const double per_cu = double(tiles) / 256, step = 0.48 * per_cu;
    return 4.0 + per_cu + double(ceil_div(p.k, 128)) * (step > 0.37 ? step : 0.37);
}

GemmPlan plan_gemm(const I8Gemm& p) {
    GemmPlan pl{};
    pl.stream = stream_rows(p);
    if (pl.stream != 0) return pl;
    pl.pack_a = !in_place(p.a, p.lda, p.k);
    pl.pack_b = !in_place(p.b, p.ldb, p.k);
    pl.ld = round_up(p.k, 128);
    double time = 0;
    pl.tiles = plan_tiles(p.m, p.n, ceil_div(p.k, 128), 1, &time);
    if (pl.pack_a || pl.pack_b) {
        const double bytes = 2 * double(pl.ld) * (double(p.m) * pl.pack_a + double(p.n) * pl.pack_b);
        pl.any = one_launch(any_time(p), time + kPackTime + bytes / 4e6);
    }
    return pl;
}

struct GemmWs {
    int8_t *a, *b;
    void* part;
    size_t bytes;
};

GemmWs carve_gemm(const I8Gemm& p, const GemmPlan& pl, void* ws) {
    Carver c{static_cast<char*>(ws)};
    GemmWs w{};
    if (p.m == 0 || p.n == 0 || p.k == 0 || pl.stream != 0 || pl.any) return w;
    if (pl.pack_a) w.a = static_cast<int8_t*>(c.take(size_t(p.m) * size_t(pl.ld)));
    if (pl.pack_b) w.b = static_cast<int8_t*>(c.take(size_t(p.n) * size_t(pl.ld)));
    w.part = c.take(part_bytes(pl.tiles, p.m, p.n));
    w.bytes = c.used;
    return w;
}

PackBytes bytes_job(const void* src, int64_t ld_src, int64_t rows, int64_t bytes, void* dst, int64_t ld) {
    return {static_cast<const int8_t*>(src), ld_src, rows, int(bytes), static_cast<int8_t*>(dst), ld};
}

// 32-bit aligned rows.
bool in_words(const I8Gemm& p) {
    auto words = [](const void* q, int64_t ld) { return reinterpret_cast<uintptr_t>(q) % 4 == 0 && ld % 4 == 0; };
    return words(p.a, p.lda) && words(p.b, p.ldb);
}

template <int R, int W, bool WORDS, typename T>
hipError_t launch_stream(const I8Gemm& p, const TileStore<T>& out, hipStream_t st) {
    const StreamArgs args{p.a, p.lda, p.b, p.ldb, int(p.m), int(p.n), int(p.k)};
    hipLaunchKernelGGL((tg_i8_stream<R, W, WORDS, T>), dim3(unsigned(ceil_div(p.n, 16))), dim3(W * 64), 0, st, args, out);
    return hipGetLastError();
}

// Eight waves of a workgroup; 16 for a few aligned rows (M = 1, cold weights, N
// x K: 8192 x 8192 14.6 us and 15.1 with 8, 4096 x 4096 6.1 and 6.5; unaligned
// 8192 x 8191 14.5 and 14.0).  Beyond 32 rows the way for any address serves
// all.
template <typename T>
hipError_t stream_typed(const I8Gemm& p, int rows, const TileStore<T>& out, hipStream_t st) {
    const bool words = in_words(p);
    switch (rows) {
        case 16: return words ? launch_stream<1, 16, true>(p, out, st) : launch_stream<1, 8, false>(p, out, st);
        case 32: return words ? launch_stream<2, 8, true>(p, out, st) : launch_stream<2, 8, false>(p, out, st);
        case 48: return launch_stream<3, 8, false>(p, out, st);
        default: return launch_stream<4, 8, false>(p, out, st);
    }
}

template <typename T>
hipError_t gemm_typed(const I8Gemm& p, void* ws, hipStream_t st) {
    const TileStore<T> out{p.a_scale, p.b_scale, nullptr, static_cast<const T*>(p.bias), static_cast<T*>(p.c), p.n};
    if (p.k == 0) return launch_join<int32_t>(nullptr, 0, p.m, p.n, out, st);
    const GemmPlan pl = plan_gemm(p);
    if (pl.stream != 0) return stream_typed(p, pl.stream, out, st);
    if (pl.any) {
        const AnyArgs args{p.a, p.lda, p.b, p.ldb, int(p.m), int(p.n), int(p.k), int(ceil_div(p.m, 64)), int(ceil_div(p.n, 64))};
        hipLaunchKernelGGL((tg_i8_any<T>), dim3(unsigned(args.tiles_m * args.tiles_n)), dim3(256), 0, st, args, out);
        return hipGetLastError();
    }
    const GemmWs w = carve_gemm(p, pl, ws);
    TileArgs t{};
    t.a = reinterpret_cast<const char*>(pl.pack_a ? w.a : p.a);
    t.b = reinterpret_cast<const char*>(pl.pack_b ? w.b : p.b);
    t.lda = pl.pack_a ? pl.ld : p.lda;
    t.ldb = pl.pack_b ? pl.ld : p.ldb;
    t.m = int(p.m);
    t.n = int(p.n);
    t.b_steps = int(ceil_div(p.k, 128));
    // A packed row is whole; beside one that is not, it only has to reach as far.
    t.tail = (pl.pack_a && pl.pack_b) || p.k % 128 == 0 ? 128 : int(round_up(p.k % 128, 16));
    if (pl.pack_a || pl.pack_b) {
        const PackBytes a = bytes_job(p.a, p.lda, pl.pack_a ? p.m : 0, p.k, w.a, pl.ld);
        const PackBytes b = bytes_job(p.b, p.ldb, pl.pack_b ? p.n : 0, p.k, w.b, pl.ld);
        const hipError_t e = launch_pack(a, b, st);
        if (e != hipSuccess) return e;
    }
    return launch_tiles<Mma::I8>(t, pl.tiles, out, w.part, st);
}

// ---- gradients -----------------------------------------------------------
//
// Both are a product of G with the 8-bit operand q, whose rows run across the
// sum; q is turned so that they run along it, in 16 bits, with its scales
// multiplied in.  bf16 gradients: q * scale rounded to bf16 (as dequantizing
// the operand to bf16 does; the result's error is that of its own rounding
// times sqrt 2).  f16: q * scale * 2^e rounded to f16, or G * scale as two bf16
// planes where the scales' range is too wide for that (known on the GPU alone:
// ScaleRange).  f32: q is exact in bf16; G * scale, rounded to f32, becomes three
// bf16 planes that hold all its 24 bits, each multiplied with q.

struct GradPlan {
    bool turn;  // one launch of tg_i8_turn
    bool pack_g;
    int planes;
    int64_t depth;  // of packed rows, in elements
    TilePlan tiles;
};

// Time of tg_i8_turn in us, as tile_time gives it for the others: a step takes
// the vector unit as long for each of a CU's tiles, and a little longer where
// they share it.  Fitted to 576 gradients (rows and columns 65 ... 4096, sums 64
// ... 2049; 13% off in the root mean square).  Chosen with it, 64% of those in
// 16 bits take one launch and 3.3 us less in the mean, half of those in f32 1.3
// us less; the worst choices lose 3 us (f32: 7 of 23, 1024 terms for a few columns).
double turn_time(const I8Grad& p) {
    const int64_t tiles = ceil_div(p.rows, 64) * ceil_div(p.cols, 64);
    if (tiles >= int64_t(1) << 23 || !turn_fits(p.transposed, p.rows, p.cols, p.depth)) return 1e30;
    // A CU holds `slots` tiles at a time; a last round takes at least one tile's time.
    const int64_t slots = p.type == TG_FLOAT32 ? 2 : 4, rest = tiles % (256 * slots);
    const double last = rest > 256 ? double(rest) / 256 : rest > 0 ? 1 : 0;
    const double per_cu = double(tiles / (256 * slots) * slots) + last, steps = double(ceil_div(p.depth, 64));
    if (p.type == TG_FLOAT32) return 3.0 + 0.38 * per_cu + steps * (1.04 * per_cu + (tiles > 256 ? 0.35 : 0));
    return 3.45 + 0.11 * per_cu + steps * (0.49 * per_cu + (tiles > 256 ? 0.18 : 0));
}

GradPlan plan_grad(const I8Grad& p) {
    GradPlan pl{};
    const int64_t size = p.type == TG_FLOAT32 ? 4 : 2;
    pl.planes = p.type == TG_FLOAT32 ? 3 : 1;
    pl.pack_g = p.type == TG_FLOAT32 || p.transposed || !in_place(p.g, p.ldg * size, p.depth * size);
    pl.depth = round_up(p.depth, 64);
    double time = 0;
    pl.tiles = plan_tiles(p.rows, p.cols, pl.depth / 64, pl.planes, &time);
    const double bytes = double(pl.depth) * (3 * double(p.cols) + (pl.pack_g ? double(size + 2 * pl.planes) * double(p.rows) : 0));
    const int launches = p.type == TG_F16 ? 2 : 1;  // before the tiles'
    pl.turn = one_launch(turn_time(p), time + kPackTime * launches + bytes / 4e6);
    return pl;
}

struct GradWs {
    void *g, *q, *part;
    ScaleRange* range;
    size_t bytes;
};

GradWs carve_grad(const I8Grad& p, const GradPlan& pl, void* ws) {
    Carver c{static_cast<char*>(ws)};
    GradWs w{};
    if (p.rows == 0 || p.cols == 0 || p.depth == 0 || pl.turn) return w;
    const int planes = p.type == TG_F16 ? 2 : pl.planes;  // f16: in case the range is wide
    if (pl.pack_g || planes > 1) w.g = c.take(size_t(p.rows) * size_t(pl.depth) * size_t(planes) * 2);
    w.q = c.take(size_t(p.cols) * size_t(pl.depth) * 2);
    if (p.type == TG_F16) w.range = static_cast<ScaleRange*>(c.take(sizeof(ScaleRange)));
    w.part = c.take(part_bytes(pl.tiles, p.rows, p.cols));
    w.bytes = c.used;
    return w;
}

template <typename T, bool TRANS>
hipError_t launch_turn(const I8Grad& p, const TileStore<T>& out, hipStream_t st) {
    using Cfg = Turn<T, TRANS>;
    const auto kernel = &tg_i8_turn<T, TRANS>;
    static const hipError_t attr = allow_lds(kernel, Cfg::LDS);
    if (attr != hipSuccess) return attr;
    const TurnArgs args{p.g, p.ldg, p.q, p.ldq, p.scale, int(p.rows), int(p.cols), int(p.depth),
                        int(ceil_div(p.rows, 64)), int(ceil_div(p.cols, 64))};
    hipLaunchKernelGGL(kernel, dim3(unsigned(args.tiles_m * args.tiles_n)), dim3(Cfg::NT), Cfg::LDS, st, args, out);
    return hipGetLastError();
}

// Lays out q in `D` and, where it has to be, G in PLANES planes of D.
template <typename T, typename D, int PLANES>
hipError_t pack_grad(const I8Grad& p, const GradPlan& pl, const GradWs& w, hipStream_t st) {
    const T* g = static_cast<const T*>(p.g);
    const float* scale_g = PLANES > 1 ? p.scale : nullptr;  // the scales go with one operand
    const PackTurned<int8_t, D, 1> q{p.q, p.ldq, p.depth, p.cols, PLANES > 1 ? nullptr : p.scale, nullptr, static_cast<D*>(w.q), pl.depth};
    if (!pl.pack_g) return launch_pack(q, PackNothing(), st);
    if (p.transposed)
        return launch_pack(q, PackTurned<T, D, PLANES>{g, p.ldg, p.depth, p.rows, scale_g, nullptr, static_cast<D*>(w.g), pl.depth}, st);
    if constexpr (PLANES > 1)
        return launch_pack(q, PackSplit<T, PLANES>{g, p.ldg, p.rows, p.depth, p.scale, static_cast<D*>(w.g), pl.depth}, st);
    else
        return launch_pack(q, bytes_job(p.g, p.ldg * 2, p.rows, p.depth * 2, w.g, pl.depth * 2), st);
}

// f16: one way or the other by the scales' range.
hipError_t pack_grad_f16(const I8Grad& p, const GradPlan& pl, const GradWs& w, hipStream_t st) {
    const f16_t* g = static_cast<const f16_t*>(p.g);
    bf16_t* wide_g = static_cast<bf16_t*>(w.g);
    using Narrow = PackTurned<int8_t, f16_t, 1>;
    using Wide = PackTurned<int8_t, bf16_t, 1>;
    const PackEither<Narrow, Wide> q{
        Narrow{p.q, p.ldq, p.depth, p.cols, p.scale, &w.range->factor, static_cast<f16_t*>(w.q), pl.depth},
        Wide{p.q, p.ldq, p.depth, p.cols, nullptr, nullptr, static_cast<bf16_t*>(w.q), pl.depth}, w.range};
    if (pl.pack_g && p.transposed) {
        using NarrowG = PackTurned<f16_t, f16_t, 1>;
        using WideG = PackTurned<f16_t, bf16_t, 2>;
        return launch_pack(q,
                           PackEither<NarrowG, WideG>{
                               NarrowG{g, p.ldg, p.depth, p.rows, nullptr, nullptr, static_cast<f16_t*>(w.g), pl.depth},
                               WideG{g, p.ldg, p.depth, p.rows, p.scale, nullptr, wide_g, pl.depth}, w.range},
                           st);
    }
    const PackSplit<f16_t, 2> wide{g, p.ldg, p.rows, p.depth, p.scale, wide_g, pl.depth};
    if (!pl.pack_g) return launch_pack(q, PackEither<PackNothing, PackSplit<f16_t, 2>>{{}, wide, w.range}, st);
    const PackBytes narrow = bytes_job(p.g, p.ldg * 2, p.rows, p.depth * 2, w.g, pl.depth * 2);
    return launch_pack(q, PackEither<PackBytes, PackSplit<f16_t, 2>>{narrow, wide, w.range}, st);
}

template <typename T>
hipError_t grad_typed(const I8Grad& p, void* ws, hipStream_t st) {
    constexpr bool F32 = std::is_same<T, float>::value, F16 = std::is_same<T, f16_t>::value;
    TileStore<T> out{nullptr, nullptr, nullptr, nullptr, static_cast<T*>(p.out), p.cols};
    if (p.depth == 0) return launch_join<float>(nullptr, 0, p.rows, p.cols, out, st);
    const GradPlan pl = plan_grad(p);
    if (pl.turn) return p.transposed ? launch_turn<T, true>(p, out, st) : launch_turn<T, false>(p, out, st);
    const GradWs w = carve_grad(p, pl, ws);
    hipError_t e = hipSuccess;
    TileArgs t{};
    if constexpr (F16) {
        hipLaunchKernelGGL(tg_i8_scale_range, dim3(1), dim3(1024), 0, st, p.scale, p.depth, w.range);
        e = hipGetLastError();
        if (e != hipSuccess) return e;
        out.all = &w.range->back;
        t.wide = &w.range->wide;
        t.wide_a = static_cast<const char*>(w.g);
        t.wide_lda = pl.depth * 2 * 2;
        e = pack_grad_f16(p, pl, w, st);
    } else {
        e = pack_grad<T, bf16_t, F32 ? 3 : 1>(p, pl, w, st);
    }
    if (e != hipSuccess) return e;
    t.a = static_cast<const char*>(pl.pack_g ? w.g : p.g);
    t.b = static_cast<const char*>(w.q);
    t.lda = pl.pack_g ? pl.depth * pl.planes * 2 : p.ldg * 2;
    t.ldb = pl.depth * 2;
    t.m = int(p.rows);
    t.n = int(p.cols);
    t.b_steps = int(pl.depth / 64);
    t.plane = pl.depth * 2;
    t.tail = pl.pack_g || p.depth % 64 == 0 ? 128 : int(p.depth % 64 * 2);
    return launch_tiles<F16 ? Mma::F16 : Mma::BF16>(t, pl.tiles, out, w.part, st);
}

// The tiles' part of a plan's name.
std::string tiles_name(const TilePlan& pl) {
    const TileTime& c = kTiles[pl.form];
    std::string name = "tiles " + std::to_string(c.bm) + "x" + std::to_string(c.bn);
    if (c.per_cu > 1) name += " per_cu " + std::to_string(c.per_cu);
    if (c.planes > 1) name += " planes " + std::to_string(c.planes);
    if (pl.slices > 1) name += " slices " + std::to_string(pl.slices);
    return name;
}

}  // namespace

std::string i8_gemm_plan(const I8Gemm& p) {
    if (p.m == 0 || p.n == 0) return "none";
    if (p.k == 0) return "bias";
    const GemmPlan pl = plan_gemm(p);
    if (pl.stream != 0) return "stream rows " + std::to_string(pl.stream) + (in_words(p) && pl.stream <= 32 ? " words" : "");
    if (pl.any) return "any";
    return tiles_name(pl.tiles) + (pl.pack_a ? " pack a" : "") + (pl.pack_b ? " pack b" : "");
}

std::string i8_grad_plan(const I8Grad& p) {
    if (p.rows == 0 || p.cols == 0) return "none";
    if (p.depth == 0) return "zero";
    const GradPlan pl = plan_grad(p);
    if (pl.turn) return "turn";
    return tiles_name(pl.tiles) + (pl.pack_g ? " pack grad_c" : "");
}

size_t i8_gemm_ws(const I8Gemm& p) { return carve_gemm(p, plan_gemm(p), nullptr).bytes; }

hipError_t i8_gemm(const I8Gemm& p, void* ws, hipStream_t st) {
    if (p.m == 0 || p.n == 0) return hipSuccess;
    return by_type(p.type, [&](auto tag) { return gemm_typed<decltype(tag)>(p, ws, st); });
}

size_t i8_grad_ws(const I8Grad& p) { return carve_grad(p, plan_grad(p), nullptr).bytes; }

hipError_t i8_grad(const I8Grad& p, void* ws, hipStream_t st) {
    if (p.rows == 0 || p.cols == 0) return hipSuccess;
    return by_type(p.type, [&](auto tag) { return grad_typed<decltype(tag)>(p, ws, st); });
}

}  // namespace tg
