// tg_layers_backward.hip -- layer norm's backward pass.
#include "tg_layers_rows.hpp"

namespace tg {
namespace {

template <typename T, typename W>
struct BackwardArgs {
    const T *gy, *h, *gh;
    int64_t ldg, ldh, ldgh;
    const W* w;
    const float *mean, *rstd;
    Dropout drop;
    T *gx, *gr;
    float* part;
    int64_t rows, cols;
};

enum class Form { PLAIN, TINY, WIDE };

// Rows that a workgroup holds at a time: 512 threads are at work on short ones
// too (bf16, 8192 x 1024: 31 us one row at a time, 24 so).
template <int NT>
constexpr int kRowsAtOnce = NT < 512 ? 512 / NT : 1;

// xh = (h - mean) * rstd, u = gy * w, gr = rstd * (u - mean(u) - xh * mean(u *
// xh)) + gh, gx = dropout(gr); each of the G parts of a workgroup adds gy * xh and
// gy of its rows (blockIdx.x * G, + gridDim.x * G, ...) in that order in registers,
// the parts' sums are added in their order, and each column's go to the
// workgroup's two rows of `part`.  A thread holds eight columns; its weights stay
// in registers, and the next row is loaded, and what it drops made, before this
// one is reduced.  A row's last group is moved back to end with the row.  TINY, rows
// below eight elements, is one group with a bound; WIDE, a row longer than NT * 8, is
// shared by blockIdx.y: every workgroup reduces all of it and stores its own
// columns (bf16, 4096 x 12288 with dropout: 166 us, floor 96).
//
// Two workgroups of 512 threads have to fit a CU, 128 registers a thread, so that
// the compiler may keep neither comparisons nor the generator's keys in registers
// over all rows; and the masks are made while the loads are on their way.  bf16, 8192
// x 4096 with dropout: 62 to 68 us (352 MB with the parts, 5.5 TB/s) and 5 for the
// parts' sum; without the two 97 together.
template <typename T, typename W, bool DROP, bool GH, int NT, Form FORM>
__global__ __launch_bounds__(NT* kRowsAtOnce<NT>, 4) void tg_layer_norm_backward_rows(BackwardArgs<T, W> p) {
    constexpr int W64 = NT / 64, G = kRowsAtOnce<NT>;
    constexpr bool TINY = FORM == Form::TINY, WIDE = FORM == Form::WIDE;
    __shared__ float red[2][2][G * W64];
    const int64_t rows = p.rows, cols = p.cols;
    const int t = threadIdx.x % NT, wave = threadIdx.x / 64;
    const int group = G > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x / NT) : 0, first = group * W64;
    // Columns fit 32 bits, and a row is the same in all lanes: addresses are one of
    // the wave's and one offset of the lane's.
    const int n_cols = int(cols), base = WIDE ? int(blockIdx.y) * (NT * 8) : 0, start = base + t * 8;
    const int at = TINY ? 0 : start <= n_cols - 8 ? start : n_cols - 8;
    const bool live = start < n_cols;
    const int again = live ? start - at : 8;  // elements of the group before this one
    const int n = TINY ? n_cols : 8;
    const Keep keep(p.drop);
    // `again` without what the compiler knows of it: eight comparisons made once
    // and kept for all rows take more registers than there are.
    auto fresh = [&] {
        int a = again;
        asm volatile("" : "+v"(a));
        return a;
    };
    // Stores the thread's group, without the columns before the workgroup's first.
    auto store = [&](auto* to, const float(&v)[8]) {
        if (!TINY && (!WIDE || at >= base)) {
            store8(to, v);
        } else {
            const int a = fresh();
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (i >= a && i < n) to[i] = static_cast<std::remove_reference_t<decltype(*to)>>(v[i]);
        }
    };
    auto load8_of = [&](const auto* from, auto& x) {
        if constexpr (TINY) x.load(from, n);
        else x.load(from);
    };
    Eight<W> wv;
    load8_of(p.w + at, wv);
    float acc_w[8] = {}, acc_b[8] = {};
    struct Row {
        Eight<T> g, h, gh;
        float mean, rstd;
        uint32_t kept;
    } x[2];
    auto load = [&](int64_t row, Row& r) {
        if (row >= rows) return;
        load8_of(p.gy + row * p.ldg + at, r.g);
        load8_of(p.h + row * p.ldh + at, r.h);
        if constexpr (GH) load8_of(p.gh + row * p.ldgh + at, r.gh);
        r.mean = p.mean[row];
        r.rstd = p.rstd[row];
        if constexpr (DROP) r.kept = keep.from(row, at);
    };
    // (h - mean) * rstd; h - mean may pass f32, half of it does not.
    auto normal = [](float h, float mean, float rstd) { return (h * 0.5f - mean * 0.5f) * (rstd * 2.0f); };
    const float inv_n = 1.0f / float(cols);
    auto finish = [&](int64_t row, const Row& r, int slot) {
        float su = 0.0f, dot = 0.0f, xh[8], u[8];
        if (WIDE) {  // the part of the row that other workgroups hold
            for (int c = t * 8; c < n_cols; c += NT * 8) {
                if (c >= base && c < base + NT * 8) continue;
                const int left = n_cols - c < 8 ? n_cols - c : 8;
                float a[8], b[8], d[8];
                load_upto8(p.gy + row * p.ldg + c, left, a);
                load_upto8(p.h + row * p.ldh + c, left, b);
                load_upto8(p.w + c, left, d);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    if (i >= left) continue;
                    su += a[i] * d[i];
                    dot += a[i] * d[i] * normal(b[i], r.mean, r.rstd);
                }
            }
        }
        const int own = fresh();
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            xh[i] = normal(to_f32(r.h.v[i]), r.mean, r.rstd);
            u[i] = to_f32(r.g.v[i]) * to_f32(wv.v[i]);
            su += i >= own ? u[i] : 0.0f;
            dot += i >= own ? u[i] * xh[i] : 0.0f;
        }
        su = wave_sum(su);
        dot = wave_sum(dot);
        if constexpr (W64 > 1) {
            if (t % 64 == 0) {
                red[slot][0][wave] = su;
                red[slot][1][wave] = dot;
            }
            __syncthreads();
            su = dot = 0.0f;
#pragma unroll
            for (int i = 0; i < W64; ++i) {
                su += red[slot][0][first + i];
                dot += red[slot][1][first + i];
            }
        }
        if (G > 1 && row >= rows) return;
        su *= inv_n;
        dot *= inv_n;
        float o[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float g = to_f32(r.g.v[i]);
            acc_w[i] += g * xh[i];
            acc_b[i] += g;
            o[i] = r.rstd * (u[i] - su - xh[i] * dot);
            if constexpr (GH) o[i] += to_f32(r.gh.v[i]);
        }
        if (!live) return;
        store(p.gr + row * cols + at, o);
        if constexpr (DROP) {
            keep.apply(r.kept, o);
            store(p.gx + row * cols + at, o);
        }
    };
    // Every part of the workgroup reaches the barriers of its first part's rows.
    const int64_t stride = int64_t(gridDim.x) * G, from = int64_t(blockIdx.x) * G;
    load(from + group, x[0]);
    for (int64_t row = from; row < rows; row += 2 * stride) {
        load(row + stride + group, x[1]);
        finish(row + group, x[0], 0);
        load(row + 2 * stride + group, x[0]);
        if (row + stride < rows) finish(row + stride + group, x[1], 1);
    }
    if constexpr (G > 1) {
        __shared__ f32x4 sums[G][4][NT];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const float* a = q < 2 ? acc_w + 4 * q : acc_b + 4 * (q - 2);
            sums[group][q][t] = f32x4{a[0], a[1], a[2], a[3]};
        }
        __syncthreads();
        if (group != 0) return;
#pragma unroll
        for (int g = 1; g < G; ++g)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                float* a = q < 2 ? acc_w + 4 * q : acc_b + 4 * (q - 2);
                const f32x4 v = sums[g][q][t];
#pragma unroll
                for (int e = 0; e < 4; ++e) a[e] += v[e];
            }
    }
    if (live) {
        float* to = p.part + int64_t(blockIdx.x) * 2 * cols + at;
        store(to, acc_w);
        store(to + cols, acc_b);
    }
}

// gw and gb: each column's sum over the parts, 32 slices of them, each in order
// with eight loads on their way, then the slices in order: the same bits in every
// run.  Columns from `cols` on are the bias's.
template <typename W>
__global__ __launch_bounds__(1024) void tg_layer_norm_sum_parts(const float* __restrict__ part, int64_t parts,
                                                                W* __restrict__ gw, W* __restrict__ gb, int64_t cols) {
    __shared__ float s[32][33];
    const int c = threadIdx.x % 32, y = threadIdx.x / 32;
    const int64_t col = int64_t(blockIdx.x) * 32 + c, wide = 2 * cols;
    float a = 0.0f;
    if (col < wide) {
        for (int64_t r = y; r < parts; r += 256) {
            float v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = r + 32 * i < parts ? part[(r + 32 * i) * wide + col] : 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) a += v[i];
        }
    }
    s[y][c] = a;
    __syncthreads();
    if (threadIdx.x < 32 && col < wide) {
        a = s[0][c];
#pragma unroll
        for (int i = 1; i < 32; ++i) a += s[i][c];
        if (col < cols) gw[col] = static_cast<W>(a);
        else gb[col - cols] = static_cast<W>(a);
    }
}

// Threads of a row.
int64_t row_threads(int64_t cols) {
    for (int64_t n = 64; n < 1024; n *= 2)
        if (cols <= n * 8) return n;
    return 1024;
}

// Workgroups along the rows, each with its parts of the sums: as many as the GPU
// holds at once.
int64_t backward_parts(int64_t rows, int64_t cols) {
    const int64_t most = cols > 4096 ? 256 : 512, at_once = row_threads(cols) < 512 ? 512 / row_threads(cols) : 1;
    const int64_t n = ceil_div(rows, at_once);
    return n < most ? n : most;
}

template <typename T, typename W, int NT, Form FORM = Form::PLAIN>
hipError_t launch_backward(const LayerNormBackward& q, float* part, hipStream_t st) {
    const int64_t parts = backward_parts(q.rows, q.cols);
    if (parts > 0) {
        const dim3 grid(unsigned(parts), unsigned(ceil_div(q.cols, NT * 8)));
        const BackwardArgs<T, W> p{static_cast<const T*>(q.grad_y), static_cast<const T*>(q.h),
                                   static_cast<const T*>(q.grad_h), q.ldg, q.ldh, q.ldgh,
                                   static_cast<const W*>(q.weight), q.mean, q.rstd, q.drop,
                                   static_cast<T*>(q.grad_x), static_cast<T*>(q.grad_residual), part, q.rows, q.cols};
        const hipError_t e = by_flag(q.drop.below > 0, [&](auto drop) {
            return by_flag(q.grad_h != nullptr, [&](auto gh) {
                hipLaunchKernelGGL((tg_layer_norm_backward_rows<T, W, decltype(drop)::value, decltype(gh)::value, NT, FORM>),
                                   grid, dim3(NT * kRowsAtOnce<NT>), 0, st, p);
                return hipGetLastError();
            });
        });
        if (e != hipSuccess) return e;
    }
    hipLaunchKernelGGL((tg_layer_norm_sum_parts<W>), dim3(unsigned(ceil_div(2 * q.cols, 32))), dim3(1024), 0, st, part,
                       parts, static_cast<W*>(q.grad_weight), static_cast<W*>(q.grad_bias), q.cols);
    return hipGetLastError();
}

template <typename T, typename W>
hipError_t backward_form(const LayerNormBackward& p, float* part, hipStream_t st) {
    if (p.cols < 8) return launch_backward<T, W, 64, Form::TINY>(p, part, st);
    switch (row_threads(p.cols)) {
        case 64: return launch_backward<T, W, 64>(p, part, st);
        case 128: return launch_backward<T, W, 128>(p, part, st);
        case 256: return launch_backward<T, W, 256>(p, part, st);
        case 512: return launch_backward<T, W, 512>(p, part, st);
    }
    if (p.cols > 8192) return launch_backward<T, W, 1024, Form::WIDE>(p, part, st);
    return launch_backward<T, W, 1024>(p, part, st);
}

}  // namespace

size_t layer_norm_backward_ws(int64_t rows, int64_t cols) {
    return size_t(backward_parts(rows, cols)) * 2 * size_t(cols) * sizeof(float);
}

hipError_t layer_norm_backward(const LayerNormBackward& p, void* ws, hipStream_t st) {
    if (p.cols == 0) return hipSuccess;
    float* part = static_cast<float*>(ws);
    return by_type(p.type, [&](auto tag) {
        using T = decltype(tag);
        return p.weight_type == p.type ? backward_form<T, T>(p, part, st) : backward_form<T, float>(p, part, st);
    });
}

}  // namespace tg
