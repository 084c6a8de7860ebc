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

// xh = (h - mean) * rstd, u = gy * w, gr = rstd * (u - mean(u) - xh * mean(u *
// xh)) + gh, gx = dropout(gr); the workgroup adds gy * xh and gy of its rows
// (blockIdx.x, + gridDim.x, ...) in that order in registers and writes those
// sums of each column to its two rows of `part`.  A thread holds eight columns;
// its weights stay in registers, and the next row is loaded before this one is
// reduced.  A row longer than NT * 8 is shared by blockIdx.y: every workgroup
// reduces all of it and stores its own columns.  A row's last group is moved
// back to end with the row; TINY, rows below eight elements, is one group with a
// bound.
template <typename T, typename W, bool DROP, bool GH, int NT, bool TINY>
__global__ __launch_bounds__(NT) void tg_layer_norm_backward_rows(BackwardArgs<T, W> p) {
    constexpr int W64 = NT / 64;
    __shared__ float red[2][2][W64];
    const int64_t rows = p.rows, cols = p.cols;
    const int t = threadIdx.x, wave = t / 64;
    const int64_t base = int64_t(blockIdx.y) * (NT * 8), start = base + int64_t(t) * 8;
    const int64_t at = TINY ? 0 : start <= cols - 8 ? start : cols - 8;
    const bool live = start < cols;
    const int again = live ? int(start - at) : 8;  // elements of the group before this one
    const int n = TINY ? int(cols) : 8;
    const Keep keep(p.drop);
    // Stores the thread's group, without the columns before the workgroup's first.
    auto store = [&](auto* to, const float(&v)[8]) {
        if (at >= base) {
            store_upto8(to, n, v);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (i >= again) to[i] = static_cast<std::remove_reference_t<decltype(*to)>>(v[i]);
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
    } x[2];
    auto load = [&](int64_t row, Row& r) {
        if (row >= rows) return;
        load8_of(p.gy + row * p.ldg + at, r.g);
        load8_of(p.h + row * p.ldh + at, r.h);
        if constexpr (GH) load8_of(p.gh + row * p.ldgh + at, r.gh);
        r.mean = p.mean[row];
        r.rstd = p.rstd[row];
    };
    // (h - mean) * rstd; h - mean may pass f32, half of it does not.
    auto normal = [](float h, float mean, float rstd) { return (h * 0.5f - mean * 0.5f) * (rstd * 2.0f); };
    const float inv_n = 1.0f / float(cols);
    auto finish = [&](int64_t row, const Row& r, int slot) {
        float su = 0.0f, dot = 0.0f, xh[8], u[8];
        if (gridDim.y > 1) {  // the part of the row that other workgroups hold
            for (int64_t c = int64_t(t) * 8; c < cols; c += NT * 8) {
                if (c >= base && c < base + NT * 8) continue;
                const int left = cols - c < 8 ? int(cols - c) : 8;
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
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            xh[i] = normal(to_f32(r.h.v[i]), r.mean, r.rstd);
            u[i] = to_f32(r.g.v[i]) * to_f32(wv.v[i]);
            const bool counts = i >= again && (!TINY || i < n);
            su += counts ? u[i] : 0.0f;
            dot += counts ? u[i] * xh[i] : 0.0f;
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
                su += red[slot][0][i];
                dot += red[slot][1][i];
            }
        }
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
            keep.apply(row, at, o);
            store(p.gx + row * cols + at, o);
        }
    };
    const int64_t stride = gridDim.x;
    load(blockIdx.x, x[0]);
    for (int64_t row = blockIdx.x; row < rows; row += 2 * stride) {
        load(row + stride, x[1]);
        finish(row, x[0], 0);
        load(row + 2 * stride, x[0]);
        if (row + stride < rows) finish(row + stride, x[1], 1);
    }
    if (live) {
        float* to = p.part + int64_t(blockIdx.x) * 2 * cols + at;
        store(to, acc_w);
        store(to + cols, acc_b);
    }
}

// gw and gb: each column's sum over the parts, 64 slices of them, each in order
// with four loads on their way, then the slices in order: the same bits in every
// run.  Columns from `cols` on are the bias's.
template <typename W>
__global__ __launch_bounds__(1024) void tg_layer_norm_sum_parts(const float* __restrict__ part, int64_t parts,
                                                                W* __restrict__ gw, W* __restrict__ gb, int64_t cols) {
    __shared__ float s[64][17];
    const int c = threadIdx.x % 16, y = threadIdx.x / 16;
    const int64_t col = int64_t(blockIdx.x) * 16 + c, wide = 2 * cols;
    float a = 0.0f;
    if (col < wide) {
        for (int64_t r = y; r < parts; r += 256) {
            float v[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = r + 64 * i < parts ? part[(r + 64 * i) * wide + col] : 0.0f;
#pragma unroll
            for (int i = 0; i < 4; ++i) a += v[i];
        }
    }
    s[y][c] = a;
    __syncthreads();
    if (threadIdx.x < 16 && col < wide) {
        a = s[0][c];
#pragma unroll
        for (int i = 1; i < 64; ++i) a += s[i][c];
        if (col < cols) gw[col] = static_cast<W>(a);
        else gb[col - cols] = static_cast<W>(a);
    }
}

// Workgroups along the rows, each with its parts of the sums: as many as the GPU
// holds at once.
int64_t backward_parts(int64_t rows, int64_t cols) {
    const int64_t most = cols > 4096 ? 256 : 512;
    return rows < most ? rows : most;
}

template <typename T, typename W, int NT, bool TINY = false>
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
                hipLaunchKernelGGL((tg_layer_norm_backward_rows<T, W, decltype(drop)::value, decltype(gh)::value, NT, TINY>),
                                   grid, dim3(NT), 0, st, p);
                return hipGetLastError();
            });
        });
        if (e != hipSuccess) return e;
    }
    hipLaunchKernelGGL((tg_layer_norm_sum_parts<W>), dim3(unsigned(ceil_div(2 * q.cols, 16))), dim3(1024), 0, st, part,
                       parts, static_cast<W*>(q.grad_weight), static_cast<W*>(q.grad_bias), q.cols);
    return hipGetLastError();
}

template <typename T, typename W>
hipError_t backward_form(const LayerNormBackward& p, float* part, hipStream_t st) {
    const int64_t groups = ceil_div(p.cols, 8);
    if (p.cols < 8) return launch_backward<T, W, 64, true>(p, part, st);
    if (groups <= 64) return launch_backward<T, W, 64>(p, part, st);
    if (groups <= 128) return launch_backward<T, W, 128>(p, part, st);
    if (groups <= 256) return launch_backward<T, W, 256>(p, part, st);
    if (groups <= 512) return launch_backward<T, W, 512>(p, part, st);
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
