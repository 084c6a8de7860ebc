// tg_i8_rows.hip -- row operators of the 8-bit layer: RMS norm with the
// residual's addition and 8-bit output, its backward pass, and rows packed to
// 8 bits with a scale and restored.
//
// All of them are bound by HBM: every input element is read once, every
// output written once, a row's values stay in registers between its reduction
// and its output.  (A copy of 1 GiB reaches 4.95 TB/s on the same GPU.)
#include <type_traits>

#include "../../include/tropical_gemm_hip.h"
#include "tg_i8.hpp"
#include "tg_i8_types.hpp"

namespace tg {
namespace {

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// One row's threads: NT lanes of a workgroup, 256 / NT rows per workgroup
// where NT is below 256.  A thread holds VPT groups of eight neighbouring
// elements, group g of thread t starting at element (g * NT + t) * 8, so the
// lanes of a wave read 1 KiB (of 16-bit elements) side by side.
template <int NT>
constexpr int kRowsPerBlock = NT < 256 ? 256 / NT : 1;
template <int NT>
constexpr int kBlock = NT < 256 ? 256 : NT;

// Squares of numbers above 2^64 pass f32.  A row whose sum of squares is not
// finite is summed again with its values times kShrink: the largest, below
// 2^128, become 2^48, of which 2^31 squares stay in f32, and the row's maximum,
// at least 2^48 in a sum of 2^31 squares that passes 2^128, becomes 2^-32.
constexpr float kHuge = __builtin_huge_valf();
constexpr float kShrink = 0x1p-80f;

// Reduces (sum, top) over the NT threads of each row; every thread gets both.
template <int NT>
__device__ __forceinline__ void row_reduce(float& sum, float& top) {
    sum = wave_sum(sum);
    top = wave_max(top);
    if constexpr (NT > 64) {
        constexpr int W = NT / 64;
        __shared__ float part[2][kRowsPerBlock<NT> * W];
        const int wave = threadIdx.x / 64, first = wave / W * W;
        if (threadIdx.x % 64 == 0) {
            part[0][wave] = sum;
            part[1][wave] = top;
        }
        __syncthreads();
        sum = part[0][first];
        top = part[1][first];
#pragma unroll
        for (int i = 1; i < W; ++i) {
            sum += part[0][first + i];
            top = max_nan(top, part[1][first + i]);
        }
    }
}

// A group of eight elements as it is loaded.
template <typename T>
struct Eight {
    typedef T t8 __attribute__((ext_vector_type(8)));
    t8 v;
    // The eight from p on, at any address.
    __device__ __forceinline__ void load(const T* p) {
        typedef uint32_t words __attribute__((ext_vector_type(sizeof(T) * 2)));
        typedef uint32_t words_any __attribute__((ext_vector_type(sizeof(T) * 2), aligned(sizeof(T))));
        v = __builtin_bit_cast(t8, words(*reinterpret_cast<const words_any*>(p)));
    }
    // The first `left` of them, zeros behind.
    __device__ __forceinline__ void load(const T* p, int64_t left) {
        if (left >= 8) {
            load(p);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = i < left ? p[i] : T(0.0f);
        }
    }
};

// v * 127 / top with one rounding: 127 / top as a sum of two numbers.  Where it
// is a whole number and a half exactly, as for half of the row's maximum, the
// result is too, and goes to the even neighbour; 127 / top rounded once misses
// one such tie in twenty.
struct Steps {
    float hi, lo;
    __device__ __forceinline__ explicit Steps(float top) {
        hi = 127.0f / top;
        lo = fmaf(-hi, top, 127.0f) / top;
    }
    __device__ __forceinline__ float of(float v) const { return fmaf(v, hi, v * lo); }
};

// h = round(x + residual); rstd = (mean h^2 + eps)^-1/2; v = h * w;
// top = max(max |v|, tiny); q = rint(v * 127 / top); scale = top * rstd / 127.
// rstd cancels in q, so q depends on no order of summation, and both
// reductions of the row are made in one pass.  NORM false: v = x, rstd = 1.
// A NaN or infinity makes the row's scale NaN or infinite with zeros in q, so
// its values are NaN, as dividing by the row's maximum gives them.
//
// VPT > 0, for rows of at least eight elements: all loads of a thread are
// issued before the first is used.  A group that would end past the row is
// moved back to end with it, so that no load depends on a branch; the elements
// it shares with the group before it are written twice, with the same values,
// and counted once.
// VPT 0: rows of any length, read again (through L2) after the reduction.
// bf16, 8192 x 8192: norm with residual 89 us (470 MB, 5.3 TB/s), without norm
// 40 us (201 MB, 5.0 TB/s); one row of 4096: 2.7 us, the loads' latency and
// the launch's (medians of 60 runs).
template <typename T, typename W, bool NORM, bool RES, int NT, int VPT>
__global__ __launch_bounds__(kBlock<NT>) void tg_i8_rows(const T* __restrict__ x, int64_t ldx,
                                                         const T* __restrict__ res, int64_t ldr,
                                                         const W* __restrict__ w, float eps,
                                                         int8_t* __restrict__ q,
                                                         float* __restrict__ scale, T* __restrict__ h,
                                                         int64_t rows, int64_t cols) {
    const int t = threadIdx.x % NT;
    const int64_t row = int64_t(blockIdx.x) * kRowsPerBlock<NT> + threadIdx.x / NT;
    const bool live = row < rows;  // every thread reaches the reduction's barrier
    const T* xr = x + row * ldx;
    const T* rr = RES ? res + row * ldr : nullptr;
    float sum = 0.0f, top = 0.0f;

    auto give = [&](int64_t at, int n, const float(&v)[8], const Steps& s) {
        int o[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int r = __float2int_rn(s.of(v[i]));
            o[i] = r > 127 ? 127 : (r < -127 ? -127 : r);
        }
        store_i8_upto8(q + row * cols + at, n, o);
    };
    // The sum of squares of the row times kShrink; every wave makes it all.
    auto shrunk_sum = [&] {
        float s = 0.0f;
        for (int64_t at = int64_t(threadIdx.x % 64) * 8; at < cols; at += 512) {
            const int n = cols - at < 8 ? int(cols - at) : 8;
            float v[8], r[8] = {};
            load_upto8(xr + at, n, v);
            if constexpr (RES) load_upto8(rr + at, n, r);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float hs = (RES ? to_f32(static_cast<T>(v[i] + r[i])) : v[i]) * kShrink;
                s += hs * hs;
            }
        }
        return wave_sum(s);
    };
    // Reduces the row, stores its scale and gives 127 / top.
    auto reduce = [&] {
        row_reduce<NT>(sum, top);
        top = max_nan(top, kI8TinyTop);
        float shrink = 1.0f;
        if constexpr (NORM) {
            if (live && !(sum < kHuge)) {
                sum = shrunk_sum();
                shrink = kShrink;
            }
        }
        if (live && t == 0) {
            if constexpr (NORM) {
                const float rstd = shrink / sqrtf(sum / float(cols > 0 ? cols : 1) + eps * shrink * shrink);
                scale[row] = top * rstd / 127.0f;
            } else {
                scale[row] = top / 127.0f;
            }
        }
        return Steps(top);
    };

    if constexpr (VPT > 0) {
        float v[VPT][8];
        auto start = [&](int g) { return int64_t(g * NT + t) * 8; };
        auto from = [&](int g) { return start(g) <= cols - 8 ? start(g) : cols - 8; };
        if (live) {
            Eight<T> a[VPT], b[VPT];
            Eight<W> f[VPT];
#pragma unroll
            for (int g = 0; g < VPT; ++g) {
                a[g].load(xr + from(g));
                if constexpr (RES) b[g].load(rr + from(g));
            }
            if constexpr (NORM) {
#pragma unroll
                for (int g = 0; g < VPT; ++g) f[g].load(w + from(g));
            }
#pragma unroll
            for (int g = 0; g < VPT; ++g) {
                const int again = int(start(g) - from(g));  // of the group before it; 8 and more: all
#pragma unroll
                for (int i = 0; i < 8; ++i) v[g][i] = to_f32(a[g].v[i]);
                if constexpr (RES) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) v[g][i] = to_f32(static_cast<T>(v[g][i] + to_f32(b[g].v[i])));
                    if (again < 8) store8(h + row * cols + from(g), v[g]);
                }
                if constexpr (NORM) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        sum += i >= again ? v[g][i] * v[g][i] : 0.0f;
                        v[g][i] *= to_f32(f[g].v[i]);
                    }
                }
#pragma unroll
                for (int i = 0; i < 8; ++i) top = max_nan(top, fabsf(v[g][i]));
            }
        }
        const Steps steps = reduce();
        if (live) {
#pragma unroll
            for (int g = 0; g < VPT; ++g)
                if (start(g) < cols) give(from(g), 8, v[g], steps);
        }
    } else {
        // One group: the (rounded) stream and its weighted values.
        auto take = [&](int64_t at, int n, float(&v)[8], bool first) {
            load_upto8(xr + at, n, v);
            if constexpr (RES) {
                float r[8];
                load_upto8(rr + at, n, r);
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = to_f32(static_cast<T>(v[i] + r[i]));
                if (first) store_upto8(h + row * cols + at, n, v);
            }
            if constexpr (NORM) {
                float g[8];
                load_upto8(w + at, n, g);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    if (first) sum += v[i] * v[i];
                    v[i] *= g[i];
                }
            }
            if (first) {
#pragma unroll
                for (int i = 0; i < 8; ++i) top = max_nan(top, fabsf(v[i]));
            }
        };
        auto each = [&](auto&& f) {
            if (!live) return;
            for (int64_t at = int64_t(t) * 8; at < cols; at += NT * 8) f(at, cols - at < 8 ? int(cols - at) : 8);
        };
        float v[8];
        each([&](int64_t at, int n) { take(at, n, v, true); });
        const Steps steps = reduce();
        each([&](int64_t at, int n) {
            take(at, n, v, false);
            give(at, n, v, steps);
        });
    }
}

template <typename T, typename W, bool NORM, bool RES, int NT, int VPT>
hipError_t launch_rows(const I8Norm& p, hipStream_t st) {
    // A launch's thread count stays below 2^32.
    constexpr int64_t kMost = int64_t(1) << 21;
    for (int64_t r0 = 0; r0 < p.rows; r0 += kMost) {
        const int64_t n = p.rows - r0 < kMost ? p.rows - r0 : kMost;
        hipLaunchKernelGGL((tg_i8_rows<T, W, NORM, RES, NT, VPT>), dim3(unsigned(ceil_div(n, kRowsPerBlock<NT>))),
                           dim3(kBlock<NT>), 0, st, static_cast<const T*>(p.x) + r0 * p.ldx, p.ldx,
                           RES ? static_cast<const T*>(p.residual) + r0 * p.ldr : nullptr, p.ldr,
                           static_cast<const W*>(p.weight), p.eps, p.q + r0 * p.cols, p.scale + r0,
                           RES ? static_cast<T*>(p.h) + r0 * p.cols : nullptr, n, p.cols);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

// Few threads a row, so that a workgroup's barrier stops few loads, and two
// groups each (three where two would leave more than a quarter of the threads
// without one, or with one they share): bf16 norm with residual of 16384 rows
// of 1024: 19.7 us, 21.1 with one group a thread on twice the threads; of 2501:
// 56.6 us as 128 x 3, 70.3 as 256 x 2; 8192 rows of 8192: 81.9 us as 512 x 2,
// 85.1 as 256 x 4, 85.0 as 1024 x 1 (each the least of 30 runs).
template <typename T, typename W, bool NORM, bool RES>
hipError_t rows_form(const I8Norm& p, hipStream_t st) {
    const int64_t groups = ceil_div(p.cols, 8);
    if (p.cols < 8) return launch_rows<T, W, NORM, RES, 64, 0>(p, st);
    if (groups <= 64) return launch_rows<T, W, NORM, RES, 64, 1>(p, st);
    if (groups <= 128) return launch_rows<T, W, NORM, RES, 64, 2>(p, st);
    if (groups <= 256) return launch_rows<T, W, NORM, RES, 128, 2>(p, st);
    if (groups <= 384) return launch_rows<T, W, NORM, RES, 128, 3>(p, st);
    if (groups <= 512) return launch_rows<T, W, NORM, RES, 256, 2>(p, st);
    if (groups <= 768) return launch_rows<T, W, NORM, RES, 256, 3>(p, st);
    if (groups <= 1024) return launch_rows<T, W, NORM, RES, 512, 2>(p, st);
    return launch_rows<T, W, NORM, RES, 1024, 0>(p, st);
}

template <typename T, typename W>
hipError_t norm_typed(const I8Norm& p, hipStream_t st) {
    return p.residual != nullptr ? rows_form<T, W, true, true>(p, st) : rows_form<T, W, true, false>(p, st);
}

// f(T()) for the element type.
template <typename F>
hipError_t by_type(int type, F&& f) {
    switch (type) {
        case TG_BF16: return f(bf16_t());
        case TG_F16: return f(f16_t());
        default: return f(float());
    }
}

// y = round(q * scale), eight elements a thread.  bf16, 8192 x 8192: 32.8 us
// behind the kernel that wrote q (201 MB, 6.1 TB/s, q still in the last cache).
template <typename T>
__global__ __launch_bounds__(256) void tg_i8_restore(const int8_t* __restrict__ q, int64_t ldq,
                                                     const float* __restrict__ scale, T* __restrict__ y,
                                                     int64_t rows, int64_t cols, int64_t groups) {
    const int64_t stride = int64_t(gridDim.x) * 256;
    for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < rows * groups; i += stride) {
        const int64_t row = i / groups, at = (i - row * groups) * 8;
        const int n = cols - at < 8 ? int(cols - at) : 8;
        const float s = scale[row];
        float v[8];
        load_i8_upto8(q + row * ldq + at, n, v);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] *= s;
        store_upto8(y + row * cols + at, n, v);
    }
}

// Backward of the norm.  u = gy * w, rstd and c = rstd^2 * mean(u * h) of each
// row, gx = rstd * (u - h * c) + gh; the workgroup adds gy * h * rstd of its
// rows (blockIdx.x, + gridDim.x, ...) in that order in registers, and writes
// that sum of each column to part[blockIdx.x].  The columns of a thread are as
// in tg_i8_rows; its weights stay in registers, and the next row is loaded
// before this one is reduced, so that loads are always on their way.  A row
// longer than NT * 8 is shared by blockIdx.y; then every workgroup reduces all
// of it, its own columns last, so that two of them may differ in the sums' last
// bit: each column is stored by its own workgroup alone.  A row's last group is
// moved back to end with the row, as in tg_i8_rows, so that no load waits for a
// branch (bf16, 8192 rows of 4095: 62 us for the whole pass with branches, 45
// so); TINY, rows below eight elements, is one group with a bound.  bf16, 8192 x 4096 with gh: 51 us (277 MB with the
// parts, 5.4 TB/s); f32, 777 x 2501: 11 us, two rows one after the other.
template <typename T, typename W, bool GH, int NT, bool TINY>
__global__ __launch_bounds__(NT) void tg_i8_norm_backward(
    const T* __restrict__ gy, int64_t ldg, const T* __restrict__ h, int64_t ldh, const W* __restrict__ w,
    float eps, const T* __restrict__ gh, int64_t ldgh, T* __restrict__ gx, float* __restrict__ part,
    int64_t rows, int64_t cols) {
    constexpr int W64 = NT / 64;
    __shared__ float red[2][2][W64];
    const int t = threadIdx.x, wave = t / 64;
    const int64_t base = int64_t(blockIdx.y) * (NT * 8), start = base + int64_t(t) * 8;
    const int64_t at = TINY ? 0 : start <= cols - 8 ? start : cols - 8;
    const bool live = start < cols;
    const int again = live ? int(start - at) : 8;  // elements of the group before this one
    const int n = TINY ? int(cols) : 8;
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
    load8_of(w + at, wv);
    float acc[8] = {};
    struct Row {
        Eight<T> g, h, gh;
    } x[2];
    auto load = [&](int64_t row, Row& r) {
        if (row >= rows) return;
        load8_of(gy + row * ldg + at, r.g);
        load8_of(h + row * ldh + at, r.h);
        if constexpr (GH) load8_of(gh + row * ldgh + at, r.gh);
    };
    const float inv_n = 1.0f / float(cols);
    float ss = 0.0f, dot = 0.0f;
    // The row's sums of h * h and u * h, of h times `shrink`, by way of
    // red[slot]: never the same slot twice in turn, so that one barrier is enough.
    auto sums = [&](int64_t row, const Row& r, float shrink, int slot) {
        ss = dot = 0.0f;
        if (gridDim.y > 1) {  // the part of the row that other workgroups hold
            for (int64_t c = int64_t(t) * 8; c < cols; c += NT * 8) {
                if (c >= base && c < base + NT * 8) continue;
                const int left = cols - c < 8 ? int(cols - c) : 8;
                float a[8], b[8], d[8];
                load_upto8(gy + row * ldg + c, left, a);
                load_upto8(h + row * ldh + c, left, b);
                load_upto8(w + c, left, d);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float hv = b[i] * shrink;
                    ss += hv * hv;
                    dot += a[i] * d[i] * hv;
                }
            }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float hv = i >= again ? to_f32(r.h.v[i]) * shrink : 0.0f;
            ss += hv * hv;
            dot += i >= again ? to_f32(r.g.v[i]) * to_f32(wv.v[i]) * hv : 0.0f;
        }
        ss = wave_sum(ss);
        dot = wave_sum(dot);
        if constexpr (W64 > 1) {
            if (t % 64 == 0) {
                red[slot][0][wave] = ss;
                red[slot][1][wave] = dot;
            }
            __syncthreads();
            ss = dot = 0.0f;
#pragma unroll
            for (int i = 0; i < W64; ++i) {
                ss += red[slot][0][i];
                dot += red[slot][1][i];
            }
        }
    };
    // Its part of the gradients.
    auto give = [&](int64_t row, const Row& r, float shrink) {
        const float rstd = 1.0f / sqrtf(ss * inv_n + eps * shrink * shrink);  // of h times `shrink`
        const float c = dot * inv_n * rstd * rstd;
        float o[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float g = to_f32(r.g.v[i]), hv = to_f32(r.h.v[i]) * shrink;
            acc[i] += g * (hv * rstd);
            o[i] = rstd * shrink * (g * to_f32(wv.v[i]) - hv * c);
            if constexpr (GH) o[i] += to_f32(r.gh.v[i]);
        }
        if (live) store(gx + row * cols + at, o);
    };
    bool huge = false;
    auto finish = [&](int64_t row, const Row& r, int flip) {
        sums(row, r, 1.0f, flip);
        huge |= !(ss < kHuge);
        give(row, r, 1.0f);
    };
    const int64_t stride = gridDim.x;
    load(blockIdx.x, x[0]);
    for (int64_t row = blockIdx.x; row < rows; row += 2 * stride) {
        load(row + stride, x[1]);
        finish(row, x[0], 0);
        load(row + 2 * stride, x[0]);
        if (row + stride < rows) finish(row + stride, x[1], 1);
    }
    // Rows whose squares passed f32 had rstd 0, and nothing of them (or a NaN, of
    // rows that are not finite) is in acc.  A second pass: as a branch of the
    // first it makes the loads on their way wait (55 us there, 69).
    if (huge) {  // the same in the whole workgroup
        __syncthreads();
        int slot = 0;  // another one each time, as above
        for (int64_t row = blockIdx.x; row < rows; row += stride, slot ^= 1) {
            load(row, x[0]);
            sums(row, x[0], 1.0f, slot);
            if (ss < kHuge) continue;
            sums(row, x[0], kShrink, slot ^= 1);
            give(row, x[0], kShrink);
        }
    }
    if (live) store(part + int64_t(blockIdx.x) * cols + at, acc);
}

// gw[j] = sum over the parts: 64 slices of them, each in order, four of its
// loads on their way at a time, then the slices in order.  The same bits in
// every run.  512 parts of 4096: 5.1 us, a launch and a few loads' latency.
template <typename W>
__global__ __launch_bounds__(1024) void tg_i8_sum_parts(const float* __restrict__ part, int64_t parts,
                                                        W* __restrict__ gw, int64_t cols) {
    __shared__ float s[64][17];
    const int c = threadIdx.x % 16, y = threadIdx.x / 16;
    const int64_t col = int64_t(blockIdx.x) * 16 + c;
    float a = 0.0f;
    if (col < cols) {
        for (int64_t r = y; r < parts; r += 256) {
            float v[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = r + 64 * i < parts ? part[(r + 64 * i) * cols + col] : 0.0f;
#pragma unroll
            for (int i = 0; i < 4; ++i) a += v[i];
        }
    }
    s[y][c] = a;
    __syncthreads();
    if (threadIdx.x < 16 && col < cols) {
        a = s[0][c];
#pragma unroll
        for (int i = 1; i < 64; ++i) a += s[i][c];
        gw[col] = static_cast<W>(a);
    }
}

// Workgroups along the rows, each with a part of the weight's gradient: as many
// as the GPU holds at once, two for each CU, or one of 1024 threads (a part
// costs cols * 8 bytes of traffic, as much as a row's gradient or two).
int64_t backward_parts(int64_t rows, int64_t cols) {
    const int64_t most = cols > 4096 ? 256 : 512;
    return rows < most ? rows : most;
}

template <typename T, typename W, int NT, bool TINY = false>
hipError_t launch_norm_backward(const I8NormBackward& p, float* part, hipStream_t st) {
    const int64_t parts = backward_parts(p.rows, p.cols);
    if (parts > 0) {
        const dim3 grid(unsigned(parts), unsigned(ceil_div(p.cols, NT * 8)));
        const auto kernel = p.grad_h != nullptr ? &tg_i8_norm_backward<T, W, true, NT, TINY>
                                                : &tg_i8_norm_backward<T, W, false, NT, TINY>;
        hipLaunchKernelGGL(kernel, grid, dim3(NT), 0, st, static_cast<const T*>(p.grad_y), p.ldg,
                           static_cast<const T*>(p.h), p.ldh, static_cast<const W*>(p.weight), p.eps,
                           static_cast<const T*>(p.grad_h), p.ldgh, static_cast<T*>(p.grad_x), part, p.rows, p.cols);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    hipLaunchKernelGGL((tg_i8_sum_parts<W>), dim3(unsigned(ceil_div(p.cols, 16))), dim3(1024), 0, st, part,
                       parts, static_cast<W*>(p.grad_weight), p.cols);
    return hipGetLastError();
}

template <typename T, typename W>
hipError_t norm_backward_typed(const I8NormBackward& p, float* part, hipStream_t st) {
    const int64_t groups = ceil_div(p.cols, 8);
    if (p.cols < 8) return launch_norm_backward<T, W, 64, true>(p, part, st);
    if (groups <= 64) return launch_norm_backward<T, W, 64>(p, part, st);
    if (groups <= 128) return launch_norm_backward<T, W, 128>(p, part, st);
    if (groups <= 256) return launch_norm_backward<T, W, 256>(p, part, st);
    if (groups <= 512) return launch_norm_backward<T, W, 512>(p, part, st);
    return launch_norm_backward<T, W, 1024>(p, part, st);
}

}  // namespace

hipError_t i8_rms_norm(const I8Norm& p, hipStream_t st) {
    if (p.rows == 0) return hipSuccess;
    return by_type(p.type, [&](auto tag) {
        using T = decltype(tag);
        return p.weight_type == p.type ? norm_typed<T, T>(p, st) : norm_typed<T, float>(p, st);
    });
}

hipError_t i8_quantize(const I8Norm& p, hipStream_t st) {
    if (p.rows == 0) return hipSuccess;
    return by_type(p.type, [&](auto tag) {
        using T = decltype(tag);
        return rows_form<T, T, false, false>(p, st);
    });
}

hipError_t i8_dequantize(int type, const int8_t* q, int64_t ldq, const float* scale, void* y,
                         int64_t rows, int64_t cols, hipStream_t st) {
    if (rows == 0 || cols == 0) return hipSuccess;
    const int64_t groups = ceil_div(cols, 8), blocks = ceil_div(rows * groups, 256);
    return by_type(type, [&](auto tag) {
        using T = decltype(tag);
        hipLaunchKernelGGL((tg_i8_restore<T>), dim3(unsigned(blocks < 65536 ? blocks : 65536)), dim3(256), 0,
                           st, q, ldq, scale, static_cast<T*>(y), rows, cols, groups);
        return hipGetLastError();
    });
}

size_t i8_rms_norm_backward_ws(int64_t rows, int64_t cols) {
    return size_t(backward_parts(rows, cols)) * size_t(cols) * sizeof(float);
}

hipError_t i8_rms_norm_backward(const I8NormBackward& p, void* ws, hipStream_t st) {
    if (p.cols == 0) return hipSuccess;
    float* part = static_cast<float*>(ws);
    return by_type(p.type, [&](auto tag) {
        using T = decltype(tag);
        return p.weight_type == p.type ? norm_backward_typed<T, T>(p, part, st)
                                       : norm_backward_typed<T, float>(p, part, st);
    });
}

}  // namespace tg
