// tg_layers.hip -- layer norm with dropout and the residual's addition in one
// pass, and dropout by itself.  Both are bound by memory:
// every input element is read once, every output written once, a row's values
// stay in registers between its reductions and its output.
#include "tg_layers_rows.hpp"

namespace tg {
namespace {

constexpr float kHuge = __builtin_huge_valf();
// Squares of numbers above 2^64 pass f32: a row whose sum of them is not finite
// is summed again with its values times kShrink (the largest become 2^48).  Those of
// numbers below 2^-63 lose bits or all of themselves: a row whose variance and eps
// together are below kFaint, and its mean below kFaintMean, is summed again with its
// values times kGrow (the least become 2^-49).  With a larger mean such a row's
// values are all equal, a step of f32 there being above the root of kFaint.
constexpr float kShrink = 0x1p-80f;
constexpr float kGrow = 0x1p100f, kFaint = 0x1p-100f, kFaintMean = 0x1p-10f;

// A row's threads: NT lanes, several rows in a workgroup where NT is below 256.
// A thread holds VPT groups of eight neighbours, group g of thread t from
// element (g * NT + t) * 8 on.
template <int NT>
constexpr int kRowsPerBlock = NT < 256 ? 256 / NT : 1;
template <int NT>
constexpr int kBlock = NT < 256 ? 256 : NT;

// Sums of N numbers over the NT threads of each row, in every one of them.  Called
// once for each N, so that one barrier is enough.
template <int NT, int N>
__device__ __forceinline__ void row_sums(float (&x)[N]) {
#pragma unroll
    for (int k = 0; k < N; ++k) x[k] = wave_sum(x[k]);
    if constexpr (NT > 64) {
        constexpr int W = NT / 64;
        __shared__ float part[N][kRowsPerBlock<NT> * W];
        const int wave = threadIdx.x / 64, first = wave / W * W;
        if (threadIdx.x % 64 == 0) {
#pragma unroll
            for (int k = 0; k < N; ++k) part[k][wave] = x[k];
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < N; ++k) {
            x[k] = part[k][first];
#pragma unroll
            for (int i = 1; i < W; ++i) x[k] += part[k][first + i];
        }
    }
}

template <typename T, typename W>
struct NormArgs {
    const T *x, *res;
    int64_t ldx, ldr;
    const W *w, *b;
    float eps;
    Dropout drop;
    T *y, *h;
    float *mean, *rstd;
    int64_t first_row, rows, cols;  // first_row: of the launch, as dropout counts
};

// h = round(dropout(x) + residual); mean and variance of h in two sums of the
// values in registers, which loses nothing where the mean is large beside the
// deviations; y = (h - mean) * rstd * w + b.  With the deviations' squares go the
// deviations themselves, whose mean is what rounding took from the mean: where that
// is one step of f32, equal values of 1000 would come out as 0.02 (eps 1e-5) and not
// as 0.  It is added where the mean is at least the standard deviation.  Below,
// the rounding of the deviations is all that it holds, and the first mean is the
// better one: sums of 16-bit values round little or not at all.  Error of the mean
// without and with it, in deviations (root mean square, 4096 normal values):
//     mean / deviation     0               0.5             1               4               1000
//     bf16            5.7e-10 2.0e-8  2.1e-8 3.3e-8  4.3e-8 3.8e-8  6.1e-8 5.9e-8  0       0
//     f32             1.8e-9  8.6e-9  2.3e-8 1.4e-8  4.4e-8 2.7e-8  1.8e-7 1.1e-7  3.4e-5  1.7e-5
//
// VPT > 0, rows of at least eight elements: all loads of a thread are issued
// before the first is used; a group that would end past the row is moved back to
// end with it, and what it shares with the group before it is counted once.
// VPT 0: any length, read again for each sum (bf16, 4096 x 12288 with dropout and
// residual: 125 us, 403 MB if read once).
//
// bf16, 8192 x 8192 with dropout and residual: 99 us (537 MB, 5.4 TB/s; 105 where
// the rows whose sums pass f32 were stored with the others, which took 82 registers;
// 62 now), 8192 x 4096 with residual only 44 (268 MB, 6.0 TB/s); one row of 4096:
// 3.2 us, the loads' latency, two reductions and the launch.
template <typename T, typename W, bool DROP, bool RES, int NT, int VPT>
__global__ __launch_bounds__(kBlock<NT>) void tg_layer_norm_rows(NormArgs<T, W> p) {
    constexpr bool STREAM = DROP || RES;  // h is not x
    const int t = threadIdx.x % NT;
    const int64_t row = int64_t(blockIdx.x) * kRowsPerBlock<NT> +
                        (kRowsPerBlock<NT> > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x / NT) : 0);  // of the wave
    const bool live = row < p.rows;  // every thread reaches the barriers
    const int64_t cols = p.cols;
    const T* xr = p.x + row * p.ldx;
    const T* rr = RES ? p.res + row * p.ldr : nullptr;
    const Keep keep(p.drop);
    const float inv_n = 1.0f / float(cols);

    // n values of the stream from `at` on, as they are stored.
    auto stream = [&](int64_t at, int n, float(&v)[8]) {
        load_upto8(xr + at, n, v);
        if constexpr (DROP) keep.apply(p.first_row + row, at, v);
        if constexpr (RES) {
            float r[8];
            load_upto8(rr + at, n, r);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] += r[i];
        }
        if constexpr (STREAM) {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = to_f32(static_cast<T>(v[i]));
        }
    };
    auto keep_stats = [&](float mean, float rstd) {
        if (t == 0) {
            p.mean[row] = mean;
            p.rstd[row] = rstd;
        }
    };
    auto out = [&](int64_t at, int n, const float(&v)[8], const float(&f)[8], const float(&b)[8], float scale,
                   float mean, float rstd) {
        float o[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i] = (v[i] * scale - mean) * rstd * f[i] + b[i];
        store_upto8(p.y + row * cols + at, n, o);
    };
    // The row's statistics and outputs with its values times `scale`, kShrink or
    // kGrow, from memory again; every wave makes all the sums.  The mean is corrected
    // as in the other rows, so that equal values have no deviations; where the
    // deviations themselves need no shrinking, they are taken as they are.
    auto again_times = [&](float scale) {
        float mean = 0.0f, var = 0.0f, v[8];
#pragma unroll 1
        for (int pass = 0; pass < 3; ++pass) {
            float sum = 0.0f, squares = 0.0f;
            for (int64_t at = int64_t(threadIdx.x % 64) * 8; at < cols; at += 512) {
                const int n = cols - at < 8 ? int(cols - at) : 8;
                stream(at, n, v);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float d = i < n ? v[i] * scale - mean : 0.0f;
                    sum += d;
                    squares += d * d;
                }
            }
            sum = wave_sum(sum) * inv_n;
            var = wave_sum(squares) * inv_n;
            if (pass == 0 || (pass == 1 && mean * mean >= var)) mean += sum;
        }
        const float back = scale == kGrow ? 1.0f / kGrow : 1.0f / kShrink;
        float whole = mean * back;  // rounding may pass the largest number
        if (fabsf(mean) < kHuge) whole = fminf(fmaxf(whole, -3.402823466e38f), 3.402823466e38f);
        const bool small = scale == kShrink && var < 0x1p-100f;
        const float use = small ? 1.0f : scale;
        const float rstd = 1.0f / sqrtf(small ? var * back * back + p.eps : var + p.eps * use * use);
        keep_stats(whole, rstd * use);
        for (int64_t at = int64_t(t) * 8; at < cols; at += NT * 8) {
            const int n = cols - at < 8 ? int(cols - at) : 8;
            float f[8], b[8] = {};
            stream(at, n, v);
            load_upto8(p.w + at, n, f);
            if (p.b != nullptr) load_upto8(p.b + at, n, b);
            out(at, n, v, f, b, use, small ? whole : mean, rstd);
        }
    };
    // Mean and rstd from the sums of the deviations from `near` and of their squares;
    // false: the row's outputs need nothing more.
    auto finish = [&](float near, const float(&sums)[2], float& mean, float& rstd) {
        if (!live) return false;
        const float off = sums[0] * inv_n, left = sums[1] - sums[0] * off;
        const float ss = left < 0.0f ? 0.0f : left;  // a NaN stays one
        const bool faint = ss * inv_n + p.eps < kFaint && fabsf(near) < kFaintMean;
        if (!(ss < kHuge) || faint) {
            again_times(faint ? kGrow : kShrink);
            return false;
        }
        mean = near * near >= ss * inv_n ? near + off : near;
        rstd = 1.0f / sqrtf(ss * inv_n + p.eps);
        keep_stats(mean, rstd);
        return true;
    };

    if constexpr (VPT > 0) {
        float v[VPT][8];
        Eight<W> f[VPT], b[VPT];
        auto start = [&](int g) { return int64_t(g * NT + t) * 8; };
        auto from = [&](int g) { return start(g) <= cols - 8 ? start(g) : cols - 8; };
        auto again = [&](int g) { return int(start(g) - from(g)); };  // of the group before it; 8 and more: all
        float s[1] = {};
        if (live) {
            Eight<T> a[VPT], r[VPT];
#pragma unroll
            for (int g = 0; g < VPT; ++g) {
                a[g].load(xr + from(g));
                if constexpr (RES) r[g].load(rr + from(g));
            }
#pragma unroll
            for (int g = 0; g < VPT; ++g) {
                f[g].load(p.w + from(g));
                if (p.b != nullptr) b[g].load(p.b + from(g));
            }
#pragma unroll
            for (int g = 0; g < VPT; ++g) {
#pragma unroll
                for (int i = 0; i < 8; ++i) v[g][i] = to_f32(a[g].v[i]);
                if constexpr (DROP)
                    if (again(g) < 8) keep.apply(p.first_row + row, from(g), v[g]);
                if constexpr (RES) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) v[g][i] += to_f32(r[g].v[i]);
                }
                if constexpr (STREAM) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) v[g][i] = to_f32(static_cast<T>(v[g][i]));
                    if (again(g) < 8) store8(p.h + row * cols + from(g), v[g]);
                }
#pragma unroll
                for (int i = 0; i < 8; ++i) s[0] += i >= again(g) ? v[g][i] : 0.0f;
            }
        }
        row_sums<NT>(s);
        const float near = s[0] * inv_n;
        float ss[2] = {};
        if (live) {
#pragma unroll
            for (int g = 0; g < VPT; ++g)
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float d = i >= again(g) ? v[g][i] - near : 0.0f;
                    ss[0] += d;
                    ss[1] += d * d;
                }
        }
        row_sums<NT>(ss);
        float mean, rstd;
        if (!finish(near, ss, mean, rstd)) return;
#pragma unroll
        for (int g = 0; g < VPT; ++g) {
            if (again(g) >= 8) continue;
            float fv[8], bv[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                fv[i] = to_f32(f[g].v[i]);
                bv[i] = p.b != nullptr ? to_f32(b[g].v[i]) : 0.0f;
            }
            out(from(g), 8, v[g], fv, bv, 1.0f, mean, rstd);
        }
    } else {
        float v[8];
        auto each = [&](auto&& f) {
            if (!live) return;
            for (int64_t at = int64_t(t) * 8; at < cols; at += NT * 8) {
                const int n = cols - at < 8 ? int(cols - at) : 8;
                stream(at, n, v);
                f(at, n);
            }
        };
        float s[1] = {}, ss[2] = {};
        each([&](int64_t at, int n) {
            if constexpr (STREAM) store_upto8(p.h + row * cols + at, n, v);
#pragma unroll
            for (int i = 0; i < 8; ++i) s[0] += i < n ? v[i] : 0.0f;
        });
        row_sums<NT>(s);
        const float near = s[0] * inv_n;
        each([&](int64_t, int n) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float d = i < n ? v[i] - near : 0.0f;
                ss[0] += d;
                ss[1] += d * d;
            }
        });
        row_sums<NT>(ss);
        float mean, rstd;
        if (!finish(near, ss, mean, rstd)) return;
        each([&](int64_t at, int n) {
            float f[8], b[8] = {};
            load_upto8(p.w + at, n, f);
            if (p.b != nullptr) load_upto8(p.b + at, n, b);
            out(at, n, v, f, b, 1.0f, mean, rstd);
        });
    }
}

template <typename T, typename W, bool DROP, bool RES, int NT, int VPT>
hipError_t launch_norm(const LayerNorm& q, hipStream_t st) {
    constexpr int64_t kMost = int64_t(1) << 21;  // a launch's thread count stays below 2^32
    for (int64_t r0 = 0; r0 < q.rows; r0 += kMost) {
        const int64_t n = q.rows - r0 < kMost ? q.rows - r0 : kMost;
        const NormArgs<T, W> p{static_cast<const T*>(q.x) + r0 * q.ldx,
                               RES ? static_cast<const T*>(q.residual) + r0 * q.ldr : nullptr,
                               q.ldx, q.ldr, static_cast<const W*>(q.weight), static_cast<const W*>(q.bias), q.eps,
                               q.drop, static_cast<T*>(q.y) + r0 * q.cols,
                               DROP || RES ? static_cast<T*>(q.h) + r0 * q.cols : nullptr,
                               q.mean + r0, q.rstd + r0, r0, n, q.cols};
        hipLaunchKernelGGL((tg_layer_norm_rows<T, W, DROP, RES, NT, VPT>), dim3(unsigned(ceil_div(n, kRowsPerBlock<NT>))),
                           dim3(kBlock<NT>), 0, st, p);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

// Two groups a thread, three where two would leave more than a quarter of the
// threads without one (bf16, 8192 rows with residual: of 2501 38.4 us as 256 x 2,
// 30.9 as 128 x 3; of 5001 93.6 as 512 x 2, 78.5 as 256 x 3).
template <typename T, typename W, bool DROP, bool RES>
hipError_t norm_form(const LayerNorm& p, hipStream_t st) {
    const int64_t groups = ceil_div(p.cols, 8);
    if (p.cols < 8) return launch_norm<T, W, DROP, RES, 64, 0>(p, st);
    if (groups <= 64) return launch_norm<T, W, DROP, RES, 64, 1>(p, st);
    if (groups <= 128) return launch_norm<T, W, DROP, RES, 64, 2>(p, st);
    if (groups <= 256) return launch_norm<T, W, DROP, RES, 128, 2>(p, st);
    if (groups <= 384) return launch_norm<T, W, DROP, RES, 128, 3>(p, st);
    if (groups <= 512) return launch_norm<T, W, DROP, RES, 256, 2>(p, st);
    if (groups <= 768) return launch_norm<T, W, DROP, RES, 256, 3>(p, st);
    if (groups <= 1024) return launch_norm<T, W, DROP, RES, 512, 2>(p, st);
    return launch_norm<T, W, DROP, RES, 1024, 0>(p, st);
}

// ---- dropout -----------------------------------------------------------------

// y = round(dropout(x) + residual), eight elements a thread; a row's last group is
// moved back to end with the row, and what it shares with the one before it is
// written twice, with the same values (bf16, 8192 x 4095 with residual: 37.7 us,
// 50.8 with bounds instead).  Rows below eight elements: one group with a bound.
// bf16, 16384 x 4096 with residual: 69 us (403 MB, 5.8 TB/s).
template <typename T, bool DROP, bool RES>
__global__ __launch_bounds__(256) void tg_dropout_rows(const T* __restrict__ x, int64_t ldx, const T* __restrict__ res,
                                                       int64_t ldr, Dropout drop, T* __restrict__ y, int64_t rows,
                                                       int64_t cols, int64_t groups) {
    const Keep keep(drop);
    const int64_t stride = int64_t(gridDim.x) * 256;
    const bool tiny = cols < 8;
    for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < rows * groups; i += stride) {
        const int64_t row = i / groups, start = (i - row * groups) * 8;
        const int64_t at = tiny || start <= cols - 8 ? start : cols - 8;
        float v[8], r[8];
        if (tiny) {
            load_part(x + row * ldx, int(cols), v);
            if constexpr (RES) load_part(res + row * ldr, int(cols), r);
        } else {
            load8(x + row * ldx + at, v);
            if constexpr (RES) load8(res + row * ldr + at, r);
        }
        if constexpr (DROP) keep.apply(row, at, v);
        if constexpr (RES) {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] += r[e];
        }
        store_upto8(y + row * cols + at, tiny ? int(cols) : 8, v);
    }
}

}  // namespace

hipError_t dropout_rows(const DropoutRows& p, hipStream_t st) {
    if (p.rows == 0 || p.cols == 0) return hipSuccess;
    const int64_t groups = ceil_div(p.cols, 8), blocks = ceil_div(p.rows * groups, 256);
    return by_type(p.type, [&](auto tag) {
        using T = decltype(tag);
        return by_flag(p.drop.below > 0, [&](auto drop) {
            return by_flag(p.residual != nullptr, [&](auto res) {
                hipLaunchKernelGGL((tg_dropout_rows<T, decltype(drop)::value, decltype(res)::value>),
                                   dim3(unsigned(blocks < 65536 ? blocks : 65536)), dim3(256), 0, st,
                                   static_cast<const T*>(p.x), p.ldx, static_cast<const T*>(p.residual), p.ldr, p.drop,
                                   static_cast<T*>(p.y), p.rows, p.cols, groups);
                return hipGetLastError();
            });
        });
    });
}

hipError_t layer_norm(const LayerNorm& p, hipStream_t st) {
    if (p.rows == 0 || p.cols == 0) return hipSuccess;
    return by_type(p.type, [&](auto tag) {
        using T = decltype(tag);
        return by_flag(p.drop.below > 0, [&](auto drop) {
            return by_flag(p.residual != nullptr, [&](auto res) {
                constexpr bool DROP = decltype(drop)::value, RES = decltype(res)::value;
                return p.weight_type == p.type ? norm_form<T, T, DROP, RES>(p, st) : norm_form<T, float, DROP, RES>(p, st);
            });
        });
    });
}

}  // namespace tg
