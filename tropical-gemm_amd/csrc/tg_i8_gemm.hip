// tg_i8_gemm.hip -- the 8-bit layer's products: rows times rows in 8-bit
// integers with scales, and the two gradients, which read one 8-bit operand.
#include "../../include/tropical_gemm_hip.h"
#include "tg_i8.hpp"
#include "tg_i8_types.hpp"

namespace tg {
namespace {

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

typedef int32_t i32x4 __attribute__((ext_vector_type(4)));

template <typename F>
hipError_t by_type(int type, F&& f) {
    switch (type) {
        case TG_BF16: return f(bf16_t());
        case TG_F16: return f(f16_t());
        default: return f(float());
    }
}

// C = (A B^T) * a_scale * b_scale + bias on 64 x 64 tiles, 64 k at a time; four
// waves of 32 x 32.  v_mfma_i32_16x16x64_i8: lane l holds 16 consecutive k of
// row l % 16 from k = (l / 16) * 16, and the outputs of column l % 16, rows
// (l / 16) * 4 ... + 3.  Operands pass through LDS byte by byte, so any
// strides, alignment and sizes are right.
template <typename T>
__global__ __launch_bounds__(256) void tg_i8_gemm_tiles(const int8_t* __restrict__ A, int64_t lda,
                                                        const float* __restrict__ sa,
                                                        const int8_t* __restrict__ B, int64_t ldb,
                                                        const float* __restrict__ sb,
                                                        const T* __restrict__ bias, T* __restrict__ C,
                                                        int64_t M, int64_t N, int64_t K, int64_t tiles_n) {
    __shared__ __align__(16) int8_t la[64][80], lb[64][80];
    const int t = threadIdx.x, lane = t % 64, wave = t / 64;
    const int64_t m0 = int64_t(blockIdx.x) / tiles_n * 64, n0 = int64_t(blockIdx.x) % tiles_n * 64;
    const int wm = wave / 2 * 32, wn = wave % 2 * 32;
    i32x4 acc[2][2] = {};
    for (int64_t k0 = 0; k0 < K; k0 += 64) {
        for (int i = t; i < 64 * 64; i += 256) {
            const int r = i / 64, k = i % 64;
            la[r][k] = m0 + r < M && k0 + k < K ? A[(m0 + r) * lda + k0 + k] : int8_t(0);
            lb[r][k] = n0 + r < N && k0 + k < K ? B[(n0 + r) * ldb + k0 + k] : int8_t(0);
        }
        __syncthreads();
        i32x4 fa[2], fb[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            fa[i] = *reinterpret_cast<const i32x4*>(&la[wm + i * 16 + lane % 16][lane / 16 * 16]);
            fb[i] = *reinterpret_cast<const i32x4*>(&lb[wn + i * 16 + lane % 16][lane / 16 * 16]);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j)
                acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fa[i], fb[j], acc[i][j], 0, 0, 0);
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int64_t m = m0 + wm + i * 16 + lane / 16 * 4 + e, n = n0 + wn + j * 16 + lane % 16;
                if (m >= M || n >= N) continue;
                float v = float(acc[i][j][e]) * sa[m] * sb[n];
                if (bias != nullptr) v += to_f32(bias[n]);
                C[m * N + n] = static_cast<T>(v);
            }
}

// out[i, j] = sum over r of G(i, r) * scale[r] * q[r, j] in f32: 64 x 64 tiles,
// 16 r at a time, 4 x 4 outputs a thread.
template <typename T, bool TRANS>
__global__ __launch_bounds__(256) void tg_i8_grad_tiles(const T* __restrict__ G, int64_t ldg,
                                                        const int8_t* __restrict__ Q, int64_t ldq,
                                                        const float* __restrict__ scale, T* __restrict__ out,
                                                        int64_t rows, int64_t cols, int64_t depth,
                                                        int64_t tiles_n) {
    __shared__ float lg[16][65], lq[16][65];
    const int t = threadIdx.x, tx = t % 16, ty = t / 16;
    const int64_t i0 = int64_t(blockIdx.x) / tiles_n * 64, j0 = int64_t(blockIdx.x) % tiles_n * 64;
    float acc[4][4] = {};
    for (int64_t r0 = 0; r0 < depth; r0 += 16) {
        for (int e = t; e < 16 * 64; e += 256) {
            const int r = TRANS ? e / 64 : e % 16, i = TRANS ? e % 64 : e / 16;
            const bool in = i0 + i < rows && r0 + r < depth;
            lg[r][i] = in ? to_f32(G[TRANS ? (r0 + r) * ldg + i0 + i : (i0 + i) * ldg + r0 + r]) : 0.0f;
            const int rq = e / 64, j = e % 64;
            lq[rq][j] = j0 + j < cols && r0 + rq < depth ? float(Q[(r0 + rq) * ldq + j0 + j]) * scale[r0 + rq] : 0.0f;
        }
        __syncthreads();
        for (int r = 0; r < 16; ++r)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] += lg[r][ty + 16 * i] * lq[r][tx + 16 * j];
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int64_t m = i0 + ty + 16 * i, n = j0 + tx + 16 * j;
            if (m < rows && n < cols) out[m * cols + n] = static_cast<T>(acc[i][j]);
        }
}

}  // namespace

size_t i8_gemm_ws(const I8Gemm&) { return 0; }

hipError_t i8_gemm(const I8Gemm& p, void*, hipStream_t st) {
    if (p.m == 0 || p.n == 0) return hipSuccess;
    return by_type(p.type, [&](auto tag) {
        using T = decltype(tag);
        const int64_t tn = ceil_div(p.n, 64);
        hipLaunchKernelGGL((tg_i8_gemm_tiles<T>), dim3(unsigned(ceil_div(p.m, 64) * tn)), dim3(256), 0, st, p.a,
                           p.lda, p.a_scale, p.b, p.ldb, p.b_scale, static_cast<const T*>(p.bias),
                           static_cast<T*>(p.c), p.m, p.n, p.k, tn);
        return hipGetLastError();
    });
}

size_t i8_grad_ws(const I8Grad&) { return 0; }

hipError_t i8_grad(const I8Grad& p, void*, hipStream_t st) {
    if (p.rows == 0 || p.cols == 0) return hipSuccess;
    return by_type(p.type, [&](auto tag) {
        using T = decltype(tag);
        const int64_t tn = ceil_div(p.cols, 64);
        const auto kernel = p.transposed ? &tg_i8_grad_tiles<T, true> : &tg_i8_grad_tiles<T, false>;
        hipLaunchKernelGGL(kernel, dim3(unsigned(ceil_div(p.rows, 64) * tn)), dim3(256), 0, st,
                           static_cast<const T*>(p.g), p.ldg, p.q, p.ldq, p.scale, static_cast<T*>(p.out),
                           p.rows, p.cols, p.depth, tn);
        return hipGetLastError();
    });
}

}  // namespace tg
