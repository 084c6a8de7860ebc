// tg_f8.hpp -- host interface of the layer in 8-bit floating point: blocks
// (tg_f8_rows.hip) and products (tg_f8_gemm.hip).  The entry points in
// tg_f8_capi.hip check the arguments first; sizes here are non-negative.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <string>

namespace tg {

constexpr int kF8Block = 128;             // elements of a row with one scale
constexpr int kF8LeastExponent = -100;    // of a scale that is made here

// The scale of row block r and column block c, as an e8m0 byte, is p[r * row + c * col].
struct F8Scale {
    const uint8_t* p;
    int64_t row, col;
};

struct F8Quantize {
    int type;  // tg_float
    const void* x;
    int64_t ldx;
    int block_rows;  // 1 or kF8Block
    uint8_t *q, *scale;  // scale: [column block][row block]
    int64_t rows, cols;
};
hipError_t f8_quantize(const F8Quantize& p, hipStream_t st);

struct F8Matrix {
    const uint8_t* q;
    int64_t ld;
    F8Scale scale;
    int block_rows;
};
hipError_t f8_dequantize(int type, const F8Matrix& q, void* y, int64_t rows, int64_t cols, hipStream_t st);

// C (m x n) = A (m x k) B^T (n x k) + bias: A's scales for 1 x 128, B's for 128 x 128.
struct F8Gemm {
    int type;
    const uint8_t* a;
    int64_t lda;
    F8Scale a_scale;
    const uint8_t* b;
    int64_t ldb;
    F8Scale b_scale;
    const void* bias;
    void* c;
    int64_t m, n, k;
};
size_t f8_gemm_ws(const F8Gemm& p);
hipError_t f8_gemm(const F8Gemm& p, void* ws, hipStream_t st);
std::string f8_gemm_plan(const F8Gemm& p);

// out (rows x cols) = sum over r < depth of G(i, r) * q[r, j] * its scale, with
// G(i, r) = g[i * ldg + r], or g[r * ldg + i] when `transposed`.
struct F8Grad {
    int type;
    const void* g;
    int64_t ldg;
    bool transposed;
    F8Matrix q;
    void* out;
    int64_t rows, cols, depth;
};
size_t f8_grad_ws(const F8Grad& p);
hipError_t f8_grad(const F8Grad& p, void* ws, hipStream_t st);
std::string f8_grad_plan(const F8Grad& p);

}  // namespace tg
