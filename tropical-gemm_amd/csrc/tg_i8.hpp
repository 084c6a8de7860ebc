// tg_i8.hpp -- host interface of the 8-bit layer's kernels: rows
// (tg_i8_rows.hip) and products (tg_i8_gemm.hip).  The entry points in
// tg_i8_capi.hip check the arguments first; sizes here are non-negative.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <string>

namespace tg {

// Least row maximum a scale is made from: a row of zeros gets zeros and a
// scale that is small and not zero.
constexpr float kI8TinyTop = 1e-30f;

struct I8Norm {
    int type, weight_type;  // tg_float
    const void *x, *residual, *weight;
    int64_t ldx, ldr;
    float eps;
    int8_t* q;
    float* scale;
    void* h;
    int64_t rows, cols;
};
hipError_t i8_rms_norm(const I8Norm& p, hipStream_t st);
// x, ldx, q, scale, rows and cols of p only.
hipError_t i8_quantize(const I8Norm& p, hipStream_t st);
hipError_t i8_dequantize(int type, const int8_t* q, int64_t ldq, const float* scale, void* y,
                         int64_t rows, int64_t cols, hipStream_t st);

struct I8NormBackward {
    int type, weight_type;
    const void *grad_y, *h, *weight, *grad_h;
    int64_t ldg, ldh, ldgh;
    float eps;
    void *grad_x, *grad_weight;
    int64_t rows, cols;
};
size_t i8_rms_norm_backward_ws(int64_t rows, int64_t cols);
hipError_t i8_rms_norm_backward(const I8NormBackward& p, void* ws, hipStream_t st);

// C (m x n) = (A (m x k) B^T (n x k)) * a_scale * b_scale + bias.
struct I8Gemm {
    int type;
    const int8_t* a;
    int64_t lda;
    const float* a_scale;
    const int8_t* b;
    int64_t ldb;
    const float* b_scale;
    const void* bias;
    void* c;
    int64_t m, n, k;
};
size_t i8_gemm_ws(const I8Gemm& p);
hipError_t i8_gemm(const I8Gemm& p, void* ws, hipStream_t st);
std::string i8_gemm_plan(const I8Gemm& p);

// out (rows x cols) = sum over r < depth of G(i, r) * scale[r] * q[r, j], with
// G(i, r) = g[i * ldg + r], or g[r * ldg + i] when `transposed`.
struct I8Grad {
    int type;
    const void* g;
    int64_t ldg;
    bool transposed;
    const int8_t* q;
    int64_t ldq;
    const float* scale;
    void* out;
    int64_t rows, cols, depth;
};
size_t i8_grad_ws(const I8Grad& p);
hipError_t i8_grad(const I8Grad& p, void* ws, hipStream_t st);
std::string i8_grad_plan(const I8Grad& p);

// out (m x n, of type) = A B^T + bias in bf16, for operands laid out as tg_i8_tiles
// takes them: rows of `steps` steps of 128 bytes (the last of `tail` that count);
// a row of A is the sum of `planes` such rows (3: for f32 alone), one behind the
// other.
struct PlaneGemm {
    int type, planes;
    const void *a, *b;
    int64_t lda, ldb;  // bytes
    int64_t steps;
    int tail;
    const void* bias;  // of type, or null
    void* out;
    int64_t m, n;
};
// Bytes for partial sums; the time of it in us.
size_t plane_gemm_ws(int64_t m, int64_t n, int64_t steps, int planes);
double plane_gemm_time(int64_t m, int64_t n, int64_t steps, int planes);
hipError_t plane_gemm(const PlaneGemm& p, void* part, hipStream_t st);
std::string plane_gemm_plan(int64_t m, int64_t n, int64_t steps, int planes);
// out = 0 (an empty sum).
hipError_t plane_gemm_zero(int type, void* out, int64_t m, int64_t n, hipStream_t st);

}  // namespace tg
