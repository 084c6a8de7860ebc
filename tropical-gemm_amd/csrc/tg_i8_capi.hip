// tg_i8_capi.hip -- C entry points of the 8-bit layer: argument checks (before
// any HIP call), device selection and dispatch.
#include <string>

#include "tg_entry.hpp"
#include "tg_i8.hpp"

namespace {

// 2^14 is the largest product of two 8-bit integers; 2^17 of them could pass
// an i32 sum.
constexpr int64_t kMostK = (int64_t(1) << 17) - 1;

// The operands laid out along the sum have row strides below 2^23 bytes.
constexpr int64_t kMostDepth = int64_t(1) << 20;

// The norm's backward pass counts a row's elements in f32 and has 64 threads
// for each column of its widest launch.
constexpr int64_t kMostBackwardCols = int64_t(1) << 24;

int check_gemm(const tg::I8Gemm& p) {
    TG_CHECK(check_type(p.type));
    TG_CHECK(check_dims({p.m, p.n, p.k}));
    if (p.k > kMostK) return bad_size("k is " + std::to_string(p.k) + ": sums of 8-bit products are exact up to k = " + std::to_string(kMostK));
    TG_CHECK(check_ld("a", p.lda, p.k));
    return check_ld("b", p.ldb, p.k);
}

// Gradient of `rows` x `cols`: g is rows x depth (or depth x rows).
int check_grad(const tg::I8Grad& p, const char* q_name) {
    TG_CHECK(check_type(p.type));
    TG_CHECK(check_dims({p.rows, p.cols, p.depth}));
    if (p.depth > kMostDepth) return bad_size("the gradient's sum has " + std::to_string(p.depth) + " terms: at most 2^20 are supported");
    TG_CHECK(check_ld("grad_c", p.ldg, p.transposed ? p.rows : p.depth));
    return check_ld(q_name, p.ldq, p.cols);
}

int run_grad(int device, const tg::I8Grad& p, const char* q_name, const char* scale_name, const char* out_name,
             void* ws, size_t ws_bytes, void* stream) {
    TG_CHECK(check_grad(p, q_name));
    const bool any = p.rows > 0 && p.cols > 0;
    TG_CHECK(check_ptr("grad_c", p.g, any && p.depth > 0));
    TG_CHECK(check_ptr(q_name, p.q, any && p.depth > 0));
    TG_CHECK(check_ptr(scale_name, p.scale, any && p.depth > 0));
    TG_CHECK(check_ptr(out_name, p.out, any));
    TG_CHECK(check_ws(tg::i8_grad_ws(p), ws, ws_bytes));
    return launched(device, "tg_i8_backward", [&] { return tg::i8_grad(p, ws, as_stream(stream)); });
}

tg::I8Grad grad_a(tg_float type, const void* grad_c, int64_t ldg, const int8_t* b, int64_t ldb,
                  const float* b_scale, void* out, int64_t m, int64_t n, int64_t k) {
    return {type, grad_c, ldg, false, b, ldb, b_scale, out, m, k, n};
}
tg::I8Grad grad_b(tg_float type, const void* grad_c, int64_t ldg, const int8_t* a, int64_t lda,
                  const float* a_scale, void* out, int64_t m, int64_t n, int64_t k) {
    return {type, grad_c, ldg, true, a, lda, a_scale, out, n, k, m};
}

}  // namespace

extern "C" {

int tg_i8_quantize(int device, tg_float type, const void* x, int64_t ldx, int8_t* q, float* scale,
                   int64_t rows, int64_t cols, void* stream) {
    return guarded([&]() -> int {
        TG_CHECK(check_type(type));
        TG_CHECK(check_dims({rows, cols}));
        TG_CHECK(check_ld("x", ldx, cols));
        TG_CHECK(check_ptr("x", x, rows > 0 && cols > 0));
        TG_CHECK(check_ptr("q", q, rows > 0 && cols > 0));
        TG_CHECK(check_ptr("scale", scale, rows > 0));
        const tg::I8Norm p{type, type, x, nullptr, nullptr, ldx, 0, 0.0f, q, scale, nullptr, rows, cols};
        return launched(device, "tg_i8_quantize", [&] { return tg::i8_quantize(p, as_stream(stream)); });
    });
}

int tg_i8_dequantize(int device, tg_float type, const int8_t* q, int64_t ldq, const float* scale, void* y,
                     int64_t rows, int64_t cols, void* stream) {
    return guarded([&]() -> int {
        TG_CHECK(check_type(type));
        TG_CHECK(check_dims({rows, cols}));
        TG_CHECK(check_ld("q", ldq, cols));
        const bool any = rows > 0 && cols > 0;
        TG_CHECK(check_ptr("q", q, any));
        TG_CHECK(check_ptr("scale", scale, any));
        TG_CHECK(check_ptr("y", y, any));
        return launched(device, "tg_i8_dequantize",
                        [&] { return tg::i8_dequantize(type, q, ldq, scale, y, rows, cols, as_stream(stream)); });
    });
}

int tg_i8_rms_norm(int device, tg_float type, tg_float weight_type, const void* x, int64_t ldx,
                   const void* residual, int64_t ldr, const void* weight, float eps, int8_t* q, float* scale,
                   void* h, int64_t rows, int64_t cols, void* stream) {
    return guarded([&]() -> int {
        TG_CHECK(check_weight_type(type, weight_type));
        TG_CHECK(check_dims({rows, cols}));
        TG_CHECK(check_ld("x", ldx, cols));
        if (residual != nullptr) TG_CHECK(check_ld("residual", ldr, cols));
        TG_CHECK(check_eps(eps));
        const bool any = rows > 0 && cols > 0;
        TG_CHECK(check_ptr("x", x, any));
        TG_CHECK(check_ptr("weight", weight, any));
        TG_CHECK(check_ptr("q", q, any));
        TG_CHECK(check_ptr("scale", scale, rows > 0));
        TG_CHECK(check_ptr("h", h, any && residual != nullptr));
        const tg::I8Norm p{type, weight_type, x, residual, weight, ldx, ldr, eps, q, scale, h, rows, cols};
        return launched(device, "tg_i8_rms_norm", [&] { return tg::i8_rms_norm(p, as_stream(stream)); });
    });
}

size_t tg_i8_rms_norm_backward_workspace_size(int64_t rows, int64_t cols) {
    return rows < 0 || cols < 0 ? size_t(-1) : tg::i8_rms_norm_backward_ws(rows, cols);
}

int tg_i8_rms_norm_backward(int device, tg_float type, tg_float weight_type, const void* grad_y, int64_t ldg,
                            const void* h, int64_t ldh, const void* weight, float eps, const void* grad_h,
                            int64_t ldgh, void* grad_x, void* grad_weight, int64_t rows, int64_t cols,
                            void* workspace, size_t workspace_bytes, void* stream) {
    return guarded([&]() -> int {
        TG_CHECK(check_weight_type(type, weight_type));
        TG_CHECK(check_dims({rows, cols}));
        TG_CHECK(check_ld("grad_y", ldg, cols));
        TG_CHECK(check_ld("h", ldh, cols));
        if (grad_h != nullptr) TG_CHECK(check_ld("grad_h", ldgh, cols));
        TG_CHECK(check_eps(eps));
        if (cols > kMostBackwardCols) return bad_size("cols is " + std::to_string(cols) + ": at most 2^24 are supported");
        const bool any = rows > 0 && cols > 0;
        TG_CHECK(check_ptr("grad_y", grad_y, any));
        TG_CHECK(check_ptr("h", h, any));
        TG_CHECK(check_ptr("weight", weight, any));
        TG_CHECK(check_ptr("grad_x", grad_x, any));
        TG_CHECK(check_ptr("grad_weight", grad_weight, cols > 0));
        TG_CHECK(check_ws(tg::i8_rms_norm_backward_ws(rows, cols), workspace, workspace_bytes));
        const tg::I8NormBackward p{type, weight_type, grad_y, h, weight, grad_h, ldg, ldh, ldgh, eps, grad_x,
                                   grad_weight, rows, cols};
        return launched(device, "tg_i8_rms_norm_backward",
                        [&] { return tg::i8_rms_norm_backward(p, workspace, as_stream(stream)); });
    });
}

size_t tg_i8_gemm_workspace_size(const int8_t* a, int64_t lda, const int8_t* b, int64_t ldb, int64_t m,
                                 int64_t n, int64_t k) {
    const tg::I8Gemm p{TG_BF16, a, lda, nullptr, b, ldb, nullptr, nullptr, nullptr, m, n, k};
    return m < 0 || n < 0 || k < 0 || k > kMostK ? size_t(-1) : tg::i8_gemm_ws(p);
}

int tg_i8_gemm(int device, tg_float type, const int8_t* a, int64_t lda, const float* a_scale, const int8_t* b,
               int64_t ldb, const float* b_scale, const void* bias, void* c, int64_t m, int64_t n, int64_t k,
               void* workspace, size_t workspace_bytes, void* stream) {
    return guarded([&]() -> int {
        const tg::I8Gemm p{type, a, lda, a_scale, b, ldb, b_scale, bias, c, m, n, k};
        TG_CHECK(check_gemm(p));
        const bool any = m > 0 && n > 0;
        TG_CHECK(check_ptr("a", a, any && k > 0));
        TG_CHECK(check_ptr("b", b, any && k > 0));
        TG_CHECK(check_ptr("a_scale", a_scale, any));
        TG_CHECK(check_ptr("b_scale", b_scale, any));
        TG_CHECK(check_ptr("c", c, any));
        TG_CHECK(check_ws(tg::i8_gemm_ws(p), workspace, workspace_bytes));
        return launched(device, "tg_i8_gemm", [&] { return tg::i8_gemm(p, workspace, as_stream(stream)); });
    });
}

const char* tg_i8_gemm_plan(const int8_t* a, int64_t lda, const int8_t* b, int64_t ldb, int64_t m, int64_t n,
                            int64_t k) {
    const tg::I8Gemm p{TG_BF16, a, lda, nullptr, b, ldb, nullptr, nullptr, nullptr, m, n, k};
    return named([&] { return check_gemm(p) == TG_OK ? tg::i8_gemm_plan(p) : std::string("invalid"); });
}

const char* tg_i8_backward_plan(tg_float type, int want_a, const void* grad_c, int64_t ldg, int64_t m, int64_t n,
                                int64_t k) {
    const tg::I8Grad p = want_a != 0 ? grad_a(type, grad_c, ldg, nullptr, k, nullptr, nullptr, m, n, k)
                                     : grad_b(type, grad_c, ldg, nullptr, k, nullptr, nullptr, m, n, k);
    return named([&] { return check_grad(p, "q") == TG_OK ? tg::i8_grad_plan(p) : std::string("invalid"); });
}

size_t tg_i8_backward_a_workspace_size(tg_float type, const void* grad_c, int64_t ldg, int64_t m, int64_t n,
                                       int64_t k) {
    return m < 0 || n < 0 || k < 0 ? size_t(-1)
                                   : tg::i8_grad_ws(grad_a(type, grad_c, ldg, nullptr, k, nullptr, nullptr, m, n, k));
}

int tg_i8_backward_a(int device, tg_float type, const void* grad_c, int64_t ldg, const int8_t* b, int64_t ldb,
                     const float* b_scale, void* grad_a_out, int64_t m, int64_t n, int64_t k, void* workspace,
                     size_t workspace_bytes, void* stream) {
    return guarded([&]() -> int {
        return run_grad(device, grad_a(type, grad_c, ldg, b, ldb, b_scale, grad_a_out, m, n, k), "b", "b_scale",
                        "grad_a", workspace, workspace_bytes, stream);
    });
}

size_t tg_i8_backward_b_workspace_size(tg_float type, const void* grad_c, int64_t ldg, int64_t m, int64_t n,
                                       int64_t k) {
    return m < 0 || n < 0 || k < 0 ? size_t(-1)
                                   : tg::i8_grad_ws(grad_b(type, grad_c, ldg, nullptr, k, nullptr, nullptr, m, n, k));
}

int tg_i8_backward_b(int device, tg_float type, const void* grad_c, int64_t ldg, const int8_t* a, int64_t lda,
                     const float* a_scale, void* grad_b_out, int64_t m, int64_t n, int64_t k, void* workspace,
                     size_t workspace_bytes, void* stream) {
    return guarded([&]() -> int {
        return run_grad(device, grad_b(type, grad_c, ldg, a, lda, a_scale, grad_b_out, m, n, k), "a", "a_scale",
                        "grad_b", workspace, workspace_bytes, stream);
    });
}

}  // extern "C"
