// tg_f8_capi.hip -- C entry points of the layer in 8-bit floating point: argument
// checks (before any HIP call), device selection and dispatch.
#include <string>

#include "tg_entry.hpp"
#include "tg_f8.hpp"

namespace {

// Tiles address a panel's rows and scales in 32 bits.
constexpr int64_t kMostSum = int64_t(1) << 20;
constexpr int64_t kMostScaleRow = int64_t(1) << 22;
constexpr int64_t kMostCols = int64_t(1) << 30;

int check_scale(const char* name, const tg::F8Scale& s) {
    if (s.row >= 0 && s.row <= kMostScaleRow && s.col >= 0 && s.col <= (int64_t(1) << 40)) return TG_OK;
    return bad_size(std::string("strides of ") + name + " are " + std::to_string(s.row) + " and " + std::to_string(s.col) +
                    ": 0 to 2^22 and 0 to 2^40 are supported");
}

// What the size functions answer for: the calls refuse the rest.
bool sizes_fit(int type, int64_t m, int64_t n, int64_t k, int64_t sum) {
    auto dim = [](int64_t d) { return d >= 0 && d <= 0x7fffffffLL; };
    return (type == TG_FLOAT32 || type == TG_BF16 || type == TG_F16) && dim(m) && dim(n) && dim(k) && sum <= kMostSum;
}

int check_block_rows(int64_t n) {
    if (n == 1 || n == tg::kF8Block) return TG_OK;
    return bad_argument("block_rows is " + std::to_string(n) + ": 1 or 128 is needed");
}

int check_gemm(const tg::F8Gemm& p) {
    TG_CHECK(check_type(p.type));
    TG_CHECK(check_dims({p.m, p.n, p.k}));
    if (p.k > kMostSum) return bad_size("k is " + std::to_string(p.k) + ": at most 2^20 is supported");
    TG_CHECK(check_ld("a", p.lda, p.k));
    TG_CHECK(check_ld("b", p.ldb, p.k));
    TG_CHECK(check_scale("a_scale", p.a_scale));
    return check_scale("b_scale", p.b_scale);
}

// Gradient of `rows` x `cols`: g is rows x depth (or depth x rows).
int check_grad(const tg::F8Grad& p, const char* q_name, const char* scale_name) {
    TG_CHECK(check_type(p.type));
    TG_CHECK(check_dims({p.rows, p.cols, p.depth}));
    if (p.depth > kMostSum) return bad_size("the gradient's sum has " + std::to_string(p.depth) + " terms: at most 2^20 are supported");
    TG_CHECK(check_ld("grad_c", p.ldg, p.transposed ? p.rows : p.depth));
    TG_CHECK(check_ld(q_name, p.q.ld, p.cols));
    return check_scale(scale_name, p.q.scale);
}

int run_grad(int device, const tg::F8Grad& p, const char* q_name, const char* scale_name, const char* out_name,
             void* ws, size_t ws_bytes, void* stream) {
    TG_CHECK(check_grad(p, q_name, scale_name));
    const bool any = p.rows > 0 && p.cols > 0;
    TG_CHECK(check_ptr("grad_c", p.g, any && p.depth > 0));
    TG_CHECK(check_ptr(q_name, p.q.q, any && p.depth > 0));
    TG_CHECK(check_ptr(scale_name, p.q.scale.p, any && p.depth > 0));
    TG_CHECK(check_ptr(out_name, p.out, any));
    TG_CHECK(check_ws(tg::f8_grad_ws(p), ws, ws_bytes));
    return launched(device, "tg_f8_backward", [&] { return tg::f8_grad(p, ws, as_stream(stream)); });
}

tg::F8Grad grad_a(tg_float type, const void* grad_c, int64_t ldg, const uint8_t* b, int64_t ldb, tg::F8Scale scale,
                  void* out, int64_t m, int64_t n, int64_t k) {
    return {type, grad_c, ldg, false, {b, ldb, scale, tg::kF8Block}, out, m, k, n};
}
tg::F8Grad grad_b(tg_float type, const void* grad_c, int64_t ldg, const uint8_t* a, int64_t lda, tg::F8Scale scale,
                  void* out, int64_t m, int64_t n, int64_t k) {
    return {type, grad_c, ldg, true, {a, lda, scale, 1}, out, n, k, m};
}

}  // namespace

extern "C" {

int tg_f8_quantize(int device, tg_float type, const void* x, int64_t ldx, int64_t block_rows, uint8_t* q,
                   uint8_t* scale, int64_t rows, int64_t cols, void* stream) {
    return guarded([&]() -> int {
        TG_CHECK(check_type(type));
        TG_CHECK(check_dims({rows, cols}));
        TG_CHECK(check_ld("x", ldx, cols));
        TG_CHECK(check_block_rows(block_rows));
        if (cols > kMostCols) return bad_size("cols is " + std::to_string(cols) + ": at most 2^30 are supported");
        const bool any = rows > 0 && cols > 0;
        TG_CHECK(check_ptr("x", x, any));
        TG_CHECK(check_ptr("q", q, any));
        TG_CHECK(check_ptr("scale", scale, any));
        const tg::F8Quantize p{type, x, ldx, int(block_rows), q, scale, rows, cols};
        return launched(device, "tg_f8_quantize", [&] { return tg::f8_quantize(p, as_stream(stream)); });
    });
}

int tg_f8_dequantize(int device, tg_float type, const uint8_t* q, int64_t ldq, const uint8_t* scale,
                     int64_t scale_row, int64_t scale_col, int64_t block_rows, void* y, int64_t rows, int64_t cols,
                     void* stream) {
    return guarded([&]() -> int {
        const tg::F8Matrix p{q, ldq, {scale, scale_row, scale_col}, int(block_rows)};
        TG_CHECK(check_type(type));
        TG_CHECK(check_dims({rows, cols}));
        TG_CHECK(check_ld("q", ldq, cols));
        TG_CHECK(check_block_rows(block_rows));
        TG_CHECK(check_scale("scale", p.scale));
        const bool any = rows > 0 && cols > 0;
        TG_CHECK(check_ptr("q", q, any));
        TG_CHECK(check_ptr("scale", scale, any));
        TG_CHECK(check_ptr("y", y, any));
        return launched(device, "tg_f8_dequantize",
                        [&] { return tg::f8_dequantize(type, p, y, rows, cols, as_stream(stream)); });
    });
}

size_t tg_f8_gemm_workspace_size(tg_float type, const uint8_t* a, int64_t lda, const uint8_t* b, int64_t ldb,
                                 int64_t m, int64_t n, int64_t k) {
    const tg::F8Gemm p{type, a, lda, {}, b, ldb, {}, nullptr, nullptr, m, n, k};
    return sizes_fit(type, m, n, k, k) ? tg::f8_gemm_ws(p) : size_t(-1);
}

int tg_f8_gemm(int device, tg_float type, const uint8_t* a, int64_t lda, const uint8_t* a_scale, int64_t a_scale_row,
               int64_t a_scale_col, const uint8_t* b, int64_t ldb, const uint8_t* b_scale, int64_t b_scale_row,
               int64_t b_scale_col, const void* bias, void* c, int64_t m, int64_t n, int64_t k, void* workspace,
               size_t workspace_bytes, void* stream) {
    return guarded([&]() -> int {
        const tg::F8Gemm p{type, a, lda, {a_scale, a_scale_row, a_scale_col}, b, ldb, {b_scale, b_scale_row, b_scale_col},
                           bias, c, m, n, k};
        TG_CHECK(check_gemm(p));
        const bool any = m > 0 && n > 0;
        TG_CHECK(check_ptr("a", a, any && k > 0));
        TG_CHECK(check_ptr("b", b, any && k > 0));
        TG_CHECK(check_ptr("a_scale", a_scale, any && k > 0));
        TG_CHECK(check_ptr("b_scale", b_scale, any && k > 0));
        TG_CHECK(check_ptr("c", c, any));
        TG_CHECK(check_ws(tg::f8_gemm_ws(p), workspace, workspace_bytes));
        return launched(device, "tg_f8_gemm", [&] { return tg::f8_gemm(p, workspace, as_stream(stream)); });
    });
}

const char* tg_f8_gemm_plan(tg_float type, const uint8_t* a, int64_t lda, const uint8_t* b, int64_t ldb, int64_t m,
                            int64_t n, int64_t k) {
    const tg::F8Gemm p{type, a, lda, {}, b, ldb, {}, nullptr, nullptr, m, n, k};
    return named([&] { return check_gemm(p) == TG_OK ? tg::f8_gemm_plan(p) : std::string("invalid"); });
}

const char* tg_f8_backward_plan(tg_float type, int want_a, const void* grad_c, int64_t ldg, int64_t m, int64_t n,
                                int64_t k) {
    const tg::F8Grad p = want_a != 0 ? grad_a(type, grad_c, ldg, nullptr, k, {}, nullptr, m, n, k)
                                     : grad_b(type, grad_c, ldg, nullptr, k, {}, nullptr, m, n, k);
    return named([&] { return check_grad(p, "q", "scale") == TG_OK ? tg::f8_grad_plan(p) : std::string("invalid"); });
}

size_t tg_f8_backward_a_workspace_size(tg_float type, const void* grad_c, int64_t ldg, int64_t m, int64_t n,
                                       int64_t k) {
    if (!sizes_fit(type, m, n, k, n)) return size_t(-1);
    return tg::f8_grad_ws(grad_a(type, grad_c, ldg, nullptr, k, {}, nullptr, m, n, k));
}

int tg_f8_backward_a(int device, tg_float type, const void* grad_c, int64_t ldg, const uint8_t* b, int64_t ldb,
                     const uint8_t* b_scale, int64_t b_scale_row, int64_t b_scale_col, void* out, int64_t m, int64_t n,
                     int64_t k, void* workspace, size_t workspace_bytes, void* stream) {
    return guarded([&]() -> int {
        return run_grad(device, grad_a(type, grad_c, ldg, b, ldb, {b_scale, b_scale_row, b_scale_col}, out, m, n, k), "b",
                        "b_scale", "grad_a", workspace, workspace_bytes, stream);
    });
}

size_t tg_f8_backward_b_workspace_size(tg_float type, const void* grad_c, int64_t ldg, int64_t m, int64_t n,
                                       int64_t k) {
    if (!sizes_fit(type, m, n, k, m)) return size_t(-1);
    return tg::f8_grad_ws(grad_b(type, grad_c, ldg, nullptr, k, {}, nullptr, m, n, k));
}

int tg_f8_backward_b(int device, tg_float type, const void* grad_c, int64_t ldg, const uint8_t* a, int64_t lda,
                     const uint8_t* a_scale, int64_t a_scale_row, int64_t a_scale_col, void* out, int64_t m, int64_t n,
                     int64_t k, void* workspace, size_t workspace_bytes, void* stream) {
    return guarded([&]() -> int {
        return run_grad(device, grad_b(type, grad_c, ldg, a, lda, {a_scale, a_scale_row, a_scale_col}, out, m, n, k), "a",
                        "a_scale", "grad_b", workspace, workspace_bytes, stream);
    });
}

}  // extern "C"
