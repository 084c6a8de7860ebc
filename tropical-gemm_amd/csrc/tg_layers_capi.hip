// tg_layers_capi.hip -- C entry points of layer norm and dropout: argument checks
// (before any HIP call), device selection and dispatch.
#include <cmath>
#include <string>

#include "tg_entry.hpp"
#include "tg_layers.hpp"

namespace {

// A row's elements are counted in f32, and a launch has 64 threads for each
// column of the weight's gradients.
constexpr int64_t kMostCols = int64_t(1) << 24;

int check_cols(int64_t cols) {
    if (cols <= kMostCols) return TG_OK;
    return bad_size("cols is " + std::to_string(cols) + ": at most 2^24 are supported");
}

int check_p(double p) {
    if (p >= 0.0 && p <= 1.0) return TG_OK;
    return bad_argument("p must lie between 0 and 1");
}

tg::Dropout dropout_of(double p, uint64_t seed, const uint64_t* seed_at, uint64_t offset) {
    const double below = std::rint(p * 65536.0);
    return {uint32_t(below), below < 65536.0 ? float(65536.0 / (65536.0 - below)) : 0.0f, seed, offset, seed_at};
}

}  // namespace

extern "C" {

int tg_dropout(int device, tg_float type, const void* x, int64_t ldx, const void* residual, int64_t ldr, double p,
               uint64_t seed, const uint64_t* seed_at, uint64_t offset, void* y, int64_t rows, int64_t cols,
               void* stream) {
    return guarded([&]() -> int {
        TG_CHECK(check_type(type));
        TG_CHECK(check_dims({rows, cols}));
        TG_CHECK(check_ld("x", ldx, cols));
        if (residual != nullptr) TG_CHECK(check_ld("residual", ldr, cols));
        TG_CHECK(check_p(p));
        const bool any = rows > 0 && cols > 0;
        TG_CHECK(check_ptr("x", x, any));
        TG_CHECK(check_ptr("y", y, any));
        const tg::DropoutRows q{type, x, residual, ldx, ldr, dropout_of(p, seed, seed_at, offset), y, rows, cols};
        return launched(device, "tg_dropout", [&] { return tg::dropout_rows(q, as_stream(stream)); });
    });
}

int tg_layer_norm(int device, tg_float type, tg_float weight_type, const void* x, int64_t ldx, const void* residual,
                  int64_t ldr, const void* weight, const void* bias, float eps, double p, uint64_t seed,
                  const uint64_t* seed_at, uint64_t offset, void* y, void* h, float* mean, float* rstd, int64_t rows,
                  int64_t cols, void* stream) {
    return guarded([&]() -> int {
        TG_CHECK(check_weight_type(type, weight_type));
        TG_CHECK(check_dims({rows, cols}));
        TG_CHECK(check_cols(cols));
        TG_CHECK(check_ld("x", ldx, cols));
        if (residual != nullptr) TG_CHECK(check_ld("residual", ldr, cols));
        TG_CHECK(check_eps(eps));
        TG_CHECK(check_p(p));
        const tg::Dropout drop = dropout_of(p, seed, seed_at, offset);
        const bool any = rows > 0 && cols > 0;
        TG_CHECK(check_ptr("x", x, any));
        TG_CHECK(check_ptr("weight", weight, any));
        TG_CHECK(check_ptr("y", y, any));
        TG_CHECK(check_ptr("h", h, any && (residual != nullptr || drop.below > 0)));
        TG_CHECK(check_ptr("mean", mean, any));
        TG_CHECK(check_ptr("rstd", rstd, any));
        const tg::LayerNorm q{type, weight_type, x, residual, weight, bias, ldx, ldr, eps, drop, y, h, mean, rstd, rows, cols};
        return launched(device, "tg_layer_norm", [&] { return tg::layer_norm(q, as_stream(stream)); });
    });
}

size_t tg_layer_norm_backward_workspace_size(int64_t rows, int64_t cols) {
    return rows < 0 || rows > 0x7fffffffLL || cols < 0 || cols > kMostCols ? size_t(-1) : tg::layer_norm_backward_ws(rows, cols);
}

int tg_layer_norm_backward(int device, tg_float type, tg_float weight_type, const void* grad_y, int64_t ldg,
                           const void* h, int64_t ldh, const float* mean, const float* rstd, const void* weight,
                           const void* grad_h, int64_t ldgh, double p, uint64_t seed, const uint64_t* seed_at,
                           uint64_t offset, void* grad_x, void* grad_residual, void* grad_weight, void* grad_bias,
                           int64_t rows, int64_t cols, void* workspace, size_t workspace_bytes, void* stream) {
    return guarded([&]() -> int {
        TG_CHECK(check_weight_type(type, weight_type));
        TG_CHECK(check_dims({rows, cols}));
        TG_CHECK(check_cols(cols));
        TG_CHECK(check_ld("grad_y", ldg, cols));
        TG_CHECK(check_ld("h", ldh, cols));
        if (grad_h != nullptr) TG_CHECK(check_ld("grad_h", ldgh, cols));
        TG_CHECK(check_p(p));
        const tg::Dropout drop = dropout_of(p, seed, seed_at, offset);
        const bool any = rows > 0 && cols > 0;
        TG_CHECK(check_ptr("grad_y", grad_y, any));
        TG_CHECK(check_ptr("h", h, any));
        TG_CHECK(check_ptr("mean", mean, any));
        TG_CHECK(check_ptr("rstd", rstd, any));
        TG_CHECK(check_ptr("weight", weight, any));
        TG_CHECK(check_ptr("grad_x", grad_x, any && drop.below > 0));
        TG_CHECK(check_ptr("grad_residual", grad_residual, any));
        TG_CHECK(check_ptr("grad_weight", grad_weight, cols > 0));
        TG_CHECK(check_ptr("grad_bias", grad_bias, cols > 0));
        TG_CHECK(check_ws(tg::layer_norm_backward_ws(rows, cols), workspace, workspace_bytes));
        const tg::LayerNormBackward q{type, weight_type, grad_y, h, weight, grad_h, ldg, ldh, ldgh, mean, rstd, drop,
                                      grad_x, grad_residual, grad_weight, grad_bias, rows, cols};
        return launched(device, "tg_layer_norm_backward",
                        [&] { return tg::layer_norm_backward(q, workspace, as_stream(stream)); });
    });
}

}  // extern "C"
