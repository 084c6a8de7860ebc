// tg_layers.hpp -- host interface of layer norm and dropout (tg_layers.hip).
// The entry points in tg_layers_capi.hip check the arguments first; sizes here
// are non-negative.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace tg {

// Which elements are dropped: those whose 16 random bits are below `below`;
// the others are multiplied by `factor`.
struct Dropout {
    uint32_t below;  // 0: none are, and nothing is multiplied
    float factor;
    uint64_t seed, offset;
    const uint64_t* seed_at;  // not null: the seed is there, on the GPU
};

struct DropoutRows {
    int type;  // tg_float
    const void *x, *residual;
    int64_t ldx, ldr;
    Dropout drop;
    void* y;
    int64_t rows, cols;
};
hipError_t dropout_rows(const DropoutRows& p, hipStream_t st);

struct LayerNorm {
    int type, weight_type;
    const void *x, *residual, *weight, *bias;
    int64_t ldx, ldr;
    float eps;
    Dropout drop;
    void *y, *h;
    float *mean, *rstd;
    int64_t rows, cols;
};
hipError_t layer_norm(const LayerNorm& p, hipStream_t st);

struct LayerNormBackward {
    int type, weight_type;
    const void *grad_y, *h, *weight, *grad_h;
    int64_t ldg, ldh, ldgh;
    const float *mean, *rstd;
    Dropout drop;
    void *grad_x, *grad_residual, *grad_weight, *grad_bias;  // grad_x null: as grad_residual
    int64_t rows, cols;
};
size_t layer_norm_backward_ws(int64_t rows, int64_t cols);
hipError_t layer_norm_backward(const LayerNormBackward& p, void* ws, hipStream_t st);

}  // namespace tg
