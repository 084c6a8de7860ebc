// tg_layers_rows.hpp -- what layer norm's forward and backward pass share.
#pragma once

#include <type_traits>

#include "../../include/tropical_gemm_hip.h"
#include "tg_dropout.hpp"
#include "tg_i8_types.hpp"
#include "tg_layers.hpp"

namespace tg {
namespace {

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// f(T()) for the element type.
template <typename F>
hipError_t by_type(int type, F&& f) {
    switch (type) {
        case TG_BF16: return f(bf16_t());
        case TG_F16: return f(f16_t());
        default: return f(float());
    }
}

// f(std::true_type()) or f(std::false_type()).
template <typename F>
hipError_t by_flag(bool flag, F&& f) {
    return flag ? f(std::true_type()) : f(std::false_type());
}

// A group of eight as it is loaded, at any address.
template <typename T>
struct Eight {
    typedef T t8 __attribute__((ext_vector_type(8)));
    t8 v;
    __device__ __forceinline__ void load(const T* p) {
        typedef uint32_t words __attribute__((ext_vector_type(sizeof(T) * 2)));
        typedef uint32_t words_any __attribute__((ext_vector_type(sizeof(T) * 2), aligned(sizeof(T))));
        v = __builtin_bit_cast(t8, words(*reinterpret_cast<const words_any*>(p)));
    }
    // The first n of them, zeros behind.
    __device__ __forceinline__ void load(const T* p, int n) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = i < n ? p[i] : T(0.0f);
    }
};

}  // namespace
}  // namespace tg
