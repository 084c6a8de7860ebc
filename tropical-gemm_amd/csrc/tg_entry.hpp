// tg_entry.hpp -- what the C entry points of the layers share: argument checks
// (before any HIP call), device selection and launch errors.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <exception>
#include <initializer_list>
#include <string>

#include "../../include/tropical_gemm_hip.h"
#include "tg_host.hpp"

namespace {

using tg::host_fail;

// No C++ exception leaves a C entry point.
template <typename F>
int guarded(F&& f) noexcept {
    try {
        return f();
    } catch (const std::exception& e) {
        try {
            return host_fail(TG_ERR_DRIVER, e.what());
        } catch (...) {
        }
    } catch (...) {
    }
    return TG_ERR_DRIVER;
}

int bad_argument(const std::string& msg) { return host_fail(TG_ERR_INVALID_ARGUMENT, msg); }
int bad_size(const std::string& msg) { return host_fail(TG_ERR_DIMENSION_MISMATCH, msg); }

int check_type(int type, const char* what = "type") {
    if (type == TG_FLOAT32 || type == TG_BF16 || type == TG_F16) return TG_OK;
    return bad_argument(std::string("unknown ") + what + " " + std::to_string(type));
}

int check_weight_type(int type, int weight_type) {
    if (int rc = check_type(type)) return rc;
    if (weight_type == type || weight_type == TG_FLOAT32) return TG_OK;
    return bad_argument("the weight's type must be the activations' or f32");
}

int check_dims(std::initializer_list<int64_t> dims) {
    for (int64_t d : dims) {
        if (d < 0) return bad_size("negative dimension");
        if (d > 0x7fffffffLL) return bad_size("dimension exceeds 2^31-1");
    }
    return TG_OK;
}

// Row strides count elements; the elements of a row are neighbours.
int check_ld(const char* name, int64_t ld, int64_t cols) {
    if (ld >= cols && ld <= (int64_t(1) << 40)) return TG_OK;
    return bad_size(std::string("row stride of ") + name + " is " + std::to_string(ld) +
                    ": at least the row's " + std::to_string(cols) + " elements (and at most 2^40) are needed");
}

int check_ptr(const char* name, const void* p, bool needed) {
    if (p != nullptr || !needed) return TG_OK;
    return bad_argument(std::string(name) + " is NULL");
}

int check_eps(float eps) {
    if (eps >= 0.0f && eps <= 3.4e38f) return TG_OK;
    return bad_argument("eps must be finite and not negative");
}

int check_ws(size_t need, const void* ws, size_t bytes) {
    if (need == 0) return TG_OK;
    if (ws == nullptr || bytes < need)
        return bad_argument("workspace too small: " + std::to_string(need) + " bytes are needed, got " +
                            std::to_string(ws == nullptr ? 0 : bytes));
    if ((reinterpret_cast<uintptr_t>(ws) & 255u) != 0) return bad_argument("workspace must be 256-byte aligned");
    return TG_OK;
}

int on_device(int device, const char* what, hipError_t (*run)(const void*), const void* arg) {
    const tg::OnDevice on(device);
    if (on.status() != TG_OK) return on.status();
    const hipError_t e = run(arg);
    return e == hipSuccess ? int(TG_OK) : tg::host_hip_fail(e, what);
}

// Runs f on the device; its launch error becomes the call's.
template <typename F>
int launched(int device, const char* what, F&& f) {
    return on_device(device, what, [](const void* p) { return (*static_cast<const F*>(p))(); }, &f);
}

hipStream_t as_stream(void* s) { return static_cast<hipStream_t>(s); }

#define TG_CHECK(expr)                    \
    do {                                  \
        if (int rc_ = (expr)) return rc_; \
    } while (0)

// A plan's name, the thread's until its next one.
template <typename F>
const char* named(F&& f) noexcept {
    try {
        static thread_local std::string name;
        name = f();
        return name.c_str();
    } catch (...) {
        return "invalid";
    }
}

}  // namespace
