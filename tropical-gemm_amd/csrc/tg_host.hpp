// tg_host.hpp -- what the C entry points share on the host: the thread's last
// error and the choice of a device (defined in tg_capi.hip).
#pragma once

#include <hip/hip_runtime.h>

#include <string>

namespace tg {

// Records msg for tg_last_error() and returns status.
int host_fail(int status, const std::string& msg);
// The same for a HIP call that failed.
int host_hip_fail(hipError_t e, const char* what);
// Checks the ordinal and makes the device current.
int host_select_device(int device);

}  // namespace tg
