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

// Checks the ordinal and makes the device the thread's current one; at its end the
// one before is current again, so that a call on a device leaves its caller where
// it was.
class OnDevice {
  public:
    explicit OnDevice(int device);
    ~OnDevice();
    OnDevice(const OnDevice&) = delete;
    OnDevice& operator=(const OnDevice&) = delete;
    int status() const { return status_; }

  private:
    int before_ = -1;  // -1: nothing to go back to
    int status_;       // initialised after before_, which it may set
};

}  // namespace tg
