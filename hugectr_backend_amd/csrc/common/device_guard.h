// The calling thread's device for the length of a C entry: the entry's own device inside, the caller's again behind it.  An error that an
// earlier HIP call left in the thread is not this entry's (its launches ask for the last error), and the entry's own stays in its status.
#pragma once
#include <hip/hip_runtime_api.h>

#include "status.h"

namespace hps {

class DeviceGuard {
 public:
  DeviceGuard() = default;
  DeviceGuard(const DeviceGuard&) = delete;
  DeviceGuard& operator=(const DeviceGuard&) = delete;
  ~DeviceGuard() {
    if (restore_ >= 0) (void)hipSetDevice(restore_);
    (void)hipGetLastError();
  }
  Status Enter(int device) {
    (void)hipGetLastError();
    int now = 0;
    const bool any = hipGetDevice(&now) == hipSuccess;
    if (any && now == device) return Status::Ok();
    int ndev = 0;
    if (!any || hipGetDeviceCount(&ndev) != hipSuccess || ndev <= 0)
      return Error(Code::kUnavailable, "this call needs a HIP device and none is visible; there is no CPU fallback");
    if (device < 0 || device >= ndev) return Error(Code::kInvalidArg, "device ", device, " is not visible (", ndev, " HIP devices)");
    const hipError_t e = hipSetDevice(device);
    if (e != hipSuccess) return Error(Code::kInternal, "selecting device ", device, " failed: ", hipGetErrorString(e));
    restore_ = now;
    return Status::Ok();
  }

 private:
  int restore_ = -1;
};

}  // namespace hps
