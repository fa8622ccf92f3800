// The calling thread's device for the length of a C entry: the entry's own device inside, the caller's again behind it.  The thread's last HIP
// error stays what it was: one that the caller's earlier calls left is still there for the caller, the entry's own is in its status alone.
// (An entry that fails while another error was pending leaves none: the runtime holds one.)
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
    if (hipPeekAtLastError() != before_) (void)hipGetLastError();
  }
  Status Enter(int device) {
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
  const hipError_t before_ = hipPeekAtLastError();
  int restore_ = -1;
};

}  // namespace hps
