// A kernel launch whose status is the launch's own.  `<<<>>>` leaves it in the thread's last error, where it cannot be told from an error that
// the caller's own earlier calls left there and that the caller has yet to look at.
#pragma once
#include <hip/hip_runtime_api.h>
#include <stdint.h>

#include <tuple>

namespace hps {

template <typename... P, typename... A>
hipError_t Launch(void (*kernel)(P...), uint32_t blocks, uint32_t threads, hipStream_t stream, A... args) {
  static_assert(sizeof...(P) == sizeof...(A), "one argument per parameter");
  std::tuple<P...> held(static_cast<P>(args)...);
  return std::apply(
      [&](P&... p) {
        void* at[] = {const_cast<void*>(static_cast<const void*>(&p))...};
        return hipLaunchKernel(reinterpret_cast<const void*>(kernel), dim3(blocks), dim3(threads), at, 0, stream);
      },
      held);
}

}  // namespace hps
