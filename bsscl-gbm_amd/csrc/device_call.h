// What the entry points on device buffers share: the current device for the
// length of a call, and errors in the place of exceptions.
#pragma once

#include <exception>
#include <new>
#include <string>

#include <hip/hip_runtime_api.h>

#include "bsscl_internal.h"

namespace bsscl {

// Makes `device` current and puts the caller's device back at the end.
class DeviceScope {
 public:
  int enter(int device) {
    hipError_t e = hipGetDevice(&before_);
    if (e == hipSuccess && device != before_) {
      e = hipSetDevice(device);
      changed_ = e == hipSuccess;
    }
    if (e == hipSuccess) return BSSCL_OK;
    (void)hipGetLastError();
    return set_error(BSSCL_EDEVICE,
                     "device " + std::to_string(device) + ": " + hipGetErrorString(e));
  }
  ~DeviceScope() {
    if (changed_) (void)hipSetDevice(before_);
  }

 private:
  int before_ = 0;
  bool changed_ = false;
};

// f() with C++ exceptions as error codes.
template <typename F>
int no_throw(F &&f) {
  try {
    return f();
  } catch (const std::bad_alloc &) {
    return set_error(BSSCL_ENOMEM, "host allocation failed");
  } catch (const std::exception &e) {
    return set_error(BSSCL_EINTERNAL, e.what());
  } catch (...) {
    return set_error(BSSCL_EINTERNAL, "unknown error");
  }
}

}  // namespace bsscl
