// What the entry points of the decode path share: statuses of refusals and launches, and the current device.
#pragma once

#include "reactor_internal.h"

namespace prom {

// The device that the reactor's stream and staging belong to is current while a call
// queues its work, whatever the calling thread had chosen.
class CurrentDevice {
 public:
  explicit CurrentDevice(int device) {
    if (hipGetDevice(&before_) == hipSuccess && before_ != device) changed_ = hipSetDevice(device) == hipSuccess;
  }
  ~CurrentDevice() {
    if (changed_) (void)hipSetDevice(before_);
  }

 private:
  int before_ = 0;
  bool changed_ = false;
};

inline int refuse(uint32_t* stage, int* detail, uint32_t s, int d) {
  set_status(stage, detail, s, d);
  return PROM_ERROR;
}

inline int invalid(uint32_t* stage, int* detail) { return refuse(stage, detail, PROM_STAGE_INIT, PROM_DETAIL_INVALID_ARGUMENT); }

inline int bad_handle(uint32_t* stage, int* detail) {
  set_status(stage, detail, PROM_STAGE_INIT, PROM_INVALID_HANDLE);
  return PROM_INVALID_HANDLE;
}

inline bool aligned(const void* p, uintptr_t to) { return ((uintptr_t)p & (to - 1)) == 0; }
inline uintptr_t dtype_size(uint32_t dtype) { return dtype == PROM_DTYPE_BF16 ? 2 : 4; }

// PROM_OK, or what the caller returns: the launch's error to a status.
inline int queued(hipError_t e, uint32_t* stage, int* detail, int path) {
  if (e == hipErrorOutOfMemory) return refuse(stage, detail, PROM_STAGE_TRANSFER_IN, PROM_DETAIL_HIP_ALLOC_FAILED);
  if (e != hipSuccess) {
    (void)hipGetLastError();
    return refuse(stage, detail, PROM_STAGE_SUBMIT, PROM_DETAIL_HIP_LAUNCH_FAILED);
  }
  set_status(stage, detail, PROM_STAGE_SUBMIT, path);
  return PROM_OK;
}

}  // namespace prom
