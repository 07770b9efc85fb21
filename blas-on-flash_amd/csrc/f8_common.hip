// f8_common.hip -- argument checks that the entry points of bof_f8.h share.
#include "f8_common.h"

namespace bof {

int refuse(const char *call, const char *why) {
  set_error(std::string(call) + ": " + why);
  return BOF_EINVAL;
}

// (the two predefined streams, 1 = legacy and 2 = per thread, belong to the current device like the null stream)
LaunchDevice::LaunchDevice(hipStream_t st) {
  hipError_t e = hipGetDevice(&before_);
  if (e != hipSuccess) { rc_ = hip_fail(e, "hipGetDevice"); return; }
  dev_ = before_;
  if (reinterpret_cast<uintptr_t>(st) > 2) {
    hipDevice_t d = 0;
    e = hipStreamGetDevice(st, &d);
    if (e != hipSuccess) { rc_ = hip_fail(e, "hipStreamGetDevice"); return; }
    dev_ = d;
  }
  if (dev_ != before_ && (e = hipSetDevice(dev_)) != hipSuccess) {
    rc_ = hip_fail(e, "hipSetDevice");
    dev_ = before_;
  }
}
LaunchDevice::~LaunchDevice() {
  if (dev_ != before_) (void) hipSetDevice(before_);
}

// One attribute query costs 0.06 us: every array of every call is looked at.
int LaunchDevice::reaches(const void *p, const char *call, const char *name) {
  hipPointerAttribute_t at{};
  const hipError_t e = hipPointerGetAttributes(&at, p);
  if (e != hipSuccess) (void) hipGetLastError();
  if (e == hipSuccess && ((at.type == hipMemoryTypeDevice && at.device == dev_) || at.type == hipMemoryTypeHost ||
                          at.type == hipMemoryTypeManaged || at.type == hipMemoryTypeUnified))
    return BOF_OK;
  return refuse(call, (std::string(name) + " is not memory of the stream's device").c_str());
}

}  // namespace bof
