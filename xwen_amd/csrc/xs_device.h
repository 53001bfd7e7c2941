// The current device of the calling thread, for the length of a call.
#ifndef XS_DEVICE_H
#define XS_DEVICE_H

#include <hip/hip_runtime.h>

namespace xs_host {

// A call runs on its context's device and leaves the thread's current one as it
// was.
struct OnDevice {
  int before = -1;
  bool ok;
  explicit OnDevice(int device) { ok = hipGetDevice(&before) == hipSuccess && (before == device || hipSetDevice(device) == hipSuccess); }
  ~OnDevice() {
    int now = -1;
    if (before >= 0 && hipGetDevice(&now) == hipSuccess && now != before) (void)hipSetDevice(before);
  }
};

}  // namespace xs_host

#endif
