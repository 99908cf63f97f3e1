// What the entry points of training check before they touch a device, and how
// they enter the call's device and stream (host only).
#pragma once

#include <hip/hip_runtime.h>

#include <atomic>
#include <cmath>
#include <cstdint>
#include <cstring>
#include <string>

#include "../../../include/mfhip.h"
#include "learn_ranges.h"
#include "mfh_status.h"

namespace mfh {
namespace checks {

inline int HipError(const char *fn, const char *what, hipError_t e) {
  (void)hipGetLastError();
  return SetError(MFH_ERR_HIP, std::string(fn) + ": " + what + ": " + hipGetErrorString(e));
}

inline int Invalid(const char *fn, const char *what) {
  return SetError(MFH_ERR_INVALID, std::string(fn) + ": " + what);
}

inline bool Aligned(const void *p, std::uintptr_t bytes) {
  return reinterpret_cast<std::uintptr_t>(p) % bytes == 0;
}

// Makes `device` current for a call and puts the caller's device back.
class OnDevice {
 public:
  ~OnDevice() {
    if (before_ >= 0)
      (void)hipSetDevice(before_);
  }
  hipError_t Set(int device) {
    int now = 0;
    hipError_t e = hipGetDevice(&now);
    if (e != hipSuccess || now == device)
      return e;
    e = hipSetDevice(device);
    if (e == hipSuccess)
      before_ = now;
    return e;
  }

 private:
  int before_ = -1;
};

// Whether device `dev` is a gfx950, looked up once per device.
inline bool IsGfx950(int dev) {
  constexpr int kMaxDevices = 64;
  static std::atomic<int> known[kMaxDevices] = {};  // 0 unknown, 1 yes, 2 no
  if (dev < 0 || dev >= kMaxDevices)
    return false;
  int k = known[dev].load(std::memory_order_relaxed);
  if (k == 0) {
    hipDeviceProp_t prop;
    if (hipGetDeviceProperties(&prop, dev) != hipSuccess) {
      (void)hipGetLastError();
      return false;
    }
    k = std::strncmp(prop.gcnArchName, "gfx950", 6) == 0 ? 1 : 2;
    known[dev].store(k, std::memory_order_relaxed);
  }
  return k == 1;
}

inline int NeedDevice(const char *fn, int dev) {
  static std::atomic<int> count{-1};
  int n = count.load(std::memory_order_relaxed);
  if (n < 0) {
    if (hipGetDeviceCount(&n) != hipSuccess) {
      (void)hipGetLastError();
      n = 0;
    }
    count.store(n, std::memory_order_relaxed);
  }
  if (n <= 0)
    return SetError(MFH_ERR_NO_DEVICE, std::string(fn) + ": no HIP device available");
  if (dev >= n)
    return SetError(MFH_ERR_NO_DEVICE, std::string(fn) + ": device ordinal out of range");
  return MFH_OK;
}

// The device of `p`; an error if it is not device memory, or (want >= 0)
// another device's.
inline int PointerDevice(const char *fn, const char *name, const void *p, int want, int *dev) {
  hipPointerAttribute_t attr;
  const hipError_t e = hipPointerGetAttributes(&attr, p);
  if (e != hipSuccess)
    (void)hipGetLastError();
  if (e != hipSuccess || (attr.type != hipMemoryTypeDevice && attr.type != hipMemoryTypeManaged))
    return Invalid(fn, (std::string(name) + " is not device memory").c_str());
  if (want >= 0 && attr.device != want)
    return Invalid(fn, (std::string(name) + " is on another device").c_str());
  if (dev)
    *dev = attr.device;
  return MFH_OK;
}

inline int StreamDevice(const char *fn, hipStream_t stream, int device) {
  // The standing streams belong to the device that is current at the launch.
  if (!stream || stream == hipStreamPerThread || stream == hipStreamLegacy)
    return MFH_OK;
  hipDevice_t dev = 0;
  const hipError_t e = hipStreamGetDevice(stream, &dev);
  if (e != hipSuccess)
    return HipError(fn, "stream", e);
  if (dev != device)
    return Invalid(fn, "the stream is another device's");
  return MFH_OK;
}

struct Named {
  const char *name;
  const void *p;
};

// Device, stream and pointers of a call: sets `on` to the device of the
// first pointer (or `want`), and checks the rest against it.
template <size_t N>
inline int Enter(const char *fn, int want, const Named (&ptrs)[N], hipStream_t stream, OnDevice *on) {
  int rc = NeedDevice(fn, want);
  if (rc != MFH_OK)
    return rc;
  int dev = want >= 0 ? want : -1;
  for (const Named &n : ptrs) {
    if (!n.p)
      continue;
    int d = dev;
    rc = PointerDevice(fn, n.name, n.p, dev, &d);
    if (rc != MFH_OK)
      return rc;
    dev = d;
  }
  if (!IsGfx950(dev))
    return SetError(MFH_ERR_NO_DEVICE, std::string(fn) + ": the device is not gfx950 (MI355X)");
  rc = StreamDevice(fn, stream, dev);
  if (rc != MFH_OK)
    return rc;
  const hipError_t e = on->Set(dev);
  return e == hipSuccess ? MFH_OK : HipError(fn, "hipSetDevice", e);
}

// Refuses a call that writes into another of its arrays.
template <size_t N> int CheckApart(const char *fn, const Span (&spans)[N]) {
  size_t a = 0, b = 0;
  if (!FindOverlap(spans, &a, &b))
    return MFH_OK;
  return Invalid(fn, (std::string(spans[a].name) + " overlaps " + spans[b].name).c_str());
}

// No tensor on a card of 288 GB has more.
constexpr uint64_t kMostElements = uint64_t(1) << 38;

inline bool Finite(float v) { return std::isfinite(v); }

}  // namespace checks
}  // namespace mfh
