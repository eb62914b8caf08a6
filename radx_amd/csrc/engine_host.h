// engine_host.h — what the host sides of the engine's translation units share: the calling
// thread's error text, argument and HIP error returns, and the choice of the device to launch on.
#ifndef RADX_ENGINE_HOST_H
#define RADX_ENGINE_HOST_H

#include <hip/hip_runtime.h>

#include <stdio.h>

namespace radx_engine __attribute__((visibility("hidden"))) {

inline thread_local char g_error[256] = "";

inline int fail(hipError_t e, const char* what) {
    snprintf(g_error, sizeof(g_error), "%s: %s", what, hipGetErrorString(e));
    return static_cast<int>(e);
}
inline int bad_arg(const char* what) {
    snprintf(g_error, sizeof(g_error), "invalid argument: %s", what);
    return static_cast<int>(hipErrorInvalidValue);
}

#define RADX_TRY(expr)                                   \
    do {                                                 \
        const hipError_t e_ = (expr);                    \
        if (e_ != hipSuccess) return fail(e_, #expr);    \
    } while (0)

class DeviceGuard {
public:
    explicit DeviceGuard(int device) {
        if (hipGetDevice(&prev_) != hipSuccess) prev_ = -1;
        if (prev_ != device) { status_ = hipSetDevice(device); changed_ = status_ == hipSuccess; }
    }
    ~DeviceGuard() { if (changed_ && prev_ >= 0) (void)hipSetDevice(prev_); }
    hipError_t status() const { return status_; }
private:
    int prev_ = -1;
    bool changed_ = false;
    hipError_t status_ = hipSuccess;
};

// The free functions take raw device pointers and no handle: each launches on the device that
// owns its buffer, whatever device is current on the calling thread.
inline int device_of(const void* p, int* device) {
    hipPointerAttribute_t attr;
    if (hipPointerGetAttributes(&attr, p) != hipSuccess) {
        (void)hipGetLastError();
        return bad_arg("buffer is not memory HIP knows (hipMalloc / hipHostMalloc)");
    }
    *device = attr.device;
    return 0;
}
#define RADX_ON_DEVICE_OF(ptr)                                     \
    int dev_ = 0;                                                  \
    if (const int rc_ = device_of((ptr), &dev_)) return rc_;       \
    DeviceGuard guard_(dev_);                                      \
    RADX_TRY(guard_.status())

}  // namespace radx_engine

#endif  // RADX_ENGINE_HOST_H
