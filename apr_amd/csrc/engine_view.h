// engine_view.h -- what a translation unit beside engine.hip needs of an engine: its GPU, its stream, and where its error text goes.
#pragma once
#include <hip/hip_runtime.h>

#include "../../include/apr.h"

namespace apr {

struct EngineView {
    int device;
    hipStream_t stream;
    int n_cus;
};
// false for a null handle
bool engine_view(const apr_engine *e, EngineView &v) noexcept;
// Keeps `text` as the engine's last error (this thread's, for a null handle) and returns `code`.
int engine_fail(apr_engine *e, int code, const char *text) noexcept;
// operators.hip, once for an engine, with its device current
bool operators_prepare() noexcept;

// Makes a device current for a scope and puts the caller's back: torch and other libraries in the process go by the current device.
class DeviceScope {
    int before_ = -1;
    bool ok_ = false;

public:
    explicit DeviceScope(int device) noexcept
    {
        if (hipGetDevice(&before_) != hipSuccess) { before_ = -1; return; }
        ok_ = before_ == device || hipSetDevice(device) == hipSuccess;
        if (before_ == device) before_ = -1;
    }
    ~DeviceScope()
    {
        if (before_ >= 0) (void)hipSetDevice(before_);
    }
    DeviceScope(const DeviceScope &) = delete;
    DeviceScope &operator=(const DeviceScope &) = delete;
    bool ok() const noexcept { return ok_; }
};

// A kernel's launch, with its own error: the thread's last error (hipGetLastError) may be of somebody else's earlier call, who has yet to
// read it.
template <typename P>
struct as_is { typedef P type; };
template <typename... P>
hipError_t launch_kernel(hipStream_t stream, void (*kernel)(P...), dim3 grid, dim3 block, unsigned lds, typename as_is<P>::type... p) noexcept
{
    void *args[] = {(void *)&p...};
    const hipError_t r = hipLaunchKernel(reinterpret_cast<const void *>(kernel), grid, block, args, lds, stream);
    if (r != hipSuccess) (void)hipGetLastError();   // this one is reported here
    return r;
}

// The launches of one call, up to the first error
class Launches {
    hipStream_t stream_;
    hipError_t error_ = hipSuccess;

public:
    explicit Launches(hipStream_t stream) noexcept : stream_(stream) {}
    template <typename... P>
    void operator()(void (*kernel)(P...), dim3 grid, dim3 block, unsigned lds, typename as_is<P>::type... p) noexcept
    {
        if (error_ == hipSuccess) error_ = launch_kernel<P...>(stream_, kernel, grid, block, lds, p...);
    }
    hipError_t error() const noexcept { return error_; }
};

}  // namespace apr
