// lv_serve_host.h — what the entry points of a serving step share on the host.
#pragma once

#include "lv_common.h"

namespace lv {

// makes a device current while it lives; the caller's is current again afterwards
struct DeviceScope {
    int before = -1;
    hipError_t error;
    explicit DeviceScope(int device)
    {
        error = hipGetDevice(&before);
        if (error == hipSuccess && before != device) error = hipSetDevice(device);
        else before = -1;
    }
    ~DeviceScope()
    {
        if (before >= 0) (void)hipSetDevice(before);
    }
    DeviceScope(const DeviceScope &) = delete;
    DeviceScope &operator=(const DeviceScope &) = delete;
};

}  // namespace lv
