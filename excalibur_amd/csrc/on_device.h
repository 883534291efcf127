#pragma once
#include <hip/hip_runtime.h>

// The entry points that hold one work on their context's device whatever device the calling thread is on.
struct exhip_on_device {
    int before = -1;
    hipError_t error = hipSuccess;
    explicit exhip_on_device(int device) {
        int now = device;
        error = hipGetDevice(&now);
        if (error == hipSuccess && now != device) {
            error = hipSetDevice(device);
            if (error == hipSuccess) before = now;
        }
    }
    ~exhip_on_device() {
        if (before >= 0) (void)hipSetDevice(before);
    }
};
