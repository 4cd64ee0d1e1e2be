// The largest dynamic LDS that a kernel may ask for: a setting of the driver's for each kernel and device.
#pragma once
#include <hip/hip_runtime_api.h>
#include <stddef.h>
#include <atomic>
#include <mutex>

// Raised to the most that was asked for, from whichever thread needs more first.  The bytes differ from call to call, so reading, setting
// and recording go under one lock: two threads side by side could otherwise leave the smaller of their values set and the larger one
// recorded, and later launches in between would skip the setting that they need.  A call whose bytes are recorded takes no lock.
struct LdsLimit {
    static constexpr int DEVICES = 64;
    std::atomic<size_t> have[DEVICES] = {};
    std::mutex mu;
    // `beside`: the kernel's static share (up to 64 KB together need no setting)
    hipError_t allow(const void *kern, size_t bytes, size_t beside = 0) {
        if (bytes + beside <= 65536) return hipSuccess;
        int dev = 0;
        if (hipError_t e = hipGetDevice(&dev)) return e;
        if (dev < 0 || dev >= DEVICES) return hipErrorInvalidDevice;
        if (have[dev].load(std::memory_order_acquire) >= bytes) return hipSuccess;
        std::lock_guard<std::mutex> lock(mu);
        if (have[dev].load(std::memory_order_relaxed) >= bytes) return hipSuccess;
        if (hipError_t e = hipFuncSetAttribute(kern, hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes)) return e;
        have[dev].store(bytes, std::memory_order_release);
        return hipSuccess;
    }
};
