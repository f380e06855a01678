// per_device.cuh -- what the host keeps for each device (host code only).
#pragma once
#include <atomic>

#include <cuda_runtime_api.h>

namespace moe_b200 {

// Lets a kernel use as much dynamic shared memory as a block of the current
// device can have.  The limit belongs to the kernel and the device, not to a
// call: set to what one call needs, another host thread may lower it between
// that call's setting and its launch, which then fails.  So it is set to the
// same, highest, value by everyone, at the kernel's first launch on a device
// (later ones save the driver's call too).  One object per kernel.
class SmemLimit {
public:
    cudaError_t open(const void* kernel) {
        int dev = 0;
        cudaError_t err = cudaGetDevice(&dev);
        if (err != cudaSuccess) return err;
        const bool kept = dev >= 0 && dev < kDevices;
        if (kept && open_[dev].load(std::memory_order_acquire)) return cudaSuccess;
        int most = 0;
        cudaFuncAttributes of_kernel{};
        err = cudaDeviceGetAttribute(&most, cudaDevAttrMaxSharedMemoryPerBlockOptin, dev);
        if (err == cudaSuccess) err = cudaFuncGetAttributes(&of_kernel, kernel);
        if (err == cudaSuccess)
            err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       most - int(of_kernel.sharedSizeBytes));
        if (err == cudaSuccess && kept) open_[dev].store(true, std::memory_order_release);
        return err;
    }

private:
    static constexpr int kDevices = 64;
    std::atomic<bool> open_[kDevices] = {};
};

}  // namespace moe_b200
