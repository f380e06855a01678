// per_device.cuh -- what the host keeps for each device (host code only).
#pragma once
#include <atomic>

#include <cuda_runtime_api.h>

namespace moe_b200 {

constexpr int kPerDevice = 64;  // devices whose values are kept

// A count that belongs to the current device: asked for by ask() (> 0) at its
// first use there.
class DeviceCount {
public:
    template <typename Ask> int get(Ask&& ask) {
        int dev = 0;
        if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kPerDevice) return ask();
        int n = known_[dev].load(std::memory_order_relaxed);
        if (n == 0) known_[dev].store(n = ask(), std::memory_order_relaxed);
        return n;
    }

private:
    std::atomic<int> known_[kPerDevice] = {};
};

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
        const bool kept = dev >= 0 && dev < kPerDevice;
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
    std::atomic<bool> open_[kPerDevice] = {};
};

}  // namespace moe_b200
