// Host-side pieces shared by the operators on caller-owned device tensors
// (leo_gated_scan.cu, leo_logits.cu): argument failures, CUDA error checks,
// the device switch of one call, and the frame that turns an exception into
// the C ABI's -1 with a message.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>
#include <exception>
#include <stdexcept>
#include <string>

#include "leo_kernels.h"

namespace leo_operator {

struct Failure : std::runtime_error {
    using std::runtime_error::runtime_error;
};

inline void require(bool ok, const char* what) {
    if (!ok) throw Failure(what);
}

inline void check(cudaError_t e, const char* what) {
    if (e != cudaSuccess) throw Failure(std::string(what) + ": " + cudaGetErrorString(e));
}

// Makes `device` current for one call and restores the caller's device.
class DeviceScope {
  public:
    explicit DeviceScope(int device) {
        check(cudaGetDevice(&previous_), "cudaGetDevice");
        if (device != previous_) {
            check(cudaSetDevice(device), "cudaSetDevice");
            switched_ = true;
        }
    }
    ~DeviceScope() {
        if (switched_) cudaSetDevice(previous_);
    }
    DeviceScope(const DeviceScope&) = delete;
    DeviceScope& operator=(const DeviceScope&) = delete;

  private:
    int previous_ = 0;
    bool switched_ = false;
};

// SMs of the current device, asked for once a device.
inline int sm_count() {
    static std::atomic<int> known[64];
    int device = 0, sms = 0;
    check(cudaGetDevice(&device), "cudaGetDevice");
    if (device < 64 && (sms = known[device].load(std::memory_order_relaxed)) > 0) return sms;
    check(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device), "SM count");
    if (device < 64) known[device].store(sms, std::memory_order_relaxed);
    return sms;
}

// Lets `kernel` have `bytes` of dynamic shared memory on the current device;
// `done` remembers for which devices that has been said.
template <typename Kernel>
void allow_shared(Kernel kernel, size_t bytes, std::atomic<uint64_t>& done) {
    int device = 0;
    check(cudaGetDevice(&device), "cudaGetDevice");
    const uint64_t bit = device < 64 ? 1ull << device : 0;
    if (done.load(std::memory_order_relaxed) & bit) return;
    check(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes), "shared memory");
    done.fetch_or(bit, std::memory_order_relaxed);
}

template <typename Body>
int guarded(Body&& body) noexcept {
    try {
        body();
        return 0;
    } catch (const std::exception& e) {
        try {
            leo_set_last_error(e.what());
        } catch (...) {
        }
        return -1;
    } catch (...) {
        return -1;
    }
}

}  // namespace leo_operator
