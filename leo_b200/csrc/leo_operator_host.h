// Host-side pieces shared by the operators on caller-owned device tensors
// (leo_gated_scan.cu, leo_logits.cu): argument failures, CUDA error checks,
// the device switch of one call, and the frame that turns an exception into
// the C ABI's -1 with a message.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

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
