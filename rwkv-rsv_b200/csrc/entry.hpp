// What the entry points that take a caller's device memory share: errors as return codes, and the caller's current device left as it was.
#pragma once
#include <cuda_runtime.h>

#include <stdexcept>
#include <string>

#include "cuda_error.hpp"

namespace rsv {

void set_last_error(const std::string& msg);  // defined with the C ABI

// Runs f; no exception leaves.
template <class F>
int entry_guarded(F&& f) {
    try {
        f();
        return 0;
    } catch (const CudaError& e) {
        set_last_error(e.what());
        return 2;
    } catch (const std::exception& e) {
        set_last_error(e.what());
        return 1;
    } catch (...) {
        set_last_error("unknown error");
        return 3;
    }
}

// Makes `device` current for a call.
class DeviceScope {
  public:
    explicit DeviceScope(int device) {
        const cudaError_t e = cudaGetDevice(&before_);
        int n = 0;
        if (e != cudaSuccess || (device != before_ && cudaGetDeviceCount(&n) != cudaSuccess)) {
            cudaGetLastError();
            throw CudaError(std::string("no CUDA device available (") + cudaGetErrorString(e) + "): this library has no CPU fallback");
        }
        if (device == before_) return;
        if (device < 0 || device >= n) throw std::runtime_error("device index out of range");
        RSV_CUDA(cudaSetDevice(device));
        changed_ = true;
    }
    ~DeviceScope() {
        if (changed_) cudaSetDevice(before_);
    }
    DeviceScope(const DeviceScope&) = delete;

  private:
    int before_ = 0;
    bool changed_ = false;
};

}  // namespace rsv
