// Shared by the policy operators: errors, the caller's device, and the launch constants.
#pragma once

#include <cuda_runtime.h>

#include <cstdint>
#include <string>

#include "policy.h"

namespace policy {

int fail(int code, const std::string& msg);
int cuda_fail(cudaError_t e, const char* what);

// The SM count of `device` and whether it is an sm_100 one, read once per process.
struct DeviceInfo {
    int sms = 0;
    int status = POLICY_OK;
};
DeviceInfo device_info(int device);

// The word of policy_stall_word, allocated at the first call; null where that fails.
int32_t* stall_word();
// POLICY_ERR_STALLED, once, after a kernel has set it.
int check_stall();

// Makes `device` the calling thread's current device for the scope and puts the caller's
// current device back when the scope ends.
class DeviceScope {
public:
    explicit DeviceScope(int device)
    {
        if (cudaGetDevice(&prev_) != cudaSuccess) {
            cudaGetLastError();
            prev_ = -1;
        }
        if (prev_ != device) {
            err_ = cudaSetDevice(device);
            switched_ = err_ == cudaSuccess && prev_ >= 0;
        }
    }
    ~DeviceScope()
    {
        if (switched_) cudaSetDevice(prev_);
    }
    DeviceScope(const DeviceScope&) = delete;
    DeviceScope& operator=(const DeviceScope&) = delete;
    cudaError_t error() const { return err_; }

private:
    int prev_ = -1;
    bool switched_ = false;
    cudaError_t err_ = cudaSuccess;
};

inline size_t dtype_bytes(int dtype) { return dtype == POLICY_F32 ? 4 : 2; }
inline bool known_dtype(int dtype) { return dtype == POLICY_F32 || dtype == POLICY_BF16; }

}  // namespace policy
