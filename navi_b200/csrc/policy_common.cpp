// Errors and device properties of the policy operators' library.
#include <mutex>

#include "policy_internal.h"

namespace policy {
namespace {

thread_local std::string g_error;

constexpr int kMaxDevices = 64;
std::mutex g_mu;
DeviceInfo g_info[kMaxDevices];
bool g_known[kMaxDevices];

}  // namespace

int fail(int code, const std::string& msg)
{
    g_error = msg;
    return code;
}

int cuda_fail(cudaError_t e, const char* what)
{
    return fail(POLICY_ERR_CUDA, std::string(what) + ": " + cudaGetErrorString(e));
}

DeviceInfo device_info(int device)
{
    DeviceInfo info;
    if (device < 0 || device >= kMaxDevices) {
        info.status = fail(POLICY_ERR_INVALID, "device must be a CUDA device index");
        return info;
    }
    std::lock_guard<std::mutex> lock(g_mu);
    if (g_known[device]) return g_info[device];
    int major = 0;
    cudaError_t e = cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, device);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&info.sms, cudaDevAttrMultiProcessorCount, device);
    if (e != cudaSuccess) {
        cudaGetLastError();
        info.status = cuda_fail(e, "cudaDeviceGetAttribute");
        return info;
    }
    if (major != 10) {
        info.status = fail(POLICY_ERR_UNSUPPORTED, "the policy operators need an sm_100 device");
        return info;
    }
    g_info[device] = info;
    g_known[device] = true;
    return info;
}

}  // namespace policy

extern "C" int policy_version(void) { return POLICY_ABI_VERSION; }
extern "C" const char* policy_last_error(void) { return policy::g_error.c_str(); }
