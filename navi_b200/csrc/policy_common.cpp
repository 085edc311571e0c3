// Errors and device properties of the policy operators' library.
#include <atomic>
#include <mutex>

#include "policy_internal.h"

namespace policy {
namespace {

thread_local std::string g_error;

constexpr int kMaxDevices = 64;
std::mutex g_mu;
DeviceInfo g_info[kMaxDevices];
bool g_known[kMaxDevices];
std::atomic<int32_t*> g_stall{nullptr};

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

int32_t* stall_word()
{
    int32_t* word = g_stall.load(std::memory_order_acquire);
    if (word) return word;
    std::lock_guard<std::mutex> lock(g_mu);
    if ((word = g_stall.load(std::memory_order_acquire))) return word;
    // the first call may be under capture, where an allocation is an error in every other mode
    cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
    cudaThreadExchangeStreamCaptureMode(&mode);
    void* p = nullptr;
    const cudaError_t e = cudaHostAlloc(&p, sizeof(int32_t), cudaHostAllocPortable | cudaHostAllocMapped);
    cudaThreadExchangeStreamCaptureMode(&mode);
    if (e != cudaSuccess) {
        cudaGetLastError();
        return nullptr;
    }
    word = static_cast<int32_t*>(p);
    *word = 0;
    g_stall.store(word, std::memory_order_release);
    return word;
}

int check_stall()
{
    int32_t* word = g_stall.load(std::memory_order_acquire);
    if (!word || !__atomic_load_n(word, __ATOMIC_ACQUIRE) || !__atomic_exchange_n(word, 0, __ATOMIC_ACQ_REL)) return POLICY_OK;
    return fail(POLICY_ERR_STALLED, "a wait inside an earlier attention kernel ran out of time: rows of its results are NaN");
}

}  // namespace policy

extern "C" volatile int32_t* policy_stall_word(void) { return policy::stall_word(); }
extern "C" int policy_version(void) { return POLICY_ABI_VERSION; }
extern "C" const char* policy_last_error(void) { return policy::g_error.c_str(); }
