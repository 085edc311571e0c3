// Runs the bounded wait of the policy kernels (policy_tcgen05.cuh) on a barrier that one thread arrives at late, or
// nothing does.
#include "policy_tcgen05.cuh"

namespace {

__device__ __forceinline__ uint64_t nanoseconds()
{
    uint64_t t;
    asm volatile("mov.u64 %0, %globaltimer;\n" : "=l"(t));
    return t;
}

// Warp 0 waits; warp 1 arrives `arrive_ns` after the start, unless that is negative.  Both loops end by themselves.
__global__ void __launch_bounds__(64) wait_kernel(long long arrive_ns, unsigned polls, int* result, int32_t* word)
{
    __shared__ __align__(8) unsigned long long barrier;
    __shared__ int broken_flag;
    volatile int* broken = &broken_flag;
    const uint32_t bar = static_cast<uint32_t>(__cvta_generic_to_shared(&barrier));
    if (threadIdx.x == 0) {
        broken_flag = 0;
        policy::bar_init(bar, 1);
    }
    __syncthreads();
    if (threadIdx.x == 0) *result = policy::bar_wait(bar, 0, broken, polls);
    if (threadIdx.x == 32 && arrive_ns >= 0) {
        const uint64_t start = nanoseconds();
        while (nanoseconds() - start < static_cast<uint64_t>(arrive_ns)) __nanosleep(1000);
        policy::bar_arrive(bar);
    }
    __syncthreads();
    if (threadIdx.x == 0) policy::report_stall(broken, word);
}

}  // namespace

// *result: whether the wait saw the arrival; *word is set to 1 where it did not.  The limit in polls of kPollNs.  Times of
// at most a second.
extern "C" int navi_check_wait(long long arrive_ns, unsigned long long limit_ns, int* result, int* word, void* stream)
{
    if (arrive_ns > 1000000000ll || limit_ns > 1000000000ull || !result || !word) return cudaErrorInvalidValue;
    wait_kernel<<<1, 64, 0, static_cast<cudaStream_t>(stream)>>>(arrive_ns, static_cast<unsigned>(limit_ns / policy::kPollNs), result, word);
    return static_cast<int>(cudaGetLastError());
}
