// The global norm of a list of gradients, and their clipping.
//
// Two launches: every block adds the squares of its chunks (32 bits within a thread's chunk, 64 bits
// from there on) into one partial sum; every block of the second launch adds the partial sums in the
// same order, which costs it a few kilobytes from L2 and saves a launch between the two, and scales
// its chunks.  The second launch starts while the first still runs (programmatic dependent launch): its
// blocks read their first chunk before they wait for the partial sums.  Memory bounds both; the second pass
// takes the chunks in the opposite order, so that it starts on what the first left in L2.  150 M values (487 MB) into other
// tensors: 249 us for the three passes, 5.9 TB/s; 1.2 M values: 8 us.
#include <cuda_bf16.h>

#include <algorithm>
#include <limits>
#include <utility>
#include <vector>

#include "policy_internal.h"

namespace policy {
namespace {

using bf16 = __nv_bfloat16;
constexpr int kThreads = 256;
// Values of a chunk: 32 per thread where there are chunks enough for every SM, else 8.
constexpr int kLongChunk = 8192, kShortChunk = 2048;
constexpr int kBlocksPerSm = 8;     // 256 threads: the SM is full
constexpr int kMaxSms = 256;         // SMs that the workspace allows for
constexpr int kTensors = 512;       // tensors of one launch (its parameters: 16 KB)
constexpr int kFewTensors = 64;     // a launch of up to this many takes 2 KB of parameters instead

struct ClipTensor {
    const void* grad;
    void* out;
    uint64_t count;
    uint32_t first_chunk;  // chunks of the launch's tensors before this one
    uint32_t dtype;        // bit 0: bf16; bit 1: every chunk is 16-byte aligned
};

template <int N, int CHUNK>
struct ClipParams {
    ClipTensor t[N];
    double* parts;
    float* norm;
    float max_norm;
    int n;
    uint32_t chunks;
    int part0;   // first partial sum of this launch (first pass)
    int n_parts; // all partial sums (second pass)
};

template <int N, int CHUNK>
__device__ __forceinline__ int find_tensor(const ClipParams<N, CHUNK>& p, uint32_t chunk)
{
    int lo = 0, hi = p.n - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (p.t[mid].first_chunk <= chunk) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

__device__ __forceinline__ double block_sum(double x)
{
    __shared__ double warp_sums[kThreads / 32];
    __shared__ double total;
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
    if ((threadIdx.x & 31) == 0) warp_sums[threadIdx.x >> 5] = x;
    __syncthreads();
    if (threadIdx.x == 0) {
        x = 0.0;
        for (int i = 0; i < kThreads / 32; ++i) x += warp_sums[i];
        total = x;
    }
    __syncthreads();
    return total;
}

__device__ __forceinline__ float2 unpack(uint32_t w)
{
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}

__device__ __forceinline__ uint32_t scale2(uint32_t w, float c)
{
    const float2 v = unpack(w);
    const __nv_bfloat162 h = __floats2bfloat162_rn(v.x * c, v.y * c);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// One chunk of a tensor, in registers where it is whole and aligned.
template <int N, int CHUNK>
struct Chunk {
    static constexpr int kWords = CHUNK / kThreads / 4;  // 16-byte words of f32; half as many of bf16
    const ClipTensor* t;
    uint64_t at;
    int n;
    bool wide;
    uint4 v[kWords];

    __device__ __forceinline__ void load(const ClipParams<N, CHUNK>& p, uint32_t chunk)
    {
        t = &p.t[find_tensor(p, chunk)];
        at = static_cast<uint64_t>(chunk - t->first_chunk) * CHUNK;
        n = static_cast<int>(min(static_cast<uint64_t>(CHUNK), t->count - at));
        wide = n == CHUNK && (t->dtype & 2u);
        if (!wide) return;
        if (t->dtype & 1u) {
            const uint4* g = reinterpret_cast<const uint4*>(static_cast<const bf16*>(t->grad) + at);
#pragma unroll
            for (int i = 0; i < kWords / 2; ++i) v[i] = g[threadIdx.x + i * kThreads];
        } else {
            const uint4* g = reinterpret_cast<const uint4*>(static_cast<const float*>(t->grad) + at);
#pragma unroll
            for (int i = 0; i < kWords; ++i) v[i] = g[threadIdx.x + i * kThreads];
        }
    }
    __device__ __forceinline__ float value(int i) const
    {
        return (t->dtype & 1u) ? __bfloat162float(static_cast<const bf16*>(t->grad)[at + i]) : static_cast<const float*>(t->grad)[at + i];
    }
    __device__ __forceinline__ float squares() const
    {
        float x = 0.f;
        if (!wide) {
            for (int i = threadIdx.x; i < n; i += kThreads) x = fmaf(value(i), value(i), x);
        } else if (t->dtype & 1u) {
#pragma unroll
            for (int i = 0; i < kWords / 2; ++i) {
                const uint32_t w[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const float2 f = unpack(w[k]);
                    x = fmaf(f.x, f.x, fmaf(f.y, f.y, x));
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < kWords; ++i) {
                const float4 f = make_float4(__uint_as_float(v[i].x), __uint_as_float(v[i].y), __uint_as_float(v[i].z), __uint_as_float(v[i].w));
                x = fmaf(f.x, f.x, fmaf(f.y, f.y, fmaf(f.z, f.z, fmaf(f.w, f.w, x))));
            }
        }
        return x;
    }
    __device__ __forceinline__ void scale(float c) const
    {
        if (c == 1.f && t->out == t->grad) return;
        if (!wide) {
            for (int i = threadIdx.x; i < n; i += kThreads) {
                if (t->dtype & 1u) static_cast<bf16*>(t->out)[at + i] = __float2bfloat16_rn(value(i) * c);
                else static_cast<float*>(t->out)[at + i] = value(i) * c;
            }
        } else if (t->dtype & 1u) {
            uint4* o = reinterpret_cast<uint4*>(static_cast<bf16*>(t->out) + at);
#pragma unroll
            for (int i = 0; i < kWords / 2; ++i)
                o[threadIdx.x + i * kThreads] = make_uint4(scale2(v[i].x, c), scale2(v[i].y, c), scale2(v[i].z, c), scale2(v[i].w, c));
        } else {
            float4* o = reinterpret_cast<float4*>(static_cast<float*>(t->out) + at);
#pragma unroll
            for (int i = 0; i < kWords; ++i)
                o[threadIdx.x + i * kThreads] = make_float4(__uint_as_float(v[i].x) * c, __uint_as_float(v[i].y) * c, __uint_as_float(v[i].z) * c,
                                                            __uint_as_float(v[i].w) * c);
        }
    }
};

template <int N, int CHUNK>
__global__ void __launch_bounds__(kThreads) clip_norm_kernel(const __grid_constant__ ClipParams<N, CHUNK> p)
{
    asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
    double sum = 0.0;
    Chunk<N, CHUNK> c;
    for (uint32_t chunk = blockIdx.x; chunk < p.chunks; chunk += gridDim.x) {
        c.load(p, chunk);
        sum += c.squares();
    }
    sum = block_sum(sum);
    if (threadIdx.x == 0) p.parts[p.part0 + blockIdx.x] = sum;
}

template <int N, int CHUNK>
__global__ void __launch_bounds__(kThreads) clip_scale_kernel(const __grid_constant__ ClipParams<N, CHUNK> p)
{
    Chunk<N, CHUNK> c;
    uint32_t k = blockIdx.x;
    c.load(p, p.chunks - 1 - k);
    asm volatile("griddepcontrol.wait;\n" ::: "memory");
    double sum = 0.0;
    for (int i = threadIdx.x; i < p.n_parts; i += kThreads) sum += p.parts[i];
    const float norm = static_cast<float>(sqrt(block_sum(sum)));
    if (p.norm && blockIdx.x == 0 && threadIdx.x == 0) *p.norm = norm;
    const float f = p.max_norm / (norm + 1e-6f);
    const float factor = f > 1.f ? 1.f : f;  // NaN stays NaN
    for (;;) {
        c.scale(factor);
        k += gridDim.x;
        if (k >= p.chunks) break;
        c.load(p, p.chunks - 1 - k);
    }
}

// --- host ----------------------------------------------------------------------

int check_grads(const policy_grad* grads, int64_t n)
{
    if (n < 0 || n > (1 << 24)) return fail(POLICY_ERR_INVALID, "n must be between 0 and 2^24");
    if (n > 0 && !grads) return fail(POLICY_ERR_INVALID, "grads must not be null");
    for (int64_t i = 0; i < n; ++i) {
        const policy_grad& g = grads[i];
        if (!known_dtype(g.dtype)) return fail(POLICY_ERR_INVALID, "dtype must be POLICY_F32 or POLICY_BF16");
        if (g.count > (1ull << 40)) return fail(POLICY_ERR_INVALID, "count must not pass 2^40");
        if (g.count && (!g.grad || !g.out)) return fail(POLICY_ERR_INVALID, "grad and out must not be null");
        const size_t e = dtype_bytes(g.dtype);
        if (reinterpret_cast<uintptr_t>(g.grad) % e || reinterpret_cast<uintptr_t>(g.out) % e)
            return fail(POLICY_ERR_INVALID, "grad and out must be aligned to their type");
    }
    return POLICY_OK;
}

// The blocks run in no order, so what one writes nobody else may read or write: no two outputs overlap, and no output
// overlaps another gradient than its own, which is at the same address.
int check_memory(const policy_grad* grads, int64_t n)
{
    using Range = std::pair<uintptr_t, uintptr_t>;
    const auto range = [](const void* p, const policy_grad& g) {
        const uintptr_t at = reinterpret_cast<uintptr_t>(p);
        return Range(at, at + g.count * dtype_bytes(g.dtype));
    };
    std::vector<Range> written;
    written.reserve(static_cast<size_t>(n));
    for (int64_t i = 0; i < n; ++i)
        if (grads[i].count) written.push_back(range(grads[i].out, grads[i]));
    std::sort(written.begin(), written.end());
    bool ok = true;
    for (size_t i = 1; i < written.size(); ++i) ok = ok && written[i - 1].second <= written[i].first;
    for (int64_t i = 0; ok && i < n; ++i) {
        if (grads[i].count == 0 || grads[i].grad == grads[i].out) continue;
        const Range read = range(grads[i].grad, grads[i]);
        // the last output that starts before the gradient ends
        const auto after = std::lower_bound(written.begin(), written.end(), Range(read.second, 0));
        ok = after == written.begin() || (after - 1)->second <= read.first;
    }
    return ok ? POLICY_OK : fail(POLICY_ERR_INVALID, "the tensors that are written must not share memory with each other or with another gradient");
}

// Takes tensors from grads[i..] for one launch; returns how many entries it consumed.
template <int N, int CHUNK>
int64_t fill_launch(const policy_grad* grads, int64_t n, ClipParams<N, CHUNK>& p)
{
    p.n = 0;
    uint64_t chunks = 0;
    int64_t i = 0;
    for (; i < n && p.n < N; ++i) {
        const policy_grad& g = grads[i];
        if (g.count == 0) continue;
        const uint64_t own = (g.count + CHUNK - 1) / CHUNK;
        if (chunks + own > std::numeric_limits<int32_t>::max()) break;  // one tensor alone always fits: count <= 2^40
        ClipTensor& t = p.t[p.n++];
        const bool wide = reinterpret_cast<uintptr_t>(g.grad) % 16 == 0 && reinterpret_cast<uintptr_t>(g.out) % 16 == 0;
        t.grad = g.grad, t.out = g.out, t.count = g.count;
        t.first_chunk = static_cast<uint32_t>(chunks);
        t.dtype = (g.dtype == POLICY_BF16 ? 1u : 0u) | (wide ? 2u : 0u);
        chunks += own;
    }
    p.chunks = static_cast<uint32_t>(chunks);
    return i;
}

template <int N, int CHUNK>
int launch_blocks(const ClipParams<N, CHUNK>& p, int sms)
{
    const uint32_t most = static_cast<uint32_t>(sms < kMaxSms ? sms : kMaxSms) * kBlocksPerSm;
    return static_cast<int>(p.chunks < most ? p.chunks : most);
}

template <int N, int CHUNK>
int launch_clip(const policy_grad* grads, int64_t n, float max_norm, float* norm, int sms, void* workspace, cudaStream_t stream)
{
    ClipParams<N, CHUNK> p;
    p.parts = static_cast<double*>(workspace);
    p.max_norm = max_norm;
    p.n_parts = 0;
    bool one_launch = false;
    for (int64_t i = 0; i < n;) {
        i += fill_launch(grads + i, n - i, p);
        if (p.chunks == 0) continue;
        if (!workspace) return fail(POLICY_ERR_INVALID, "workspace must not be null");
        p.part0 = p.n_parts;
        const int blocks = launch_blocks(p, sms);
        clip_norm_kernel<<<blocks, kThreads, 0, stream>>>(p);
        const cudaError_t e = cudaGetLastError();
        if (e != cudaSuccess) return cuda_fail(e, "clip_norm_kernel");
        one_launch = p.n_parts == 0;
        p.n_parts += blocks;
    }
    if (p.n_parts == 0) {
        const cudaError_t e = cudaMemsetAsync(norm, 0, sizeof(float), stream);
        return e == cudaSuccess ? POLICY_OK : cuda_fail(e, "cudaMemsetAsync");
    }
    p.norm = norm;
    // With several launches the first scaling one may start only when every sum is written, which the launch
    // before it alone does not say; the gradients of a later one are not read before it starts.
    bool first = one_launch;
    for (int64_t i = 0; i < n;) {
        i += fill_launch(grads + i, n - i, p);
        if (p.chunks == 0) continue;
        cudaLaunchAttribute early{};
        early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
        early.val.programmaticStreamSerializationAllowed = first;
        cudaLaunchConfig_t config{};
        config.gridDim = launch_blocks(p, sms), config.blockDim = kThreads, config.stream = stream;
        config.attrs = &early, config.numAttrs = 1;
        const cudaError_t e = cudaLaunchKernelEx(&config, clip_scale_kernel<N, CHUNK>, p);
        if (e != cudaSuccess) return cuda_fail(e, "clip_scale_kernel");
        first = false;
        p.norm = nullptr;
    }
    return POLICY_OK;
}

int run_clip(const policy_grad* grads, int64_t n, float max_norm, float* norm, int device, void* workspace, cudaStream_t stream)
{
    int rc = check_grads(grads, n);
    if (rc != POLICY_OK || (rc = check_memory(grads, n)) != POLICY_OK) return rc;
    if (!(max_norm >= 0.f)) return fail(POLICY_ERR_INVALID, "max_norm must not be negative");
    if (!norm) return fail(POLICY_ERR_INVALID, "norm must not be null");
    const DeviceInfo info = device_info(device);
    if (info.status != POLICY_OK) return info.status;
    DeviceScope scope(device);
    if (scope.error() != cudaSuccess) return cuda_fail(scope.error(), "cudaSetDevice");
    uint64_t values = 0;
    for (int64_t i = 0; i < n; ++i) values += grads[i].count;
    const bool few = values < static_cast<uint64_t>(info.sms) * 4 * kLongChunk;
    if (n <= kFewTensors)
        return few ? launch_clip<kFewTensors, kShortChunk>(grads, n, max_norm, norm, info.sms, workspace, stream)
                   : launch_clip<kFewTensors, kLongChunk>(grads, n, max_norm, norm, info.sms, workspace, stream);
    return few ? launch_clip<kTensors, kShortChunk>(grads, n, max_norm, norm, info.sms, workspace, stream)
               : launch_clip<kTensors, kLongChunk>(grads, n, max_norm, norm, info.sms, workspace, stream);
}

}  // namespace
}  // namespace policy

using namespace policy;

extern "C" uint64_t policy_clip_grad_workspace_bytes(const policy_grad* grads, int64_t n)
try {
    if (check_grads(grads, n) != POLICY_OK) return 0;
    // one launch for every kTensors non-empty tensors, at most the resident blocks of a full device each
    const int64_t launches = (n + kTensors - 1) / kTensors + 1;
    return static_cast<uint64_t>(launches) * kMaxSms * kBlocksPerSm * sizeof(double);
} catch (...) {
    return 0;
}

extern "C" int policy_clip_grad_norm(const policy_grad* grads, int64_t n, float max_norm, float* norm, int device, void* workspace,
                                     void* stream)
try {
    return run_clip(grads, n, max_norm, norm, device, workspace, static_cast<cudaStream_t>(stream));
} catch (...) {
    return POLICY_ERR_INVALID;
}
