// What the cross attention kernels share.
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

#include "policy_mma.cuh"

namespace policy {

struct AttnParams {
    const void* q;
    const void* k;
    const void* v;
    const void* dout;
    int64_t qs[3], ks[3], vs[3], ds[3];
    const uint8_t* mask;
    int64_t mask_stride;
    const int32_t* lengths;
    void* out;
    float2* stats;    // of a row: exponent of reference, 1 / sum (0: no visible key)
    void* rest;       // bf16: what the rounding of out left off
    const float* delta;
    void* dq;
    void* dk;
    void* dv;
    float* part;      // f32 parts of a split launch
    float* part_ml;   // forward: the parts' (maximum, sum)
    int64_t q_count;  // values of q, and of k: the parts' strides
    int64_t k_count;
    int lq, lk, heads, kv_heads, group, dim, rows;
    int tiles;        // row tiles (forward, dq) or key tiles (dk, dv) of the grid
    int splits;
    int stages;       // of key tiles in shared memory (forward)
    float scale, scale_log2;
    int32_t* stalled;  // tcgen05: the host's word for a wait that ran out
};

__device__ __forceinline__ float exp2_fast(float x)
{
    float y;  // relative error below 2^-22; 0 for -inf
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// The rows of one (batch, key head): offsets of row r in a strided [batch][lq][heads][dim]
// tensor and in the contiguous one.
struct Rows {
    int64_t b;
    int hk, group;
    __device__ __forceinline__ int64_t at(const int64_t (&s)[3], int r) const
    {
        const int l = r / group;
        return b * s[0] + l * s[1] + (static_cast<int64_t>(hk) * group + (r - l * group)) * s[2];
    }
    // index of the row in [batch][lq][heads]
    __device__ __forceinline__ int64_t index(const AttnParams& p, int r) const
    {
        const int l = r / group;
        return (b * p.lq + l) * p.heads + static_cast<int64_t>(hk) * group + (r - l * group);
    }
};

__device__ __forceinline__ int visible_keys(const AttnParams& p, int64_t b)
{
    if (!p.lengths) return p.lk;
    return min(max(__ldg(p.lengths + b), 0), p.lk);
}

// Whether at most one key of batch b is visible, n being visible_keys: the softmax of one score is constant, and its
// gradient is 0, not a rounding of it.  For a whole warp; reads the mask up to the second visible key, as a rule in its
// first 512 bytes.
__device__ __forceinline__ bool lone_key(const AttnParams& p, int64_t b, int n)
{
    if (n <= 1 || !p.mask) return n <= 1;
    const uint8_t* mask = p.mask + b * p.mask_stride;
    const int lane = threadIdx.x & 31;
    const auto ones = [](uint32_t w) { return __popc(__vsetne4(w, 0u)); };
    int at = 0, seen = 0;
    if (reinterpret_cast<uintptr_t>(mask) % 16 == 0) {
        for (; at + 512 <= n && seen < 2; at += 512) {
            const uint4 w = __ldg(reinterpret_cast<const uint4*>(mask + at) + lane);
            seen += __reduce_add_sync(0xffffffffu, ones(w.x) + ones(w.y) + ones(w.z) + ones(w.w));
        }
    }
    for (; at < n && seen < 2; at += 256) {
        int mine = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int key = at + i * 32 + lane;
            if (key < n) mine += __ldg(mask + key) != 0;
        }
        seen += __reduce_add_sync(0xffffffffu, mine);
    }
    return seen < 2;
}

__device__ __forceinline__ float round_bf16(float x) { return __bfloat162float(__float2bfloat16_rn(x)); }

// 4 values of a row
template <typename T>
__device__ __forceinline__ void store4(T* p, float a, float b, float c, float d);
template <>
__device__ __forceinline__ void store4<float>(float* p, float a, float b, float c, float d)
{
    *reinterpret_cast<float4*>(p) = make_float4(a, b, c, d);
}
template <>
__device__ __forceinline__ void store4<bf16>(bf16* p, float a, float b, float c, float d)
{
    *reinterpret_cast<uint2*>(p) = make_uint2(Mma<bf16>::pack(a, b), Mma<bf16>::pack(c, d));
}

// 4 values of an output, and what their rounding leaves off where that is wanted
template <typename T>
__device__ __forceinline__ void store_out(const AttnParams& p, int64_t at, float a, float b, float c, float d)
{
    store4(static_cast<T*>(p.out) + at, a, b, c, d);
    if constexpr (sizeof(T) == 2) {
        if (p.rest)
            store4(static_cast<T*>(p.rest) + at, a - round_bf16(a), b - round_bf16(b), c - round_bf16(c), d - round_bf16(d));
    }
}

// A row's weights are 2^(c s - x) y.
__device__ __forceinline__ float2 row_stats(float reference, float sum)
{
    return make_float2(reference, sum == 0.f ? 0.f : 1.f / sum);
}

// The forward on the tensor cores of tcgen05 (policy_attention_tc.cu): bf16, tiles of 256 rows.
constexpr int kTcRows = 256;
constexpr int kTcKeys = 128;
// Whether the strides of k and v fit the copies' descriptors (policy_map.h).
bool attend_tc_takes(const AttnParams& p);
int launch_attend_tc(const AttnParams& p, int64_t bh, int sms, int device, cudaStream_t stream);

// The gradients on tcgen05 (policy_attention_grad_tc.cu): bf16; dk and dv (keys) or dq.  Takes groups that divide 64
// and strides that fit the copies' descriptors; p.tiles counts tiles of grad_tc_tile keys or rows.
bool attend_grad_tc_takes(const AttnParams& p);
int grad_tc_tile(bool keys, int dim);
constexpr int kGradTcStream = 64;  // rows or keys that stream past at a time
int launch_attend_grad_tc(const AttnParams& p, bool keys, int64_t bh, int sms, int device, cudaStream_t stream);

}  // namespace policy
