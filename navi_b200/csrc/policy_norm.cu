// Per-head RMS norm of queries and keys with the rotation by the token's angles, and its gradient.
//
//   u = w x r,  r = 1 / sqrt(mean(x^2) + eps);   y = R u, R the rotation of the first values
// and, since R is orthogonal,
//   g = R^T dy,  dw = sum over rows of g x r,  dx = r w g - r^3 x mean(w g x).
// Memory bounds both: one read of x (and dy) and one write.  A row belongs to dim / 8 neighbouring
// lanes with 8 values each, so that a rotation's partner values sit rotary / 16 lanes away and are
// shuffled, not read again; a thread takes up to four heads of one token, which share the token's
// cosines and sines.  Everything between the read and the one rounding at the store is in 32 bits.
#include <cuda_bf16.h>

#include <limits>

#include "policy_internal.h"

namespace policy {
namespace {

using bf16 = __nv_bfloat16;
constexpr int kThreads = 256;
constexpr int kHeads = 4;  // heads of a token per thread

struct NormSide {
    const void* x;
    const void* dy;
    void* y;  // forward: y, backward: dx
    const float* weight;
    const float* table;
    const int32_t* positions;
    int64_t xs[3], ds[3];
    int64_t table_rows;
    int64_t units;      // (batch, token, group of kHeads heads)
    float* part;        // backward: [blocks][dim], null without dweight
    float* dweight;
    int tokens, heads, chunks;
    int blocks;
};

struct NormParams {
    NormSide side[2];
    int dim, rotary, lanes;  // lanes per row, a power of two
    float eps;
};

template <typename T>
__device__ __forceinline__ void load8(float (&v)[8], const T* p);
template <>
__device__ __forceinline__ void load8<float>(float (&v)[8], const float* p)
{
    const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
}
template <>
__device__ __forceinline__ void load8<bf16>(float (&v)[8], const bf16* p)
{
    const uint4 a = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[2 * i] = __uint_as_float(w[i] << 16);
        v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&v)[8]);
template <>
__device__ __forceinline__ void store8<float>(float* p, const float (&v)[8])
{
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
    *reinterpret_cast<float4*>(p + 4) = make_float4(v[4], v[5], v[6], v[7]);
}
template <>
__device__ __forceinline__ void store8<bf16>(bf16* p, const float (&v)[8])
{
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
}

__device__ __forceinline__ float row_sum(float x, int lanes)
{
    for (int d = 1; d < lanes; d <<= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
    return x;
}

// A lane's place in its row and the token it works on.
struct Place {
    int sub;            // lane of the row
    int pair;           // lane that holds the rotation's other value, or this one
    bool in_dim, low;   // low: the first half of a rotated pair
    __device__ __forceinline__ Place(const NormParams& p)
    {
        const int lane = threadIdx.x & 31, half = p.rotary / 16;
        sub = lane & (p.lanes - 1);
        in_dim = sub * 8 < p.dim;
        low = sub < half;
        pair = low ? lane + half : sub < 2 * half ? lane - half : lane;
    }
};

// The cosines and signed sines of a lane's 8 values: y = u cos + other sin.  Returns false for a
// position outside the table.
__device__ __forceinline__ bool angles(const NormParams& p, const NormSide& s, const Place& at, int64_t b, int token, bool active,
                                       float (&cs)[8], float (&sn)[8])
{
    const int half = p.rotary / 16;
    int64_t pos = token;
    if (s.positions && active) pos = s.positions[b * s.tokens + token];
    const bool inside = pos >= 0 && pos < s.table_rows;
    if (active && inside && at.sub < 2 * half) {
        const float* row = s.table + pos * p.rotary + (at.low ? at.sub : at.sub - half) * 8;
        load8(cs, row);
        load8(sn, row + p.rotary / 2);
        if (at.low) {
#pragma unroll
            for (int i = 0; i < 8; ++i) sn[i] = -sn[i];
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) cs[i] = 1.f, sn[i] = 0.f;
    }
    return inside;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) qk_norm_kernel(const __grid_constant__ NormParams p)
{
    const bool second = blockIdx.x >= p.side[0].blocks;
    const NormSide& s = p.side[second ? 1 : 0];
    const int block = second ? blockIdx.x - p.side[0].blocks : blockIdx.x;
    const Place at(p);
    const int rows = kThreads / p.lanes;
    float w[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = 1.f;
    if (s.weight && at.in_dim) load8(w, s.weight + at.sub * 8);

    for (int64_t base = static_cast<int64_t>(block) * rows; base < s.units; base += static_cast<int64_t>(s.blocks) * rows) {
        const int64_t unit = base + threadIdx.x / p.lanes;
        const bool active = unit < s.units && at.in_dim;
        const int64_t bt = unit < s.units ? unit / s.chunks : 0;
        const int h0 = unit < s.units ? static_cast<int>(unit - bt * s.chunks) * kHeads : 0;
        const int64_t b = bt / s.tokens;
        const int token = static_cast<int>(bt - b * s.tokens);
        const T* x = static_cast<const T*>(s.x) + b * s.xs[0] + token * s.xs[1] + h0 * s.xs[2] + at.sub * 8;
        T* y = static_cast<T*>(s.y) + (bt * s.heads + h0) * p.dim + at.sub * 8;
        float v[kHeads][8];
#pragma unroll
        for (int h = 0; h < kHeads; ++h) {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[h][i] = 0.f;
            if (active && h0 + h < s.heads) load8(v[h], x + h * s.xs[2]);
        }
        float cs[8], sn[8];
        bool inside = true;
        if (s.table) inside = angles(p, s, at, b, token, active, cs, sn);
#pragma unroll
        for (int h = 0; h < kHeads; ++h) {
            float sum = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) sum = fmaf(v[h][i], v[h][i], sum);
            const float r = rsqrtf(row_sum(sum, p.lanes) / p.dim + p.eps);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[h][i] = v[h][i] * r * w[i];
            if (s.table) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float other = __shfl_sync(0xffffffffu, v[h][i], at.pair);
                    v[h][i] = inside ? fmaf(v[h][i], cs[i], other * sn[i]) : NAN;
                }
            }
            if (active && h0 + h < s.heads) store8(y + h * p.dim, v[h]);
        }
    }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) qk_norm_grad_kernel(const __grid_constant__ NormParams p)
{
    __shared__ float sums[kThreads * 8];
    const bool second = blockIdx.x >= p.side[0].blocks;
    const NormSide& s = p.side[second ? 1 : 0];
    const int block = second ? blockIdx.x - p.side[0].blocks : blockIdx.x;
    const Place at(p);
    const int rows = kThreads / p.lanes;
    float w[8], dw[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = 1.f, dw[i] = 0.f;
    if (s.weight && at.in_dim) load8(w, s.weight + at.sub * 8);

    for (int64_t base = static_cast<int64_t>(block) * rows; base < s.units; base += static_cast<int64_t>(s.blocks) * rows) {
        const int64_t unit = base + threadIdx.x / p.lanes;
        const bool active = unit < s.units && at.in_dim;
        const int64_t bt = unit < s.units ? unit / s.chunks : 0;
        const int h0 = unit < s.units ? static_cast<int>(unit - bt * s.chunks) * kHeads : 0;
        const int64_t b = bt / s.tokens;
        const int token = static_cast<int>(bt - b * s.tokens);
        const T* x = static_cast<const T*>(s.x) + b * s.xs[0] + token * s.xs[1] + h0 * s.xs[2] + at.sub * 8;
        const T* dy = static_cast<const T*>(s.dy) + b * s.ds[0] + token * s.ds[1] + h0 * s.ds[2] + at.sub * 8;
        T* dx = static_cast<T*>(s.y) + (bt * s.heads + h0) * p.dim + at.sub * 8;
        float cs[8], sn[8];
        bool inside = true;
        if (s.table) inside = angles(p, s, at, b, token, active, cs, sn);
#pragma unroll
        for (int h = 0; h < kHeads; ++h) {
            const bool on = active && h0 + h < s.heads;
            float v[8], g[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = g[i] = 0.f;
            if (on) {
                load8(v, x + h * s.xs[2]);
                load8(g, dy + h * s.ds[2]);
            }
            if (s.table) {  // the rotation back: the sines change sign
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float other = __shfl_sync(0xffffffffu, g[i], at.pair);
                    g[i] = inside ? fmaf(g[i], cs[i], -other * sn[i]) : on ? NAN : 0.f;
                }
            }
            float sum = 0.f, dot = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                sum = fmaf(v[i], v[i], sum);
                dot = fmaf(v[i] * w[i], g[i], dot);
            }
            const float r = rsqrtf(row_sum(sum, p.lanes) / p.dim + p.eps);
            const float f = r * r * r * (row_sum(dot, p.lanes) / p.dim);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if (on) dw[i] = fmaf(g[i], v[i] * r, dw[i]);
                v[i] = fmaf(r * w[i], g[i], -f * v[i]);
            }
            if (on) store8(dx + h * p.dim, v);
        }
    }
    if (!s.part) return;
    // the block's rows, in order
#pragma unroll
    for (int i = 0; i < 8; ++i) sums[(threadIdx.x / p.lanes) * p.lanes * 8 + at.sub * 8 + i] = dw[i];
    __syncthreads();
    for (int d = threadIdx.x; d < p.dim; d += kThreads) {
        float x = 0.f;
        for (int r = 0; r < rows; ++r) x += sums[r * p.lanes * 8 + d];
        s.part[static_cast<int64_t>(block) * p.dim + d] = x;
    }
}

// dweight[d] = sum of the blocks' parts: one block per (side, 32 columns), 32 threads to a column.
__global__ void __launch_bounds__(1024) norm_weight_kernel(const __grid_constant__ NormParams p)
{
    __shared__ float sums[32][33];
    const NormSide& s = p.side[blockIdx.y];
    if (!s.part) return;
    const int d = blockIdx.x * 32 + (threadIdx.x & 31), r0 = threadIdx.x >> 5;
    float x = 0.f;
    if (d < p.dim)
        for (int r = r0; r < s.blocks; r += 32) x += s.part[static_cast<int64_t>(r) * p.dim + d];
    sums[r0][threadIdx.x & 31] = x;
    __syncthreads();
    if (r0 == 0 && d < p.dim) {
        x = 0.f;
        for (int r = 0; r < 32; ++r) x += sums[r][threadIdx.x];
        s.dweight[d] = x;
    }
}

// --- host ----------------------------------------------------------------------

constexpr int64_t kMaxInt = std::numeric_limits<int32_t>::max();

bool aligned_rows(const void* p, const int64_t (&s)[3], size_t e)
{
    bool ok = p && reinterpret_cast<uintptr_t>(p) % 16 == 0;
    for (int64_t x : s) ok = ok && (x * static_cast<int64_t>(e)) % 16 == 0;
    return ok;
}

int check_norm(const policy_qk_norm* a)
{
    if (!a) return fail(POLICY_ERR_INVALID, "args must not be null");
    if (!known_dtype(a->dtype)) return fail(POLICY_ERR_INVALID, "dtype must be POLICY_F32 or POLICY_BF16");
    if (a->dim < 8 || a->dim > 256 || a->dim % 8 != 0) return fail(POLICY_ERR_INVALID, "dim must be a multiple of 8 from 8 to 256");
    if (a->rotary < 0 || a->rotary > a->dim || a->rotary % 16 != 0)
        return fail(POLICY_ERR_INVALID, "rotary must be a multiple of 16 from 0 to dim");
    if (!(a->eps >= 0.f)) return fail(POLICY_ERR_INVALID, "eps must not be negative");
    if (a->batch < 0 || a->batch > kMaxInt) return fail(POLICY_ERR_INVALID, "batch must be between 0 and 2^31 - 1");
    for (const policy_norm_side& s : a->side) {
        if (s.tokens < 0 || s.tokens > kMaxInt) return fail(POLICY_ERR_INVALID, "tokens must be between 0 and 2^31 - 1");
        if (s.heads < 1 || s.heads > 65536) return fail(POLICY_ERR_INVALID, "heads must be between 1 and 65536");
        if (a->rotary > 0 && s.table_rows < 0) return fail(POLICY_ERR_INVALID, "table_rows must not be negative");
    }
    return POLICY_OK;
}

int check_norm_pointers(const policy_qk_norm* a, bool backward)
{
    int rc = check_norm(a);
    if (rc != POLICY_OK) return rc;
    const size_t e = dtype_bytes(a->dtype);
    const int64_t none[3] = {0, 0, 0};
    for (const policy_norm_side& s : a->side) {
        if (a->batch == 0 || s.tokens == 0) continue;
        if (!aligned_rows(s.x, s.strides, e)) return fail(POLICY_ERR_INVALID, "x must not be null and must have 16-byte aligned rows");
        if (!backward && !aligned_rows(s.y, none, e)) return fail(POLICY_ERR_INVALID, "y must not be null and must be 16-byte aligned");
        if (backward) {
            if (!aligned_rows(s.dy, s.dy_strides, e)) return fail(POLICY_ERR_INVALID, "dy must not be null and must have 16-byte aligned rows");
            if (!aligned_rows(s.dx, none, e)) return fail(POLICY_ERR_INVALID, "dx must not be null and must be 16-byte aligned");
        }
        if (s.weight && !aligned_rows(s.weight, none, 4)) return fail(POLICY_ERR_INVALID, "weight must be 16-byte aligned");
        if (a->rotary > 0 && !aligned_rows(s.table, none, 4)) return fail(POLICY_ERR_INVALID, "table must not be null and must be 16-byte aligned");
    }
    return POLICY_OK;
}

// Blocks of each side: enough to fill the device several times over; at most one per group of rows.
constexpr int kBlocksPerSm = 8;

NormParams make_norm(const policy_qk_norm& a, int sms, bool backward)
{
    NormParams p{};
    p.dim = a.dim, p.rotary = a.rotary, p.eps = a.eps;
    p.lanes = 1;
    while (p.lanes * 8 < a.dim) p.lanes *= 2;
    const int rows = kThreads / p.lanes;
    int64_t total = 0;
    for (int i = 0; i < 2; ++i) {
        const policy_norm_side& s = a.side[i];
        NormSide& d = p.side[i];
        d.x = s.x, d.dy = s.dy, d.y = backward ? s.dx : s.y;
        d.weight = s.weight, d.table = a.rotary ? s.table : nullptr, d.positions = s.positions;
        for (int k = 0; k < 3; ++k) d.xs[k] = s.strides[k], d.ds[k] = s.dy_strides[k];
        d.table_rows = s.table_rows;
        d.tokens = static_cast<int>(s.tokens), d.heads = s.heads;
        d.chunks = (s.heads + kHeads - 1) / kHeads;
        d.units = a.batch * s.tokens * d.chunks;
        total += d.units;
    }
    for (NormSide& d : p.side) {
        const int64_t most = (d.units + rows - 1) / rows;
        // a side's share of the resident blocks, by its rows
        int64_t share = total ? (static_cast<int64_t>(sms) * kBlocksPerSm * d.units + total - 1) / total : 0;
        d.blocks = static_cast<int>(share < most ? share : most);
    }
    return p;
}

size_t align256(size_t n) { return (n + 255) & ~static_cast<size_t>(255); }

int run_norm(const policy_qk_norm* a, bool backward, cudaStream_t stream)
{
    int rc = check_norm_pointers(a, backward);
    if (rc != POLICY_OK) return rc;
    const DeviceInfo info = device_info(a->device);
    if (info.status != POLICY_OK) return info.status;
    DeviceScope scope(a->device);
    if (scope.error() != cudaSuccess) return cuda_fail(scope.error(), "cudaSetDevice");
    NormParams p = make_norm(*a, info.sms, backward);
    const int blocks = p.side[0].blocks + p.side[1].blocks;
    bool weights = false;
    if (backward) {
        char* ws = static_cast<char*>(a->workspace);
        for (int i = 0; i < 2; ++i) {
            if (!a->side[i].dweight) continue;
            if (!ws && p.side[i].blocks) return fail(POLICY_ERR_INVALID, "workspace must not be null");
            p.side[i].dweight = a->side[i].dweight;
            // without rows the pointer only says that the (empty) sum is wanted
            p.side[i].part = p.side[i].blocks ? reinterpret_cast<float*>(ws) : a->side[i].dweight;
            if (p.side[i].blocks) ws += align256(sizeof(float) * p.side[i].blocks * p.dim);
            weights = true;
        }
    }
    const bool f32 = a->dtype == POLICY_F32;
    if (blocks > 0) {
        if (!backward) {
            if (f32) qk_norm_kernel<float><<<blocks, kThreads, 0, stream>>>(p);
            else qk_norm_kernel<bf16><<<blocks, kThreads, 0, stream>>>(p);
        } else {
            if (f32) qk_norm_grad_kernel<float><<<blocks, kThreads, 0, stream>>>(p);
            else qk_norm_grad_kernel<bf16><<<blocks, kThreads, 0, stream>>>(p);
        }
        const cudaError_t e = cudaGetLastError();
        if (e != cudaSuccess) return cuda_fail(e, "qk_norm_kernel");
    }
    if (weights) {
        norm_weight_kernel<<<dim3((p.dim + 31) / 32, 2), 1024, 0, stream>>>(p);
        const cudaError_t e = cudaGetLastError();
        if (e != cudaSuccess) return cuda_fail(e, "norm_weight_kernel");
    }
    return POLICY_OK;
}

}  // namespace
}  // namespace policy

using namespace policy;

extern "C" uint64_t policy_qk_norm_workspace_bytes(const policy_qk_norm* a)
try {
    if (check_norm(a) != POLICY_OK) return 0;
    const DeviceInfo info = device_info(a->device);
    if (info.status != POLICY_OK) return 0;
    const NormParams p = make_norm(*a, info.sms, true);
    return align256(sizeof(float) * p.side[0].blocks * p.dim) + align256(sizeof(float) * p.side[1].blocks * p.dim);
} catch (...) {
    return 0;
}

extern "C" int policy_qk_norm_rotary(const policy_qk_norm* a, void* stream)
try {
    return run_norm(a, false, static_cast<cudaStream_t>(stream));
} catch (...) {
    return POLICY_ERR_INVALID;
}

extern "C" int policy_qk_norm_rotary_backward(const policy_qk_norm* a, void* stream)
try {
    return run_norm(a, true, static_cast<cudaStream_t>(stream));
} catch (...) {
    return POLICY_ERR_INVALID;
}
