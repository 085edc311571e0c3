// Per-head RMS norm of queries and keys with the rotation by the token's angles, and its gradient.
//
//   u = w x r,  r = 1 / sqrt(mean(x^2) + eps);   y = R u, R the rotation of the first values
// and, since R is orthogonal,
//   g = R^T dy,  dw = sum over rows of g x r,  dx = r w g - r^3 x mean(w g x).
// Memory bounds both: one read of x (and dy) and one write.  A row belongs to LANES neighbouring
// lanes with 8 values each, so that a rotation's partner values sit rotary / 16 lanes away and are
// shuffled, not read again.  A thread keeps one token and up to HEADS of its heads and walks over
// batches: without positions the token's cosines and sines (four times the bytes of a bfloat16
// value each) are read once for all of them, and the next batch's rows are read while this one's
// are worked on.  Everything between the read and the one rounding at the store is in 32 bits, two
// values to an instruction (the f32x2 forms), since at 16 bits a value the issue slots come next
// after memory.
#include <cuda_bf16.h>

#include <cmath>
#include <limits>

#include "policy_internal.h"

namespace policy {
namespace {

using bf16 = __nv_bfloat16;
constexpr int kThreads = 256;

struct NormSide {
    const void* x;
    const void* dy;
    void* y;  // forward: y, backward: dx
    const float* weight;
    const float* table;
    const int32_t* positions;
    int64_t xs[3], ds[3];
    int64_t table_rows;
    float* part;        // backward: [blocks][dim], null without dweight
    float* dweight;
    int tokens, heads;
    int chunks;         // groups of HEADS heads
    int splits;         // batch ranges
    int blocks;
};

struct NormParams {
    NormSide side[2];
    int batch, dim, rotary;
    float eps, inv_dim;
};

// two f32 values in a register pair
using F2 = unsigned long long;
__device__ __forceinline__ F2 pair(float a, float b)
{
    F2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float2 both(F2 v)
{
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b)
{
    F2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c)
{
    F2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ F2 shuffle2(F2 v, int lane)
{
    const float2 f = both(v);
    return pair(__shfl_sync(0xffffffffu, f.x, lane), __shfl_sync(0xffffffffu, f.y, lane));
}

// 8 values as they lie in memory
template <typename T>
struct Raw;
template <>
struct Raw<float> {
    float4 a, b;
    __device__ __forceinline__ void load(const float* p)
    {
        a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
    }
    __device__ __forceinline__ void clear() { a = b = make_float4(0.f, 0.f, 0.f, 0.f); }
    __device__ __forceinline__ void get(F2 (&v)[4]) const
    {
        v[0] = pair(a.x, a.y), v[1] = pair(a.z, a.w), v[2] = pair(b.x, b.y), v[3] = pair(b.z, b.w);
    }
    static __device__ __forceinline__ void store(float* p, const F2 (&v)[4])
    {
        const float2 x = both(v[0]), y = both(v[1]), z = both(v[2]), w = both(v[3]);
        *reinterpret_cast<float4*>(p) = make_float4(x.x, x.y, y.x, y.y);
        *reinterpret_cast<float4*>(p + 4) = make_float4(z.x, z.y, w.x, w.y);
    }
};
template <>
struct Raw<bf16> {
    uint4 a;
    __device__ __forceinline__ void load(const bf16* p) { a = *reinterpret_cast<const uint4*>(p); }
    __device__ __forceinline__ void clear() { a = make_uint4(0u, 0u, 0u, 0u); }
    static __device__ __forceinline__ F2 one(uint32_t w)
    {
        return pair(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
    }
    __device__ __forceinline__ void get(F2 (&v)[4]) const { v[0] = one(a.x), v[1] = one(a.y), v[2] = one(a.z), v[3] = one(a.w); }
    static __device__ __forceinline__ void store(bf16* p, const F2 (&v)[4])
    {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = both(v[i]);
            const __nv_bfloat162 h = __floats2bfloat162_rn(f.x, f.y);
            w[i] = *reinterpret_cast<const uint32_t*>(&h);
        }
        *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    }
};

template <int LANES>
__device__ __forceinline__ float row_sum(F2 x)
{
    const float2 f = both(x);
    float s = f.x + f.y;
#pragma unroll
    for (int d = 1; d < LANES; d <<= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
    return s;
}

// What a thread works on: its lane of the row, its token and heads, and its range of batches.
template <int LANES, int HEADS>
struct Work {
    int sub;              // lane of the row
    int other;            // lane that holds the rotation's other value, or this one
    bool low, turned;     // in the first half of a rotated pair, in either
    bool active;
    int token, h0, heads; // heads of this thread that exist
    int b0, b1;
    __device__ __forceinline__ Work(const NormParams& p, const NormSide& s, int block)
    {
        const int lane = threadIdx.x & 31, half = p.rotary / 16;
        sub = lane & (LANES - 1);
        low = sub < half;
        turned = sub < 2 * half;
        other = low ? lane + half : turned ? lane - half : lane;
        const int64_t unit = static_cast<int64_t>(block) * (kThreads / LANES) + threadIdx.x / LANES;
        const int64_t row = unit / s.chunks;
        h0 = static_cast<int>(unit - row * s.chunks) * HEADS;
        const int split = static_cast<int>(row / s.tokens);
        token = static_cast<int>(row - static_cast<int64_t>(split) * s.tokens);
        active = split < s.splits && sub * 8 < p.dim;
        heads = active ? min(HEADS, s.heads - h0) : 0;
        // every lane of a warp takes part in the shuffles of as many rounds as the longest range has
        b0 = split < s.splits ? static_cast<int>(static_cast<int64_t>(p.batch) * split / s.splits) : 0;
        b1 = split < s.splits ? static_cast<int>(static_cast<int64_t>(p.batch) * (split + 1) / s.splits) : 0;
    }
};

// The cosines and signed sines of a lane's 8 values, y = u cos + other sin; false for a position
// outside the table.
template <int LANES, int HEADS>
__device__ __forceinline__ bool angles(const NormParams& p, const NormSide& s, const Work<LANES, HEADS>& at, int64_t pos, F2 (&cs)[4],
                                       F2 (&sn)[4])
{
    const bool inside = pos >= 0 && pos < s.table_rows;
    if (at.active && inside && at.turned) {
        const float* row = s.table + pos * p.rotary + (at.low ? at.sub : at.sub - p.rotary / 16) * 8;
        Raw<float> c, n;
        c.load(row);
        n.load(row + p.rotary / 2);
        c.get(cs);
        n.get(sn);
        const float sign = at.low ? -1.f : 1.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) sn[i] = mul2(sn[i], pair(sign, sign));
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) cs[i] = pair(1.f, 1.f), sn[i] = pair(0.f, 0.f);
    }
    return inside;
}

__device__ __forceinline__ void load_weight(F2 (&w)[4], const NormSide& s, int sub, bool active)
{
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = pair(1.f, 1.f);
    if (s.weight && active) {
        Raw<float> r;
        r.load(s.weight + sub * 8);
        r.get(w);
    }
}

// Rows that a thread works on at a time: HEADS heads of its token in kRows / HEADS batches.
constexpr int kRows = 4;

template <typename T, int LANES, int HEADS>
__global__ void __launch_bounds__(kThreads) qk_norm_kernel(const __grid_constant__ NormParams p)
{
    constexpr int BATCHES = kRows / HEADS;
    const bool second = blockIdx.x >= p.side[0].blocks;
    const NormSide& s = p.side[second ? 1 : 0];
    const Work<LANES, HEADS> at(p, s, second ? blockIdx.x - p.side[0].blocks : blockIdx.x);
    F2 w[4], cs[4], sn[4];
    load_weight(w, s, at.sub, at.active);
    bool inside = true;
    if (s.table && !s.positions) inside = angles(p, s, at, at.token, cs, sn);

    const int rounds = __reduce_max_sync(0xffffffffu, (at.b1 - at.b0 + BATCHES - 1) / BATCHES);
    const T* x = static_cast<const T*>(s.x) + at.b0 * s.xs[0] + at.token * s.xs[1] + at.h0 * s.xs[2] + at.sub * 8;
    const int64_t y_step = static_cast<int64_t>(s.tokens) * s.heads * p.dim;
    T* y = static_cast<T*>(s.y) + at.b0 * y_step + (static_cast<int64_t>(at.token) * s.heads + at.h0) * p.dim + at.sub * 8;
    Raw<T> next[kRows];
    int next_pos[BATCHES] = {};
    const auto here = [&](int i, int u) { return at.b0 + i * BATCHES + u < at.b1; };
    const auto fetch = [&](int i) {
#pragma unroll
        for (int u = 0; u < BATCHES; ++u) {
            const int64_t b = i * BATCHES + u;
#pragma unroll
            for (int h = 0; h < HEADS; ++h) {
                if (here(i, u) && h < at.heads) next[u * HEADS + h].load(x + b * s.xs[0] + h * s.xs[2]);
                else next[u * HEADS + h].clear();
            }
            if (s.positions && here(i, u)) next_pos[u] = s.positions[(at.b0 + b) * s.tokens + at.token];
        }
    };
    fetch(0);
    for (int i = 0; i < rounds; ++i) {
        F2 v[kRows][4];
        int pos[BATCHES];
#pragma unroll
        for (int k = 0; k < kRows; ++k) next[k].get(v[k]);
#pragma unroll
        for (int u = 0; u < BATCHES; ++u) pos[u] = next_pos[u];
        if (i + 1 < rounds) fetch(i + 1);
#pragma unroll
        for (int u = 0; u < BATCHES; ++u) {
            if (s.positions) inside = angles(p, s, at, pos[u], cs, sn);
#pragma unroll
            for (int h = 0; h < HEADS; ++h) {
                F2(&z)[4] = v[u * HEADS + h];
                F2 sum = mul2(z[0], z[0]);
#pragma unroll
                for (int k = 1; k < 4; ++k) sum = fma2(z[k], z[k], sum);
                const float r = rsqrtf(fmaf(row_sum<LANES>(sum), p.inv_dim, p.eps));
                const F2 r2 = pair(r, r);
#pragma unroll
                for (int k = 0; k < 4; ++k) z[k] = mul2(mul2(z[k], r2), w[k]);
                if (s.table) {
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const F2 o = shuffle2(z[k], at.other);
                        z[k] = fma2(z[k], cs[k], mul2(o, sn[k]));
                        if (!inside) z[k] = pair(NAN, NAN);
                    }
                }
                if (h < at.heads && here(i, u)) Raw<T>::store(y + (i * BATCHES + u) * y_step + h * p.dim, z);
            }
        }
    }
}

template <typename T, int LANES, int HEADS>
__global__ void __launch_bounds__(kThreads) qk_norm_grad_kernel(const __grid_constant__ NormParams p)
{
    constexpr int BATCHES = kRows / HEADS;
    __shared__ float sums[kThreads * 8];
    const bool second = blockIdx.x >= p.side[0].blocks;
    const NormSide& s = p.side[second ? 1 : 0];
    const int block = second ? blockIdx.x - p.side[0].blocks : blockIdx.x;
    const Work<LANES, HEADS> at(p, s, block);
    F2 w[4], dw[4], cs[4], sn[4];
    load_weight(w, s, at.sub, at.active);
#pragma unroll
    for (int k = 0; k < 4; ++k) dw[k] = pair(0.f, 0.f);
    bool inside = true;
    if (s.table && !s.positions) inside = angles(p, s, at, at.token, cs, sn);

    const int rounds = __reduce_max_sync(0xffffffffu, (at.b1 - at.b0 + BATCHES - 1) / BATCHES);
    const T* x = static_cast<const T*>(s.x) + at.b0 * s.xs[0] + at.token * s.xs[1] + at.h0 * s.xs[2] + at.sub * 8;
    const T* dy = static_cast<const T*>(s.dy) + at.b0 * s.ds[0] + at.token * s.ds[1] + at.h0 * s.ds[2] + at.sub * 8;
    const int64_t dx_step = static_cast<int64_t>(s.tokens) * s.heads * p.dim;
    T* dx = static_cast<T*>(s.y) + at.b0 * dx_step + (static_cast<int64_t>(at.token) * s.heads + at.h0) * p.dim + at.sub * 8;
    for (int i = 0; i < rounds; ++i) {
        Raw<T> rx[kRows], rg[kRows];
        int pos[BATCHES];
#pragma unroll
        for (int u = 0; u < BATCHES; ++u) {
            const int64_t b = i * BATCHES + u;
            const bool on = at.b0 + b < at.b1;
            pos[u] = at.token;
            if (s.positions && on) pos[u] = s.positions[(at.b0 + b) * s.tokens + at.token];
#pragma unroll
            for (int h = 0; h < HEADS; ++h) {
                const int k = u * HEADS + h;
                if (on && h < at.heads) {
                    rx[k].load(x + b * s.xs[0] + h * s.xs[2]);
                    rg[k].load(dy + b * s.ds[0] + h * s.ds[2]);
                } else {
                    rx[k].clear();
                    rg[k].clear();
                }
            }
        }
#pragma unroll
        for (int u = 0; u < BATCHES; ++u) {
            const int64_t b = i * BATCHES + u;
            if (s.positions) inside = angles(p, s, at, pos[u], cs, sn);
#pragma unroll
            for (int h = 0; h < HEADS; ++h) {
                const bool here = at.b0 + b < at.b1 && h < at.heads;
                F2 v[4], g[4];
                rx[u * HEADS + h].get(v);
                rg[u * HEADS + h].get(g);
                if (s.table) {  // the rotation back: the sines change sign
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const F2 o = shuffle2(g[k], at.other);
                        g[k] = fma2(g[k], cs[k], mul2(mul2(o, sn[k]), pair(-1.f, -1.f)));
                        if (!inside && here) g[k] = pair(NAN, NAN);
                    }
                }
                F2 sum = mul2(v[0], v[0]), dot = mul2(mul2(v[0], w[0]), g[0]);
#pragma unroll
                for (int k = 1; k < 4; ++k) {
                    sum = fma2(v[k], v[k], sum);
                    dot = fma2(mul2(v[k], w[k]), g[k], dot);
                }
                const float r = rsqrtf(fmaf(row_sum<LANES>(sum), p.inv_dim, p.eps));
                const float f = -r * r * r * (row_sum<LANES>(dot) * p.inv_dim);
                const F2 r2 = pair(r, r), f2 = pair(f, f);
                if (here) {
                    F2 d[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const F2 gr = mul2(g[k], r2);
                        dw[k] = fma2(gr, v[k], dw[k]);
                        d[k] = fma2(gr, w[k], mul2(f2, v[k]));
                    }
                    Raw<T>::store(dx + b * dx_step + h * p.dim, d);
                }
            }
        }
    }
    if (!s.part) return;
    // the block's rows, in order
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const float2 f = both(dw[k]);
        float* at_row = sums + (threadIdx.x / LANES) * (LANES * 8) + at.sub * 8 + 2 * k;
        at_row[0] = f.x, at_row[1] = f.y;
    }
    __syncthreads();
    for (int d = threadIdx.x; d < p.dim; d += kThreads) {
        float t = 0.f;
        for (int r = 0; r < kThreads / LANES; ++r) t += sums[r * (LANES * 8) + d];
        s.part[static_cast<int64_t>(block) * p.dim + d] = t;
    }
}

// dweight[d] = sum of the blocks' parts: a block to 8 columns (one 32-byte sector) of a side, 128 threads to a
// column, so that the few thousand parts are a few dependent reads.
__global__ void __launch_bounds__(1024) norm_weight_kernel(const __grid_constant__ NormParams p)
{
    __shared__ float sums[128][9];
    const NormSide& s = p.side[blockIdx.y];
    if (!s.part) return;
    const int column = threadIdx.x & 7, first = threadIdx.x >> 3, d = blockIdx.x * 8 + column;
    float x = 0.f;
#pragma unroll 4
    for (int r = first; r < s.blocks; r += 128) x += s.part[static_cast<int64_t>(r) * p.dim + d];
    sums[first][column] = x;
    __syncthreads();
    for (int n = 64; n > 0; n >>= 1) {
        if (first < n) sums[first][column] += sums[first + n][column];
        __syncthreads();
    }
    if (first == 0) s.dweight[d] = sums[0][column];
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

// Lanes of a row and heads of a thread.  A wider group than the dim needs leaves lanes idle, so the
// lanes follow the dim; the heads follow the side with more rows (heads that a side does not have
// are not worked on).
struct NormShape {
    int lanes, heads;
};

NormShape norm_shape(const policy_qk_norm& a)
{
    NormShape s{4, 4};
    while (s.lanes * 8 < a.dim) s.lanes *= 2;
    const policy_norm_side& big = a.side[0].tokens * a.side[0].heads > a.side[1].tokens * a.side[1].heads ? a.side[0] : a.side[1];
    if (big.heads <= 2) s.heads = big.heads;
    return s;
}

// Threads' ranges of batches: as long as they leave the device kRounds full sets of blocks.
constexpr int kBlocksPerSm = 8;
constexpr int kRounds = 2;

int make_norm(const policy_qk_norm& a, int sms, bool backward, NormParams& p)
{
    p = NormParams{};
    const NormShape shape = norm_shape(a);
    p.batch = static_cast<int>(a.batch), p.dim = a.dim, p.rotary = a.rotary, p.eps = a.eps;
    p.inv_dim = 1.f / static_cast<float>(a.dim);
    const int64_t groups = kThreads / shape.lanes;
    int64_t total = 0;
    for (int i = 0; i < 2; ++i) {
        const policy_norm_side& s = a.side[i];
        NormSide& d = p.side[i];
        d.x = s.x, d.dy = s.dy, d.y = backward ? s.dx : s.y;
        d.weight = s.weight, d.table = a.rotary ? s.table : nullptr, d.positions = a.rotary ? s.positions : nullptr;
        for (int k = 0; k < 3; ++k) d.xs[k] = s.strides[k], d.ds[k] = s.dy_strides[k];
        d.table_rows = s.table_rows;
        d.tokens = static_cast<int>(s.tokens), d.heads = s.heads;
        d.chunks = (s.heads + shape.heads - 1) / shape.heads;
        total += a.batch * s.tokens * d.chunks;
    }
    const int64_t want = static_cast<int64_t>(sms) * kBlocksPerSm * kRounds * groups;
    const int64_t round = kRows / shape.heads;  // batches at a time
    const int64_t length = total / want > 1 ? (total / want + round - 1) / round * round : 1;  // batches of a thread
    for (NormSide& d : p.side) {
        d.splits = static_cast<int>((a.batch + length - 1) / length);
        const int64_t blocks = (static_cast<int64_t>(d.splits) * d.tokens * d.chunks + groups - 1) / groups;
        if (blocks > kMaxInt / 2) return fail(POLICY_ERR_INVALID, "the launch would need over 2^30 blocks");
        d.blocks = static_cast<int>(blocks);
    }
    return POLICY_OK;
}

template <typename T, int LANES, int HEADS>
void launch_norm(const NormParams& p, bool backward, unsigned blocks, cudaStream_t stream)
{
    if (backward) qk_norm_grad_kernel<T, LANES, HEADS><<<blocks, kThreads, 0, stream>>>(p);
    else qk_norm_kernel<T, LANES, HEADS><<<blocks, kThreads, 0, stream>>>(p);
}

template <typename T, int LANES>
void launch_norm(const NormParams& p, int heads, bool backward, unsigned blocks, cudaStream_t stream)
{
    if (heads == 1) launch_norm<T, LANES, 1>(p, backward, blocks, stream);
    else if (heads == 2) launch_norm<T, LANES, 2>(p, backward, blocks, stream);
    else launch_norm<T, LANES, 4>(p, backward, blocks, stream);
}

template <typename T>
void launch_norm(const NormParams& p, const NormShape& s, bool backward, unsigned blocks, cudaStream_t stream)
{
    if (s.lanes == 4) launch_norm<T, 4>(p, s.heads, backward, blocks, stream);
    else if (s.lanes == 8) launch_norm<T, 8>(p, s.heads, backward, blocks, stream);
    else if (s.lanes == 16) launch_norm<T, 16>(p, s.heads, backward, blocks, stream);
    else launch_norm<T, 32>(p, s.heads, backward, blocks, stream);
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
    NormParams p;
    if ((rc = make_norm(*a, info.sms, backward, p)) != POLICY_OK) return rc;
    const unsigned blocks = static_cast<unsigned>(p.side[0].blocks) + static_cast<unsigned>(p.side[1].blocks);
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
    if (blocks > 0) {
        const NormShape shape = norm_shape(*a);
        if (a->dtype == POLICY_F32) launch_norm<float>(p, shape, backward, blocks, stream);
        else launch_norm<bf16>(p, shape, backward, blocks, stream);
        const cudaError_t e = cudaGetLastError();
        if (e != cudaSuccess) return cuda_fail(e, "qk_norm_kernel");
    }
    if (weights) {
        norm_weight_kernel<<<dim3(p.dim / 8, 2), 1024, 0, stream>>>(p);
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
    NormParams p;
    if (make_norm(*a, info.sms, true, p) != POLICY_OK) return 0;
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
