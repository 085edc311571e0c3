// Per-head RMS norm of queries and keys with the rotation by the token's angles, and its gradient.
//
//   u = w x r,  r = 1 / sqrt(mean(x^2) + eps);   y = R u, R the rotation of the first values
// and, since R is orthogonal,
//   g = R^T dy,  dw = sum over rows of g x r,  dx = r w g - r^3 x mean(w g x).
// Memory bounds both: one read of x (and dy) and one write; 64 x 12,288 tokens x 2 heads x 64 in bf16 take 70 us (5.8 TB/s),
// 112 us with gradients (1,024 x 192 tokens x 8 heads, 5.8 TB/s; 142 us with positions, whose angles come from L2).  A row belongs to LANES neighbouring
// lanes with 8 values each, so that a rotation's partner values sit rotary / 16 lanes away and are
// shuffled, not read again.  A thread keeps one token and up to HEADS of its heads and walks over
// batches: without positions the token's cosines and sines (four times the bytes of a bfloat16
// value each) are read once for all of them, and the next batch's rows are read while this one's
// are worked on.  Everything between the read and the one rounding at the store is in 32 bits, two
// values to an instruction (the f32x2 forms), since at 16 bits a value the issue slots come next
// after memory.
#include <atomic>
#include <cmath>
#include <limits>

#include "policy_internal.h"
#include "policy_mma.cuh"

namespace policy {
namespace {

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
    static constexpr int kPieces = 2;  // of 16 bytes
    // by way of L1: the two halves of a sector are two copies
    static __device__ __forceinline__ void copy(uint32_t dst, const float* src, bool take)
    {
        asm volatile("cp.async.ca.shared.global [%0], [%1], 16, %2;\n" ::"r"(dst), "l"(src), "r"(take ? 16 : 0) : "memory");
    }
    float4 a, b;
    __device__ __forceinline__ void fill(float v) { a = b = make_float4(v, v, v, v); }
    __device__ __forceinline__ void take(const uint4* ring)
    {
        a = *reinterpret_cast<const float4*>(ring), b = *reinterpret_cast<const float4*>(ring + kThreads);
    }
    __device__ __forceinline__ void load(const float* p)
    {
        a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
    }
    __device__ __forceinline__ Raw from(int lane) const
    {
        Raw r;
        r.a.x = __shfl_sync(0xffffffffu, a.x, lane), r.a.y = __shfl_sync(0xffffffffu, a.y, lane);
        r.a.z = __shfl_sync(0xffffffffu, a.z, lane), r.a.w = __shfl_sync(0xffffffffu, a.w, lane);
        r.b.x = __shfl_sync(0xffffffffu, b.x, lane), r.b.y = __shfl_sync(0xffffffffu, b.y, lane);
        r.b.z = __shfl_sync(0xffffffffu, b.z, lane), r.b.w = __shfl_sync(0xffffffffu, b.w, lane);
        return r;
    }
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
    static constexpr int kPieces = 1;
    static __device__ __forceinline__ void copy(uint32_t dst, const bf16* src, bool take) { copy16(dst, src, take); }
    uint4 a;
    __device__ __forceinline__ void take(const uint4* ring) { a = *ring; }
    // the values of another lane, two to a shuffle
    __device__ __forceinline__ Raw from(int lane) const
    {
        Raw r;
        r.a.x = __shfl_sync(0xffffffffu, a.x, lane), r.a.y = __shfl_sync(0xffffffffu, a.y, lane);
        r.a.z = __shfl_sync(0xffffffffu, a.z, lane), r.a.w = __shfl_sync(0xffffffffu, a.w, lane);
        return r;
    }
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

// The cosines and sines of a lane's 8 values, y = u cos + other sin: the sine is negative in the first half of a
// pair (backward: in the second).  Outside the table both are NaN, and so is every value that they meet.
struct Angles {
    Raw<float> c, n;
    template <int LANES, int HEADS>
    __device__ __forceinline__ void load(const NormParams& p, const NormSide& s, const Work<LANES, HEADS>& at, int pos)
    {
        const bool inside = pos >= 0 && pos < s.table_rows;
        if (at.active && inside && at.turned) {
            const float* row = s.table + static_cast<int64_t>(pos) * p.rotary + (at.low ? at.sub : at.sub - p.rotary / 16) * 8;
            c.load(row);
            n.load(row + p.rotary / 2);
        } else {
            c.fill(inside || !at.active ? 1.f : NAN);
            n.fill(0.f);
        }
    }
    __device__ __forceinline__ void get(bool negative, F2 (&cs)[4], F2 (&sn)[4]) const
    {
        c.get(cs);
        n.get(sn);
        const float sign = negative ? -1.f : 1.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) sn[i] = mul2(sn[i], pair(sign, sign));
    }
};

// The positions of a thread's token, batch by batch: the angles of the next round are read while this round's rows
// are worked on, the position after it at the same time.
template <int LANES, int HEADS>
struct Positions {
    const NormParams& p;
    const NormSide& s;
    const Work<LANES, HEADS>& at;
    Angles now;
    int following;
    __device__ __forceinline__ int position(int i) const
    {
        const int64_t b = at.b0 + i;
        return !s.positions ? at.token : b < at.b1 ? s.positions[b * s.tokens + at.token] : 0;
    }
    __device__ __forceinline__ Positions(const NormParams& p_, const NormSide& s_, const Work<LANES, HEADS>& at_) : p(p_), s(s_), at(at_)
    {
        now.load(p, s, at, position(0));
        following = position(1);
    }
    __device__ __forceinline__ Angles next(int i)
    {
        const Angles current = now;
        now.load(p, s, at, following);
        following = position(i + 2);
        return current;
    }
};

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

// Rows that a thread works on at a time: HEADS heads of its token, in as many batches as make kRows of them (one with
// positions, where each batch has its own angles).
template <typename T>
constexpr int kRows = sizeof(T) == 2 ? 4 : 2;

// The rows of the next rounds come by asynchronous copies into the thread's own places of a ring in shared memory
// (no other thread reads them, so no barrier): with the rows in registers instead, too few bytes were on their way
// (16 warps an SM, 4.5 TB/s).  TENSORS: x, or x and dy.
template <typename T, int HEADS, int TENSORS, bool POSITIONS>
struct Ring {
    static constexpr int BATCHES = POSITIONS ? 1 : kRows<T> / HEADS;
    static constexpr int ROWS = BATCHES * HEADS;
    static constexpr int kPieces = TENSORS * ROWS * Raw<T>::kPieces;  // 16-byte places of a stage
    static constexpr int kStages = kPieces <= 4 ? 4 : sizeof(T) == 4 ? 2 : 3;
    static constexpr size_t kBytes = sizeof(uint4) * kStages * kPieces * kThreads;

    uint4* mine;
    const T* x[TENSORS];
    int64_t batch[TENSORS], head[TENSORS];  // strides
    int b0, b1, heads;

    __device__ __forceinline__ void issue(int i)
    {
        uint4* to = mine + (i % kStages) * kPieces * kThreads;
#pragma unroll
        for (int t = 0; t < TENSORS; ++t) {
#pragma unroll
            for (int u = 0; u < BATCHES; ++u) {
                const int64_t b = static_cast<int64_t>(i) * BATCHES + u;
                const bool on = b0 + b < b1;
#pragma unroll
                for (int h = 0; h < HEADS; ++h) {
                    const bool take = on && h < heads;
                    const T* from = take ? x[t] + b * batch[t] + h * head[t] : x[t];
#pragma unroll
                    for (int c = 0; c < Raw<T>::kPieces; ++c, to += kThreads) Raw<T>::copy(smem_addr(to), from + c * (16 / sizeof(T)), take);
                }
            }
        }
        copy_commit();
    }
    __device__ __forceinline__ void start()
    {
#pragma unroll
        for (int i = 0; i < kStages - 1; ++i) issue(i);
    }
    // the rows of round i are there, and the round kStages - 1 later is on its way
    __device__ __forceinline__ const uint4* round(int i)
    {
        copy_wait<kStages - 2>();
        return mine + (i % kStages) * kPieces * kThreads;
    }
};

template <typename T, int LANES, int HEADS, bool POSITIONS>
__global__ void __launch_bounds__(kThreads, sizeof(T) == 2 && !POSITIONS ? 3 : 2) qk_norm_kernel(const __grid_constant__ NormParams p)
{
    using R = Ring<T, HEADS, 1, POSITIONS>;
    extern __shared__ uint4 ring_memory[];
    const bool second = blockIdx.x >= p.side[0].blocks;
    const NormSide& s = p.side[second ? 1 : 0];
    const Work<LANES, HEADS> at(p, s, second ? blockIdx.x - p.side[0].blocks : blockIdx.x);
    const int rounds = __reduce_max_sync(0xffffffffu, (at.b1 - at.b0 + R::BATCHES - 1) / R::BATCHES);
    const T* x = static_cast<const T*>(s.x) + at.b0 * s.xs[0] + at.token * s.xs[1] + at.h0 * s.xs[2] + at.sub * 8;
    R ring{ring_memory + threadIdx.x, {x}, {s.xs[0]}, {s.xs[2]}, at.b0, at.b1, at.heads};
    ring.start();
    const int64_t y_step = static_cast<int64_t>(s.tokens) * s.heads * p.dim;
    T* y = static_cast<T*>(s.y) + at.b0 * y_step + (static_cast<int64_t>(at.token) * s.heads + at.h0) * p.dim + at.sub * 8;

    // y = r (x (w cos) + other x (other w sin)): the products with the weights are made once for all rows of a token
    F2 w[4], wo[4], cs[4], sn[4];
    load_weight(w, s, at.sub, at.active);
#pragma unroll
    for (int k = 0; k < 4; ++k) wo[k] = shuffle2(w[k], at.other);
    const auto turn = [&](const Angles& a) {
        a.get(at.low, cs, sn);
#pragma unroll
        for (int k = 0; k < 4; ++k) cs[k] = mul2(cs[k], w[k]), sn[k] = mul2(sn[k], wo[k]);
    };
    const auto work = [&](int i) {
        Raw<T> raw[R::ROWS];
        const uint4* rows = ring.round(i);
#pragma unroll
        for (int k = 0; k < R::ROWS; ++k) raw[k].take(rows + k * Raw<T>::kPieces * kThreads);
        ring.issue(i + R::kStages - 1);
#pragma unroll
        for (int u = 0; u < R::BATCHES; ++u) {
            const int64_t b = i * R::BATCHES + u;
#pragma unroll
            for (int h = 0; h < HEADS; ++h) {
                F2 z[4];
                raw[u * HEADS + h].get(z);
                F2 sum = mul2(z[0], z[0]);
#pragma unroll
                for (int k = 1; k < 4; ++k) sum = fma2(z[k], z[k], sum);
                const float r = rsqrtf(fmaf(row_sum<LANES>(sum), p.inv_dim, p.eps));
                const F2 r2 = pair(r, r);
                if (s.table) {
                    F2 o[4];
                    raw[u * HEADS + h].from(at.other).get(o);
#pragma unroll
                    for (int k = 0; k < 4; ++k) z[k] = mul2(fma2(o[k], sn[k], mul2(z[k], cs[k])), r2);
                } else {
#pragma unroll
                    for (int k = 0; k < 4; ++k) z[k] = mul2(mul2(z[k], r2), cs[k]);
                }
                if (h < at.heads && at.b0 + b < at.b1) Raw<T>::store(y + b * y_step + h * p.dim, z);
            }
        }
    };
    if constexpr (POSITIONS) {
        Positions<LANES, HEADS> positions(p, s, at);
        for (int i = 0; i < rounds; ++i) {
            turn(positions.next(i));
            work(i);
        }
    } else {
        if (s.table) {
            Angles a;
            a.load(p, s, at, at.token);
            turn(a);
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k) cs[k] = w[k], sn[k] = pair(0.f, 0.f);
        }
        for (int i = 0; i < rounds; ++i) work(i);
    }
}

template <typename T, int LANES, int HEADS, bool POSITIONS>
__global__ void __launch_bounds__(kThreads, 2) qk_norm_grad_kernel(const __grid_constant__ NormParams p)
{
    using R = Ring<T, HEADS, 2, POSITIONS>;
    extern __shared__ uint4 ring_memory[];
    const bool second = blockIdx.x >= p.side[0].blocks;
    const NormSide& s = p.side[second ? 1 : 0];
    const int block = second ? blockIdx.x - p.side[0].blocks : blockIdx.x;
    const Work<LANES, HEADS> at(p, s, block);
    const int rounds = __reduce_max_sync(0xffffffffu, (at.b1 - at.b0 + R::BATCHES - 1) / R::BATCHES);
    const T* x = static_cast<const T*>(s.x) + at.b0 * s.xs[0] + at.token * s.xs[1] + at.h0 * s.xs[2] + at.sub * 8;
    const T* dy = static_cast<const T*>(s.dy) + at.b0 * s.ds[0] + at.token * s.ds[1] + at.h0 * s.ds[2] + at.sub * 8;
    R ring{ring_memory + threadIdx.x, {x, dy}, {s.xs[0], s.ds[0]}, {s.xs[2], s.ds[2]}, at.b0, at.b1, at.heads};
    ring.start();
    const int64_t dx_step = static_cast<int64_t>(s.tokens) * s.heads * p.dim;
    T* dx = static_cast<T*>(s.y) + at.b0 * dx_step + (static_cast<int64_t>(at.token) * s.heads + at.h0) * p.dim + at.sub * 8;

    F2 w[4], dw[4], cs[4], sn[4];
    load_weight(w, s, at.sub, at.active);
#pragma unroll
    for (int k = 0; k < 4; ++k) dw[k] = pair(0.f, 0.f);
    const auto work = [&](int i) {
        Raw<T> rx[R::ROWS], rg[R::ROWS];
        const uint4* rows = ring.round(i);
#pragma unroll
        for (int k = 0; k < R::ROWS; ++k) {
            rx[k].take(rows + k * Raw<T>::kPieces * kThreads);
            rg[k].take(rows + (R::ROWS + k) * Raw<T>::kPieces * kThreads);
        }
        ring.issue(i + R::kStages - 1);
#pragma unroll
        for (int u = 0; u < R::BATCHES; ++u) {
            const int64_t b = i * R::BATCHES + u;
#pragma unroll
            for (int h = 0; h < HEADS; ++h) {
                F2 v[4], g[4], gw[4];
                rx[u * HEADS + h].get(v);
                rg[u * HEADS + h].get(g);
                if (s.table) {
                    F2 o[4];
                    rg[u * HEADS + h].from(at.other).get(o);
#pragma unroll
                    for (int k = 0; k < 4; ++k) g[k] = fma2(o[k], sn[k], mul2(g[k], cs[k]));
                }
#pragma unroll
                for (int k = 0; k < 4; ++k) gw[k] = mul2(g[k], w[k]);
                F2 sum = mul2(v[0], v[0]), dot = mul2(v[0], gw[0]);
#pragma unroll
                for (int k = 1; k < 4; ++k) {
                    sum = fma2(v[k], v[k], sum);
                    dot = fma2(v[k], gw[k], dot);
                }
                const float r = rsqrtf(fmaf(row_sum<LANES>(sum), p.inv_dim, p.eps));
                const float f = -r * r * r * (row_sum<LANES>(dot) * p.inv_dim);
                const F2 r2 = pair(r, r), f2 = pair(f, f);
                if (h < at.heads && at.b0 + b < at.b1) {
                    F2 d[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        dw[k] = fma2(mul2(g[k], r2), v[k], dw[k]);
                        d[k] = fma2(gw[k], r2, mul2(f2, v[k]));
                    }
                    Raw<T>::store(dx + b * dx_step + h * p.dim, d);
                }
            }
        }
    };
    // the rotation back: the sines change sign
    if constexpr (POSITIONS) {
        Positions<LANES, HEADS> positions(p, s, at);
        for (int i = 0; i < rounds; ++i) {
            positions.next(i).get(!at.low, cs, sn);
            work(i);
        }
    } else {
        if (s.table) {
            Angles a;
            a.load(p, s, at, at.token);
            a.get(!at.low, cs, sn);
        }
        for (int i = 0; i < rounds; ++i) work(i);
    }
    if (!s.part) return;
    copy_wait<0>();
    __syncthreads();
    // the block's rows, in order
    float* sums = reinterpret_cast<float*>(ring_memory);
    static_assert(R::kBytes >= sizeof(float) * kThreads * 8, "the ring holds the sums");
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
    NormShape s{4, a.dtype == POLICY_F32 ? kRows<float> : kRows<bf16>};
    while (s.lanes * 8 < a.dim) s.lanes *= 2;
    const policy_norm_side& big = a.side[0].tokens * a.side[0].heads > a.side[1].tokens * a.side[1].heads ? a.side[0] : a.side[1];
    if (big.heads < s.heads && big.heads <= 2) s.heads = big.heads;
    return s;
}

// Threads' ranges of batches: as long as they leave each SM this many blocks.
constexpr int kBlocksPerSm = 8;

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
    const int64_t want = static_cast<int64_t>(sms) * kBlocksPerSm * groups;
    const int64_t round = (a.dtype == POLICY_F32 ? kRows<float> : kRows<bf16>) / shape.heads;  // batches at a time
    const int64_t length = total / want > 1 ? (total / want + round - 1) / round * round : 1;  // batches of a thread
    for (NormSide& d : p.side) {
        d.splits = static_cast<int>((a.batch + length - 1) / length);
        const int64_t blocks = (static_cast<int64_t>(d.splits) * d.tokens * d.chunks + groups - 1) / groups;
        if (blocks > kMaxInt / 2) return fail(POLICY_ERR_INVALID, "the launch would need over 2^30 blocks");
        d.blocks = static_cast<int>(blocks);
    }
    return POLICY_OK;
}

template <typename K>
int launch_ring(K kernel, size_t bytes, const NormParams& p, unsigned blocks, int device, std::atomic<uint64_t>& done, cudaStream_t stream)
{
    const uint64_t bit = device < 64 ? 1ull << device : 0ull;
    if (!bit || !(done.load(std::memory_order_relaxed) & bit)) {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes));
        if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute");
        done.fetch_or(bit, std::memory_order_relaxed);
    }
    kernel<<<blocks, kThreads, bytes, stream>>>(p);
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? POLICY_OK : cuda_fail(e, "qk_norm_kernel");
}

template <typename T, int LANES, int HEADS, bool POSITIONS>
int launch_norm(const NormParams& p, bool backward, unsigned blocks, int device, cudaStream_t stream)
{
    static std::atomic<uint64_t> done{0}, done_grad{0};
    if (backward)
        return launch_ring(qk_norm_grad_kernel<T, LANES, HEADS, POSITIONS>, Ring<T, HEADS, 2, POSITIONS>::kBytes, p, blocks, device, done_grad, stream);
    return launch_ring(qk_norm_kernel<T, LANES, HEADS, POSITIONS>, Ring<T, HEADS, 1, POSITIONS>::kBytes, p, blocks, device, done, stream);
}

template <typename T, int LANES, int HEADS>
int launch_norm(const NormParams& p, bool backward, unsigned blocks, int device, cudaStream_t stream)
{
    if (p.side[0].positions || p.side[1].positions) return launch_norm<T, LANES, HEADS, true>(p, backward, blocks, device, stream);
    return launch_norm<T, LANES, HEADS, false>(p, backward, blocks, device, stream);
}

template <typename T, int LANES>
int launch_norm(const NormParams& p, int heads, bool backward, unsigned blocks, int device, cudaStream_t stream)
{
    if (heads == 1) return launch_norm<T, LANES, 1>(p, backward, blocks, device, stream);
    if (sizeof(T) == 4 || heads == 2) return launch_norm<T, LANES, 2>(p, backward, blocks, device, stream);
    if constexpr (sizeof(T) == 2) return launch_norm<T, LANES, 4>(p, backward, blocks, device, stream);
    return POLICY_ERR_INVALID;
}

template <typename T>
int launch_norm(const NormParams& p, const NormShape& s, bool backward, unsigned blocks, int device, cudaStream_t stream)
{
    if (s.lanes == 4) return launch_norm<T, 4>(p, s.heads, backward, blocks, device, stream);
    if (s.lanes == 8) return launch_norm<T, 8>(p, s.heads, backward, blocks, device, stream);
    if (s.lanes == 16) return launch_norm<T, 16>(p, s.heads, backward, blocks, device, stream);
    return launch_norm<T, 32>(p, s.heads, backward, blocks, device, stream);
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
        rc = a->dtype == POLICY_F32 ? launch_norm<float>(p, shape, backward, blocks, a->device, stream)
                                    : launch_norm<bf16>(p, shape, backward, blocks, a->device, stream);
        if (rc != POLICY_OK) return rc;
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
