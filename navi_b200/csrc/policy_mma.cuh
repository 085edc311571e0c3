// Warp matrix products on shared-memory tiles for the two input types.
//
// A warp multiplies A [16 x KS] by B [KS x 8] into C [16 x 8] f32.  Lane l holds of C the
// rows l/4 and l/4 + 8, columns 2 (l%4) and 2 (l%4) + 1.
//   bf16: KS = 16, one product per step.
//   f32:  KS = 8, each operand split into a TF32 value and a TF32 remainder and the three
//         larger of the four partial products added (relative error about 2^-21 per product,
//         where a single TF32 product would keep 2^-11).
#pragma once

#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cstdint>

namespace policy {

using bf16 = __nv_bfloat16;

__device__ __forceinline__ uint32_t smem_addr(const void* p)
{
    return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}

// 16 bytes from global to shared memory; zeros when !take (nothing is read then).
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool take)
{
    const int n = take ? 16 : 0;
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;\n" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait()
{
    asm volatile("cp.async.wait_group %0;\n" ::"n"(N) : "memory");
}

template <typename T>
struct Mma;

template <>
struct Mma<bf16> {
    static constexpr int KS = 16;
    static constexpr int VEC = 8;   // values in 16 bytes
    static constexpr int PAD = 8;   // row padding: consecutive rows start 16 bytes apart modulo 128
    static constexpr bool kExact = false;
    struct A { uint32_t r[4]; };
    struct B { uint32_t r[2]; };

    static __device__ __forceinline__ void mma(float (&c)[4], const A& a, const B& b)
    {
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a.r[0]), "r"(a.r[1]), "r"(a.r[2]), "r"(a.r[3]), "r"(b.r[0]), "r"(b.r[1]));
    }
    // A at `tile` = (m0, k0) of a row-major [m][k] tile
    static __device__ __forceinline__ void load_a(A& a, const bf16* tile, int pitch, int lane)
    {
        const uint32_t p = smem_addr(tile + (lane & 15) * pitch + (lane >> 4) * 8);
        asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];\n"
                     : "=r"(a.r[0]), "=r"(a.r[1]), "=r"(a.r[2]), "=r"(a.r[3]) : "r"(p) : "memory");
    }
    // the B's of columns n0.. and n0 + 8.. from a tile stored [n][k] at (n0, k0)
    static __device__ __forceinline__ void load_b_nk(B& b0, B& b1, const bf16* tile, int pitch, int lane)
    {
        const uint32_t p = smem_addr(tile + ((lane & 7) + ((lane >> 4) << 3)) * pitch + ((lane >> 3) & 1) * 8);
        asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];\n"
                     : "=r"(b0.r[0]), "=r"(b0.r[1]), "=r"(b1.r[0]), "=r"(b1.r[1]) : "r"(p) : "memory");
    }
    // the same from a tile stored [k][n] at (k0, n0)
    static __device__ __forceinline__ void load_b_kn(B& b0, B& b1, const bf16* tile, int pitch, int lane)
    {
        const uint32_t p = smem_addr(tile + (lane & 15) * pitch + (lane >> 4) * 8);
        asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];\n"
                     : "=r"(b0.r[0]), "=r"(b0.r[1]), "=r"(b1.r[0]), "=r"(b1.r[1]) : "r"(p) : "memory");
    }
    // A of k step `step` from the C's of a [16 x n] product, rounded to bf16: the weights enter
    // the second product in the type of the values that they weigh, as a relative error of 2^-9
    // each that averages over the keys
    template <int N>
    static __device__ __forceinline__ void from_c(A& a, const float (&c)[N][4], int step)
    {
        a.r[0] = pack(c[2 * step][0], c[2 * step][1]);
        a.r[1] = pack(c[2 * step][2], c[2 * step][3]);
        a.r[2] = pack(c[2 * step + 1][0], c[2 * step + 1][1]);
        a.r[3] = pack(c[2 * step + 1][2], c[2 * step + 1][3]);
    }
    // The rounded weights back, for the sum that divides them: so they add up to 1, and what their roundings leave is off by
    // the spread of the values, not by their mean (which do . out would carry into every weight's gradient: rows of dq
    // off by more than their own size).
    template <int N>
    static __device__ __forceinline__ void to_c(float (&c)[N][4], const A& a, int step)
    {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float* at = c[2 * step + (i >> 1)] + 2 * (i & 1);
            at[0] = __uint_as_float(a.r[i] << 16), at[1] = __uint_as_float(a.r[i] & 0xffff0000u);
        }
    }
    // what that rounding leaves off, again as an A: both products together have the weights to 2^-17
    template <int N>
    static __device__ __forceinline__ void rest_of_c(A& a, const float (&c)[N][4], int step)
    {
        a.r[0] = pack(left_off(c[2 * step][0]), left_off(c[2 * step][1]));
        a.r[1] = pack(left_off(c[2 * step][2]), left_off(c[2 * step][3]));
        a.r[2] = pack(left_off(c[2 * step + 1][0]), left_off(c[2 * step + 1][1]));
        a.r[3] = pack(left_off(c[2 * step + 1][2]), left_off(c[2 * step + 1][3]));
    }
    static __device__ __forceinline__ float left_off(float x) { return x - __bfloat162float(__float2bfloat16_rn(x)); }
    static __device__ __forceinline__ uint32_t pack(float lo, float hi)
    {
        const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<const uint32_t*>(&v);
    }
    static __device__ __forceinline__ void store2(bf16* p, float a, float b) { *reinterpret_cast<uint32_t*>(p) = pack(a, b); }
};

// The k order inside a step is free as long as A and B share it: slot i < 4 holds k = 2i and
// slot i + 4 holds k = 2i + 1, so that a C tile is an A tile without moving a value between lanes.
template <>
struct Mma<float> {
    static constexpr int KS = 8;
    static constexpr int VEC = 4;
    static constexpr int PAD = 4;
    static constexpr bool kExact = true;
    struct A { float r[4]; };
    struct B { float r[2]; };

    // hi: the value rounded to TF32's 11 bits (half away from zero), by integers: the conversion instruction runs at
    // a fraction of their rate.  lo: what is left, of which the tensor core drops all below 2^-22 of the value.  An
    // infinite value leaves inf - inf and so gives NaN.
    static __device__ __forceinline__ void split(float x, uint32_t& hi, uint32_t& lo)
    {
        hi = (__float_as_uint(x) + 0x1000u) & 0xffffe000u;
        lo = __float_as_uint(x - __uint_as_float(hi));
    }
    static __device__ __forceinline__ void mma1(float (&c)[4], const uint32_t (&a)[4], const uint32_t (&b)[2])
    {
        asm volatile(
            "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
    }
    static __device__ __forceinline__ void mma(float (&c)[4], const A& a, const B& b)
    {
        uint32_t ah[4], al[4], bh[2], bl[2];
#pragma unroll
        for (int i = 0; i < 4; ++i) split(a.r[i], ah[i], al[i]);
#pragma unroll
        for (int i = 0; i < 2; ++i) split(b.r[i], bh[i], bl[i]);
        mma1(c, al, bh);
        mma1(c, ah, bl);
        mma1(c, ah, bh);
    }
    static __device__ __forceinline__ void load_a(A& a, const float* tile, int pitch, int lane)
    {
        const float* p = tile + (lane >> 2) * pitch + (lane & 3) * 2;
        const float2 x = *reinterpret_cast<const float2*>(p);
        const float2 y = *reinterpret_cast<const float2*>(p + 8 * pitch);
        a.r[0] = x.x, a.r[1] = y.x, a.r[2] = x.y, a.r[3] = y.y;
    }
    static __device__ __forceinline__ void load_b_nk(B& b0, B& b1, const float* tile, int pitch, int lane)
    {
        const float* p = tile + (lane >> 2) * pitch + (lane & 3) * 2;
        const float2 x = *reinterpret_cast<const float2*>(p);
        const float2 y = *reinterpret_cast<const float2*>(p + 8 * pitch);
        b0.r[0] = x.x, b0.r[1] = x.y, b1.r[0] = y.x, b1.r[1] = y.y;
    }
    static __device__ __forceinline__ void load_b_kn(B& b0, B& b1, const float* tile, int pitch, int lane)
    {
        const float* p = tile + (lane & 3) * 2 * pitch + (lane >> 2);
        b0.r[0] = p[0], b0.r[1] = p[pitch], b1.r[0] = p[8], b1.r[1] = p[pitch + 8];
    }
    template <int N>
    static __device__ __forceinline__ void from_c(A& a, const float (&c)[N][4], int step)
    {
        a.r[0] = c[step][0], a.r[1] = c[step][2], a.r[2] = c[step][1], a.r[3] = c[step][3];
    }
    template <int N>
    static __device__ __forceinline__ void to_c(float (&)[N][4], const A&, int) {}
    static __device__ __forceinline__ void store2(float* p, float a, float b)
    {
        *reinterpret_cast<float2*>(p) = make_float2(a, b);
    }
};

__device__ __forceinline__ float quad_max(float v)
{
    v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 1));
    return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 2));
}
__device__ __forceinline__ float quad_sum(float v)
{
    v += __shfl_xor_sync(0xffffffffu, v, 1);
    return v + __shfl_xor_sync(0xffffffffu, v, 2);
}

}  // namespace policy
