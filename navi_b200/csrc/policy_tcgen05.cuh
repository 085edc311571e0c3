// The fifth-generation tensor core from one block: barriers, tensor memory, matrix descriptors.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include <cstdint>

namespace policy {

// --- shared-memory barriers ------------------------------------------------------

__device__ __forceinline__ void bar_init(uint32_t bar, uint32_t arrivals)
{
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;\n" ::"r"(bar), "r"(arrivals) : "memory");
}
__device__ __forceinline__ void bar_arrive(uint32_t bar)
{
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];\n" ::"r"(bar) : "memory");
}
// One arrival for a warp whose lanes have all come here (arrivals on one barrier are served one by one).
__device__ __forceinline__ void warp_arrive(uint32_t bar)
{
    __syncwarp();
    if ((threadIdx.x & 31) == 0) bar_arrive(bar);
}
// One arrival, after which the phase also waits for `bytes` of copies.
__device__ __forceinline__ void bar_expect(uint32_t bar, uint32_t bytes)
{
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n" ::"r"(bar), "r"(bytes) : "memory");
}
// Whether the phase is over; the hardware holds the thread for some microseconds until it is.
__device__ __forceinline__ bool bar_try(uint32_t bar, uint32_t parity)
{
    uint32_t done;
    asm volatile(
        "{\n.reg .pred p;\n"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n"
        "selp.u32 %0, 1, 0, p;\n}\n"
        : "=r"(done) : "r"(bar), "r"(parity), "r"(20000u) : "memory");
    return done != 0;
}

// A wait lasts as long as a few tiles' work, microseconds.  One of two seconds' polls can only come from a defect: it
// raises the block's flag, on which every role leaves its loop, and the host's word at the end.  It counts polls, not the
// clock, which goes on while a context is paused (by a debugger, or for another process).
constexpr uint32_t kPollNs = 32'768;  // how long a poll that fails is held (measured)
constexpr uint32_t kWaitPolls = 2'000'000'000 / kPollNs;

__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity, volatile int* broken, uint32_t polls = kWaitPolls)
{
    if (bar_try(bar, parity)) return true;
#pragma unroll 1
    for (uint32_t n = 0; n < polls; ++n) {
        if (bar_try(bar, parity)) return true;
        if (*broken) return false;
    }
    *broken = 1;
    return false;
}

// The same for a whole warp, with one answer.
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile int* broken)
{
    return __all_sync(0xffffffffu, bar_wait(bar, parity, broken));
}

// By one thread of the block after its last barrier: tells the host that a wait ran out.
__device__ __forceinline__ void report_stall(const volatile int* broken, int32_t* word)
{
    if (!*broken) return;
    *static_cast<volatile int32_t*>(word) = 1;
    __threadfence_system();
}

// Makes what the calling thread wrote to shared memory visible to the tensor core.
__device__ __forceinline__ void fence_async_shared() { asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory"); }

// --- tensor memory ---------------------------------------------------------------

// One warp allocates, the same warp frees.
__device__ __forceinline__ void tmem_alloc(uint32_t dst, uint32_t columns)
{
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(dst), "r"(columns) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n");
}
__device__ __forceinline__ void tmem_free(uint32_t tmem, uint32_t columns)
{
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(columns));
}
__device__ __forceinline__ void fence_before_sync() { asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory"); }
__device__ __forceinline__ void fence_after_sync() { asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_load() { asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_store() { asm volatile("tcgen05.wait::st.sync.aligned;\n" ::: "memory"); }

// 32 columns of the calling warp's 32 lanes: thread l gets lane l.  Complete after tmem_wait_load.
__device__ __forceinline__ void tmem_load32(float* v, uint32_t tmem)
{
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n"
        : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]), "=f"(v[9]),
          "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]), "=f"(v[16]), "=f"(v[17]), "=f"(v[18]),
          "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]), "=f"(v[24]), "=f"(v[25]), "=f"(v[26]), "=f"(v[27]),
          "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31])
        : "r"(tmem)
        : "memory");
}
__device__ __forceinline__ void tmem_store32(uint32_t tmem, const float* v)
{
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};\n" ::"f"(v[0]),
        "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]), "f"(v[8]), "f"(v[9]), "f"(v[10]), "f"(v[11]),
        "f"(v[12]), "f"(v[13]), "f"(v[14]), "f"(v[15]), "f"(v[16]), "f"(v[17]), "f"(v[18]), "f"(v[19]), "f"(v[20]), "f"(v[21]),
        "f"(v[22]), "f"(v[23]), "f"(v[24]), "f"(v[25]), "f"(v[26]), "f"(v[27]), "f"(v[28]), "f"(v[29]), "f"(v[30]), "f"(v[31]),
        "r"(tmem)
        : "memory");
}
__device__ __forceinline__ void tmem_load8(float* v, uint32_t tmem)
{
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];\n"
                 : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7])
                 : "r"(tmem)
                 : "memory");
}
__device__ __forceinline__ void tmem_store8(uint32_t tmem, const float* v)
{
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%8], {%0,%1,%2,%3,%4,%5,%6,%7};\n" ::"f"(v[0]), "f"(v[1]), "f"(v[2]),
                 "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]), "r"(tmem)
                 : "memory");
}
__device__ __forceinline__ void tmem_store16(uint32_t tmem, const uint32_t* v)
{
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};\n" ::"r"(v[0]),
        "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]),
        "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(tmem)
        : "memory");
}

// --- products --------------------------------------------------------------------
//
// Operand tiles lie in shared memory as blocks of 64 bf16 columns: a block's row is 128 bytes, and its
// 16-byte pieces are permuted by the row (piece c of row r at c ^ (r & 7)), the 128-byte swizzle.

constexpr uint32_t kBlockRow = 128;  // bytes

__device__ __forceinline__ uint32_t swizzled(int row, int piece) { return row * kBlockRow + ((piece ^ (row & 7)) << 4); }

// The matrix descriptor of a swizzled tile.  Its low word holds the address and `next_block`, the bytes from one
// 64-column block to the next, used where the blocks run along the product's M or N; its high word says that
// rows advance 8 at a time by 1,024 bytes.  Advancing the address adds its sixteenth to the low word.
__device__ __forceinline__ uint32_t tile_descriptor(uint32_t addr, uint32_t next_block)
{
    return ((addr & 0x3ffffu) >> 4) | (next_block >> 4) << 16;
}
constexpr uint32_t kDescriptorHigh = 1024u >> 4 | 1u << 14 | 2u << 29;

// bf16 x bf16 -> f32, M x N; transposed_x: the operand is stored with its M (or N) axis contiguous.
__host__ __device__ constexpr uint32_t bf16_product(int m, int n, bool transposed_a, bool transposed_b)
{
    return 1u << 4 | 1u << 7 | 1u << 10 | static_cast<uint32_t>(transposed_a) << 15 | static_cast<uint32_t>(transposed_b) << 16 |
           static_cast<uint32_t>(n >> 3) << 17 | static_cast<uint32_t>(m >> 4) << 24;
}

// One lane of a converged warp.  The compiler knows that one lane at most goes on; under a plain test of the lane
// it would have to issue the products, whose operands sit in the warp's uniform registers, in a loop over lanes.
__device__ __forceinline__ bool elected()
{
    uint32_t one;
    asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xffffffff;\nselp.u32 %0, 1, 0, p;\n}\n" : "=r"(one));
    return one != 0;
}

// d (+)= a b, 16 deep, both operands in shared memory.  One elected thread issues all products of a block, which
// the tensor core runs in the order of issue.
__device__ __forceinline__ void product_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t kind, bool add)
{
    asm volatile(
        "{\n.reg .pred p;\n.reg .b64 x, y;\nsetp.ne.u32 p, %4, 0;\n"
        "mov.b64 x, {%1, %5};\nmov.b64 y, {%2, %5};\n"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %3, p;\n}\n" ::"r"(d), "r"(a), "r"(b), "r"(kind), "r"(static_cast<uint32_t>(add)),
        "n"(kDescriptorHigh)
        : "memory");
}
// the same with a in tensor memory: two bf16 of a row in each column
__device__ __forceinline__ void product_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t kind, bool add)
{
    asm volatile(
        "{\n.reg .pred p;\n.reg .b64 y;\nsetp.ne.u32 p, %4, 0;\n"
        "mov.b64 y, {%2, %5};\n"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], y, %3, p;\n}\n" ::"r"(d), "r"(a), "r"(b), "r"(kind), "r"(static_cast<uint32_t>(add)),
        "n"(kDescriptorHigh)
        : "memory");
}
// One arrival at `bar` when every product issued so far by the calling thread is complete.
__device__ __forceinline__ void products_arrive(uint32_t bar)
{
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n" ::"r"(bar) : "memory");
}

// --- copies and arithmetic --------------------------------------------------------

// A tile by TMA: 64 columns from `column` of the map's heads and tokens from (head, token) on; counts its bytes at `bar`.
__device__ __forceinline__ void copy_tile(uint32_t dst, const CUtensorMap* map, int column, int head, int token, int batch, uint32_t bar)
{
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];\n" ::"r"(dst),
        "l"(map), "r"(column), "r"(head), "r"(token), "r"(batch), "r"(bar)
        : "memory");
}

// two f32 to an instruction
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c)
{
    float2 r;
    asm("{\n.reg .b64 x, y, z;\nmov.b64 x, {%2, %3};\nmov.b64 y, {%4, %5};\nmov.b64 z, {%6, %7};\n"
        "fma.rn.f32x2 x, x, y, z;\nmov.b64 {%0, %1}, x;\n}\n"
        : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return r;
}
// sum += the two bf16 of w, in f32: without unpacking them first, which cost the forward pass 2 to 3 %
__device__ __forceinline__ void add_bf16(float2& sum, uint32_t w)
{
    asm("{\n.reg .b16 lo, hi;\nmov.b32 {lo, hi}, %2;\nadd.rn.f32.bf16 %0, lo, %0;\nadd.rn.f32.bf16 %1, hi, %1;\n}\n"
        : "+f"(sum.x), "+f"(sum.y) : "r"(w));
}
__device__ __forceinline__ float2 same(float v) { return make_float2(v, v); }

}  // namespace policy
