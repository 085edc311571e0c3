// The gradients of cross attention for many rows, on the tcgen05 tensor cores (bf16).
//
// Both kernels keep one tile pair X and stream another, Y, past it:
//   kKeys (dk, dv): X = 128 keys' K and V, Y = 64 rows' Q and dO;
//   else (dq):      X = 128 rows' Q and dO, Y = 64 keys' K and V.
// For every Y:  S = X_a Y_a^T,  T = X_b Y_b^T  (128 x 64, f32 in tensor memory), then a thread to a row of X
//   p = 2^(c s - x_i) y_i,   ds = p (t - D_i)
// written as bf16 over S and T (0.0024 of the gradients' norm off with it, 0.0017 of that from their own rounding), and
// the products  dv += P dO, dk += dS Q  (or dq += dS K) with the left operand from tensor memory.  dv, dk and dq stay in
// tensor memory for the whole item.  A block has two sets (one where tensor memory has no room for two: dk and dv at dim
// 128), each with 4 warps and its own product-issuing thread, so that one set's products run during the other's
// arithmetic.  Blocks are persistent, one per SM.
//
// All tiles come by TMA, a row tile as 64 / group tokens x group heads.  One warp follows the copies of Y: for dq
// it zeroes K's invisible rows (0 x NaN would be NaN) and says which keys are visible, for dk and dv it brings the
// rows' statistics.  (S may be reading a row of K while it is zeroed: that column of S is not used.)  Bound by the products: at 64 columns the two SS products read shared memory faster than its
// 128 bytes a clock (48 clocks per 16 deep instead of 32).  Measured, 8 x 4,096 rows x 768 keys x 64, 8 / 4 heads: dk and dv
// 195 us, dq 177 us, 410 us with D (314 TFLOP/s); the chain products - weights - products of a tile is what is left.
#include <atomic>
#include <limits>

#include "policy_attention.cuh"
#include "policy_internal.h"
#include "policy_map.h"
#include "policy_tcgen05.cuh"

namespace policy {
namespace {

constexpr int kThreads = 384;
constexpr int kWarps = 8;    // then copies, statistics, products of either set
constexpr int kX = 128;      // rows of an X tile
constexpr int kY = kGradTcStream;  // rows of a Y tile

template <bool kKeys, int DP>
struct GradTc {
    static constexpr int kSets = kKeys && DP == 128 ? 1 : 2;
    static constexpr int kBlocks = DP / 64;
    static constexpr uint32_t kXBlock = kX * kBlockRow, kYBlock = kY * kBlockRow;
    static constexpr uint32_t kXTile = kBlocks * kXBlock, kYTile = kBlocks * kYBlock;  // one operand
    static constexpr int kStages = DP == 64 ? 4 : kKeys ? 3 : 2;
    static constexpr uint32_t kXAt = 0;  // [set][a, b]
    static constexpr uint32_t kYAt = 2 * kSets * kXTile;  // [stage][a, b]
    static constexpr uint32_t kSide = kYAt + 2 * kStages * kYTile;  // per stage: 64 x (exponent, D), or 64 bits of visibility
    static constexpr uint32_t kStore = kSide + kStages * kY * 8;    // 32 rows x 128 bytes for each warp
    static constexpr uint32_t kBars = kStore + kSets * 4 * 32 * kBlockRow;
    static constexpr uint32_t kBytes = kBars + 256;
    static constexpr uint32_t kAligned = kBytes + 1024;
    // columns of tensor memory, per set: S, T (P and dS over them), sums
    static constexpr int kSums = kKeys ? 2 : 1;
    static constexpr int kColumns = 2 * kY + kSums * DP;
    static_assert(kSets * kColumns <= 512, "tensor memory");
};

enum Bar { kXFull, kXEmpty = kXFull + 2, kSFull = kXEmpty + 2, kWFull = kSFull + 2, kAccFull = kWFull + 2, kAccEmpty = kAccFull + 2, kLast = kAccEmpty + 2, kYFull = kLast + 2 };
// then Y full, Y ready (followed up), Y empty: kStages each

struct GradMaps {
    CUtensorMap q, dout, k, v;
};

template <bool kKeys, int DP>
struct GradItem {
    using S = GradTc<kKeys, DP>;
    int split, x0, t0, t1, n;
    Rows rows;
    __device__ __forceinline__ GradItem(const AttnParams& p, int item)
    {
        split = item % p.splits;
        const int tile = (item / p.splits) % p.tiles;
        const int bh = item / p.splits / p.tiles;
        rows = Rows{bh / p.kv_heads, bh % p.kv_heads, p.group};
        x0 = tile * kX * S::kSets;
        n = visible_keys(p, rows.b);
        int tiles = ((kKeys ? p.rows : n) + kY - 1) / kY;
        if (kKeys && x0 >= n) tiles = 0;  // no key of the tile is visible
        t0 = static_cast<int>(static_cast<int64_t>(tiles) * split / p.splits);
        t1 = static_cast<int>(static_cast<int64_t>(tiles) * (split + 1) / p.splits);
    }
    __device__ __forceinline__ bool has(const AttnParams& p, int i) const { return x0 + i * kX < (kKeys ? p.lk : p.rows); }
};

template <bool kKeys, int DP>
__global__ void __launch_bounds__(kThreads, 1) attend_grad_tc_kernel(const __grid_constant__ AttnParams p, const __grid_constant__ GradMaps maps, int items)
{
    using S = GradTc<kKeys, DP>;
    using Item = GradItem<kKeys, DP>;
    extern __shared__ unsigned char raw[];
    __shared__ uint32_t tmem_at;
    __shared__ int broken_flag;
    volatile int* broken = &broken_flag;
    const uint32_t base = (smem_addr(raw) + 1023u) & ~1023u;
    unsigned char* smem = raw + (base - smem_addr(raw));
    const auto bar = [&](int i) { return base + S::kBars + 8u * i; };
    constexpr int ST = S::kStages, kSets = S::kSets;
    constexpr int kYReady = kYFull + ST, kYEmpty = kYReady + ST, kAll = kYEmpty + ST;
    static_assert(kAll * 8 <= 256, "barriers");
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        broken_flag = 0;
        for (int i = 0; i < 2; ++i) {
            bar_init(bar(kXFull + i), 1);
            bar_init(bar(kXEmpty + i), 4);
            bar_init(bar(kSFull + i), 1);
            bar_init(bar(kWFull + i), 4);
            bar_init(bar(kAccFull + i), 1);
            bar_init(bar(kAccEmpty + i), 4);
            bar_init(bar(kLast + i), 1);
        }
        for (int i = 0; i < ST; ++i) {
            bar_init(bar(kYFull + i), 1);
            bar_init(bar(kYReady + i), 1);
            bar_init(bar(kYEmpty + i), kSets);
        }
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    }
    if (warp == kWarps + 2) tmem_alloc(smem_addr(&tmem_at), 512);
    fence_before_sync();
    __syncthreads();
    fence_after_sync();
    const uint32_t tmem = tmem_at;

    if (warp == kWarps) {
        // --- copies ---
        if (elected()) {
            const int q_tokens = kX / p.group, y_tokens = kY / p.group;
            uint32_t uses = 0, x_uses[2] = {0u, 0u};
            bool ok = true;
            for (int it = blockIdx.x; it < items && ok; it += gridDim.x) {
                const Item item(p, it);
                if (item.t0 >= item.t1) continue;
                const int b = static_cast<int>(item.rows.b);
                const int kb = p.ks[0] ? b : 0, kh = p.ks[2] ? item.rows.hk : 0, vb = p.vs[0] ? b : 0, vh = p.vs[2] ? item.rows.hk : 0;
                const int qb = p.qs[0] ? b : 0, qh = p.qs[2] ? item.rows.hk * p.group : 0;
                const int db = p.ds[0] ? b : 0, dh = p.ds[2] ? item.rows.hk * p.group : 0;
#pragma unroll
                for (int i = 0; i < kSets; ++i) {
                    if (!item.has(p, i)) continue;
                    if (!(ok = bar_wait(bar(kXEmpty + i), (x_uses[i] & 1u) ^ 1u, broken))) break;
                    ++x_uses[i];
                    bar_expect(bar(kXFull + i), 2 * S::kXTile);
                    const uint32_t at = base + S::kXAt + 2 * i * S::kXTile;
                    for (int c = 0; c < S::kBlocks; ++c) {
                        if (kKeys) {
                            copy_tile(at + c * S::kXBlock, &maps.k, c * 64, kh, item.x0 + i * kX, kb, bar(kXFull + i));
                            copy_tile(at + S::kXTile + c * S::kXBlock, &maps.v, c * 64, vh, item.x0 + i * kX, vb, bar(kXFull + i));
                        } else {
                            const int token = item.x0 / p.group + i * q_tokens;
                            copy_tile(at + c * S::kXBlock, &maps.q, c * 64, qh, token, qb, bar(kXFull + i));
                            copy_tile(at + S::kXTile + c * S::kXBlock, &maps.dout, c * 64, dh, token, db, bar(kXFull + i));
                        }
                    }
                }
                for (int t = item.t0; t < item.t1 && ok; ++t, ++uses) {
                    const int st = uses % ST;
                    if (!(ok = bar_wait(bar(kYEmpty + st), ((uses / ST) & 1u) ^ 1u, broken))) break;
                    bar_expect(bar(kYFull + st), 2 * S::kYTile);
                    const uint32_t at = base + S::kYAt + 2 * st * S::kYTile;
                    for (int c = 0; c < S::kBlocks; ++c) {
                        if (kKeys) {
                            copy_tile(at + c * S::kYBlock, &maps.q, c * 64, qh, t * y_tokens, qb, bar(kYFull + st));
                            copy_tile(at + S::kYTile + c * S::kYBlock, &maps.dout, c * 64, dh, t * y_tokens, db, bar(kYFull + st));
                        } else {
                            copy_tile(at + c * S::kYBlock, &maps.k, c * 64, kh, t * kY, kb, bar(kYFull + st));
                            copy_tile(at + S::kYTile + c * S::kYBlock, &maps.v, c * 64, vh, t * kY, vb, bar(kYFull + st));
                        }
                    }
                }
            }
            if (!ok) {  // copies that nobody will wait for must not outlive the block
                volatile int quiet = 0;
                for (uint32_t u = uses > ST ? uses - ST : 0; u < uses; ++u) bar_wait(bar(kYFull + u % ST), (u / ST) & 1u, &quiet);
                for (int i = 0; i < kSets; ++i)
                    if (x_uses[i]) bar_wait(bar(kXFull + i), (x_uses[i] - 1) & 1u, &quiet);
            }
        }
        __syncwarp();
    } else if (warp == kWarps + 1) {
        // --- what belongs to a Y tile beside its values ---
        uint32_t uses = 0;
        bool ok = true;
        for (int it = blockIdx.x; it < items && ok; it += gridDim.x) {
            const Item item(p, it);
            const uint8_t* mask = p.mask ? p.mask + item.rows.b * p.mask_stride : nullptr;
            float2 next[2];  // kKeys: of rows lane and lane + 32; else: whether keys lane and lane + 32 are visible, in x
            const auto fetch = [&](int t) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int r = t * kY + h * 32 + lane;
                    if (kKeys) {
                        next[h] = make_float2(INFINITY, 0.f);  // a weight of 0
                        if (r < p.rows) {
                            const int64_t row = item.rows.index(p, r);
                            const float2 st = p.stats[row];
                            // one exponent for both: its rounding is far below that of the weights
                            if (st.y != 0.f) next[h] = make_float2(st.x - log2f(st.y), p.delta[row]);
                        }
                    } else {
                        bool on = r < item.n;
                        if (mask && on) on = __ldg(mask + r) != 0;
                        next[h].x = on ? 1.f : 0.f;
                    }
                }
            };
            if (item.t0 < item.t1) fetch(item.t0);
            for (int t = item.t0; t < item.t1; ++t, ++uses) {
                const int st = uses % ST;
                if (!(ok = warp_wait(bar(kYFull + st), (uses / ST) & 1u, broken))) break;
                unsigned char* side = smem + S::kSide + st * kY * 8;
                if (kKeys) {
                    reinterpret_cast<float2*>(side)[lane] = next[0];
                    reinterpret_cast<float2*>(side)[lane + 32] = next[1];
                } else {
                    const uint32_t w0 = __ballot_sync(0xffffffffu, next[0].x != 0.f), w1 = __ballot_sync(0xffffffffu, next[1].x != 0.f);
                    if (lane == 0) *reinterpret_cast<uint2*>(side) = make_uint2(w0, w1);
                    if ((w0 & w1) != 0xffffffffu) {
                        unsigned char* tile = smem + S::kYAt + 2 * st * S::kYTile;
#pragma unroll
                        for (int g = 0; g < kY / 4; ++g) {  // 4 rows at a time, 8 lanes to a row
                            const int row = g * 4 + (lane >> 3);
                            if (((row < 32 ? w0 : w1) >> (row & 31)) & 1u) continue;
#pragma unroll
                            for (int c = 0; c < S::kBlocks; ++c)
                                *reinterpret_cast<uint4*>(tile + c * S::kYBlock + swizzled(row, lane & 7)) = make_uint4(0u, 0u, 0u, 0u);
                        }
                    }
                    fence_async_shared();
                }
                warp_arrive(bar(kYReady + st));
                if (t + 1 < item.t1) fetch(t + 1);
            }
        }
    } else if (warp >= kWarps + 2) {
        // --- products of one set ---
        const int i = warp - (kWarps + 2);
        if (i < kSets && elected()) {
            const uint32_t inner = bf16_product(kX, kY, false, false);
            const uint32_t outer = bf16_product(kX, (p.dim + 15) & ~15, false, true);
            const uint32_t x_at = tile_descriptor(base + S::kXAt + 2 * i * S::kXTile, 0);
            const uint32_t y_inner = tile_descriptor(base + S::kYAt, 0), y_outer = tile_descriptor(base + S::kYAt, S::kYBlock);
            const uint32_t ts = tmem + i * S::kColumns, tt = ts + kY, acc = tt + kY;
            uint32_t uses = 0, done = 0, tiles = 0;
            bool ok = true;
            for (int it = blockIdx.x; it < items && ok; it += gridDim.x) {
                const Item item(p, it);
                if (item.t0 >= item.t1) continue;
                if (!item.has(p, i)) {  // the stages wait for both sets: one after the other, as they come
                    for (int t = item.t0; t < item.t1; ++t, ++uses) {
                        if (!(ok = bar_wait(bar(kYReady + uses % ST), (uses / ST) & 1u, broken))) break;
                        bar_arrive(bar(kYEmpty + uses % ST));
                    }
                    continue;
                }
                if (!(ok = bar_wait(bar(kXFull + i), done & 1u, broken))) break;
                for (int t = item.t0; t < item.t1; ++t, ++uses, ++tiles) {
                    const int st = uses % ST;
                    const uint32_t y = 2 * st * (S::kYTile >> 4);
                    if (!(ok = bar_wait(bar(kYFull + st), (uses / ST) & 1u, broken))) break;
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
#pragma unroll
                        for (int s = 0; s < DP / 16; ++s)
                            product_ss(h ? tt : ts, x_at + ((h * S::kXTile + (s >> 2) * S::kXBlock + (s & 3) * 32u) >> 4),
                                       y_inner + y + ((h * S::kYTile + (s >> 2) * S::kYBlock + (s & 3) * 32u) >> 4), inner, s > 0);
                    }
                    products_arrive(bar(kSFull + i));
                    if (!(ok = bar_wait(bar(kYReady + st), (uses / ST) & 1u, broken))) break;
                    if (t == item.t0 && !(ok = bar_wait(bar(kAccEmpty + i), (done & 1u) ^ 1u, broken))) break;
                    if (!(ok = bar_wait(bar(kWFull + i), tiles & 1u, broken))) break;
                    fence_after_sync();
#pragma unroll
                    for (int s = 0; s < kY / 16; ++s) {
                        const uint32_t at = y + s * (16 * kBlockRow >> 4);
                        product_ts(acc, tt + s * 8, y_outer + at, outer, t > item.t0 || s > 0);                                           // dS Y_a
                        if (kKeys) product_ts(acc + DP, ts + s * 8, y_outer + at + (S::kYTile >> 4), outer, t > item.t0 || s > 0);       // P Y_b
                    }
                    products_arrive(bar(kYEmpty + st));
                }
                if (!ok) break;
                products_arrive(bar(kAccFull + i));
                ++done;
            }
            if (!ok) {  // tensor memory is freed after the products that are still running
                volatile int quiet = 0;
                products_arrive(bar(kLast + i));
                bar_wait(bar(kLast + i), 0, &quiet);
            }
        }
        __syncwarp();
    } else if ((warp >> 2) < kSets) {
        // --- weights: a thread to a row of X ---
        const int i = warp >> 2;
        const int lane_row = (warp & 3) * 32 + lane;
        const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
        const uint32_t ts = tmem + lanes + i * S::kColumns, tt = ts + kY, acc = tt + kY;
        const float c = p.scale_log2;
        uint32_t uses = 0, tiles = 0, done = 0;
        for (int it = blockIdx.x; it < items; it += gridDim.x) {
            const Item item(p, it);
            if (!item.has(p, i)) {
                uses += item.t1 - item.t0;
                continue;
            }
            const int r = item.x0 + i * kX + lane_row;
            const bool in = r < (kKeys ? p.lk : p.rows);
            const bool any = item.t0 < item.t1;
            bool on = false;                  // kKeys: the key is visible
            float exponent = INFINITY, delta = 0.f;  // else: of the row
            if (kKeys) {
                on = r < item.n;
                if (p.mask && on) on = __ldg(p.mask + item.rows.b * p.mask_stride + r) != 0;
            } else if (in) {
                const int64_t row = item.rows.index(p, r);
                const float2 st = p.stats[row];
                if (st.y != 0.f) exponent = st.x - log2f(st.y), delta = p.delta[row];
            }
            const bool slope = !lone_key(p, item.rows.b, item.n) && (kKeys ? on : exponent != INFINITY);
            bool ok = __all_sync(0xffffffffu, !*broken);
            for (int t = item.t0; t < item.t1 && ok; ++t, ++uses, ++tiles) {
                const int st = uses % ST;
                if (!(ok = warp_wait(bar(kSFull + i), tiles & 1u, broken))) break;
                if (!(ok = warp_wait(bar(kYReady + st), (uses / ST) & 1u, broken))) break;
                fence_after_sync();
                const float4* side = reinterpret_cast<const float4*>(smem + S::kSide + st * kY * 8);
                uint2 vis = make_uint2(0xffffffffu, 0xffffffffu);
                if (!kKeys) vis = *reinterpret_cast<const uint2*>(side);
#pragma unroll
                for (int h = 0; h < 2; ++h) {  // 32 columns at a time
                    float s[32], d[32];
                    tmem_load32(s, ts + h * 32);
                    tmem_load32(d, tt + h * 32);
                    tmem_wait_load();
                    uint32_t wp[16], wd[16];
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        float e0 = exponent, e1 = exponent, d0 = delta, d1 = delta;
                        if (kKeys) {
                            const float4 x = side[h * 16 + j];
                            e0 = x.x, d0 = x.y, e1 = x.z, d1 = x.w;
                        }
                        float p0 = exp2_fast(fmaf(s[2 * j], c, -e0)), p1 = exp2_fast(fmaf(s[2 * j + 1], c, -e1));
                        const bool on0 = kKeys ? on : (((h ? vis.y : vis.x) >> (2 * j)) & 1u), on1 = kKeys ? on : (((h ? vis.y : vis.x) >> (2 * j + 1)) & 1u);
                        const float g0 = on0 && slope ? p0 * (d[2 * j] - d0) : 0.f, g1 = on1 && slope ? p1 * (d[2 * j + 1] - d1) : 0.f;
                        wd[j] = Mma<bf16>::pack(g0, g1);
                        if (kKeys) wp[j] = Mma<bf16>::pack(on ? p0 : 0.f, on ? p1 : 0.f);
                    }
                    // P and dS lie over the columns of S and T that are in registers already: 16 of every 32
                    if (kKeys) tmem_store16(ts + h * 16, wp);
                    tmem_store16(tt + h * 16, wd);
                }
                tmem_wait_store();
                fence_before_sync();
                warp_arrive(bar(kWFull + i));
            }
            if (ok && any) {
                ok = warp_wait(bar(kAccFull + i), done & 1u, broken);
                ++done;
                fence_after_sync();
            }
            const int64_t row = kKeys ? (item.rows.b * p.lk + (in ? r : p.lk - 1)) * p.kv_heads + item.rows.hk
                                      : item.rows.index(p, in ? r : p.rows - 1);
            unsigned char* store = smem + S::kStore + warp * 32 * kBlockRow;
#pragma unroll 1
            for (int q = 0; q < S::kSums * S::kBlocks; ++q) {
                const int sum = q / S::kBlocks, block = q % S::kBlocks;
                float o[64];
                if (ok && any) {
                    tmem_load32(o, acc + q * 64);
                    tmem_load32(o + 32, acc + q * 64 + 32);
                    tmem_wait_load();
                    if (q == S::kSums * S::kBlocks - 1) {
                        fence_before_sync();
                        warp_arrive(bar(kAccEmpty + i));
                        warp_arrive(bar(kXEmpty + i));
                    }
                }
                // dk and dq carry the scale; an invisible key has no gradient, nor does a row that sees none
                const float f = sum == 0 ? p.scale : 1.f;
                const bool some = ok && any && (!kKeys || on);
#pragma unroll
                for (int j = 0; j < 64; ++j) o[j] = some ? o[j] * f : ok ? 0.f : NAN;
                if (p.splits == 1) {
                    void* tensor = kKeys ? sum ? p.dv : p.dk : p.dq;
                    __syncwarp();
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        uint32_t w[4];
#pragma unroll
                        for (int k = 0; k < 4; ++k) w[k] = Mma<bf16>::pack(o[j * 8 + 2 * k], o[j * 8 + 2 * k + 1]);
                        *reinterpret_cast<uint4*>(store + swizzled(lane, j)) = make_uint4(w[0], w[1], w[2], w[3]);
                    }
                    __syncwarp();
                    const int col = block * 64 + (lane & 7) * 8;
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const int from = j * 4 + (lane >> 3);
                        const int64_t to_row = __shfl_sync(0xffffffffu, row, from);
                        const uint4 w = *reinterpret_cast<const uint4*>(store + swizzled(from, lane & 7));
                        if (r - lane + from < (kKeys ? p.lk : p.rows) && col < p.dim)
                            *reinterpret_cast<uint4*>(static_cast<bf16*>(tensor) + to_row * p.dim + col) = w;
                    }
                } else if (in) {
                    float* g = p.part + (kKeys ? (2 * item.split + sum) * p.k_count : item.split * p.q_count) + row * p.dim + block * 64;
#pragma unroll
                    for (int j = 0; j < 64; j += 4) {
                        if (block * 64 + j >= p.dim) break;
                        store4(g + j, o[j], o[j + 1], o[j + 2], o[j + 3]);
                    }
                }
            }
        }
    }
    fence_before_sync();
    __syncthreads();
    if (warp == kWarps + 2) {
        fence_after_sync();
        tmem_free(tmem, 512);
        if (lane == 0) report_stall(broken, p.stalled);
    }
}

// --- host ------------------------------------------------------------------------

template <bool kKeys, int DP>
int launch(const AttnParams& p, const GradMaps& maps, int64_t items, int sms, int device, cudaStream_t stream)
{
    using S = GradTc<kKeys, DP>;
    if (items > std::numeric_limits<int32_t>::max() - 4096)
        return fail(POLICY_ERR_INVALID, "policy_cross_attention_backward: more than 2^31 - 4096 tiles");
    static std::atomic<uint64_t> done{0};
    const uint64_t bit = device < 64 ? 1ull << device : 0ull;
    if (!bit || !(done.load(std::memory_order_relaxed) & bit)) {
        const cudaError_t e =
            cudaFuncSetAttribute(attend_grad_tc_kernel<kKeys, DP>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(S::kAligned));
        if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute");
        done.fetch_or(bit, std::memory_order_relaxed);
    }
    const int grid = static_cast<int>(items < sms ? items : sms);
    attend_grad_tc_kernel<kKeys, DP><<<grid, kThreads, S::kAligned, stream>>>(p, maps, static_cast<int>(items));
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? POLICY_OK : cuda_fail(e, "attend_grad_tc_kernel");
}

}  // namespace

bool attend_grad_tc_takes(const AttnParams& p)
{
    const int64_t batch = p.q_count / p.lq / p.heads / p.dim;
    const int64_t q_shape[3] = {batch, p.lq, p.heads}, k_shape[3] = {batch, p.lk, p.kv_heads};
    return kY % p.group == 0 && map_takes(q_shape, p.qs, p.group) && map_takes(q_shape, p.ds, p.group) && map_takes(k_shape, p.ks, 1) &&
           map_takes(k_shape, p.vs, 1);
}

int grad_tc_tile(bool keys, int dim) { return keys && dim > 64 ? kX : 2 * kX; }

int launch_attend_grad_tc(const AttnParams& p, bool keys, int64_t bh, int sms, int device, cudaStream_t stream)
{
    const int64_t batch = bh / p.kv_heads;
    const int64_t q_shape[3] = {batch, p.lq, p.heads}, k_shape[3] = {batch, p.lk, p.kv_heads};
    const int q_tokens = (keys ? kY : kX) / p.group, k_tokens = keys ? kX : kY;
    GradMaps maps;
    int rc = make_map(&maps.q, p.q, q_shape, p.qs, p.dim, q_tokens, p.group);
    if (rc == POLICY_OK) rc = make_map(&maps.dout, p.dout, q_shape, p.ds, p.dim, q_tokens, p.group);
    if (rc == POLICY_OK) rc = make_map(&maps.k, p.k, k_shape, p.ks, p.dim, k_tokens, 1);
    if (rc == POLICY_OK) rc = make_map(&maps.v, p.v, k_shape, p.vs, p.dim, k_tokens, 1);
    if (rc != POLICY_OK) return rc;
    const int64_t items = bh * p.tiles * p.splits;
    if (keys)
        return p.dim <= 64 ? launch<true, 64>(p, maps, items, sms, device, stream) : launch<true, 128>(p, maps, items, sms, device, stream);
    return p.dim <= 64 ? launch<false, 64>(p, maps, items, sms, device, stream) : launch<false, 128>(p, maps, items, sms, device, stream);
}

}  // namespace policy
