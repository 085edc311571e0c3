// The forward pass of cross attention for many rows, on the tcgen05 tensor cores (bf16).
//
// A block keeps 256 rows, two tiles of 128, and walks over key tiles of 128; it is persistent, one per
// SM, and takes (batch, key head, rows, key range) items in turn.  Four roles:
//   3 warps copy: K, V and the next item's rows, masked keys and missing rows as zeros;
//   1 thread issues the products S = Q K^T (shared x shared) and O += P V (P from tensor memory);
//   2 x 4 warps, one set per row tile, do the softmax, a thread to a row: no exchange between lanes.
// Tensor memory, all 512 columns: S of both tiles (128 columns of f32 each, over which P is written as 64
// columns of bf16 pairs) and O of both.  While one set exponentiates, the other tile's products run.
//
// O is kept relative to a reference maximum that follows the running one only when it falls 8 (a factor of
// 256) behind: the sums stay exact in f32 and P below 2^8 in bf16, and almost no tile pays for rescaling O.
// The exponentials bound it (128 x 128 per tile and row tile at 16 a clock and SM, as long as the products
// take at dim 128 and twice that at 64).
#include <atomic>
#include <limits>

#include "policy_attention.cuh"
#include "policy_internal.h"
#include "policy_tcgen05.cuh"

namespace policy {
namespace {

constexpr int kThreads = 384;
constexpr int kCopyThreads = 96;
constexpr int kTile = 128;  // rows of a tile, and keys of one
constexpr float kLag = 8.f;

template <int DP>
struct TcShape {
    static constexpr int kBlocks = DP / 64;  // 64-column blocks
    static constexpr uint32_t kBlock = kTile * kBlockRow;
    static constexpr uint32_t kTileBytes = kBlocks * kBlock;
    static constexpr int kStages = DP == 64 ? 4 : 2;
    static constexpr uint32_t kQ = 0;
    static constexpr uint32_t kK = 2 * kTileBytes;
    static constexpr uint32_t kV = kK + kStages * kTileBytes;
    static constexpr uint32_t kVisible = kV + kStages * kTileBytes;  // a slot more than stages: see the copies
    static constexpr uint32_t kBars = kVisible + (kStages + 1) * kTile;
    static constexpr uint32_t kBytes = kBars + 256;
    static constexpr uint32_t kAligned = kBytes + 1024;
};

// Barriers, 8 bytes each from kBars.
enum Bar { kQFull, kQEmpty, kSFull, kPFull = kSFull + 2, kOFull = kPFull + 2, kOEmpty = kOFull + 2, kKFull = kOEmpty + 2 };
// then K full, K empty, V full, V empty: kStages each

struct Item {
    int split, r0, t0, t1, n;
    Rows rows;
    __device__ __forceinline__ Item(const AttnParams& p, int item)
    {
        split = item % p.splits;
        const int tile = (item / p.splits) % p.tiles;
        const int bh = item / p.splits / p.tiles;
        rows = Rows{bh / p.kv_heads, bh % p.kv_heads, p.group};
        r0 = tile * kTcRows;
        n = visible_keys(p, rows.b);
        const int tiles = (n + kTile - 1) / kTile;
        t0 = static_cast<int>(static_cast<int64_t>(tiles) * split / p.splits);
        t1 = static_cast<int>(static_cast<int64_t>(tiles) * (split + 1) / p.splits);
    }
};

// two f32 to an instruction
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c)
{
    float2 r;
    asm("{\n.reg .b64 x, y, z;\nmov.b64 x, {%2, %3};\nmov.b64 y, {%4, %5};\nmov.b64 z, {%6, %7};\n"
        "fma.rn.f32x2 x, x, y, z;\nmov.b64 {%0, %1}, x;\n}\n"
        : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return r;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b)
{
    float2 r;
    asm("{\n.reg .b64 x, y;\nmov.b64 x, {%2, %3};\nmov.b64 y, {%4, %5};\nadd.rn.f32x2 x, x, y;\nmov.b64 {%0, %1}, x;\n}\n"
        : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return r;
}

template <int DP>
__global__ void __launch_bounds__(kThreads, 1) attend_tc_kernel(const __grid_constant__ AttnParams p, int items)
{
    using S = TcShape<DP>;
    extern __shared__ unsigned char raw[];
    __shared__ uint32_t tmem_at;
    __shared__ int broken_flag;
    volatile int* broken = &broken_flag;
    // the swizzle goes by address bits: tiles start on 1,024 bytes
    const uint32_t base = (smem_addr(raw) + 1023u) & ~1023u;
    unsigned char* smem = raw + (base - smem_addr(raw));
    const uint32_t bars = base + S::kBars;
    const auto bar = [&](int i) { return bars + 8u * i; };
    constexpr int ST = S::kStages;
    constexpr int kKEmpty = kKFull + ST, kVFull = kKEmpty + ST, kVEmpty = kVFull + ST, kAll = kVEmpty + ST;
    static_assert(kAll * 8 < 256, "barriers");
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        broken_flag = 0;
        bar_init(bar(kQFull), kCopyThreads);
        bar_init(bar(kQEmpty), 1);
        for (int i = 0; i < 2; ++i) {
            bar_init(bar(kSFull + i), 1);
            bar_init(bar(kPFull + i), kTile);
            bar_init(bar(kOFull + i), 1);
            bar_init(bar(kOEmpty + i), kTile);
        }
        for (int i = 0; i < ST; ++i) {
            bar_init(bar(kKFull + i), kCopyThreads);
            bar_init(bar(kKEmpty + i), 1);
            bar_init(bar(kVFull + i), kCopyThreads);
            bar_init(bar(kVEmpty + i), 1);
        }
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    }
    if (warp == 11) tmem_alloc(smem_addr(&tmem_at), 512);
    fence_before_sync();
    __syncthreads();
    fence_after_sync();
    const uint32_t tmem = tmem_at;

    if (warp >= 8 && warp < 11) {
        // --- copies: 8 lanes to a row's 64-column block, 4 rows to a warp ---
        const int piece = lane & 7, row0 = (warp - 8) * 4 + (lane >> 3);
        constexpr int kGroups = (kTile / 4 + 2) / 3;  // groups of 4 rows, every third to this warp
        uint32_t pending[2] = {0u, 0u};  // barriers of the copies issued and not announced, oldest first
        const auto announce = [&](uint32_t b) {
            fence_async_shared();
            bar_arrive(b);
        };
        const auto drain = [&] {
            copy_wait<0>();
            if (pending[0]) announce(pending[0]);
            if (pending[1]) announce(pending[1]);
            pending[0] = pending[1] = 0u;
        };
        // Before a wait that is not over at once, everything issued is announced: what the wait is for
        // may need it.
        const auto acquire = [&](uint32_t b, uint32_t parity) {
            if (bar_try(b, parity)) return true;
            drain();
            return bar_wait(b, parity, broken);
        };
        const auto issued = [&](uint32_t b) {
            copy_commit();
            copy_wait<2>();
            if (pending[0]) announce(pending[0]);
            pending[0] = pending[1];
            pending[1] = b;
        };
        uint32_t q_uses = 0, tile_uses = 0;
        bool ok = true;
        for (int it = blockIdx.x; it < items && ok; it += gridDim.x) {
            const Item item(p, it);
            if (item.t0 >= item.t1) continue;
            if (!(ok = acquire(bar(kQEmpty), (q_uses & 1u) ^ 1u))) break;
            ++q_uses;
            {
                const bf16* q = static_cast<const bf16*>(p.q);
                for (int r = row0; r < kTcRows; r += 12) {
                    const bool in = item.r0 + r < p.rows;
                    const bf16* src = q + (in ? item.rows.at(p.qs, item.r0 + r) : 0);
                    const uint32_t dst = base + S::kQ + (r >= kTile ? S::kTileBytes : 0u);
#pragma unroll
                    for (int b = 0; b < S::kBlocks; ++b) {
                        const int c = b * 64 + piece * 8;
                        const bool take = in && c < p.dim;
                        copy16(dst + b * S::kBlock + swizzled(r & (kTile - 1), piece), take ? src + c : q, take);
                    }
                }
            }
            issued(bar(kQFull));
            const bf16* k = static_cast<const bf16*>(p.k) + item.rows.b * p.ks[0] + item.rows.hk * p.ks[2];
            const bf16* v = static_cast<const bf16*>(p.v) + item.rows.b * p.vs[0] + item.rows.hk * p.vs[2];
            const uint8_t* mask = p.mask ? p.mask + item.rows.b * p.mask_stride : nullptr;
            const auto visible = [&](int t) {
                uint32_t bits = 0;
#pragma unroll
                for (int g = 0; g < kGroups; ++g) {
                    const int r = row0 + g * 12, key = t * kTile + r;
                    bool on = r < kTile && key < item.n;
                    if (mask && on) on = __ldg(mask + key) != 0;
                    bits |= static_cast<uint32_t>(on) << g;
                }
                return bits;
            };
            uint32_t bits = visible(item.t0);
            for (int t = item.t0; t < item.t1; ++t, ++tile_uses) {
                const int st = tile_uses % ST;
                const uint32_t parity = ((tile_uses / ST) & 1u) ^ 1u;
                const uint32_t next = t + 1 < item.t1 ? visible(t + 1) : 0u;
                const auto copy_rows = [&](const bf16* src, const int64_t step, uint32_t dst) {
#pragma unroll
                    for (int g = 0; g < kGroups; ++g) {
                        const int r = row0 + g * 12;
                        if (r >= kTile) break;
                        const bool on = (bits >> g) & 1u;
                        const bf16* row = src + (on ? (t * static_cast<int64_t>(kTile) + r) * step : 0);
#pragma unroll
                        for (int b = 0; b < S::kBlocks; ++b) {
                            const int c = b * 64 + piece * 8;
                            const bool take = on && c < p.dim;
                            copy16(dst + b * S::kBlock + swizzled(r, piece), take ? row + c : src, take);
                        }
                    }
                };
                // The slot of this tile's visibility is that of the tile kStages + 1 before: the products of
                // the tile kStages before are over (its stage is empty), and they waited for the weights of the
                // one before them, which were the last to read that slot.
                if (!(ok = acquire(bar(kKEmpty + st), parity))) break;
                if (piece == 0) {
                    uint8_t* slot = smem + S::kVisible + (tile_uses % (ST + 1)) * kTile;
#pragma unroll
                    for (int g = 0; g < kGroups; ++g)
                        if (row0 + g * 12 < kTile) slot[row0 + g * 12] = (bits >> g) & 1u;
                }
                copy_rows(k, p.ks[1], base + S::kK + st * S::kTileBytes);
                issued(bar(kKFull + st));
                if (!(ok = acquire(bar(kVEmpty + st), parity))) break;
                copy_rows(v, p.vs[1], base + S::kV + st * S::kTileBytes);
                issued(bar(kVFull + st));
                bits = next;
            }
        }
        drain();
    } else if (warp == 11) {
        // --- products ---
        if (lane == 0) {
            const uint32_t scores = bf16_product(kTile, kTile, false, false);
            const int columns = (p.dim + 15) & ~15;
            const uint32_t values = bf16_product(kTile, columns, false, true);
            const int steps = columns / 16;
            const auto issue_scores = [&](int i, int st) {
                const uint32_t a = base + S::kQ + i * S::kTileBytes, b = base + S::kK + st * S::kTileBytes;
                for (int s = 0; s < steps; ++s) {
                    const uint32_t at = (s >> 2) * S::kBlock + (s & 3) * 32u;
                    product_ss(tmem + i * kTile, tile_descriptor(a + at, 0), tile_descriptor(b + at, 0), scores, s > 0);
                }
            };
            const auto issue_values = [&](int i, int st, bool add) {
                const uint32_t b = base + S::kV + st * S::kTileBytes;
                for (int s = 0; s < kTile / 16; ++s)
                    product_ts(tmem + 2 * kTile + i * DP, tmem + i * kTile + s * 8, tile_descriptor(b + s * 16 * kBlockRow, S::kBlock), values,
                               add || s > 0);
            };
            uint32_t q_uses = 0, tile_uses = 0, weights[2] = {0u, 0u}, outs[2] = {0u, 0u};
            bool ok = true;
            for (int it = blockIdx.x; it < items && ok; it += gridDim.x) {
                const Item item(p, it);
                if (item.t0 >= item.t1) continue;
                const int count = item.r0 + kTile < p.rows ? 2 : 1;
                if (!(ok = bar_wait(bar(kQFull), q_uses & 1u, broken))) break;
                ++q_uses;
                int st = tile_uses % ST;
                if (!(ok = bar_wait(bar(kKFull + st), (tile_uses / ST) & 1u, broken))) break;
                for (int i = 0; i < count; ++i) {
                    issue_scores(i, st);
                    products_arrive(bar(kSFull + i));
                }
                products_arrive(bar(kKEmpty + st));
                if (item.t0 + 1 == item.t1) products_arrive(bar(kQEmpty));
                for (int t = item.t0; t < item.t1 && ok; ++t, ++tile_uses) {
                    st = tile_uses % ST;
                    const bool more = t + 1 < item.t1;
                    const int nx = (tile_uses + 1) % ST;
                    if (!(ok = bar_wait(bar(kVFull + st), (tile_uses / ST) & 1u, broken))) break;
                    if (more && !(ok = bar_wait(bar(kKFull + nx), ((tile_uses + 1) / ST) & 1u, broken))) break;
                    for (int i = 0; i < count; ++i) {
                        if (t == item.t0) {  // the item before has left O
                            if (!(ok = bar_wait(bar(kOEmpty + i), (outs[i] & 1u) ^ 1u, broken))) break;
                            ++outs[i];
                        }
                        if (!(ok = bar_wait(bar(kPFull + i), weights[i] & 1u, broken))) break;
                        ++weights[i];
                        fence_after_sync();
                        issue_values(i, st, t > item.t0);
                        if (more) {
                            issue_scores(i, nx);
                            products_arrive(bar(kSFull + i));
                        } else {
                            products_arrive(bar(kOFull + i));
                        }
                    }
                    if (!ok) break;
                    products_arrive(bar(kVEmpty + st));
                    if (more) {
                        products_arrive(bar(kKEmpty + nx));
                        if (t + 2 == item.t1) products_arrive(bar(kQEmpty));
                    }
                }
            }
        }
        __syncwarp();
    } else {
        // --- softmax: a thread to a row ---
        const int i = warp >> 2;
        const int lane_row = (warp & 3) * 32 + lane;
        const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
        const uint32_t ts = tmem + lanes + i * kTile, to = tmem + lanes + 2 * kTile + i * DP;
        const float c = p.scale_log2;
        uint32_t tile_uses = 0, score_uses = 0, out_uses = 0;
        for (int it = blockIdx.x; it < items; it += gridDim.x) {
            const Item item(p, it);
            const int r = item.r0 + i * kTile + lane_row;
            if (item.r0 + i * kTile >= p.rows) {  // the whole set has no rows here
                tile_uses += item.t1 - item.t0;
                continue;
            }
            float m = -INFINITY, l = 0.f, top = -INFINITY;  // m: the reference of l, P and O; top: the running maximum
            bool ok = __all_sync(0xffffffffu, !*broken);
            for (int t = item.t0; t < item.t1 && ok; ++t, ++tile_uses) {
                if (!(ok = warp_wait(bar(kSFull + i), score_uses & 1u, broken))) break;
                ++score_uses;
                fence_after_sync();
                float s[kTile];
#pragma unroll
                for (int q = 0; q < 4; ++q) tmem_load32(s + q * 32, ts + q * 32);
                tmem_wait_load();
                if (p.mask || (t + 1) * kTile > item.n) {
                    const uint4* vis = reinterpret_cast<const uint4*>(smem + S::kVisible + (tile_uses % (ST + 1)) * kTile);
#pragma unroll
                    for (int q = 0; q < kTile / 16; ++q) {
                        const uint4 w = vis[q];
                        const uint32_t x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                        for (int j = 0; j < 16; ++j)
                            if (!((x[j >> 2] >> ((j & 3) * 8)) & 1u)) s[q * 16 + j] = -INFINITY;
                    }
                }
                float x[4] = {top, s[0], s[1], s[2]};
#pragma unroll
                for (int j = 3; j < kTile; ++j) x[j & 3] = fmaxf(x[j & 3], s[j]);
                top = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
                // in units of the exponent; before the first tile O holds nothing
                const bool behind = (top - m) * c > kLag;
                if (t == item.t0) {
                    m = top;
                } else if (__any_sync(0xffffffffu, behind)) {
                    const float a = top == -INFINITY ? 1.f : exp2_fast((m - top) * c);
                    m = top;
                    l *= a;
                    // in small pieces: this runs while a row of S is held
#pragma unroll 1
                    for (int q = 0; q < DP / 8; ++q) {
                        float o[8];
                        tmem_load8(o, to + q * 8);
                        tmem_wait_load();
#pragma unroll
                        for (int j = 0; j < 8; ++j) o[j] *= a;
                        tmem_store8(to + q * 8, o);
                    }
                }
                const float b = m == -INFINITY ? 0.f : m * c;
                const float2 c2 = make_float2(c, c), b2 = make_float2(-b, -b);
                float2 sum = make_float2(0.f, 0.f);
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    uint32_t w[16];
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        float2 e = fma2(make_float2(s[q * 32 + 2 * j], s[q * 32 + 2 * j + 1]), c2, b2);
                        e.x = exp2_fast(e.x);
                        e.y = exp2_fast(e.y);
                        sum = add2(sum, e);
                        w[j] = Mma<bf16>::pack(e.x, e.y);
                    }
                    tmem_store16(ts + q * 16, w);
                }
                l += sum.x + sum.y;
                tmem_wait_store();
                fence_before_sync();
                bar_arrive(bar(kPFull + i));
            }
            const bool any = item.t0 < item.t1;
            if (ok && any) {
                ok = warp_wait(bar(kOFull + i), out_uses & 1u, broken);
                ++out_uses;
                fence_after_sync();
            }
            const float inv = !ok ? NAN : l == 0.f ? 0.f : p.splits == 1 ? 1.f / l : 1.f;
            const bool in = r < p.rows;
            const int64_t row = item.rows.index(p, in ? r : p.rows - 1);
            for (int q = 0; q < DP / 32; ++q) {
                float o[32];
                if (ok && any) {
                    tmem_load32(o, to + q * 32);
                    tmem_wait_load();
                    if (q == DP / 32 - 1) {
                        fence_before_sync();
                        bar_arrive(bar(kOEmpty + i));
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < 32; ++j) o[j] = 0.f;
                }
                if (!in) continue;
                if (p.splits == 1) {
                    bf16* g = static_cast<bf16*>(p.out) + row * p.dim + q * 32;
#pragma unroll
                    for (int j = 0; j < 32; j += 8) {
                        if (q * 32 + j >= p.dim) break;
                        *reinterpret_cast<uint4*>(g + j) =
                            make_uint4(Mma<bf16>::pack(o[j] * inv, o[j + 1] * inv), Mma<bf16>::pack(o[j + 2] * inv, o[j + 3] * inv),
                                       Mma<bf16>::pack(o[j + 4] * inv, o[j + 5] * inv), Mma<bf16>::pack(o[j + 6] * inv, o[j + 7] * inv));
                    }
                } else {
                    float* g = p.part + item.split * p.q_count + row * p.dim + q * 32;
#pragma unroll
                    for (int j = 0; j < 32; j += 4) {
                        if (q * 32 + j >= p.dim) break;
                        store4(g + j, o[j] * inv, o[j + 1] * inv, o[j + 2] * inv, o[j + 3] * inv);
                    }
                }
            }
            if (!in) continue;
            if (p.splits > 1) {
                float* ml = p.part_ml + 2 * (item.split * (p.q_count / p.dim) + row);
                ml[0] = m, ml[1] = ok ? l : NAN;
            } else if (p.lse) {
                p.lse[row] = !ok ? NAN : l == 0.f ? INFINITY : (m == -INFINITY ? 0.f : m * c) + log2f(l);
            }
        }
    }
    fence_before_sync();
    __syncthreads();
    if (warp == 11) {
        if (*broken) {  // products may still be running: tensor memory is freed after them
            if (lane == 0) {
                const uint32_t last = bar(kAll);
                bar_init(last, 1);
                products_arrive(last);
                *broken = 0;
                bar_wait(last, 0, broken);
            }
            __syncwarp();
        }
        fence_after_sync();
        tmem_free(tmem, 512);
    }
}

template <int DP>
int launch_dim(const AttnParams& p, int items, int sms, int device, cudaStream_t stream)
{
    using S = TcShape<DP>;
    static std::atomic<uint64_t> done{0};
    const uint64_t bit = device < 64 ? 1ull << device : 0ull;
    if (!bit || !(done.load(std::memory_order_relaxed) & bit)) {
        const cudaError_t e = cudaFuncSetAttribute(attend_tc_kernel<DP>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(S::kAligned));
        if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute");
        done.fetch_or(bit, std::memory_order_relaxed);
    }
    attend_tc_kernel<DP><<<items < sms ? items : sms, kThreads, S::kAligned, stream>>>(p, items);
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? POLICY_OK : cuda_fail(e, "attend_tc_kernel");
}

}  // namespace

int launch_attend_tc(const AttnParams& p, int64_t bh, int sms, int device, cudaStream_t stream)
{
    const int64_t items = bh * p.tiles * p.splits;
    if (items > std::numeric_limits<int32_t>::max() - 4096)
        return fail(POLICY_ERR_INVALID, "policy_cross_attention: more than 2^31 - 4096 tiles of rows");
    return p.dim <= 64 ? launch_dim<64>(p, static_cast<int>(items), sms, device, stream)
                       : launch_dim<128>(p, static_cast<int>(items), sms, device, stream);
}

}  // namespace policy
