// The forward pass of cross attention for many rows, on the tcgen05 tensor cores (bf16).
//
// A block keeps 256 rows, two tiles of 128, and walks over key tiles of 128; it is persistent, one per
// SM, and takes (batch, key head, rows, key range) items in turn.  Its roles:
//   one thread copies K and V tiles by TMA (zeros past the last key and the last value of a head);
//   one warp, where there is a mask or there are lengths, zeroes the invisible rows of V that have come in
//     (0 x NaN would be NaN) and says which keys of the tile are visible; K needs none, its scores are replaced;
//   one thread for each row tile issues its products S = Q K^T (shared x shared) and O += P V (P from tensor
//     memory): a single thread for both would wait for one tile's softmax while the other's is ready;
//   2 x 4 warps, one set per row tile, do the softmax, a thread to a row: no exchange between lanes.  A set
//     copies its next item's rows as soon as the last product that reads the present ones is over.
// Tensor memory, all 512 columns: S of both tiles, 128 columns of f32 each, O of both, and P as 64 columns of
// bf16 pairs: at dim 64 apart, so that the next S is made as soon as this one has been read; at dim 128 over S.
// While one set exponentiates, the other tile's products run; the first half of P's keys is handed over while
// the second is still being made.
//
// O is kept relative to a reference maximum that follows the running one only when it falls 8 (a factor of
// 256) behind: the sums lose nothing in f32, P stays below 2^8 in bf16, and almost no tile pays for rescaling O.
// Measured: 16 x 8 heads of 12,288 rows x 768 keys x 128 in 753 us, 821 TFLOP/s; 4 x 8 heads of 12,288 rows and keys: 1,085
// TFLOP/s; 8 x 8 heads of 4,096 x 768 x 64: 433 TFLOP/s.  What is left of the tensor cores' rate goes to the softmax between a tile's two products.
// The special function unit gives 16 exponentials a clock and SM: as many clocks for a tile as its products
// take at dim 128, twice as many at 64.  Replacing a part of them by polynomials on the multiply-add pipes was
// slower at every share (2 of 8: 2 % at 12,288 x 768 x 128; 4 of 8: 14 %): the issue slots are the scarcer.
#include <atomic>
#include <limits>

#include "policy_attention.cuh"
#include "policy_internal.h"
#include "policy_map.h"
#include "policy_tcgen05.cuh"

namespace policy {
namespace {

constexpr int kThreads = 384;
constexpr int kSoftmaxWarps = 8;  // then copies, visibility, products of either row tile
constexpr int kTile = 128;        // rows of a tile, and keys of one
constexpr float kLag = 8.f;

template <int DP>
struct TcShape {
    static constexpr int kBlocks = DP / 64;  // 64-column blocks
    static constexpr uint32_t kBlock = kTile * kBlockRow;
    static constexpr uint32_t kTileBytes = kBlocks * kBlock;
    static constexpr int kStages = DP == 64 ? 3 : 2;
    // columns of tensor memory
    static constexpr bool kApart = DP == 64;
    static constexpr int kOutputs = 2 * kTile, kWeights = kApart ? kOutputs + 2 * DP : 0, kWeightStep = kApart ? kTile / 2 : kTile;
    static constexpr uint32_t kQ = 0;
    static constexpr uint32_t kK = 2 * kTileBytes;
    static constexpr uint32_t kV = kK + kStages * kTileBytes;
    static constexpr uint32_t kVisible = kV + kStages * kTileBytes;  // a bit per key, 16 bytes a stage
    static constexpr uint32_t kStore = kVisible + 1024;  // 32 rows x 128 bytes for each softmax warp
    static constexpr uint32_t kBars = kStore + kSoftmaxWarps * 32 * kBlockRow;
    static constexpr uint32_t kBytes = kBars + 512;
    static constexpr uint32_t kAligned = kBytes + 1024;
};

// Barriers, 8 bytes each from kBars.
enum Bar {
    kQFull,
    kSFull = kQFull + 2,
    kSFree = kSFull + 2,
    kPFull = kSFree + 2,  // two halves of the keys for each tile
    kPFree = kPFull + 4,
    kOFull = kPFree + 2,
    kOEmpty = kOFull + 2,
    kLast = kOEmpty + 2,
    kTurn = kLast + 2,  // one for each softmax warp
    kKFull = kTurn + kSoftmaxWarps
};
// then K full, K empty, V copied, V clean, V empty: kStages each

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
    __device__ __forceinline__ bool has(const AttnParams& p, int i) const { return r0 + i * kTile < p.rows; }
};

template <int DP>
__global__ void __launch_bounds__(kThreads, 1)
    attend_tc_kernel(const __grid_constant__ AttnParams p, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                     int items)
{
    using S = TcShape<DP>;
    extern __shared__ unsigned char raw[];
    __shared__ uint32_t tmem_at;
    __shared__ int broken_flag;
    volatile int* broken = &broken_flag;
    // the swizzle goes by address bits: tiles start on 1,024 bytes
    const uint32_t base = (smem_addr(raw) + 1023u) & ~1023u;
    unsigned char* smem = raw + (base - smem_addr(raw));
    const auto bar = [&](int i) { return base + S::kBars + 8u * i; };
    constexpr int ST = S::kStages;
    constexpr int kKEmpty = kKFull + ST, kVCopied = kKEmpty + ST, kVClean = kVCopied + ST, kVEmpty = kVClean + ST, kAll = kVEmpty + ST;
    static_assert(kAll * 8 <= 512, "barriers");
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const bool hidden = p.mask || p.lengths;  // keys that exist may be invisible
    const int v_ready = hidden ? kVClean : kVCopied;

    if (threadIdx.x == 0) {
        broken_flag = 0;
        for (int i = 0; i < 2; ++i) {
            bar_init(bar(kQFull + i), 4);
            bar_init(bar(kSFull + i), 1);
            bar_init(bar(kSFree + i), 4);
            bar_init(bar(kPFull + 2 * i), 4);
            bar_init(bar(kPFull + 2 * i + 1), 4);
            bar_init(bar(kPFree + i), 1);
            bar_init(bar(kOFull + i), 1);
            bar_init(bar(kOEmpty + i), 4);
            bar_init(bar(kLast + i), 1);
        }
        for (int i = 0; i < kSoftmaxWarps; ++i) bar_init(bar(kTurn + i), 1);
        for (int i = 0; i < ST; ++i) {
            bar_init(bar(kKFull + i), 1);
            bar_init(bar(kKEmpty + i), 2);
            bar_init(bar(kVCopied + i), 1);
            bar_init(bar(kVClean + i), 1);
            bar_init(bar(kVEmpty + i), 2);
        }
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    }
    if (warp == kSoftmaxWarps + 2) tmem_alloc(smem_addr(&tmem_at), 512);
    fence_before_sync();
    __syncthreads();
    fence_after_sync();
    const uint32_t tmem = tmem_at;

    if (warp == kSoftmaxWarps) {
        // --- copies of K and V ---
        if (elected()) {
            uint32_t uses = 0, v_uses = 0;
            bool ok = true;
            for (int it = blockIdx.x; it < items && ok; it += gridDim.x) {
                const Item item(p, it);
                const int kb = p.ks[0] ? static_cast<int>(item.rows.b) : 0, kh = p.ks[2] ? item.rows.hk : 0;
                const int vb = p.vs[0] ? static_cast<int>(item.rows.b) : 0, vh = p.vs[2] ? item.rows.hk : 0;
                for (int t = item.t0; t < item.t1; ++t) {
                    const int st = uses % ST;
                    const uint32_t parity = ((uses / ST) & 1u) ^ 1u;
                    if (!(ok = bar_wait(bar(kKEmpty + st), parity, broken))) break;
                    bar_expect(bar(kKFull + st), S::kTileBytes);
                    for (int b = 0; b < S::kBlocks; ++b)
                        copy_tile(base + S::kK + st * S::kTileBytes + b * S::kBlock, &map_k, b * 64, kh, t * kTile, kb, bar(kKFull + st));
                    ++uses;
                    if (!(ok = bar_wait(bar(kVEmpty + st), parity, broken))) break;
                    bar_expect(bar(kVCopied + st), S::kTileBytes);
                    for (int b = 0; b < S::kBlocks; ++b)
                        copy_tile(base + S::kV + st * S::kTileBytes + b * S::kBlock, &map_v, b * 64, vh, t * kTile, vb, bar(kVCopied + st));
                    ++v_uses;
                }
            }
            if (!ok) {  // copies that nobody will wait for must not outlive the block
                volatile int quiet = 0;
                for (uint32_t u = uses > ST ? uses - ST : 0; u < uses; ++u) bar_wait(bar(kKFull + u % ST), (u / ST) & 1u, &quiet);
                for (uint32_t u = v_uses > ST ? v_uses - ST : 0; u < v_uses; ++u) bar_wait(bar(kVCopied + u % ST), (u / ST) & 1u, &quiet);
            }
        }
        __syncwarp();
    } else if (warp == kSoftmaxWarps + 1) {
        // --- visibility ---
        uint32_t uses = 0;
        bool ok = hidden;
        for (int it = blockIdx.x; it < items && ok; it += gridDim.x) {
            const Item item(p, it);
            const uint8_t* mask = p.mask ? p.mask + item.rows.b * p.mask_stride : nullptr;
            const auto visible = [&](int t) {  // bit g: key 32 g + lane of the tile
                uint32_t bits = 0;
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const int key = t * kTile + g * 32 + lane;
                    bool on = key < item.n;
                    if (mask && on) on = __ldg(mask + key) != 0;
                    bits |= static_cast<uint32_t>(on) << g;
                }
                return bits;
            };
            uint32_t bits = item.t0 < item.t1 ? visible(item.t0) : 0u;
            for (int t = item.t0; t < item.t1; ++t, ++uses) {
                const int st = uses % ST;
                if (!(ok = warp_wait(bar(kVCopied + st), (uses / ST) & 1u, broken))) break;
                uint32_t words[4];
#pragma unroll
                for (int g = 0; g < 4; ++g) words[g] = __ballot_sync(0xffffffffu, (bits >> g) & 1u);
                if (lane == 0)
                    *reinterpret_cast<uint4*>(smem + S::kVisible + st * 16) = make_uint4(words[0], words[1], words[2], words[3]);
                if ((words[0] & words[1] & words[2] & words[3]) != 0xffffffffu) {
                    unsigned char* tile = smem + S::kV + st * S::kTileBytes;
#pragma unroll
                    for (int g = 0; g < 32; ++g) {  // 4 rows at a time, 8 lanes to a row
                        const int row = g * 4 + (lane >> 3);
                        if ((words[g >> 3] >> (row & 31)) & 1u) continue;
#pragma unroll
                        for (int b = 0; b < S::kBlocks; ++b)
                            *reinterpret_cast<uint4*>(tile + b * S::kBlock + swizzled(row, lane & 7)) = make_uint4(0u, 0u, 0u, 0u);
                    }
                }
                fence_async_shared();
                warp_arrive(bar(kVClean + st));
                if (t + 1 < item.t1) bits = visible(t + 1);
            }
        }
    } else if (warp >= kSoftmaxWarps + 2) {
        // --- products of one row tile ---
        if (elected()) {
            const int i = warp - (kSoftmaxWarps + 2);
            const uint32_t scores = bf16_product(kTile, kTile, false, false);
            const uint32_t values = bf16_product(kTile, (p.dim + 15) & ~15, false, true);
            const uint32_t rows_at = tile_descriptor(base + S::kQ + i * S::kTileBytes, 0), keys_at = tile_descriptor(base + S::kK, 0);
            const uint32_t values_at = tile_descriptor(base + S::kV, S::kBlock);
            const uint32_t ts = tmem + i * kTile, to = tmem + S::kOutputs + i * DP, tp = tmem + S::kWeights + i * S::kWeightStep;
            uint32_t uses = 0, items_done = 0, tiles_done = 0;  // tiles of all items; items and tiles of this set
            bool ok = true;
            // S of the tile in stage `use % ST`, once it is there and the last S is out of the way
            const auto make_scores = [&](uint32_t use) {
                const int st = use % ST;
                if (!(ok = bar_wait(bar(kKFull + st), (use / ST) & 1u, broken))) return;
                if (S::kApart && tiles_done + (use - uses) > 0) {
                    if (!(ok = bar_wait(bar(kSFree + i), (tiles_done + (use - uses) - 1) & 1u, broken))) return;
                    fence_after_sync();
                }
                const uint32_t k = keys_at + st * (S::kTileBytes >> 4);
#pragma unroll
                for (int s = 0; s < DP / 16; ++s) {
                    const uint32_t at = ((s >> 2) * S::kBlock + (s & 3) * 32u) >> 4;
                    product_ss(ts, rows_at + at, k + at, scores, s > 0);
                }
                products_arrive(bar(kSFull + i));
                products_arrive(bar(kKEmpty + st));
            };
            for (int it = blockIdx.x; it < items && ok; it += gridDim.x) {
                const Item item(p, it);
                if (!item.has(p, i)) {  // the stages wait for both sets: one after the other, as they come
                    for (int t = item.t0; t < item.t1 && ok; ++t, ++uses) {
                        const int st = uses % ST;
                        if (!(ok = bar_wait(bar(kKFull + st), (uses / ST) & 1u, broken))) break;
                        bar_arrive(bar(kKEmpty + st));
                        if (!(ok = bar_wait(bar(v_ready + st), (uses / ST) & 1u, broken))) break;
                        bar_arrive(bar(kVEmpty + st));
                    }
                    continue;
                }
                if (item.t0 >= item.t1) continue;
                if (!(ok = bar_wait(bar(kQFull + i), items_done & 1u, broken))) break;
                make_scores(uses);
                for (int t = item.t0; t < item.t1 && ok; ++t) {
                    const int st = uses % ST;
                    const bool more = t + 1 < item.t1;
                    if (S::kApart && more) make_scores(uses + 1);
                    if (!ok || !(ok = bar_wait(bar(v_ready + st), (uses / ST) & 1u, broken))) break;
                    // the item before has left O
                    if (t == item.t0 && !(ok = bar_wait(bar(kOEmpty + i), (items_done & 1u) ^ 1u, broken))) break;
                    constexpr int kSteps = kTile / 16 / 2;
                    for (int half = 0; half < 2 && ok; ++half) {
                        if (!(ok = bar_wait(bar(kPFull + 2 * i + half), tiles_done & 1u, broken))) break;
                        fence_after_sync();
                        const uint32_t v = values_at + st * (S::kTileBytes >> 4) + half * kSteps * (16 * kBlockRow >> 4);
#pragma unroll
                        for (int s = 0; s < kSteps; ++s)
                            product_ts(to, tp + half * kSteps * 8 + s * 8, v + s * (16 * kBlockRow >> 4), values, t > item.t0 || half > 0 || s > 0);
                    }
                    if (!ok) break;
                    if (S::kApart) products_arrive(bar(kPFree + i));
                    products_arrive(bar(kVEmpty + st));
                    if (!more) products_arrive(bar(kOFull + i));
                    ++uses, ++tiles_done;
                    if (!S::kApart && more) make_scores(uses);
                }
                ++items_done;
            }
            if (!ok) {  // tensor memory is freed after the products that are still running
                volatile int quiet = 0;
                products_arrive(bar(kLast + i));
                bar_wait(bar(kLast + i), 0, &quiet);
            }
        }
        __syncwarp();
    } else {
        // --- softmax: a thread to a row ---
        const int i = warp >> 2;
        const int lane_row = (warp & 3) * 32 + lane;
        const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
        const uint32_t ts = tmem + lanes + i * kTile, to = tmem + lanes + S::kOutputs + i * DP;
        const uint32_t tp = tmem + lanes + S::kWeights + i * S::kWeightStep;
        const float c = p.scale_log2;
        uint32_t uses = 0, score_uses = 0, out_uses = 0;  // tiles of all sets, of this one, and its items
        uint32_t turns = 0;  // tiles that both sets work on

        // the next item from `it` on that has work for this set, or `items`
        const auto next_item = [&](int it) {
            for (; it < items; it += gridDim.x) {
                const Item item(p, it);
                if (item.t0 < item.t1 && item.has(p, i)) return it;
            }
            return items;
        };
        const auto copy_rows = [&](int it) {  // 8 lanes to a row's 64-column block, 4 rows at a time
            const Item item(p, it);
            const bf16* q = static_cast<const bf16*>(p.q);
            const uint32_t dst = base + S::kQ + i * S::kTileBytes;
            const int piece = lane & 7;
#pragma unroll
            for (int g = 0; g < 8; ++g) {
                const int row = (warp & 3) * 32 + g * 4 + (lane >> 3), r = item.r0 + i * kTile + row;
                const bool in = r < p.rows;
                const bf16* src = q + (in ? item.rows.at(p.qs, r) : 0);
#pragma unroll
                for (int b = 0; b < S::kBlocks; ++b) {
                    const int col = b * 64 + piece * 8;
                    const bool take = in && col < p.dim;
                    copy16(dst + b * S::kBlock + swizzled(row, piece), take ? src + col : q, take);
                }
            }
            copy_commit();
        };
        const auto rows_ready = [&] {
            copy_wait<0>();
            fence_async_shared();
            warp_arrive(bar(kQFull + i));
        };
        {
            const int first = next_item(blockIdx.x);
            if (first < items) {
                copy_rows(first);
                rows_ready();
            }
        }
        for (int it = blockIdx.x; it < items; it += gridDim.x) {
            const Item item(p, it);
            const int r = item.r0 + i * kTile + lane_row;
            if (!item.has(p, i)) {
                uses += item.t1 - item.t0;
                continue;
            }
            float m = -INFINITY, l = 0.f, top = -INFINITY;  // m: the reference of l, P and O; top: the running maximum
            bool ok = __all_sync(0xffffffffu, !*broken);
            for (int t = item.t0; t < item.t1 && ok; ++t, ++uses) {
                if (!(ok = warp_wait(bar(kSFull + i), score_uses & 1u, broken))) break;
                ++score_uses;
                fence_after_sync();
                // S is read twice, 32 columns ahead of the work: for the maximum, and for the weights.  A whole row in
                // registers spilled, and was 17 % slower at dim 128.
                float s[64];
                tmem_load32(s, ts);
                int ahead = items;
                if (t + 1 == item.t1) {
                    ahead = next_item(it + gridDim.x);
                    if (ahead < items) copy_rows(ahead);
                }
                const bool whole = !p.mask && (t + 1) * kTile <= item.n;
                uint32_t vis[4];
                if (!whole) {
                    if (p.mask) {
                        const int st = uses % ST;
                        if (!(ok = warp_wait(bar(kVClean + st), (uses / ST) & 1u, broken))) break;
                        const uint4 w = *reinterpret_cast<const uint4*>(smem + S::kVisible + st * 16);
                        vis[0] = w.x, vis[1] = w.y, vis[2] = w.z, vis[3] = w.w;
                    } else {
#pragma unroll
                        for (int q = 0; q < 4; ++q) {
                            const int left = item.n - t * kTile - q * 32;
                            vis[q] = left >= 32 ? 0xffffffffu : left <= 0 ? 0u : (1u << left) - 1u;
                        }
                    }
                }
                float x[4] = {top, top, top, top};
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    float* now = s + (q & 1) * 32;
                    tmem_wait_load();
                    if (q < 3) tmem_load32(s + ((q + 1) & 1) * 32, ts + (q + 1) * 32);
                    if (!whole) {
#pragma unroll
                        for (int j = 0; j < 32; ++j)
                            if (!((vis[q] >> j) & 1u)) now[j] = -INFINITY;
                        tmem_store32(ts + q * 32, now);
                    }
#pragma unroll
                    for (int j = 0; j < 32; j += 2) x[(j >> 1) & 3] = fmaxf(x[(j >> 1) & 3], fmaxf(now[j], now[j + 1]));
                }
                if (!whole) tmem_wait_store();
                tmem_load32(s, ts);
                top = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
                if (S::kApart && score_uses > 1) {  // the products with the weights before these are over
                    if (!(ok = warp_wait(bar(kPFree + i), (score_uses & 1u), broken))) break;
                    fence_after_sync();
                }
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
                const float2 c2 = same(c), b2 = same(m == -INFINITY ? 0.f : -m * c);
                float2 sum = same(0.f);
                // The two sets take turns at the exponentials, warp by warp: side by side they would be twice as slow
                // each, and then leave the special function unit idle while both wait for their products.
                const bool both = item.has(p, 1);
                if (both) {
                    if (!(ok = warp_wait(bar(kTurn + warp), (turns & 1u) ^ (i == 0 ? 1u : 0u), broken))) break;
                    ++turns;
                }
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    uint32_t w[16];
                    float* now = s + (q & 1) * 32;
                    tmem_wait_load();
                    if (q < 3) {
                        tmem_load32(s + ((q + 1) & 1) * 32, ts + (q + 1) * 32);
                    } else if (S::kApart) {
                        fence_before_sync();
                        warp_arrive(bar(kSFree + i));
                    }
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        float2 e = fma2(make_float2(now[2 * j], now[2 * j + 1]), c2, b2);
                        e = make_float2(exp2_fast(e.x), exp2_fast(e.y));
                        w[j] = Mma<bf16>::pack(e.x, e.y);
                        add_bf16(sum, w[j]);  // the sum is of the weights that multiply v
                    }
                    tmem_store16(tp + q * 16, w);
                    if (q & 1) {
                        tmem_wait_store();
                        fence_before_sync();
                        warp_arrive(bar(kPFull + 2 * i + (q >> 1)));
                    }
                }
                if (both) warp_arrive(bar(kTurn + (warp ^ 4)));
                l += sum.x + sum.y;
                if (ahead < items) rows_ready();
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
            unsigned char* store = smem + S::kStore + warp * 32 * kBlockRow;
            for (int q = 0; q < DP / 64; ++q) {
                float o[64];
                if (ok && any) {
                    tmem_load32(o, to + q * 64);
                    tmem_load32(o + 32, to + q * 64 + 32);
                    tmem_wait_load();
                    if (q == DP / 64 - 1) {
                        fence_before_sync();
                        warp_arrive(bar(kOEmpty + i));
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < 64; ++j) o[j] = 0.f;
                }
                if (p.splits == 1) {
                    // through shared memory, so that 8 lanes write a row's 128 bytes: a thread's own row would be 16
                    // bytes in each of 32 places at a time
                    const auto put = [&](void* tensor) {
                        __syncwarp();
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            uint32_t w[4];
#pragma unroll
                            for (int k = 0; k < 4; ++k) w[k] = Mma<bf16>::pack(o[j * 8 + 2 * k], o[j * 8 + 2 * k + 1]);
                            *reinterpret_cast<uint4*>(store + swizzled(lane, j)) = make_uint4(w[0], w[1], w[2], w[3]);
                        }
                        __syncwarp();
                        const int col = q * 64 + (lane & 7) * 8;
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            const int from = j * 4 + (lane >> 3);
                            const int64_t to_row = __shfl_sync(0xffffffffu, row, from);
                            const uint4 w = *reinterpret_cast<const uint4*>(store + swizzled(from, lane & 7));
                            if (r - lane + from < p.rows && col < p.dim)
                                *reinterpret_cast<uint4*>(static_cast<bf16*>(tensor) + to_row * p.dim + col) = w;
                        }
                    };
#pragma unroll
                    for (int j = 0; j < 64; ++j) o[j] *= inv;
                    put(p.out);
                    if (p.rest) {
#pragma unroll
                        for (int j = 0; j < 64; ++j) o[j] -= round_bf16(o[j]);
                        put(p.rest);
                    }
                } else if (in) {
                    float* g = p.part + item.split * p.q_count + row * p.dim + q * 64;
#pragma unroll
                    for (int j = 0; j < 64; j += 4) {
                        if (q * 64 + j >= p.dim) break;
                        store4(g + j, o[j] * inv, o[j + 1] * inv, o[j + 2] * inv, o[j + 3] * inv);
                    }
                }
            }
            if (!in) continue;
            if (p.splits > 1) {
                float* ml = p.part_ml + 2 * (item.split * (p.q_count / p.dim) + row);
                ml[0] = m, ml[1] = ok ? l : NAN;
            } else if (p.stats) {
                p.stats[row] = ok ? row_stats(m == -INFINITY ? 0.f : m * c, l) : same(NAN);
            }
        }
    }
    fence_before_sync();
    __syncthreads();
    if (warp == kSoftmaxWarps + 2) {
        fence_after_sync();
        tmem_free(tmem, 512);
        if (lane == 0) report_stall(broken, p.stalled);
    }
}

// --- host ------------------------------------------------------------------------

template <int DP>
int launch_dim(const AttnParams& p, const CUtensorMap& map_k, const CUtensorMap& map_v, int items, int sms, int device, cudaStream_t stream)
{
    using S = TcShape<DP>;
    static std::atomic<uint64_t> done{0};
    const uint64_t bit = device < 64 ? 1ull << device : 0ull;
    if (!bit || !(done.load(std::memory_order_relaxed) & bit)) {
        const cudaError_t e = cudaFuncSetAttribute(attend_tc_kernel<DP>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(S::kAligned));
        if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute");
        done.fetch_or(bit, std::memory_order_relaxed);
    }
    attend_tc_kernel<DP><<<items < sms ? items : sms, kThreads, S::kAligned, stream>>>(p, map_k, map_v, items);
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? POLICY_OK : cuda_fail(e, "attend_tc_kernel");
}

}  // namespace

bool attend_tc_takes(const AttnParams& p)
{
    const int64_t shape[3] = {p.k_count / p.lk / p.kv_heads / p.dim, p.lk, p.kv_heads};
    return map_takes(shape, p.ks, 1) && map_takes(shape, p.vs, 1);
}

int launch_attend_tc(const AttnParams& p, int64_t bh, int sms, int device, cudaStream_t stream)
{
    const int64_t items = bh * p.tiles * p.splits;
    if (items > std::numeric_limits<int32_t>::max() - 4096)
        return fail(POLICY_ERR_INVALID, "policy_cross_attention: more than 2^31 - 4096 tiles of rows");
    const int64_t batch = bh / p.kv_heads;
    const int64_t shape[3] = {batch, p.lk, p.kv_heads};
    CUtensorMap map_k, map_v;
    int rc = make_map(&map_k, p.k, shape, p.ks, p.dim, kTile, 1);
    if (rc == POLICY_OK) rc = make_map(&map_v, p.v, shape, p.vs, p.dim, kTile, 1);
    if (rc != POLICY_OK) return rc;
    return p.dim <= 64 ? launch_dim<64>(p, map_k, map_v, static_cast<int>(items), sms, device, stream)
                       : launch_dim<128>(p, map_k, map_v, static_cast<int>(items), sms, device, stream);
}

}  // namespace policy
