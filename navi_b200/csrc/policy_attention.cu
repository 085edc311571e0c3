// Cross attention of a policy's queries to the tokens of a ray fan, and its gradients.
//
// Layout.  The query heads that share a key head are rows of one matrix: row r of
// (batch, key head) is query r / group, head r % group, so one key tile serves the whole
// group and the gradients of a shared key head need no second pass.
//
// Forward: one pass over the keys with the running maximum and sum of the softmax
//   m' = max(m, max_j s_j),  a = 2^(c (m - m')),  l' = a l + sum_j 2^(c (s_j - m')),  o' = a o + sum_j 2^(..) v_j
// with c = scale log2(e).  Rows beyond the last and keys that are not visible are zeros in
// shared memory, so nothing that masked keys hold reaches a product.
//
// Gradient: p_ij = 2^(c s_ij - x_i) y_i (the forward's reference exponent and reciprocal sum), D_i = do_i . o_i, ds_ij = p_ij (do_i . v_j - D_i);
//   dv_j = sum_i p_ij do_i,  dk_j = scale sum_i ds_ij q_i,  dq_i = scale sum_j ds_ij k_j.
// Up to 16 rows one kernel reads each key and value once and makes all three gradients; with
// more rows one kernel makes dk and dv (a key tile stays, rows stream), one dq (rows stay,
// keys stream).  No sum uses an atomic: work split over a long axis writes f32 parts that a
// second kernel adds in order.
#include <cmath>
#include <atomic>
#include <limits>

#include "policy_attention.cuh"
#include "policy_internal.h"

namespace policy {
namespace {

// rows r0 .. r0 + N - 1 of a query-shaped tensor into a [N][PITCH] tile; zeros past the last row and value
template <typename T, int DP, int PITCH, int N, int THREADS>
__device__ __forceinline__ void load_rows(T* tile, const T* g, const int64_t (&s)[3], const Rows& rows, int r0, int n_rows,
                                          int dim)
{
    using M = Mma<T>;
    constexpr int CH = DP / M::VEC;
    for (int i = threadIdx.x; i < N * CH; i += THREADS) {
        const int r = i / CH, c = (i % CH) * M::VEC;
        const bool take = r0 + r < n_rows && c < dim;
        copy16(smem_addr(tile + r * PITCH + c), take ? g + rows.at(s, r0 + r) + c : g, take);
    }
}

// Streams key and value tiles.  A thread copies the same 16-byte column of every
// (THREADS / CH)-th row of a tile; the rows' visibility is read one tile ahead.
template <typename T, int DP, int PITCH, int KT, int THREADS>
struct KeyLoader {
    using M = Mma<T>;
    static constexpr int CH = DP / M::VEC;
    static constexpr int STEP = THREADS / CH;
    static constexpr int N = KT / STEP;
    static_assert(THREADS % CH == 0 && KT % STEP == 0 && N <= 32, "tile shape");

    const T* k;
    const T* v;
    int64_t ks, vs;
    const uint8_t* mask;
    int n;  // keys below n may be visible
    int row, col;
    bool in_dim;

    __device__ __forceinline__ KeyLoader(const AttnParams& p, int64_t b, int hk, int visible)
    {
        row = threadIdx.x / CH;
        col = (threadIdx.x % CH) * M::VEC;
        in_dim = col < p.dim;
        k = static_cast<const T*>(p.k) + b * p.ks[0] + hk * p.ks[2] + (in_dim ? col : 0);
        v = static_cast<const T*>(p.v) + b * p.vs[0] + hk * p.vs[2] + (in_dim ? col : 0);
        ks = p.ks[1];
        vs = p.vs[1];
        mask = p.mask ? p.mask + b * p.mask_stride : nullptr;
        n = visible;
    }
    __device__ __forceinline__ uint32_t visible(int key0) const
    {
        uint32_t bits = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int key = key0 + row + i * STEP;
            bool on = key < n;
            if (mask && on) on = __ldg(mask + key) != 0;
            bits |= static_cast<uint32_t>(on) << i;
        }
        return bits;
    }
    __device__ __forceinline__ void issue(T* sk, T* sv, uint8_t* svis, int key0, uint32_t bits) const
    {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int r = row + i * STEP;
            const bool on = (bits >> i) & 1u;
            const bool take = on && in_dim;
            const int64_t key = take ? key0 + r : 0;
            copy16(smem_addr(sk + r * PITCH + col), k + key * ks, take);
            copy16(smem_addr(sv + r * PITCH + col), v + key * vs, take);
            if (col == 0) svis[r] = on;
        }
    }
};

// c += a b over the k steps; f32 sums the tile apart and adds it rounded to nearest, since the
// tensor core truncates every accumulation and a long chain of truncations is a bias
//
// f32 also leaves out the steps and columns that hold nothing but the padding of the dim, of the last key tile or of
// the last row tile (`used` of STEPS here, the same for the whole warp): its three products and the splitting make
// them dear, 33 % at dim 96 and most of the time at 3 keys.  Tiles without padding run code without these
// branches, which keep steps from overlapping (20 % at dim 64).
template <bool V>
struct Flag {
    static constexpr bool value = V;
};
template <typename T, typename F>
__device__ __forceinline__ void with_padding(bool padded, F&& f)
{
    if constexpr (Mma<T>::kExact) {
        if (padded) f(Flag<true>{});
        else f(Flag<false>{});
    } else {
        f(Flag<false>{});
    }
}

// f32 adds up this many k steps apart before it adds them, rounded to nearest, to the sum.
constexpr int kFlush = 4;

// c0 and c1 += a with the two B tiles that load(b0, b1, kk) brings, in f32 kFlush steps apart: with the 8 of a 64-key tile in
// one chain, out was off by 2^-20 of its size where values have one sign.
// `rest`, where not null, holds what a's rounding to bf16 left off: a second product with the same b.
template <typename T, int STEPS, bool PADDED, typename LoadB>
__device__ __forceinline__ void accumulate(float (&c0)[4], float (&c1)[4], const typename Mma<T>::A (&a)[STEPS], int used, LoadB&& load,
                                           const typename Mma<T>::A* rest = nullptr)
{
    using M = Mma<T>;
    if constexpr (M::kExact) {
#pragma unroll
        for (int k0 = 0; k0 < STEPS; k0 += kFlush) {
            if (PADDED && k0 >= used) break;
            float t0[4] = {0.f, 0.f, 0.f, 0.f}, t1[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int kk = k0; kk < k0 + kFlush && kk < STEPS; ++kk) {
                if (PADDED && kk >= used) break;
                typename M::B b0, b1;
                load(b0, b1, kk);
                M::mma(t0, a[kk], b0);
                M::mma(t1, a[kk], b1);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) c0[i] += t0[i], c1[i] += t1[i];
        }
    } else {
#pragma unroll
        for (int kk = 0; kk < STEPS; ++kk) {
            typename M::B b0, b1;
            load(b0, b1, kk);
            M::mma(c0, a[kk], b0);
            M::mma(c1, a[kk], b1);
            if (rest) {
                M::mma(c0, rest[kk], b0);
                M::mma(c1, rest[kk], b1);
            }
        }
    }
}

// The products of a 16-row A with N pairs of B tiles, k step by k step: c (+)= a b.  f32 adds up kFlush steps apart
// here too.
template <typename T, int STEPS, bool PADDED, int N, typename Step>
__device__ __forceinline__ void multiply(float (&c)[N][4], int dim, Step&& step)
{
    if constexpr (Mma<T>::kExact) {
#pragma unroll
        for (int k0 = 0; k0 < STEPS; k0 += kFlush) {
            float t[N][4] = {};
#pragma unroll
            for (int kk = k0; kk < k0 + kFlush && kk < STEPS; ++kk)
                if (!PADDED || kk * Mma<T>::KS < dim) step(t, kk);
#pragma unroll
            for (int j = 0; j < N; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i) c[j][i] += t[j][i];
        }
    } else {
#pragma unroll
        for (int kk = 0; kk < STEPS; ++kk) step(c, kk);
    }
}

template <typename T, int DP, int WM, int WN, int KT>
struct FwdShape {
    static constexpr int THREADS = WM * WN * 32;
    static constexpr int ROWS = WM * 16;
    static constexpr int PITCH = DP + Mma<T>::PAD;
    static constexpr int STAGES = 2;
    static_assert(THREADS % (DP / 4) == 0, "a thread keeps its columns");
    // one stage does where there is one tile, and leaves room for more blocks
    static size_t bytes(int stages)
    {
        const size_t stream = kQ + 2 * stages * kTile + stages * KT;
        return stream > kMerge ? stream : kMerge;
    }
    static constexpr size_t kTile = sizeof(T) * KT * PITCH;
    static constexpr size_t kQ = sizeof(T) * ROWS * PITCH;
    static constexpr int OPITCH = DP + 4;
    static constexpr size_t kMerge = sizeof(float) * WN * ROWS * (OPITCH + 2);
};

// WM warps along the rows (16 each), WN along the keys of a tile.  With few rows memory bounds it: one query with 4
// heads to a key head over 64 x 12,288 keys of 64 in bf16 takes 72 us for 404 MB, 5.6 TB/s; in f32 195 us, bound by the
// three TF32 products and the splitting of every operand (35 TFLOP/s where rows are many).
//
// TWO (bf16, up to kFewKeysFwd keys): the weights enter the product with v as two bf16 parts, since the gradients take
// do . out from it, where a weight's rounding does not cancel against the exact one beside it; with many keys the
// roundings average out, and the second product costs 13 % at 64 keys and 37 % where rows and keys are many.
constexpr int kFewKeysFwd = 32;

template <typename T, int DP, int WM, int WN, int KT, bool TWO>
__global__ void __launch_bounds__(WM * WN * 32) attend_kernel(const AttnParams p)
{
    using M = Mma<T>;
    using S = FwdShape<T, DP, WM, WN, KT>;
    constexpr int KS = M::KS, STEPS = DP / KS, KSL = KT / WN, PITCH = S::PITCH;
    constexpr bool QREG = STEPS * 4 <= 32;
    extern __shared__ __align__(128) unsigned char smem[];
    T* sq = reinterpret_cast<T*>(smem);
    T* sk = sq + S::ROWS * PITCH;
    T* sv = sk + p.stages * KT * PITCH;
    uint8_t* svis = reinterpret_cast<uint8_t*>(sv + p.stages * KT * PITCH);

    const int split = blockIdx.x % p.splits;
    const int tile = (blockIdx.x / p.splits) % p.tiles;
    const int bh = blockIdx.x / p.splits / p.tiles;
    const Rows rows{bh / p.kv_heads, bh % p.kv_heads, p.group};
    const int r0 = tile * S::ROWS;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int wm = warp % WM, wn = warp / WM;

    const int n = visible_keys(p, rows.b);
    const int tiles = (n + KT - 1) / KT;
    const int t0 = static_cast<int>(static_cast<int64_t>(tiles) * split / p.splits);
    const int t1 = static_cast<int>(static_cast<int64_t>(tiles) * (split + 1) / p.splits);

    const KeyLoader<T, DP, PITCH, KT, S::THREADS> loader(p, rows.b, rows.hk, n);
    load_rows<T, DP, PITCH, S::ROWS, S::THREADS>(sq, static_cast<const T*>(p.q), p.qs, rows, r0, p.rows, p.dim);
    uint32_t bits = 0;
    if (t0 < t1) {
        loader.issue(sk, sv, svis, t0 * KT, loader.visible(t0 * KT));
        if (t0 + 1 < t1) bits = loader.visible((t0 + 1) * KT);
    }
    copy_commit();

    typename M::A qf[QREG ? STEPS : 1];
    float o[DP / 8][4];
#pragma unroll
    for (int j = 0; j < DP / 8; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[j][i] = 0.f;
    float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
    const float c = p.scale_log2;

    for (int t = t0; t < t1; ++t) {
        const int st = (t - t0) & 1;
        copy_wait<0>();
        __syncthreads();
        if (t + 1 < t1) {
            const int nx = st ^ 1;
            loader.issue(sk + nx * KT * PITCH, sv + nx * KT * PITCH, svis + nx * KT, (t + 1) * KT, bits);
            if (t + 2 < t1) bits = loader.visible((t + 2) * KT);
        }
        copy_commit();
        if constexpr (QREG) {
            if (t == t0) {
#pragma unroll
                for (int kk = 0; kk < STEPS; ++kk) M::load_a(qf[kk], sq + wm * 16 * PITCH + kk * KS, PITCH, lane);
            }
        }
        const T* tk = sk + st * KT * PITCH + wn * KSL * PITCH;
        const T* tv = sv + st * KT * PITCH + wn * KSL * PITCH;
        float s[KSL / 8][4];
#pragma unroll
        for (int j = 0; j < KSL / 8; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) s[j][i] = 0.f;
        const int left = min(n - t * KT, KT) - wn * KSL;  // keys of this warp's part of the tile
        const bool padded = p.dim < DP || left < KSL;
        with_padding<T>(padded, [&](auto pad) {
            multiply<T, STEPS, pad.value>(s, p.dim, [&](float (&x)[KSL / 8][4], int kk) {
                typename M::A a;
                if constexpr (QREG) a = qf[kk];
                else M::load_a(a, sq + wm * 16 * PITCH + kk * KS, PITCH, lane);
#pragma unroll
                for (int j = 0; j < KSL / 16; ++j) {
                    if (pad.value && j * 16 >= left) break;
                    typename M::B b0, b1;
                    M::load_b_nk(b0, b1, tk + j * 16 * PITCH + kk * KS, PITCH, lane);
                    M::mma(x[2 * j], a, b0);
                    M::mma(x[2 * j + 1], a, b1);
                }
            });
        });
        if (p.mask || (t + 1) * KT > n) {
            const uint8_t* vis = svis + st * KT + wn * KSL + (lane & 3) * 2;
#pragma unroll
            for (int j = 0; j < KSL / 8; ++j) {
                const uchar2 on = *reinterpret_cast<const uchar2*>(vis + j * 8);
                if (!on.x) s[j][0] = s[j][2] = -INFINITY;
                if (!on.y) s[j][1] = s[j][3] = -INFINITY;
            }
        }
        float x0 = m0, x1 = m1;
#pragma unroll
        for (int j = 0; j < KSL / 8; ++j) {
            x0 = fmaxf(x0, fmaxf(s[j][0], s[j][1]));
            x1 = fmaxf(x1, fmaxf(s[j][2], s[j][3]));
        }
        x0 = quad_max(x0), x1 = quad_max(x1);
        const float b0 = x0 == -INFINITY ? 0.f : x0 * c, b1 = x1 == -INFINITY ? 0.f : x1 * c;
        const float a0 = exp2_fast(fmaf(m0, c, -b0)), a1 = exp2_fast(fmaf(m1, c, -b1));
        m0 = x0, m1 = x1;
        l0 *= a0, l1 *= a1;
#pragma unroll
        for (int j = 0; j < KSL / 8; ++j) {
            s[j][0] = exp2_fast(fmaf(s[j][0], c, -b0));
            s[j][1] = exp2_fast(fmaf(s[j][1], c, -b0));
            s[j][2] = exp2_fast(fmaf(s[j][2], c, -b1));
            s[j][3] = exp2_fast(fmaf(s[j][3], c, -b1));
        }
        typename M::A pf[KSL / KS];
#pragma unroll
        for (int kk = 0; kk < KSL / KS; ++kk) {
            M::from_c(pf[kk], s, kk);
            if constexpr (!TWO) M::to_c(s, pf[kk], kk);
        }
#pragma unroll
        for (int j = 0; j < KSL / 8; ++j) {
            l0 += s[j][0] + s[j][1];
            l1 += s[j][2] + s[j][3];
        }
        typename M::A pr[TWO ? KSL / KS : 1];
        if constexpr (TWO) {
#pragma unroll
            for (int kk = 0; kk < KSL / KS; ++kk) M::rest_of_c(pr[kk], s, kk);
        }
        with_padding<T>(padded, [&](auto pad) {
#pragma unroll
            for (int j = 0; j < DP / 16; ++j) {
                if (pad.value && j * 16 >= p.dim) break;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    o[2 * j + h][0] *= a0, o[2 * j + h][1] *= a0;
                    o[2 * j + h][2] *= a1, o[2 * j + h][3] *= a1;
                }
                accumulate<T, KSL / KS, pad.value>(o[2 * j], o[2 * j + 1], pf, (left + KS - 1) / KS, [&](typename M::B& b0_, typename M::B& b1_, int kk) {
                    M::load_b_kn(b0_, b1_, tv + kk * KS * PITCH + j * 16, PITCH, lane);
                }, TWO ? pr : nullptr);
            }
        });
    }

    // the warps along the keys meet in shared memory, and the rows leave it in whole vectors
    copy_wait<0>();
    __syncthreads();
    float* so = reinterpret_cast<float*>(smem);
    float* sm = so + WN * S::ROWS * S::OPITCH;
    float* sl = sm + WN * S::ROWS;
    l0 = quad_sum(l0), l1 = quad_sum(l1);
    {
        const int r = wn * S::ROWS + wm * 16 + (lane >> 2);
        float* w = so + r * S::OPITCH + (lane & 3) * 2;
#pragma unroll
        for (int j = 0; j < DP / 8; ++j) {
            *reinterpret_cast<float2*>(w + j * 8) = make_float2(o[j][0], o[j][1]);
            *reinterpret_cast<float2*>(w + 8 * S::OPITCH + j * 8) = make_float2(o[j][2], o[j][3]);
        }
        if ((lane & 3) == 0) sm[r] = m0, sl[r] = l0, sm[r + 8] = m1, sl[r + 8] = l1;
    }
    __syncthreads();
    constexpr int CHUNKS = DP / 4;  // a thread keeps its columns
    for (int i = threadIdx.x; i < S::ROWS * CHUNKS; i += S::THREADS) {
        const int r = i / CHUNKS, d = (i % CHUNKS) * 4;
        if (r0 + r >= p.rows || d >= p.dim) break;
        float m = sm[r];
#pragma unroll
        for (int w = 1; w < WN; ++w) m = fmaxf(m, sm[w * S::ROWS + r]);
        const float base = m == -INFINITY ? 0.f : m * c;
        float l = 0.f;
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < WN; ++w) {
            const float f = exp2_fast(fmaf(sm[w * S::ROWS + r], c, -base));
            const float4 y = *reinterpret_cast<const float4*>(so + (w * S::ROWS + r) * S::OPITCH + d);
            l = fmaf(f, sl[w * S::ROWS + r], l);
            x.x = fmaf(f, y.x, x.x), x.y = fmaf(f, y.y, x.y), x.z = fmaf(f, y.z, x.z), x.w = fmaf(f, y.w, x.w);
        }
        const int64_t row = rows.index(p, r0 + r);
        if (p.splits == 1) {
            const float inv = l == 0.f ? 0.f : 1.f / l;
            store_out<T>(p, row * p.dim + d, x.x * inv, x.y * inv, x.z * inv, x.w * inv);
            if (d == 0 && p.stats) p.stats[row] = row_stats(base, l);
        } else {
            store4(p.part + split * p.q_count + row * p.dim + d, x.x, x.y, x.z, x.w);
            if (d == 0) {
                float* ml = p.part_ml + 2 * (split * (p.q_count / p.dim) + row);
                ml[0] = m, ml[1] = l;
            }
        }
    }
}

// Joins the parts of a forward launch split over the keys: a block to a row, its threads in groups of
// `lanes` (a power of two, 4 values each), which share out the parts.
constexpr int kJoinThreads = 128;

template <typename T>
__global__ void __launch_bounds__(kJoinThreads) attend_join_kernel(const AttnParams p, int lanes)
{
    __shared__ float4 sums[kJoinThreads];
    __shared__ float2 stats[kJoinThreads];
    const int64_t n_rows = p.q_count / p.dim, row = blockIdx.x;
    const int d = (threadIdx.x & (lanes - 1)) * 4, first = threadIdx.x / lanes, groups = kJoinThreads / lanes;
    const float c = p.scale_log2;
    const float2* ml = reinterpret_cast<const float2*>(p.part_ml) + row;
    const float* part = p.part + row * p.dim + d;
    float m = -INFINITY, l = 0.f;
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
    if (d < p.dim) {
#pragma unroll 4
        for (int s = first; s < p.splits; s += groups) {
            const float2 v = ml[s * n_rows];
            const float4 y = *reinterpret_cast<const float4*>(part + s * p.q_count);
            const float top = fmaxf(m, v.x);
            const float base = top == -INFINITY ? 0.f : top * c;
            const float a = exp2_fast(fmaf(m, c, -base)), f = exp2_fast(fmaf(v.x, c, -base));
            m = top;
            l = fmaf(l, a, f * v.y);
            x.x = fmaf(x.x, a, f * y.x), x.y = fmaf(x.y, a, f * y.y), x.z = fmaf(x.z, a, f * y.z), x.w = fmaf(x.w, a, f * y.w);
        }
    }
    sums[threadIdx.x] = x;
    stats[threadIdx.x] = make_float2(m, l);
    __syncthreads();
    if (first != 0 || d >= p.dim) return;
    float top = -INFINITY;
    for (int g = 0; g < groups; ++g) top = fmaxf(top, stats[g * lanes + threadIdx.x].x);
    const float base = top == -INFINITY ? 0.f : top * c;
    l = 0.f;
    x = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int g = 0; g < groups; ++g) {
        const float2 v = stats[g * lanes + threadIdx.x];
        const float4 y = sums[g * lanes + threadIdx.x];
        const float f = exp2_fast(fmaf(v.x, c, -base));
        l = fmaf(f, v.y, l);
        x.x = fmaf(f, y.x, x.x), x.y = fmaf(f, y.y, x.y), x.z = fmaf(f, y.z, x.z), x.w = fmaf(f, y.w, x.w);
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    store_out<T>(p, row * p.dim + d, x.x * inv, x.y * inv, x.z * inv, x.w * inv);
    if (d == 0 && p.stats) p.stats[row] = row_stats(base, l);
}

// --- gradients -----------------------------------------------------------------

// D_i = do_i . o_i of a row, b and its rest (or null) together being o: 8 lanes to a row.
template <typename T>
__device__ __forceinline__ float row_dot(const T* a, const T* b, const T* rest, int dim, int sub)
{
    float x = 0.f;
    for (int d = sub * 4; d < dim; d += 32) {
        if constexpr (sizeof(T) == 4) {
            const float4 u = *reinterpret_cast<const float4*>(a + d), w = *reinterpret_cast<const float4*>(b + d);
            x = fmaf(u.x, w.x, fmaf(u.y, w.y, fmaf(u.z, w.z, fmaf(u.w, w.w, x))));
        } else {
            const uint2 u = *reinterpret_cast<const uint2*>(a + d), w = *reinterpret_cast<const uint2*>(b + d);
            const float2 u0 = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u.x));
            const float2 u1 = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u.y));
            const float2 w0 = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w.x));
            const float2 w1 = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w.y));
            x = fmaf(u0.x, w0.x, fmaf(u0.y, w0.y, fmaf(u1.x, w1.x, fmaf(u1.y, w1.y, x))));
            if (rest) {
                const uint2 z = *reinterpret_cast<const uint2*>(rest + d);
                const float2 z0 = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&z.x));
                const float2 z1 = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&z.y));
                x = fmaf(u0.x, z0.x, fmaf(u0.y, z0.y, fmaf(u1.x, z1.x, fmaf(u1.y, z1.y, x))));
            }
        }
    }
    x += __shfl_xor_sync(0xffffffffu, x, 1);
    x += __shfl_xor_sync(0xffffffffu, x, 2);
    return x + __shfl_xor_sync(0xffffffffu, x, 4);
}

template <typename T>
__global__ void __launch_bounds__(256) attend_delta_kernel(const AttnParams p, float* delta)
{
    const int64_t i = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) >> 3;
    const int64_t n_rows = p.q_count / p.dim;
    const int64_t row = min(i, n_rows - 1);
    const int h = static_cast<int>(row % p.heads);
    const int64_t bl = row / p.heads, b = bl / p.lq, l = bl - b * p.lq;
    const T* g = static_cast<const T*>(p.dout) + b * p.ds[0] + l * p.ds[1] + h * p.ds[2];
    const T* rest = p.rest ? static_cast<const T*>(p.rest) + row * p.dim : nullptr;
    const float x = row_dot(g, static_cast<const T*>(p.out) + row * p.dim, rest, p.dim, threadIdx.x & 7);
    if (i < n_rows && (threadIdx.x & 7) == 0) delta[row] = x;
}

template <typename T, int DP, int NW>
struct GradShape {
    static constexpr int THREADS = NW * 32;
    static constexpr int KT = NW * 16;
    static constexpr int PITCH = DP + Mma<T>::PAD;
    static constexpr int TP = sizeof(T) == 2 ? 24 : 20;  // pitch of a warp's 16 x 16 transpose
    static constexpr int OPITCH = DP + 4;
    static constexpr size_t kKeys = sizeof(T) * KT * PITCH;
    // all gradients, 16 rows
    static constexpr size_t kMerge = sizeof(float) * NW * 16 * OPITCH;
    static constexpr size_t few_bytes(bool two)
    {
        const size_t stream = 4 * kKeys + sizeof(T) * (2 * 16 * PITCH + (two ? 2 : 1) * NW * 16 * TP) + 2 * KT + 16 * 3 * sizeof(float);
        return stream > kMerge ? stream : kMerge;
    }
    // dk and dv: RT rows stream
    static constexpr int RT = 32;
    static constexpr size_t kKeyGrad = 2 * kKeys + 4 * sizeof(T) * RT * PITCH + 6 * RT * sizeof(float) + KT;
    // dq: 16 NW rows stay, QT keys stream
    static constexpr int QT = 32;
    static constexpr size_t kQueryStream = 2 * kKeys + 4 * sizeof(T) * QT * PITCH + 2 * QT;
    static constexpr size_t kQueryGrad = kQueryStream > kMerge ? kQueryStream : kMerge;
};

// A warp's 16 keys x 16 DP gradient C tiles through its own 16 rows of a shared tile to global memory.
template <typename T, int DP, int PITCH>
__device__ __forceinline__ void store_key_rows(const T* tile, T* g, int64_t row_values, int key0, int lk, int dim, int lane)
{
    using M = Mma<T>;
    constexpr int CH = DP / M::VEC;
    for (int i = lane; i < 16 * CH; i += 32) {
        const int r = i / CH, c = (i % CH) * M::VEC;
        if (key0 + r < lk && c < dim)
            *reinterpret_cast<uint4*>(g + (key0 + r) * row_values + c) = *reinterpret_cast<const uint4*>(tile + r * PITCH + c);
    }
}

// All three gradients of up to 16 rows: K and V are read once; dk and dv of a key tile are whole when it
// has passed, dq is summed over the tiles.  Memory bounds it: 1,024 x 8 heads of 16 rows and 192 keys of 64 in bf16
// take 188 us for 823 MB, 4.4 TB/s; what is left above the memory's rate is the chain scores - weights -
// three products of a tile, which 16 resident warps do not hide.
//
// TWO (bf16, up to kTwoKeys keys): the weights and their gradients enter the products as two bf16 parts.  With few keys
// the roundings do not average out, and were 1.5 times the output's own; with many the second products cost 24 %.
constexpr int kTwoKeys = 64;

template <typename T, int DP, int NW, bool TWO>
__global__ void __launch_bounds__(NW * 32) attend_grad_few_kernel(const AttnParams p)
{
    using M = Mma<T>;
    using S = GradShape<T, DP, NW>;
    constexpr int KS = M::KS, STEPS = DP / KS, PITCH = S::PITCH, KT = S::KT, RS = 16 / KS;
    extern __shared__ __align__(128) unsigned char smem[];
    T* sk = reinterpret_cast<T*>(smem);
    T* sv = sk + 2 * KT * PITCH;
    T* sq = sv + 2 * KT * PITCH;
    T* sdo = sq + 16 * PITCH;
    T* str = sdo + 16 * PITCH;
    float2* sstats = reinterpret_cast<float2*>(str + (TWO ? 2 : 1) * NW * 16 * S::TP);
    float* sdelta = reinterpret_cast<float*>(sstats + 16);
    uint8_t* svis = reinterpret_cast<uint8_t*>(sdelta + 16);

    const int split = blockIdx.x % p.splits;
    const int bh = blockIdx.x / p.splits;
    const Rows rows{bh / p.kv_heads, bh % p.kv_heads, p.group};
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int n = visible_keys(p, rows.b);
    const int tiles = (p.lk + KT - 1) / KT;
    const int t0 = static_cast<int>(static_cast<int64_t>(tiles) * split / p.splits);
    const int t1 = static_cast<int>(static_cast<int64_t>(tiles) * (split + 1) / p.splits);

    const KeyLoader<T, DP, PITCH, KT, S::THREADS> loader(p, rows.b, rows.hk, n);
    load_rows<T, DP, PITCH, 16, S::THREADS>(sq, static_cast<const T*>(p.q), p.qs, rows, 0, p.rows, p.dim);
    load_rows<T, DP, PITCH, 16, S::THREADS>(sdo, static_cast<const T*>(p.dout), p.ds, rows, 0, p.rows, p.dim);
    loader.issue(sk, sv, svis, t0 * KT, loader.visible(t0 * KT));
    uint32_t bits = t0 + 1 < t1 ? loader.visible((t0 + 1) * KT) : 0u;
    copy_commit();
    for (int r = threadIdx.x >> 3; r < 16; r += S::THREADS / 8) {
        const int rr = min(r, p.rows - 1);
        const int64_t row = rows.index(p, rr);
        const float x = row_dot(static_cast<const T*>(p.dout) + rows.at(p.ds, rr), static_cast<const T*>(p.out) + row * p.dim,
                                p.rest ? static_cast<const T*>(p.rest) + row * p.dim : nullptr, p.dim, threadIdx.x & 7);
        if ((threadIdx.x & 7) == 0) {
            sstats[r] = r < p.rows ? p.stats[row] : make_float2(0.f, 0.f);
            sdelta[r] = r < p.rows ? x : 0.f;
        }
    }
    const bool lone = lone_key(p, rows.b, n);

    float dq[DP / 8][4];
#pragma unroll
    for (int j = 0; j < DP / 8; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) dq[j][i] = 0.f;
    T* tr = str + warp * 16 * S::TP;
    const int64_t key_row = static_cast<int64_t>(p.kv_heads) * p.dim;
    T* gk = static_cast<T*>(p.dk) + (rows.b * p.lk * p.kv_heads + rows.hk) * p.dim;
    T* gv = static_cast<T*>(p.dv) + (rows.b * p.lk * p.kv_heads + rows.hk) * p.dim;

    for (int t = t0; t < t1; ++t) {
        const int st = (t - t0) & 1;
        copy_wait<0>();
        __syncthreads();
        if (t + 1 < t1) {
            const int nx = st ^ 1;
            loader.issue(sk + nx * KT * PITCH, sv + nx * KT * PITCH, svis + nx * KT, (t + 1) * KT, bits);
            if (t + 2 < t1) bits = loader.visible((t + 2) * KT);
        }
        copy_commit();
        T* tk = sk + (st * KT + warp * 16) * PITCH;
        T* tv = sv + (st * KT + warp * 16) * PITCH;
        float s[2][4] = {}, dp[2][4] = {};  // [16 keys] x [16 rows]
        const bool live = t * KT + warp * 16 < n;  // some key of the warp's may be visible
        const bool padded = !live || p.dim < DP || p.rows <= 8;
        with_padding<T>(padded, [&](auto pad) {
            const auto product = [&](float (&out)[2][4], const T* a_tile, const T* b_tile) {
                multiply<T, STEPS, pad.value>(out, live ? p.dim : 0, [&](float (&x)[2][4], int kk) {
                    typename M::A a;
                    typename M::B b0, b1;
                    M::load_a(a, a_tile + kk * KS, PITCH, lane);
                    M::load_b_nk(b0, b1, b_tile + kk * KS, PITCH, lane);
                    M::mma(x[0], a, b0);
                    M::mma(x[1], a, b1);
                });
            };
            product(s, tk, sq);
            product(dp, tv, sdo);
        });
        const bool on0 = svis[st * KT + warp * 16 + (lane >> 2)], on1 = svis[st * KT + warp * 16 + (lane >> 2) + 8];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int r = j * 8 + (lane & 3) * 2 + (i & 1);
                const float2 st_r = sstats[r];
                const bool on = (i < 2 ? on0 : on1) && st_r.y != 0.f;
                const float w = exp2_fast(fmaf(s[j][i], p.scale_log2, -st_r.x)) * st_r.y;
                s[j][i] = on ? w : 0.f;
                dp[j][i] = on && !lone ? w * (dp[j][i] - sdelta[r]) : 0.f;
                const int key = (lane >> 2) + (i < 2 ? 0 : 8);
                if constexpr (TWO) {
                    tr[r * S::TP + key] = __float2bfloat16_rn(dp[j][i]);
                    tr[(NW * 16 + r) * S::TP + key] = __float2bfloat16_rn(M::left_off(dp[j][i]));
                } else {
                    tr[r * S::TP + key] = dp[j][i];
                }
            }
        }
        __syncwarp();
        typename M::A df[RS], pf[RS], kf[RS], dr[RS], pr[RS], kr[RS];
#pragma unroll
        for (int kk = 0; kk < RS; ++kk) {
            M::load_a(df[kk], tr + kk * KS, S::TP, lane);
            M::from_c(pf[kk], s, kk);
            M::from_c(kf[kk], dp, kk);
            if constexpr (TWO) {
                M::load_a(dr[kk], tr + NW * 16 * S::TP + kk * KS, S::TP, lane);
                M::rest_of_c(pr[kk], s, kk);
                M::rest_of_c(kr[kk], dp, kk);
            }
        }
        with_padding<T>(padded, [&](auto pad) {
#pragma unroll
            for (int j = 0; j < DP / 16; ++j) {
                if (pad.value && j * 16 >= p.dim) break;
                accumulate<T, RS, pad.value>(dq[2 * j], dq[2 * j + 1], df, live ? RS : 0, [&](typename M::B& b0, typename M::B& b1, int kk) {
                    M::load_b_kn(b0, b1, tk + kk * KS * PITCH + j * 16, PITCH, lane);
                }, TWO ? dr : nullptr);
            }
            __syncwarp();
#pragma unroll
            for (int j = 0; j < DP / 16; ++j) {
                if (pad.value && j * 16 >= p.dim) break;
                float x[2][4] = {}, y[2][4] = {};
                const int used = live ? (p.rows + KS - 1) / KS : 0;
                accumulate<T, RS, pad.value>(x[0], x[1], pf, used, [&](typename M::B& b0, typename M::B& b1, int kk) {
                    M::load_b_kn(b0, b1, sdo + kk * KS * PITCH + j * 16, PITCH, lane);
                }, TWO ? pr : nullptr);
                accumulate<T, RS, pad.value>(y[0], y[1], kf, used, [&](typename M::B& b0, typename M::B& b1, int kk) {
                    M::load_b_kn(b0, b1, sq + kk * KS * PITCH + j * 16, PITCH, lane);
                }, TWO ? kr : nullptr);
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int at = (lane >> 2) * PITCH + j * 16 + h * 8 + (lane & 3) * 2;
                    M::store2(tv + at, on0 ? x[h][0] : 0.f, on0 ? x[h][1] : 0.f);
                    M::store2(tv + at + 8 * PITCH, on1 ? x[h][2] : 0.f, on1 ? x[h][3] : 0.f);
                    M::store2(tk + at, on0 ? y[h][0] * p.scale : 0.f, on0 ? y[h][1] * p.scale : 0.f);
                    M::store2(tk + at + 8 * PITCH, on1 ? y[h][2] * p.scale : 0.f, on1 ? y[h][3] * p.scale : 0.f);
                }
            }
        });
        __syncwarp();
        const int key0 = t * KT + warp * 16;
        store_key_rows<T, DP, PITCH>(tv, gv, key_row, key0, p.lk, p.dim, lane);
        store_key_rows<T, DP, PITCH>(tk, gk, key_row, key0, p.lk, p.dim, lane);
    }

    copy_wait<0>();
    __syncthreads();
    float* so = reinterpret_cast<float*>(smem);
    {
        float* w = so + (warp * 16 + (lane >> 2)) * S::OPITCH + (lane & 3) * 2;
#pragma unroll
        for (int j = 0; j < DP / 8; ++j) {
            *reinterpret_cast<float2*>(w + j * 8) = make_float2(dq[j][0], dq[j][1]);
            *reinterpret_cast<float2*>(w + 8 * S::OPITCH + j * 8) = make_float2(dq[j][2], dq[j][3]);
        }
    }
    __syncthreads();
    constexpr int CHUNKS = DP / 4;
    for (int i = threadIdx.x; i < 16 * CHUNKS; i += S::THREADS) {
        const int r = i / CHUNKS, d = (i % CHUNKS) * 4;
        if (r >= p.rows || d >= p.dim) break;
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            const float4 y = *reinterpret_cast<const float4*>(so + (w * 16 + r) * S::OPITCH + d);
            x.x += y.x, x.y += y.y, x.z += y.z, x.w += y.w;
        }
        x.x *= p.scale, x.y *= p.scale, x.z *= p.scale, x.w *= p.scale;
        const int64_t at = rows.index(p, r) * p.dim + d;
        if (p.splits == 1) store4(static_cast<T*>(p.dq) + at, x.x, x.y, x.z, x.w);
        else store4(p.part + split * p.q_count + at, x.x, x.y, x.z, x.w);
    }
}

// dk and dv of 16 NW keys: the keys stay in shared memory, rows stream past them.  In bf16 the weights and their gradients
// enter the products as one bf16 part, here and for dq: the gradients are 0.0024 of their norm off with it, 0.0017 of that
// from their own rounding.
template <typename T, int DP, int NW>
__global__ void __launch_bounds__(NW * 32) attend_grad_keys_kernel(const AttnParams p)
{
    using M = Mma<T>;
    using S = GradShape<T, DP, NW>;
    constexpr int KS = M::KS, STEPS = DP / KS, PITCH = S::PITCH, KT = S::KT, RT = S::RT, RS = RT / KS;
    extern __shared__ __align__(128) unsigned char smem[];
    T* sk = reinterpret_cast<T*>(smem);
    T* sv = sk + KT * PITCH;
    T* sq = sv + KT * PITCH;
    T* sdo = sq + 2 * RT * PITCH;
    float2* sstats = reinterpret_cast<float2*>(sdo + 2 * RT * PITCH);
    float* sdelta = reinterpret_cast<float*>(sstats + 2 * RT);
    uint8_t* svis = reinterpret_cast<uint8_t*>(sdelta + 2 * RT);

    const int split = blockIdx.x % p.splits;
    const int tile = (blockIdx.x / p.splits) % p.tiles;
    const int bh = blockIdx.x / p.splits / p.tiles;
    const Rows rows{bh / p.kv_heads, bh % p.kv_heads, p.group};
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int n = visible_keys(p, rows.b);
    const int row_tiles = (p.rows + RT - 1) / RT;
    const int t0 = static_cast<int>(static_cast<int64_t>(row_tiles) * split / p.splits);
    const int t1 = static_cast<int>(static_cast<int64_t>(row_tiles) * (split + 1) / p.splits);

    const KeyLoader<T, DP, PITCH, KT, S::THREADS> loader(p, rows.b, rows.hk, n);
    loader.issue(sk, sv, svis, tile * KT, loader.visible(tile * KT));
    auto issue = [&](int t, int st) {
        load_rows<T, DP, PITCH, RT, S::THREADS>(sq + st * RT * PITCH, static_cast<const T*>(p.q), p.qs, rows, t * RT, p.rows, p.dim);
        load_rows<T, DP, PITCH, RT, S::THREADS>(sdo + st * RT * PITCH, static_cast<const T*>(p.dout), p.ds, rows, t * RT, p.rows, p.dim);
        for (int i = threadIdx.x; i < RT; i += S::THREADS) {
            const int r = t * RT + i;
            const bool take = r < p.rows;
            const int64_t row = take ? rows.index(p, r) : 0;
            asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;\n" ::"r"(smem_addr(sstats + st * RT + i)), "l"(p.stats + row),
                         "r"(take ? 8 : 0) : "memory");
            asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;\n" ::"r"(smem_addr(sdelta + st * RT + i)), "l"(p.delta + row),
                         "r"(take ? 4 : 0) : "memory");
        }
    };
    if (t0 < t1) issue(t0, 0);
    copy_commit();
    const bool lone = lone_key(p, rows.b, n);

    float dk[DP / 8][4], dv[DP / 8][4];
#pragma unroll
    for (int j = 0; j < DP / 8; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) dk[j][i] = dv[j][i] = 0.f;
    T* tk = sk + warp * 16 * PITCH;
    T* tv = sv + warp * 16 * PITCH;
    bool on0 = false, on1 = false;

    for (int t = t0; t < t1; ++t) {
        const int st = (t - t0) & 1;
        copy_wait<0>();
        __syncthreads();
        if (t + 1 < t1) issue(t + 1, st ^ 1);
        copy_commit();
        on0 = svis[warp * 16 + (lane >> 2)], on1 = svis[warp * 16 + (lane >> 2) + 8];
        const T* tq = sq + st * RT * PITCH;
        const T* td = sdo + st * RT * PITCH;
        float s[RT / 8][4] = {}, dp[RT / 8][4] = {};  // [16 keys] x [RT rows]
        const int left = p.rows - t * RT;
        const bool padded = p.dim < DP || left < RT;
        with_padding<T>(padded, [&](auto pad) {
            const auto product = [&](float (&out)[RT / 8][4], const T* a_tile, const T* b_tile) {
                multiply<T, STEPS, pad.value>(out, p.dim, [&](float (&x)[RT / 8][4], int kk) {
                    typename M::A a;
                    M::load_a(a, a_tile + kk * KS, PITCH, lane);
#pragma unroll
                    for (int j = 0; j < RT / 16; ++j) {
                        if (pad.value && j * 16 >= left) break;
                        typename M::B b0, b1;
                        M::load_b_nk(b0, b1, b_tile + j * 16 * PITCH + kk * KS, PITCH, lane);
                        M::mma(x[2 * j], a, b0);
                        M::mma(x[2 * j + 1], a, b1);
                    }
                });
            };
            product(s, tk, tq);
            product(dp, tv, td);
        });
#pragma unroll
        for (int j = 0; j < RT / 8; ++j) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int r = j * 8 + (lane & 3) * 2 + (i & 1);
                const float2 st_r = sstats[st * RT + r];
                const bool on = (i < 2 ? on0 : on1) && st_r.y != 0.f;
                const float w = exp2_fast(fmaf(s[j][i], p.scale_log2, -st_r.x)) * st_r.y;
                s[j][i] = on ? w : 0.f;
                dp[j][i] = on && !lone ? w * (dp[j][i] - sdelta[st * RT + r]) : 0.f;
            }
        }
        typename M::A pf[RS], df[RS];
#pragma unroll
        for (int kk = 0; kk < RS; ++kk) {
            M::from_c(pf[kk], s, kk);
            M::from_c(df[kk], dp, kk);
        }
        with_padding<T>(padded, [&](auto pad) {
#pragma unroll
            for (int j = 0; j < DP / 16; ++j) {
                if (pad.value && j * 16 >= p.dim) break;
                const int used = (left + KS - 1) / KS;
                accumulate<T, RS, pad.value>(dv[2 * j], dv[2 * j + 1], pf, used, [&](typename M::B& b0, typename M::B& b1, int kk) {
                    M::load_b_kn(b0, b1, td + kk * KS * PITCH + j * 16, PITCH, lane);
                });
                accumulate<T, RS, pad.value>(dk[2 * j], dk[2 * j + 1], df, used, [&](typename M::B& b0, typename M::B& b1, int kk) {
                    M::load_b_kn(b0, b1, tq + kk * KS * PITCH + j * 16, PITCH, lane);
                });
            }
        });
    }
    copy_wait<0>();
    __syncthreads();
    const int key0 = tile * KT + warp * 16;
    if (p.splits == 1) {
#pragma unroll
        for (int j = 0; j < DP / 8; ++j) {
            const int at = (lane >> 2) * PITCH + j * 8 + (lane & 3) * 2;
            M::store2(tv + at, on0 ? dv[j][0] : 0.f, on0 ? dv[j][1] : 0.f);
            M::store2(tv + at + 8 * PITCH, on1 ? dv[j][2] : 0.f, on1 ? dv[j][3] : 0.f);
            M::store2(tk + at, on0 ? dk[j][0] * p.scale : 0.f, on0 ? dk[j][1] * p.scale : 0.f);
            M::store2(tk + at + 8 * PITCH, on1 ? dk[j][2] * p.scale : 0.f, on1 ? dk[j][3] * p.scale : 0.f);
        }
        __syncwarp();
        const int64_t key_row = static_cast<int64_t>(p.kv_heads) * p.dim;
        const int64_t base = (rows.b * p.lk * p.kv_heads + rows.hk) * p.dim;
        store_key_rows<T, DP, PITCH>(tv, static_cast<T*>(p.dv) + base, key_row, key0, p.lk, p.dim, lane);
        store_key_rows<T, DP, PITCH>(tk, static_cast<T*>(p.dk) + base, key_row, key0, p.lk, p.dim, lane);
    } else {
        float* part = p.part + 2 * split * p.k_count;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int key = key0 + (lane >> 2) + 8 * h;
            const bool on = h ? on1 : on0;
            if (key >= p.lk) continue;
            float* at = part + ((rows.b * p.lk + key) * p.kv_heads + rows.hk) * p.dim + (lane & 3) * 2;
#pragma unroll
            for (int j = 0; j < DP / 8; ++j) {
                if (j * 8 >= p.dim) break;
                const float2 k2 = on ? make_float2(dk[j][2 * h] * p.scale, dk[j][2 * h + 1] * p.scale) : make_float2(0.f, 0.f);
                const float2 v2 = on ? make_float2(dv[j][2 * h], dv[j][2 * h + 1]) : make_float2(0.f, 0.f);
                *reinterpret_cast<float2*>(at + j * 8) = k2;
                *reinterpret_cast<float2*>(at + p.k_count + j * 8) = v2;
            }
        }
    }
}

// dq of 16 NW rows: the rows stay, keys stream.
template <typename T, int DP, int NW>
__global__ void __launch_bounds__(NW * 32) attend_grad_queries_kernel(const AttnParams p)
{
    using M = Mma<T>;
    using S = GradShape<T, DP, NW>;
    constexpr int KS = M::KS, STEPS = DP / KS, PITCH = S::PITCH, KT = S::QT, ROWS = NW * 16;
    extern __shared__ __align__(128) unsigned char smem[];
    T* sq = reinterpret_cast<T*>(smem);
    T* sdo = sq + ROWS * PITCH;
    T* sk = sdo + ROWS * PITCH;
    T* sv = sk + 2 * KT * PITCH;
    uint8_t* svis = reinterpret_cast<uint8_t*>(sv + 2 * KT * PITCH);

    const int split = blockIdx.x % p.splits;
    const int tile = (blockIdx.x / p.splits) % p.tiles;
    const int bh = blockIdx.x / p.splits / p.tiles;
    const Rows rows{bh / p.kv_heads, bh % p.kv_heads, p.group};
    const int r0 = tile * ROWS;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int n = visible_keys(p, rows.b);
    const int tiles = (n + KT - 1) / KT;
    const int t0 = static_cast<int>(static_cast<int64_t>(tiles) * split / p.splits);
    const int t1 = static_cast<int>(static_cast<int64_t>(tiles) * (split + 1) / p.splits);

    const KeyLoader<T, DP, PITCH, KT, S::THREADS> loader(p, rows.b, rows.hk, n);
    load_rows<T, DP, PITCH, ROWS, S::THREADS>(sq, static_cast<const T*>(p.q), p.qs, rows, r0, p.rows, p.dim);
    load_rows<T, DP, PITCH, ROWS, S::THREADS>(sdo, static_cast<const T*>(p.dout), p.ds, rows, r0, p.rows, p.dim);
    uint32_t bits = 0;
    if (t0 < t1) {
        loader.issue(sk, sv, svis, t0 * KT, loader.visible(t0 * KT));
        if (t0 + 1 < t1) bits = loader.visible((t0 + 1) * KT);
    }
    copy_commit();
    float2 stats[2];
    float delta[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int r = r0 + warp * 16 + (lane >> 2) + 8 * h;
        const int64_t row = rows.index(p, min(r, p.rows - 1));
        stats[h] = r < p.rows ? p.stats[row] : make_float2(0.f, 0.f);
        delta[h] = r < p.rows ? p.delta[row] : 0.f;
    }
    if (lone_key(p, rows.b, n)) stats[0].y = stats[1].y = 0.f;  // no gradient
    float dq[DP / 8][4];
#pragma unroll
    for (int j = 0; j < DP / 8; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) dq[j][i] = 0.f;

    for (int t = t0; t < t1; ++t) {
        const int st = (t - t0) & 1;
        copy_wait<0>();
        __syncthreads();
        if (t + 1 < t1) {
            const int nx = st ^ 1;
            loader.issue(sk + nx * KT * PITCH, sv + nx * KT * PITCH, svis + nx * KT, (t + 1) * KT, bits);
            if (t + 2 < t1) bits = loader.visible((t + 2) * KT);
        }
        copy_commit();
        const T* tk = sk + st * KT * PITCH;
        const T* tv = sv + st * KT * PITCH;
        float s[KT / 8][4] = {}, dp[KT / 8][4] = {};  // [16 rows] x [KT keys]
        const int left = n - t * KT;
        const bool padded = p.dim < DP || left < KT;
        with_padding<T>(padded, [&](auto pad) {
            const auto product = [&](float (&out)[KT / 8][4], const T* a_tile, const T* b_tile) {
                multiply<T, STEPS, pad.value>(out, p.dim, [&](float (&x)[KT / 8][4], int kk) {
                    typename M::A a;
                    M::load_a(a, a_tile + warp * 16 * PITCH + kk * KS, PITCH, lane);
#pragma unroll
                    for (int j = 0; j < KT / 16; ++j) {
                        if (pad.value && j * 16 >= left) break;
                        typename M::B b0, b1;
                        M::load_b_nk(b0, b1, b_tile + j * 16 * PITCH + kk * KS, PITCH, lane);
                        M::mma(x[2 * j], a, b0);
                        M::mma(x[2 * j + 1], a, b1);
                    }
                });
            };
            product(s, sq, tk);
            product(dp, sdo, tv);
        });
#pragma unroll
        for (int j = 0; j < KT / 8; ++j) {
            const uchar2 vis = *reinterpret_cast<const uchar2*>(svis + st * KT + j * 8 + (lane & 3) * 2);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int h = i >> 1;
                const bool on = ((i & 1) ? vis.y : vis.x) && stats[h].y != 0.f;
                const float w = exp2_fast(fmaf(s[j][i], p.scale_log2, -stats[h].x)) * stats[h].y;
                dp[j][i] = on ? w * (dp[j][i] - delta[h]) : 0.f;
            }
        }
        typename M::A df[KT / KS];
#pragma unroll
        for (int kk = 0; kk < KT / KS; ++kk) M::from_c(df[kk], dp, kk);
        with_padding<T>(padded, [&](auto pad) {
#pragma unroll
            for (int j = 0; j < DP / 16; ++j) {
                if (pad.value && j * 16 >= p.dim) break;
                accumulate<T, KT / KS, pad.value>(dq[2 * j], dq[2 * j + 1], df, (left + KS - 1) / KS, [&](typename M::B& b0, typename M::B& b1, int kk) {
                    M::load_b_kn(b0, b1, tk + kk * KS * PITCH + j * 16, PITCH, lane);
                });
            }
        });
    }
    copy_wait<0>();
    __syncthreads();
    float* so = reinterpret_cast<float*>(smem);
    {
        float* w = so + (warp * 16 + (lane >> 2)) * S::OPITCH + (lane & 3) * 2;
#pragma unroll
        for (int j = 0; j < DP / 8; ++j) {
            *reinterpret_cast<float2*>(w + j * 8) = make_float2(dq[j][0], dq[j][1]);
            *reinterpret_cast<float2*>(w + 8 * S::OPITCH + j * 8) = make_float2(dq[j][2], dq[j][3]);
        }
    }
    __syncthreads();
    constexpr int CHUNKS = DP / 4;
    for (int i = threadIdx.x; i < ROWS * CHUNKS; i += S::THREADS) {
        const int r = i / CHUNKS, d = (i % CHUNKS) * 4;
        if (r0 + r >= p.rows || d >= p.dim) break;
        const float4 x = *reinterpret_cast<const float4*>(so + r * S::OPITCH + d);
        const int64_t at = rows.index(p, r0 + r) * p.dim + d;
        if (p.splits == 1) store4(static_cast<T*>(p.dq) + at, x.x * p.scale, x.y * p.scale, x.z * p.scale, x.w * p.scale);
        else store4(p.part + split * p.q_count + at, x.x * p.scale, x.y * p.scale, x.z * p.scale, x.w * p.scale);
    }
}

// out[i] = sum over the splits of part[s * stride + i], in order; 4 values per thread.
template <typename T>
__global__ void __launch_bounds__(256) add_parts_kernel(const float* part, int64_t stride, int splits, int64_t count, T* out)
{
    const int64_t i = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) * 4;
    if (i >= count) return;
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int s = 0; s < splits; ++s) {
        const float4 y = *reinterpret_cast<const float4*>(part + s * stride + i);
        x.x += y.x, x.y += y.y, x.z += y.z, x.w += y.w;
    }
    store4(out + i, x.x, x.y, x.z, x.w);
}

template <typename T>
__global__ void __launch_bounds__(256) zero_kernel(T* out, T* rest, int64_t count, float2* stats, int64_t rows)
{
    const int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
    if (i * 4 < count) store4(out + i * 4, 0.f, 0.f, 0.f, 0.f);
    if (rest && i * 4 < count) store4(rest + i * 4, 0.f, 0.f, 0.f, 0.f);
    if (stats && i < rows) stats[i] = make_float2(0.f, 0.f);
}

// --- host ----------------------------------------------------------------------

constexpr int64_t kMaxGrid = std::numeric_limits<int32_t>::max();

int check_strides(const char* name, const void* ptr, const int64_t (&s)[3], size_t e)
{
    if (!ptr) return fail(POLICY_ERR_INVALID, std::string(name) + " must not be null");
    bool ok = reinterpret_cast<uintptr_t>(ptr) % 16 == 0;
    for (int64_t x : s) ok = ok && (x * static_cast<int64_t>(e)) % 16 == 0;
    if (!ok) return fail(POLICY_ERR_INVALID, std::string(name) + " must have 16-byte aligned rows");
    return POLICY_OK;
}

int check_sizes(const policy_attention* a)
{
    if (!a) return fail(POLICY_ERR_INVALID, "args must not be null");
    if (!known_dtype(a->dtype)) return fail(POLICY_ERR_INVALID, "dtype must be POLICY_F32 or POLICY_BF16");
    if (a->batch < 0 || a->lq < 0 || a->lk < 0) return fail(POLICY_ERR_INVALID, "batch, lq and lk must not be negative");
    if (a->heads < 1 || a->kv_heads < 1 || a->heads % a->kv_heads != 0)
        return fail(POLICY_ERR_INVALID, "heads must be a positive multiple of kv_heads");
    if (a->dim < 8 || a->dim > 128 || a->dim % 8 != 0) return fail(POLICY_ERR_INVALID, "dim must be a multiple of 8 from 8 to 128");
    if (!(a->scale > 0.f) || !std::isfinite(a->scale)) return fail(POLICY_ERR_INVALID, "scale must be positive and finite");
    const int64_t group = a->heads / a->kv_heads;
    // row and key indexes are 32-bit inside a (batch, key head); offsets are 64-bit
    if (a->lk > kMaxGrid - 256 || a->lq > (kMaxGrid - 256) / group)
        return fail(POLICY_ERR_INVALID, "lq * heads / kv_heads and lk must stay below 2^31 - 256");
    if (a->batch > kMaxGrid / a->kv_heads) return fail(POLICY_ERR_INVALID, "batch * kv_heads must stay below 2^31");
    return POLICY_OK;
}

int check_output(const char* name, const void* ptr)
{
    if (ptr && reinterpret_cast<uintptr_t>(ptr) % 16 == 0) return POLICY_OK;
    return fail(POLICY_ERR_INVALID, std::string(name) + " must not be null and must be 16-byte aligned");
}

int check_args(const policy_attention* a, bool backward)
{
    int rc = check_sizes(a);
    if (rc != POLICY_OK || a->batch == 0) return rc;
    const size_t e = dtype_bytes(a->dtype);
    if (a->lq > 0) {
        if ((rc = check_strides("q", a->q, a->q_strides, e)) != POLICY_OK) return rc;
        if ((rc = check_output("out", a->out)) != POLICY_OK) return rc;
        if (a->stats && (rc = check_output("stats", a->stats)) != POLICY_OK) return rc;
        if (a->out_rest && (rc = check_output("out_rest", a->out_rest)) != POLICY_OK) return rc;
    }
    if (a->lk > 0) {
        if ((rc = check_strides("k", a->k, a->k_strides, e)) != POLICY_OK) return rc;
        if ((rc = check_strides("v", a->v, a->v_strides, e)) != POLICY_OK) return rc;
    }
    if (!backward) return POLICY_OK;
    if (a->lq > 0) {
        if ((rc = check_strides("dout", a->dout, a->dout_strides, e)) != POLICY_OK) return rc;
        if ((rc = check_output("stats", a->stats)) != POLICY_OK) return rc;
        if ((rc = check_output("dq", a->dq)) != POLICY_OK) return rc;
    }
    if (a->lk > 0) {
        if ((rc = check_output("dk", a->dk)) != POLICY_OK) return rc;
        if ((rc = check_output("dv", a->dv)) != POLICY_OK) return rc;
    }
    return POLICY_OK;
}

AttnParams make_params(const policy_attention& a)
{
    AttnParams p{};
    p.q = a.q, p.k = a.k, p.v = a.v, p.dout = a.dout;
    for (int i = 0; i < 3; ++i) p.qs[i] = a.q_strides[i], p.ks[i] = a.k_strides[i], p.vs[i] = a.v_strides[i], p.ds[i] = a.dout_strides[i];
    p.mask = a.key_mask, p.mask_stride = a.key_mask_stride, p.lengths = a.key_lengths;
    p.out = a.out, p.rest = a.dtype == POLICY_BF16 ? a.out_rest : nullptr, p.stats = reinterpret_cast<float2*>(a.stats), p.dq = a.dq, p.dk = a.dk, p.dv = a.dv;
    p.q_count = a.batch * a.lq * a.heads * a.dim;
    p.k_count = a.batch * a.lk * a.kv_heads * a.dim;
    p.lq = static_cast<int>(a.lq), p.lk = static_cast<int>(a.lk);
    p.heads = a.heads, p.kv_heads = a.kv_heads, p.group = a.heads / a.kv_heads, p.dim = a.dim;
    p.rows = static_cast<int>(a.lq) * p.group;
    p.splits = 1;
    p.scale = a.scale;
    p.scale_log2 = a.scale * 1.4426950408889634f;
    return p;
}

// How a call is laid out: tiles, splits and workspace, from the sizes alone.
struct Plan {
    int dp = 0;              // padded head dimension: 32, 64 or 128
    bool tc = false;         // forward on tcgen05
    int fwd_rows = 0;        // rows of a forward tile: 16, 32 or 64, or 256 with tcgen05
    int fwd_keys = 0;
    int fwd_splits = 1;
    bool few = false;        // gradients in one kernel
    bool grad_tc = false;    // gradients on tcgen05
    int grad_warps = 0;
    int few_splits = 1, key_splits = 1, query_splits = 1;
    size_t fwd_bytes = 0, grad_bytes = 0;
};

int ceil_div(int64_t a, int64_t b) { return static_cast<int>((a + b - 1) / b); }
size_t align256(size_t n) { return (n + 255) & ~static_cast<size_t>(255); }

// How many parts a long axis of `tiles` tiles is split into when there are `blocks` blocks: as many as keep one
// full set of resident blocks, none shorter than `least` tiles (a shorter one costs more in parts than it gives).
int choose_splits(int64_t blocks, int tiles, int64_t resident, int least)
{
    const int64_t want = resident / (blocks > 0 ? blocks : 1);
    const int64_t most = tiles / least;
    const int64_t n = want < most ? want : most;
    return static_cast<int>(n > 1 ? n : 1);
}

// Blocks of `bytes` of shared memory that are resident on the device, at most `most` an SM (their registers).
int64_t resident_blocks(size_t bytes, int most, int sms)
{
    const int n = static_cast<int>((228 * 1024) / (bytes + 1024));
    return static_cast<int64_t>(sms) * (n < 1 ? 1 : n < most ? n : most);
}

size_t fwd_bytes(bool f32, int dp, int rows, int keys)
{
    const size_t pitch = f32 ? 4 * (dp + 4) : 2 * (dp + 8);
    return pitch * (rows + 4 * keys);
}

// Above this many rows bf16 runs on tcgen05.  Forward, 64 x 48 rows x 700 keys x 64: 42 us here, 60 us there; 64 rows x
// 2,000 keys: 99 and 124 us; 256 tokens of 2 shared heads and more: half the time there.  Gradients, 64 x 64 rows x 2,000
// keys: 374 and 363 us; 256 x 20 rows x 700 keys: 407 and 498 us.  Not measured below 700 keys, nor between 65 and 255
// rows, where tcgen05's tiles of 128 keys and 256 rows are more or less padding.
constexpr int kTcMinRows = 64;

Plan make_plan(const policy_attention& a, int sms)
{
    Plan pl;
    const bool f32 = a.dtype == POLICY_F32;
    const int64_t rows = a.lq * (a.heads / a.kv_heads);
    const int64_t bh = a.batch * a.kv_heads;
    pl.dp = a.dim <= 32 ? 32 : a.dim <= 64 ? 64 : 128;
    pl.fwd_rows = rows <= 16 ? 16 : rows <= 32 ? 32 : 64;
    if (f32) pl.fwd_keys = pl.dp == 128 ? 32 : 64;
    else pl.fwd_keys = 64;
    pl.tc = !f32 && rows > kTcMinRows && attend_tc_takes(make_params(a));
    if (pl.tc) pl.fwd_rows = kTcRows, pl.fwd_keys = kTcKeys;
    pl.grad_warps = f32 && pl.dp == 128 ? 2 : 4;
    const int64_t q_count = a.batch * a.lq * a.heads * a.dim, k_count = a.batch * a.lk * a.kv_heads * a.dim;
    if (bh == 0) return pl;
    const int64_t fwd_resident = pl.tc ? sms : resident_blocks(fwd_bytes(f32, pl.dp, pl.fwd_rows, pl.fwd_keys), 5, sms);
    pl.fwd_splits = choose_splits(bh * ceil_div(rows, pl.fwd_rows), ceil_div(a.lk, pl.fwd_keys), fwd_resident, pl.tc ? 2 : 4);
    if (pl.fwd_splits > 1)
        pl.fwd_bytes = align256(sizeof(float) * pl.fwd_splits * q_count) + align256(sizeof(float) * 2 * pl.fwd_splits * (q_count / a.dim));
    pl.few = rows <= 16;
    const int kt = pl.grad_warps * 16;
    if (pl.few) {
        pl.few_splits = choose_splits(bh, ceil_div(a.lk, kt), resident_blocks(fwd_bytes(f32, pl.dp, 32, kt), 4, sms), 4);
        if (pl.few_splits > 1) pl.grad_bytes = align256(sizeof(float) * pl.few_splits * q_count);
    } else {
        pl.grad_bytes = align256(sizeof(float) * (q_count / a.dim));
        pl.grad_tc = !f32 && rows > kTcMinRows && attend_grad_tc_takes(make_params(a));
        if (pl.grad_tc) {
            // items differ in length where lengths do: two for each SM
            pl.key_splits = choose_splits(bh * ceil_div(a.lk, grad_tc_tile(true, a.dim)), ceil_div(rows, kGradTcStream), 2 * sms, 4);
            pl.query_splits = choose_splits(bh * ceil_div(rows, grad_tc_tile(false, a.dim)), ceil_div(a.lk, kGradTcStream), sms, 4);
        } else {
            pl.key_splits = choose_splits(bh * ceil_div(a.lk, kt), ceil_div(rows, 32), 4 * sms, 2);
            pl.query_splits = choose_splits(bh * ceil_div(rows, kt), ceil_div(a.lk, 32), 4 * sms, 4);
        }
        if (pl.key_splits > 1) pl.grad_bytes += align256(sizeof(float) * 2 * pl.key_splits * k_count);
        if (pl.query_splits > 1) pl.grad_bytes += align256(sizeof(float) * pl.query_splits * q_count);
    }
    return pl;
}

int launch_blocks(int64_t n, const char* what, unsigned& grid)
{
    if (n > kMaxGrid) return fail(POLICY_ERR_INVALID, std::string(what) + ": the launch would need over 2^31 - 1 blocks");
    grid = static_cast<unsigned>(n);
    return POLICY_OK;
}

// A kernel's shared-memory allowance is set once per device.
template <typename K>
int allow_shared(K kernel, size_t bytes, int device, std::atomic<uint64_t>& done)
{
    if (bytes <= 48 * 1024) return POLICY_OK;
    const uint64_t bit = device < 64 ? 1ull << device : 0ull;
    if (bit && (done.load(std::memory_order_relaxed) & bit)) return POLICY_OK;
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes));
    if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute");
    done.fetch_or(bit, std::memory_order_relaxed);
    return POLICY_OK;
}

int launched(const char* what)
{
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? POLICY_OK : cuda_fail(e, what);
}

template <typename T, int DP, int WM, int WN, int KT, bool TWO>
int launch_fwd_tile(AttnParams p, int64_t bh, int device, cudaStream_t stream)
{
    using S = FwdShape<T, DP, WM, WN, KT>;
    static std::atomic<uint64_t> done{0};
    int rc = allow_shared(attend_kernel<T, DP, WM, WN, KT, TWO>, S::bytes(S::STAGES), device, done);
    if (rc != POLICY_OK) return rc;
    unsigned grid = 0;
    if ((rc = launch_blocks(bh * p.tiles * p.splits, "policy_cross_attention", grid)) != POLICY_OK) return rc;
    p.stages = p.lk <= KT ? 1 : S::STAGES;
    attend_kernel<T, DP, WM, WN, KT, TWO><<<grid, S::THREADS, S::bytes(p.stages), stream>>>(p);
    return launched("attend_kernel");
}

// Up to 16 and up to 32 keys have tiles of their own, with all warps along the rows: a tile of 64 computes and joins
// keys that are not there, and its shared memory keeps blocks away.  1,024 x 8 heads of 16 rows of 64, in bf16 with 16
// keys 50 us with the larger tile and 25 here, with 24 keys 52 and 31; in f32 92 and 43, 105 and 62; 32 rows and 32 keys
// of 64 in bf16 75 and 54, in f32 144 and 97; 8,132 x 4 rows and 3 keys of 64 in f32 18.8 and 16.5.  f32 tiles of dim 128
// hold 32 keys as they are.
template <typename T, int DP, int WM, int WN, int KT>
int launch_fwd(const AttnParams& p, int64_t bh, int device, cudaStream_t stream)
{
    constexpr bool kTwo = sizeof(T) == 2;
    constexpr int kLeast = WM * 32 / (DP / Mma<T>::VEC) > 16 ? 32 : 16;  // a thread loads a key at least
    if (p.lk <= 16) return launch_fwd_tile<T, DP, WM, 1, kLeast, kTwo>(p, bh, device, stream);
    if constexpr (KT > kFewKeysFwd)
        if (p.lk <= kFewKeysFwd) return launch_fwd_tile<T, DP, WM, 1, kFewKeysFwd, kTwo>(p, bh, device, stream);
    return launch_fwd_tile<T, DP, WM, WN, KT, false>(p, bh, device, stream);
}

template <typename T, int DP>
int launch_fwd_rows(const AttnParams& p, const Plan& pl, int64_t bh, int device, cudaStream_t stream)
{
    constexpr bool f32 = sizeof(T) == 4;
    if constexpr (f32 && DP == 128) {
        if (pl.fwd_rows == 16) return launch_fwd<T, DP, 1, 2, 32>(p, bh, device, stream);
        if (pl.fwd_rows == 32) return launch_fwd<T, DP, 2, 1, 32>(p, bh, device, stream);
        return launch_fwd<T, DP, 4, 1, 32>(p, bh, device, stream);
    } else {
        constexpr int KN = 64;
        if (pl.fwd_rows == 16) return launch_fwd<T, DP, 1, 4, KN>(p, bh, device, stream);
        if (pl.fwd_rows == 32) return launch_fwd<T, DP, 2, 2, KN>(p, bh, device, stream);
        return launch_fwd<T, DP, 4, 1, 64>(p, bh, device, stream);
    }
}

int set_stall_word(AttnParams& p)
{
    p.stalled = stall_word();
    return p.stalled ? POLICY_OK : fail(POLICY_ERR_CUDA, "cudaHostAlloc failed");
}

template <typename T>
int run_forward(const policy_attention& a, const Plan& pl, int sms, cudaStream_t stream)
{
    AttnParams p = make_params(a);
    const int64_t bh = a.batch * a.kv_heads;
    p.tiles = ceil_div(p.rows, pl.fwd_rows);
    p.splits = pl.fwd_splits;
    if (p.splits > 1) {
        p.part = static_cast<float*>(a.workspace);
        p.part_ml = reinterpret_cast<float*>(static_cast<char*>(a.workspace) + align256(sizeof(float) * p.splits * p.q_count));
    }
    int rc = pl.tc ? set_stall_word(p) : POLICY_OK;
    if (rc != POLICY_OK) return rc;
    rc = pl.tc         ? launch_attend_tc(p, bh, sms, a.device, stream)
             : pl.dp == 32 ? launch_fwd_rows<T, 32>(p, pl, bh, a.device, stream)
             : pl.dp == 64 ? launch_fwd_rows<T, 64>(p, pl, bh, a.device, stream)
                           : launch_fwd_rows<T, 128>(p, pl, bh, a.device, stream);
    if (rc != POLICY_OK || p.splits == 1) return rc;
    unsigned grid = 0;
    if ((rc = launch_blocks(p.q_count / p.dim, "policy_cross_attention", grid)) != POLICY_OK) return rc;
    int lanes = 2;
    while (lanes * 4 < p.dim) lanes *= 2;
    attend_join_kernel<T><<<grid, kJoinThreads, 0, stream>>>(p, lanes);
    return launched("attend_join_kernel");
}

template <typename T, typename K>
int launch_grad(K kernel, size_t bytes, std::atomic<uint64_t>& done, const AttnParams& p, int64_t blocks, int threads, int device,
                cudaStream_t stream, const char* what)
{
    int rc = allow_shared(kernel, bytes, device, done);
    if (rc != POLICY_OK) return rc;
    unsigned grid = 0;
    if ((rc = launch_blocks(blocks, what, grid)) != POLICY_OK) return rc;
    kernel<<<grid, threads, bytes, stream>>>(p);
    return launched(what);
}

template <typename T>
int add_parts(const float* part, int64_t stride, int splits, int64_t count, void* out, cudaStream_t stream)
{
    unsigned grid = 0;
    const int rc = launch_blocks((count / 4 + 255) / 256, "policy_cross_attention_backward", grid);
    if (rc != POLICY_OK) return rc;
    add_parts_kernel<T><<<grid, 256, 0, stream>>>(part, stride, splits, count, static_cast<T*>(out));
    return launched("add_parts_kernel");
}

template <typename T, int DP, int NW>
int run_backward_dim(const policy_attention& a, const Plan& pl, int sms, cudaStream_t stream)
{
    using S = GradShape<T, DP, NW>;
    static std::atomic<uint64_t> done_few{0}, done_two{0}, done_keys{0}, done_queries{0};
    AttnParams p = make_params(a);
    const int64_t bh = a.batch * a.kv_heads;
    int rc = POLICY_OK;
    if (pl.few) {
        p.splits = pl.few_splits;
        p.part = static_cast<float*>(a.workspace);
        constexpr bool kTwo = sizeof(T) == 2;
        if (kTwo && p.lk <= kTwoKeys)
            rc = launch_grad<T>(attend_grad_few_kernel<T, DP, NW, kTwo>, S::few_bytes(kTwo), done_two, p, bh * p.splits, S::THREADS, a.device,
                                stream, "attend_grad_few_kernel");
        else
            rc = launch_grad<T>(attend_grad_few_kernel<T, DP, NW, false>, S::few_bytes(false), done_few, p, bh * p.splits, S::THREADS, a.device,
                                stream, "attend_grad_few_kernel");
        if (rc == POLICY_OK && p.splits > 1) rc = add_parts<T>(p.part, p.q_count, p.splits, p.q_count, p.dq, stream);
        return rc;
    }
    char* ws = static_cast<char*>(a.workspace);
    float* delta = reinterpret_cast<float*>(ws);
    ws += align256(sizeof(float) * (p.q_count / p.dim));
    unsigned grid = 0;
    if ((rc = launch_blocks((p.q_count / p.dim + 31) / 32, "attend_delta_kernel", grid)) != POLICY_OK) return rc;
    attend_delta_kernel<T><<<grid, 256, 0, stream>>>(p, delta);
    if ((rc = launched("attend_delta_kernel")) != POLICY_OK) return rc;
    p.delta = delta;
    if (pl.grad_tc && (rc = set_stall_word(p)) != POLICY_OK) return rc;

    p.splits = pl.key_splits;
    p.tiles = ceil_div(p.lk, pl.grad_tc ? grad_tc_tile(true, p.dim) : S::KT);
    p.part = reinterpret_cast<float*>(ws);
    if (pl.grad_tc) rc = launch_attend_grad_tc(p, true, bh, sms, a.device, stream);
    else rc = launch_grad<T>(attend_grad_keys_kernel<T, DP, NW>, S::kKeyGrad, done_keys, p, bh * p.tiles * p.splits, S::THREADS, a.device,
                        stream, "attend_grad_keys_kernel");
    if (rc != POLICY_OK) return rc;
    if (p.splits > 1) {
        if ((rc = add_parts<T>(p.part, 2 * p.k_count, p.splits, p.k_count, p.dk, stream)) != POLICY_OK) return rc;
        if ((rc = add_parts<T>(p.part + p.k_count, 2 * p.k_count, p.splits, p.k_count, p.dv, stream)) != POLICY_OK) return rc;
        ws += align256(sizeof(float) * 2 * p.splits * p.k_count);
    }
    p.splits = pl.query_splits;
    p.tiles = ceil_div(p.rows, pl.grad_tc ? grad_tc_tile(false, p.dim) : NW * 16);
    p.part = reinterpret_cast<float*>(ws);
    if (pl.grad_tc) rc = launch_attend_grad_tc(p, false, bh, sms, a.device, stream);
    else rc = launch_grad<T>(attend_grad_queries_kernel<T, DP, NW>, S::kQueryGrad, done_queries, p, bh * p.tiles * p.splits, S::THREADS,
                        a.device, stream, "attend_grad_queries_kernel");
    if (rc == POLICY_OK && p.splits > 1) rc = add_parts<T>(p.part, p.q_count, p.splits, p.q_count, p.dq, stream);
    return rc;
}

template <typename T>
int zero(void* out, void* rest, int64_t count, float* stats, int64_t rows, cudaStream_t stream)
{
    const int64_t n = count / 4 > rows ? count / 4 : rows;
    if (n == 0) return POLICY_OK;
    unsigned grid = 0;
    const int rc = launch_blocks((n + 255) / 256, "policy_cross_attention", grid);
    if (rc != POLICY_OK) return rc;
    zero_kernel<T><<<grid, 256, 0, stream>>>(static_cast<T*>(out), static_cast<T*>(rest), count, reinterpret_cast<float2*>(stats), rows);
    return launched("zero_kernel");
}

template <typename T>
int forward(const policy_attention& a, int sms, cudaStream_t stream)
{
    const int64_t rows = a.batch * a.lq * a.heads;
    if (rows == 0) return POLICY_OK;
    if (a.lk == 0) return zero<T>(a.out, a.out_rest, rows * a.dim, a.stats, rows, stream);
    const Plan pl = make_plan(a, sms);
    if (pl.fwd_bytes && !a.workspace) return fail(POLICY_ERR_INVALID, "workspace must not be null");
    return run_forward<T>(a, pl, sms, stream);
}

template <typename T>
int backward(const policy_attention& a, int sms, cudaStream_t stream)
{
    if (a.batch == 0) return POLICY_OK;
    const int64_t k_count = a.batch * a.lk * a.kv_heads * a.dim;
    if (a.lq == 0) {
        const int rc = zero<T>(a.dk, nullptr, k_count, nullptr, 0, stream);
        return rc != POLICY_OK ? rc : zero<T>(a.dv, nullptr, k_count, nullptr, 0, stream);
    }
    if (a.lk == 0) return zero<T>(a.dq, nullptr, a.batch * a.lq * a.heads * a.dim, nullptr, 0, stream);
    const Plan pl = make_plan(a, sms);
    if (pl.grad_bytes && !a.workspace) return fail(POLICY_ERR_INVALID, "workspace must not be null");
    if (pl.dp == 32) return run_backward_dim<T, 32, 4>(a, pl, sms, stream);
    if (pl.dp == 64) return run_backward_dim<T, 64, 4>(a, pl, sms, stream);
    return run_backward_dim<T, 128, sizeof(T) == 4 ? 2 : 4>(a, pl, sms, stream);
}

template <typename F>
int entry(const policy_attention* a, bool is_backward, F&& run)
{
    const int rc = check_args(a, is_backward);
    if (rc != POLICY_OK) return rc;
    const DeviceInfo info = device_info(a->device);
    if (info.status != POLICY_OK) return info.status;
    const int stalled = check_stall();
    if (stalled != POLICY_OK) return stalled;
    DeviceScope scope(a->device);
    if (scope.error() != cudaSuccess) return cuda_fail(scope.error(), "cudaSetDevice");
    return run(info.sms);
}

}  // namespace
}  // namespace policy

using namespace policy;

extern "C" uint64_t policy_cross_attention_workspace_bytes(const policy_attention* a, int backward)
try {
    if (check_sizes(a) != POLICY_OK) return 0;
    const DeviceInfo info = device_info(a->device);
    if (info.status != POLICY_OK) return 0;
    if (a->lq == 0 || a->lk == 0) return 0;
    const Plan pl = make_plan(*a, info.sms);
    return backward ? pl.grad_bytes : pl.fwd_bytes;
} catch (...) {
    return 0;
}

extern "C" int policy_cross_attention(const policy_attention* a, void* stream)
try {
    return entry(a, false, [&](int sms) {
        auto st = static_cast<cudaStream_t>(stream);
        return a->dtype == POLICY_F32 ? forward<float>(*a, sms, st) : forward<bf16>(*a, sms, st);
    });
} catch (...) {
    return POLICY_ERR_INVALID;
}

extern "C" int policy_cross_attention_backward(const policy_attention* a, void* stream)
try {
    return entry(a, true, [&](int sms) {
        auto st = static_cast<cudaStream_t>(stream);
        return a->dtype == POLICY_F32 ? backward<float>(*a, sms, st) : backward<bf16>(*a, sms, st);
    });
} catch (...) {
    return POLICY_ERR_INVALID;
}
