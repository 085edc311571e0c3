/*
 * policy.h — C ABI of the operators of a policy that reads ray fans.
 *
 * Library: navi_b200/_lib/libnavi_policy.so (sm_100a).  The conventions are those of
 * tsdf.h: every function returns POLICY_OK (0) or a negative policy_status, with the
 * text of the calling thread's last error in policy_last_error(); device pointers are
 * plain CUDA device addresses; `stream` is a cudaStream_t; calls are asynchronous on it,
 * never synchronise the host, allocate no device memory and leave the caller's current
 * device as it was.  Scratch is the caller's: `workspace`, 256-byte aligned, of the size
 * that the matching *_workspace_bytes function gives.  Strides are in elements.
 *
 * No entry point has a counterpart in the reference, whose policy is eager PyTorch
 * (projects/actor/src/navi_actor).
 */
#ifndef NAVI_B200_POLICY_H
#define NAVI_B200_POLICY_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define POLICY_ABI_VERSION 1

#if defined(__GNUC__)
#define POLICY_API __attribute__((visibility("default")))
#else
#define POLICY_API
#endif

typedef enum policy_status {
    POLICY_OK = 0,
    POLICY_ERR_INVALID = -1,     /* bad argument (null pointer, size, alignment, range) */
    POLICY_ERR_CUDA = -3,        /* a CUDA runtime call failed */
    POLICY_ERR_UNSUPPORTED = -5, /* device is not sm_100 */
    POLICY_ERR_STALLED = -6      /* a wait inside an earlier attention kernel ran out: its rows are NaN */
} policy_status;

typedef enum policy_dtype {
    POLICY_F32 = 0,
    POLICY_BF16 = 1
} policy_dtype;

POLICY_API int policy_version(void);
POLICY_API const char* policy_last_error(void);

/* --- cross attention -------------------------------------------------------
 * q [batch][lq][heads][dim] attends to k, v [batch][lk][kv_heads][dim]; query head h
 * reads key head h / (heads / kv_heads).  Key j of batch b is visible when
 * j < key_lengths[b] (null: all; values outside 0..lk are clamped) and
 * key_mask[b * key_mask_stride + j] != 0 (null: all).  What k and v hold at keys that are
 * not visible does not reach any output (NaN and infinities included), and their
 * gradients are 0.
 *   s_ij = scale * q_i . k_j        p_ij = exp(s_ij) / sum_j exp(s_ij)        out_i = sum_j p_ij v_j
 * A query whose largest score is -inf (no visible key among others) gives 0 and receives
 * gradient 0.  Scores, statistics and sums are held in 32 bits.
 *
 * dim is a multiple of 8, 8 to 128.  q, k, v and dout have element stride 1 along dim,
 * 16-byte aligned rows (base address, and strides times the element size).  out, dq, dk
 * and dv are contiguous; For the backward pass the
 * forward writes, where the pointers are not null, stats [batch][lq][heads][2] f32 (the exponent that its
 * weights are relative to, in base 2, and the reciprocal of the sum of the weights as they multiply v, 0 for a
 * query that gives 0: a single logarithm of the sum would carry its own rounding into every weight), and with POLICY_BF16 out_rest, bf16 in
 * the layout of out: what the rounding of out left off (dout . out in 8 bits would be the largest error of dq
 * and dk where a query sees few keys; null in the backward: taken as 0). */
typedef struct policy_attention {
    int32_t device;
    int32_t dtype;
    int64_t batch, lq, lk;
    int32_t heads, kv_heads, dim;
    float scale;
    const void* q;
    const void* k;
    const void* v;
    int64_t q_strides[3]; /* batch, token, head */
    int64_t k_strides[3];
    int64_t v_strides[3];
    const uint8_t* key_mask;
    int64_t key_mask_stride;
    const int32_t* key_lengths;
    void* out;
    float* stats;
    void* out_rest;
    /* backward only */
    const void* dout;
    int64_t dout_strides[3];
    void* dq;
    void* dk;
    void* dv;
    void* workspace;
} policy_attention;

/* A wait inside a kernel is bounded.  One that runs out, which only a defect could cause, leaves NaN in
 * the rows that it belongs to and sets this word, in pinned host memory that every device sees, to 1.  The next
 * call of policy_cross_attention or policy_cross_attention_backward clears it and returns
 * POLICY_ERR_STALLED; a caller that has synchronised with its last call may read it.  Null without a
 * CUDA device. */
POLICY_API volatile int32_t* policy_stall_word(void);

POLICY_API uint64_t policy_cross_attention_workspace_bytes(const policy_attention* args, int backward);
POLICY_API int policy_cross_attention(const policy_attention* args, void* stream);
POLICY_API int policy_cross_attention_backward(const policy_attention* args, void* stream);

/* --- norms of queries and keys with rotation --------------------------------
 * For every row x [dim] of q and k (index 0 and 1 below; each may have 0 tokens):
 *   u = weight * x / sqrt(mean(x^2) + eps),
 * then the first `rotary` values of u are turned: with n = rotary / 2 and the cosines c
 * and sines s of the row's table entry,
 *   y_i = u_i c_i - u_{i+n} s_i,  y_{i+n} = u_{i+n} c_i + u_i s_i  (i < n), the rest as is.
 * table [table_rows][2][n] f32 (cosines, then sines); a row's entry is its token index,
 * or positions[b * tokens + token] when positions is not null.  A position outside the
 * table gives a row of NaN, forward and backward.  weight [dim] f32, null for ones.
 *
 * dim is a multiple of 8, 8 to 256; rotary a multiple of 16 (0: no rotation), at most dim.
 * x and dy have element stride 1 along dim and 16-byte aligned rows; y and dx are
 * contiguous.  Backward reads x and dy, writes dx and, when not null, dweight [dim] f32
 * (the sum over all rows, in an order that depends on the sizes alone). */
typedef struct policy_norm_side {
    const void* x;        /* [batch][tokens][heads][dim] */
    int64_t strides[3];   /* batch, token, head */
    int64_t tokens;
    int32_t heads;
    int32_t reserved;
    const float* weight;
    const float* table;
    int64_t table_rows;
    const int32_t* positions;
    void* y;              /* forward */
    const void* dy;       /* backward */
    int64_t dy_strides[3];
    void* dx;
    float* dweight;
} policy_norm_side;

typedef struct policy_qk_norm {
    int32_t device;
    int32_t dtype;
    int64_t batch;
    int32_t dim;
    int32_t rotary;
    float eps;
    int32_t reserved;
    policy_norm_side side[2];
    void* workspace;      /* backward with dweight */
} policy_qk_norm;

POLICY_API uint64_t policy_qk_norm_workspace_bytes(const policy_qk_norm* args);
POLICY_API int policy_qk_norm_rotary(const policy_qk_norm* args, void* stream);
POLICY_API int policy_qk_norm_rotary_backward(const policy_qk_norm* args, void* stream);

/* --- global gradient norm and clipping --------------------------------------
 *   norm = sqrt(sum of squares of all values),  c = min(1, max_norm / (norm + 1e-6)),
 *   out = c * grad  (out may be grad itself).
 * The norm is summed in 32 bits per thread and 64 bits across threads, in an order that
 * depends on the sizes and alignments alone.  A norm that is not finite scales by what
 * the formula gives (an infinite norm by 0, NaN by NaN).  norm receives one f32.  No two
 * outputs overlap, and an output overlaps no gradient but its own, which is then at the
 * same address: POLICY_ERR_INVALID otherwise. */
typedef struct policy_grad {
    const void* grad;
    void* out;
    uint64_t count;
    int32_t dtype;
    int32_t reserved;
} policy_grad;

POLICY_API uint64_t policy_clip_grad_workspace_bytes(const policy_grad* grads, int64_t n);
POLICY_API int policy_clip_grad_norm(const policy_grad* grads, int64_t n, float max_norm, float* norm, int device,
                                     void* workspace, void* stream);

#ifdef __cplusplus
}
#endif

#endif
