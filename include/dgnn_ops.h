/*
 * dgnn_ops.h -- C ABI of libdgnn_ops.so: operators on DEVICE tensors for predictors that are not the reference's own network.
 *
 * The leaf pool and the search take any predictor (dgnn_predict_fn, dgnn_host.h).  The engine behind dgnn.h evaluates one family of
 * networks -- 3x3 convolutions with folded batch norm, two heads -- as fused kernels; a predictor of another shape is put together from
 * the operators here:
 *
 *   dgnn_dense           y = act(alpha1 * x W^T + alpha2 * z + bias): the reference's dense layer (src/libdg_nn/layers/dense.rs:197-220)
 *                        and the epilogue of its convolutions (layers/conv2d.rs:171-220) at any size, in fp16 or bf16
 *   dgnn_group_norm      group norm over channels-last maps with an activation and a skip input, where folded batch norm does not apply
 *   dgnn_adjust_logits   penalties for repeated tokens, biases and masks on logits, before a soft-max or a sampler; what the reference does
 *                        to a policy after the boundary (src/libdg_mcts/pool/policy_helper.rs:87-134) with a bit mask of legal moves
 *
 * Conventions
 *   - those of dgnn.h: plain C types, a status code from every call (DGNN_OK ... of dgnn.h, texts: dgnn_status_string of
 *     libdgnn_hip.so), nothing aborts, no process-global current device: `device` is an argument and the caller's current device is
 *     left as it was;
 *   - data pointers are device memory of `device`, the caller's; strides count elements and are >= 0; the innermost stride is 1.  Rows that
 *     are only read may repeat (stride 0) or overlap, rows that are written may not.  Pointers are aligned to their element, no more is needed;
 *   - a call enqueues its kernels on `hip_stream` (a hipStream_t of `device`, NULL = its default stream) and returns; it allocates
 *     nothing, waits for nothing and may be captured into a graph.  Work memory, where an operator needs any, is the caller's and is
 *     the call's alone until its kernels have run;
 *   - arguments are checked before anything is enqueued: DGNN_BAD_ARGUMENT / DGNN_UNSUPPORTED leave the outputs untouched;
 *   - forward only: the engine evaluates networks, it does not train them;
 *   - any number of threads may call at once.
 */
#ifndef DGNN_OPS_H
#define DGNN_OPS_H

#include "dgnn.h"

#ifdef __cplusplus
extern "C" {
#endif

/* element types */
#define DGNN_F16   0
#define DGNN_BF16  1
#define DGNN_F32   2
#define DGNN_I32   3
#define DGNN_I64   4

/* activations; gelu is the exact one, v * Phi(v) */
#define DGNN_ACT_IDENTITY  0
#define DGNN_ACT_RELU      1   /* v < 0 ? 0 : v (a NaN stays) */
#define DGNN_ACT_TANH      2
#define DGNN_ACT_GELU      3
#define DGNN_ACT_SILU      4   /* v / (1 + exp(-v)) */

/* The hipError_t of the most recent DGNN_HIP_ERROR of this library on the calling thread (0 if none). */
int dgnn_ops_last_hip_error(void);

/* ---- y[m][n] = act(alpha1 * sum_k x[m][k] * w[n][k] + alpha2 * z[m][n] + bias[n]) -------------------------------------------------- */
typedef struct dgnn_dense_args {
    const void* x;          /* [m][k], row stride ldx */
    const void* w;          /* [n][k], row stride ldw: one row per output, as dense.rs:182-189 transposes its matrix */
    const void* bias;       /* [n] or NULL */
    const void* z;          /* [m][n] of out_type, row stride ldz (0: one row for all), or NULL; may be y itself */
    void* y;                /* [m][n] of out_type, row stride ldy; overlaps neither x nor w */
    void* workspace;        /* dgnn_dense_workspace bytes, 256-byte aligned, apart from every operand; NULL where that is 0 */
    int64_t workspace_bytes;
    int64_t m, n, k;        /* 0 <= each < 2^31; k == 0: the sum is 0 */
    int64_t ldx, ldw, ldz, ldy;
    float alpha1, alpha2;   /* alpha2 counts only with z */
    int32_t type;           /* of x and w: DGNN_F16 or DGNN_BF16; products are summed in fp32 */
    int32_t out_type;       /* of y and z: `type`, or DGNN_F32.  One rounding, at the end */
    int32_t bias_type;      /* `type` or DGNN_F32 */
    int32_t activation;
} dgnn_dense_args;
/* What the call with these arguments needs (pointers and strides as they will be; workspace and workspace_bytes are not read): room for the
 * sums of several shares of k where there are few outputs, and for copies of x and w where their rows are not 16-byte aligned. */
int dgnn_dense_workspace(const dgnn_dense_args* args, int64_t* bytes);
int dgnn_dense(int device, void* hip_stream, const dgnn_dense_args* args);

/* ---- group norm, channels last -----------------------------------------------------------------------------------------------------
 * Sample i, group g: mean and (biased) variance over p positions x c / groups channels, in fp32; then
 *   y[i][q][j] = act((x[i][q][j] - mean) / sqrt(variance + eps) * weight[j] + bias[j] + z[i][q][j]),
 * weight 1, bias 0 and z 0 where the pointer is NULL.  One rounding, at the end.  y may be x or z with the same strides. */
typedef struct dgnn_group_norm_args {
    const void* x;          /* [n][p][c], strides x_n, x_p */
    const void* weight;     /* [c] of affine_type, or NULL */
    const void* bias;       /* [c] of affine_type, or NULL */
    const void* z;          /* [n][p][c] of `type`, strides z_n, z_p (0: repeated), or NULL */
    void* y;                /* [n][p][c] of `type`, strides y_n, y_p */
    void* workspace;        /* dgnn_group_norm_workspace bytes, 256-byte aligned, apart from every operand; NULL where that is 0 */
    int64_t workspace_bytes;
    int64_t n, p, c, groups;
    int64_t x_n, x_p, z_n, z_p, y_n, y_p;
    float eps;              /* >= 0 */
    int32_t type;           /* of x, z, y: DGNN_F16, DGNN_BF16 or DGNN_F32 */
    int32_t affine_type;    /* `type` or DGNN_F32 */
    int32_t activation;
} dgnn_group_norm_args;
/* What the call with these arguments needs (pointers and strides as they will be; workspace and workspace_bytes are not read). */
int dgnn_group_norm_workspace(const dgnn_group_norm_args* args, int64_t* bytes);
int dgnn_group_norm(int device, void* hip_stream, const dgnn_group_norm_args* args);

/* ---- logits: penalties, biases, masks ------------------------------------------------------------------------------------------------
 * Row i has a history of tokens, its first `lengths[i]` entries (none without `history`), of which the first `prompt_lengths[i]` were
 * given and the others are the answer so far.  seen = v occurs in it; count = how often v occurs in the answer part.  In fp32:
 *   l = logits[i][v]
 *   seen:  l = l > 0 ? l / repetition : l * repetition
 *   l = l - frequency * count - (count > 0 ? presence : 0)
 *   l = l + bias[v]
 *   mask bit clear: l = -infinity, whatever it was
 * and one rounding to the output's type.  A row whose mask leaves nothing is -infinity throughout.  Tokens outside 0 .. v-1 (padding)
 * count for nothing; lengths are taken as clamped to 0 .. t, prompt lengths to 0 .. length. */
typedef struct dgnn_logits_args {
    const void* logits;             /* [b][v], row stride ld_logits */
    void* out;                      /* [b][v], row stride ld_out; may be logits itself (same type and stride) */
    const uint32_t* mask;           /* [b][(v + 31) / 32], row stride ld_mask (0: one for all), or NULL.  Bit v % 32 of word v / 32 set: v is allowed */
    const void* bias;               /* [b][v], row stride ld_bias (0: one for all), or NULL */
    const void* history;            /* [b][t] of history_type, row stride ld_history, or NULL */
    const int32_t* lengths;         /* [b] or NULL: t */
    const int32_t* prompt_lengths;  /* [b] or NULL: 0 */
    const float* repetition;        /* [b] or NULL: repetition_all in every row; > 0 */
    const float* presence;          /* [b] or NULL: presence_all */
    const float* frequency;         /* [b] or NULL: frequency_all */
    int64_t b, v, t;
    int64_t ld_logits, ld_out, ld_mask, ld_bias, ld_history;
    float repetition_all, presence_all, frequency_all;
    int32_t type;                   /* of logits: DGNN_F16, DGNN_BF16 or DGNN_F32 */
    int32_t out_type;               /* `type` or DGNN_F32 */
    int32_t bias_type;              /* `type` or DGNN_F32 */
    int32_t history_type;           /* DGNN_I32 or DGNN_I64 */
} dgnn_logits_args;
int dgnn_adjust_logits(int device, void* hip_stream, const dgnn_logits_args* args);

#ifdef __cplusplus
}
#endif

#endif /* DGNN_OPS_H */
