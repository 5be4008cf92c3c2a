/*
 * luminav_ops.h -- C ABI of the operators around the LuminaV step (libluminav_ops.so): layer norm,
 * log probabilities of given tokens, and distillation from a teacher's top logits, forward and
 * backward.
 *
 * Plain pointers and sizes only. Every pointer is a device (HBM) pointer on the current HIP device;
 * `stream` is a hipStream_t passed as void* (NULL = default stream). Calls are asynchronous on
 * `stream`, allocate nothing and wait for nothing, so they can be captured into a HIP graph.
 * Sums and statistics are f32 whatever the tensors' type. A call repeated on the same memory gives the
 * same bits: no result depends on the order of atomics or on timing. Layer norm's rows give the same
 * bits anywhere and in any number; its columns' sums depend on the number of rows. Over rows of logits
 * the most likely tokens and the largest logit are the same everywhere, but the last bits of what is
 * summed over a row depend on the number of rows, which decides how a row is cut, and for 16-bit logits
 * on the half of a 4-byte word that the row begins at: equal rows of an odd vocabulary may differ in
 * them between even and odd row numbers, and a packed copy from a view.
 *
 * Matrices are rows x width, elements of a row contiguous, rows `*_stride` elements apart, at any
 * element offset (no alignment beyond the element's own).
 *
 * dtype and status codes are those of luminav_hip.h: 0 f32, 1 bf16, 2 f16; 0 success, -1 null
 * pointer, -3 invalid argument, -4 launch failed.
 */
#ifndef LUMINAV_OPS_H
#define LUMINAV_OPS_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define LV_OPS_MAX_TOP 128      /* most alternatives lv_token_log_probs_forward returns per row */
#define LV_OPS_MAX_TEACHER 1024 /* most teacher logits per row */

/* y = (x - mean) * rstd * weight + bias over the last axis, mean and rstd = (var + eps)^-1/2 per
 * row. weight and bias may be NULL (1 and 0). Backward, with g = dy * weight and
 * xhat = (x - mean) * rstd:
 *   dx = rstd * (g - mean(g) - xhat * mean(g * xhat)), dweight = sum over rows of dy * xhat,
 *   dbias = sum over rows of dy.
 * out is y (forward) or dx (backward, NULL: not wanted); dweight and dbias may be NULL (not
 * wanted). weight, bias, dweight and dbias are of weight_dtype. */
typedef struct lv_layer_norm_args {
    const void *x;
    const void *dy;     /* backward only */
    void *out;
    const void *weight;
    const void *bias;   /* forward only */
    float *mean;        /* [rows]: written by forward, read by backward */
    float *rstd;
    void *dweight;      /* backward only */
    void *dbias;
    uint64_t rows;
    uint64_t width;     /* 1 to 2^30 */
    int64_t x_stride;
    int64_t dy_stride;
    int64_t out_stride;
    float eps;
    int32_t dtype;
    int32_t weight_dtype;
    int32_t reserved;
} lv_layer_norm_args;

int lv_layer_norm_forward(const lv_layer_norm_args *args, void *stream);
/* Workspace: lv_layer_norm_workspace_bytes(args) bytes of any content, 256-byte aligned; 0 when no
 * weight gradient is wanted. */
size_t lv_layer_norm_workspace_bytes(const lv_layer_norm_args *args);
int lv_layer_norm_backward(const lv_layer_norm_args *args, void *workspace, size_t workspace_bytes, void *stream);

/* The operators over logits: rows x vocab, p = softmax(logits / temperature). A token outside
 * [0, vocab) (the customary -100) names nothing. stats[r] = { max, log sum } : the row's largest
 * logit m and log sum_j exp((logits_j - m) / temperature). The two stay apart because their sum
 * would lose the second one where m is large (a row masked with the type's lowest value).
 *
 * lv_token_log_probs_forward: log_probs[r] = log p of tokens[r] (0 if it names nothing),
 *   entropy[r] = -sum p log p, stats[r], and the `count` most likely tokens of every row with their
 *   log probabilities, the lowest index first among equals.
 * lv_token_log_probs_backward: grad = d/dlogits of sum d_log_probs * log_probs + d_entropy *
 *   entropy (either may be NULL), from forward's stats and entropy:
 *   grad_j = (d_log_probs (1[j = token] - p_j) - d_entropy p_j (log p_j + entropy)) / temperature.
 * lv_distill_forward: with q = softmax of teacher_logits / temperature over the row's `count`
 *   teacher_tokens that name something, loss[r] = temperature^2 * sum q (log q - log p) and stats[r].
 *   A row without any, or whose teacher logits are all -inf, has loss 0.
 * lv_distill_backward: grad_j = temperature * w (p_j - sum of q over the entries naming j), from
 *   forward's stats, w = weight * row_weight[r] (row_weight may be NULL: 1); 0 in a row without q.
 * lv_distill_loss_and_grad: both in one call; stats are not returned.
 *
 * Rows of -inf logits alone have no distribution: stats -inf, log_probs and alternatives' -inf,
 * entropy 0, loss +inf, gradient 0. A row that holds NaN or +inf: log_probs, entropy, the log sum,
 * loss and gradient NaN, its alternatives tokens 0, 1, ... with NaN.
 * Workspaces: the *_workspace_bytes functions (0: none, may be NULL), any content, 256-byte
 * aligned. */
typedef struct lv_logits_args {
    const void *logits;
    const int64_t *tokens;          /* [rows], token_log_probs */
    const int64_t *teacher_tokens;  /* [rows, count], distill */
    const void *teacher_logits;     /* [rows, count] of teacher_dtype, distill */
    const float *row_weight;        /* [rows] or NULL, distill */
    const float *d_log_probs;       /* [rows] or NULL, token_log_probs backward */
    const float *d_entropy;         /* [rows] or NULL, token_log_probs backward */
    float *out;                     /* [rows]: log_probs or loss */
    float *entropy;                 /* [rows], token_log_probs: written by forward, read by backward */
    float *stats;                   /* [rows, 2]: written by forward, read by backward */
    float *top_log_probs;           /* [rows, count], token_log_probs forward */
    int64_t *top_tokens;            /* [rows, count], token_log_probs forward */
    void *grad;                     /* rows x vocab of dtype */
    uint64_t rows;
    uint64_t vocab;                 /* 1 to 2^30 */
    int64_t stride;                 /* of logits */
    int64_t grad_stride;
    float temperature;              /* > 0, finite */
    float weight;
    int32_t count;                  /* alternatives (0 to 128, at most vocab) or teacher logits (1 to 1024) */
    int32_t dtype;
    int32_t teacher_dtype;
    int32_t reserved;
} lv_logits_args;

size_t lv_token_log_probs_workspace_bytes(const lv_logits_args *args);
int lv_token_log_probs_forward(const lv_logits_args *args, void *workspace, size_t workspace_bytes, void *stream);
int lv_token_log_probs_backward(const lv_logits_args *args, void *stream);
size_t lv_distill_workspace_bytes(const lv_logits_args *args);
int lv_distill_forward(const lv_logits_args *args, void *workspace, size_t workspace_bytes, void *stream);
int lv_distill_backward(const lv_logits_args *args, void *stream);
int lv_distill_loss_and_grad(const lv_logits_args *args, void *workspace, size_t workspace_bytes, void *stream);

/* Description of the last error of these functions on this thread ("" if none). */
const char *lv_ops_last_error(void);

#ifdef __cplusplus
}
#endif

#endif /* LUMINAV_OPS_H */
