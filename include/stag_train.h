/*
 * stag_train.h -- C ABI of libstag_train.so: the operators that LEARN node classifiers on MI355X (gfx950), next to
 * libstag_hip.so, which evaluates them.
 *
 * A node classifier is a logistic regression over the packed one-hot row of an aligned sequence (the rows of
 * stag_encode_a2m*).  The reference fits one per tree node on the CPU (stag/create_db.py:127-145, an L1-penalised
 * LogisticRegression); these entry points are one step of that fit for all K classifiers of a table at once:
 *
 *   stag_row_scores_dev       s = scale * X T + b        (X: packed rows, T: coefficients; the sum of run_logistic_prediction,
 *                                                         stag/classify.py:22-27, for many rows and classifiers)
 *   stag_sibling_loss_dev     loss and dloss/ds of "this sibling or one of the others"
 *   stag_row_scores_grad_dev  dT = scale * X^T G, db = sum G
 *   stag_adamw_dev            AdamW with an optional L1 shrinkage, for many tensors in one launch
 *
 * A table is an embedding table: row f holds the K coefficients of token f (= 5 * column + symbol), and a packed row is
 * the sorted list of a sequence's tokens, so the score is an embedding lookup summed over the row's tokens.
 *
 * Conventions as in stag_hip.h: plain C types, 0 or a negative STAG_E_* (stag_train_last_error() then describes it,
 * thread-local), the caller owns every buffer and the library keeps no pointer after a call.  All pointers named d_* are
 * DEVICE pointers on the current device; calls enqueue work on `stream` (a hipStream_t as void*; NULL = the null stream),
 * allocate nothing and do not synchronise, so they can be captured into a HIP graph.  d_work is scratch memory of at
 * least the bytes that the matching *_workspace function returns, 256-byte aligned; its contents are not kept between
 * calls, and two calls that may run at the same time need two of them.  Outputs and d_work share memory with nothing else
 * that a call takes.  Results do not depend on timing: equal inputs give equal bits.
 *
 * Sizes: 0 <= m < 2^31 rows of a batch, 1 <= k <= 2^20 classifiers, 1 <= n_features <= 2^27; the strides of tables, scores and
 * gradients are at least k and at most 2^21 values.  What is larger, or needs more workgroups than a launch has, is refused.
 * Rows of tables and gradients that all begin at a multiple of 16 bytes (32-bit values) or 8 are read faster.
 */
#ifndef STAG_TRAIN_H
#define STAG_TRAIN_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#ifndef STAG_OK
#define STAG_OK 0
#define STAG_E_INVALID (-1) /* bad argument */
#define STAG_E_HIP (-2)     /* a HIP runtime call failed */
#endif

/* types of tables, gradients and parameters */
#define STAG_F32 0
#define STAG_BF16 1
#define STAG_F16 2

const char *stag_train_last_error(void);

/* Bytes of d_work for the two calls below; negative: STAG_E_INVALID. */
int64_t stag_row_scores_workspace(int64_t m, int32_t n_features, int32_t k, int32_t type);
int64_t stag_row_scores_grad_workspace(int64_t m, int32_t n_features, int32_t k, int32_t type);

/*
 * scores[i][c] = scale * (sum of table[f][c] over the features f of row r_i) + bias[c],   i < m, c < k
 *
 * d_bits: n packed rows, row r at d_bits + r * row_stride words (row_stride a multiple of 4, at least the words of
 * n_features, rows 16-byte aligned; bit f of a row is bit f & 31 of its word f >> 5; bits from n_features on are ignored).
 * r_i = d_rows[i], or i when d_rows is NULL (then m <= n).  The same row may be named more than once; an index outside
 * 0..n-1 marks padding, whose scores are 0.  table[f][c] = d_table[f * table_stride + c], of `type`; d_bias (k values)
 * may be NULL; scores[i][c] = d_scores[i * score_stride + c], 32-bit.
 * Sums are held in 32 bits; 32-bit coefficients count with their 24 bits, or to 2^-133 where that is coarser.  Only the
 * coefficients of features that a row has enter its score, so infinities and NaN elsewhere in the table do not reach it.
 */
int stag_row_scores_dev(const uint32_t *d_bits, int64_t n, int64_t row_stride, int32_t n_features, const int32_t *d_rows,
                        int64_t m, const void *d_table, int32_t type, int64_t table_stride, const float *d_bias, int32_t k,
                        float scale, float *d_scores, int64_t score_stride, void *d_work, int64_t work_bytes, void *stream);

/*
 * The gradient of the above: table_grad[f][c] = scale * (sum of grad[i][c] over the i whose row has feature f),
 * bias_grad[c] = sum of grad[i][c] over all i.  Rows that are padding take part in neither, whatever d_grad holds for
 * them.  A row named twice counts twice.  d_table_grad and d_bias_grad are overwritten, 32-bit; either may be NULL.
 */
int stag_row_scores_grad_dev(const uint32_t *d_bits, int64_t n, int64_t row_stride, int32_t n_features, const int32_t *d_rows,
                             int64_t m, const void *d_grad, int32_t type, int64_t grad_stride, int32_t k, float scale,
                             float *d_table_grad, int64_t table_grad_stride, float *d_bias_grad, void *d_work,
                             int64_t work_bytes, void *stream);

/*
 * Logistic loss of siblings.  Row i trains the columns lo_i <= c < hi_i, {lo_i, hi_i} = d_siblings[2 i], [2 i + 1] (cut to
 * 0..k; NULL: all k), with target 1 for c == d_label[i] and 0 for the others (a label outside the range: all are 0):
 *   loss[c]    = scale * sum_i w_i softplus(c == label_i ? -s : s),   s = scores[i][c]
 *   grad[i][c] = scale * w_i * (sigmoid(s) - target), and 0 in the columns that the row does not train, where scores are not read.
 * w_i = d_weight[i], or 1 when NULL.  loss: k 32-bit values; grad: of `type`.  Either may be NULL.
 */
int64_t stag_sibling_loss_workspace(int64_t m, int32_t k);
int stag_sibling_loss_dev(const float *d_scores, int64_t score_stride, int64_t m, int32_t k, const int32_t *d_label,
                          const int32_t *d_siblings, const float *d_weight, float scale, float *d_loss, void *d_grad,
                          int32_t type, int64_t grad_stride, void *d_work, int64_t work_bytes, void *stream);

/*
 * One AdamW step over n tensors in one launch.  For every value, with t = *d_step + 1:
 *   m = beta1 m + (1 - beta1) g;   v = beta2 v + (1 - beta2) g^2;   d = sqrt(v / (1 - beta2^t)) + eps
 *   p = p (1 - lr weight_decay) - lr m / ((1 - beta1^t) d);   with l1 > 0 then  p = sign(p) max(|p| - lr l1 / d, 0)
 * and t is stored to *d_step.  Computed in 32 bits, subnormal numbers included; p is rounded to its type at the end, to nearest.
 * A square below 2^-149 is 0: with eps = 0 a value whose gradients were all under 2^-70 may become infinite or NaN.
 *
 * The last is the proximal step of l1 * |p| in the metric of the update, so that a point at rest has
 * |mean gradient| <= l1: the LASSO's condition.
 *
 * States lie in two flat arrays, tensor j's from place state_at (a multiple of 256) on; all of them together hold
 * state_values values.  state_bits 32: d_m, d_v are floats.  state_bits 8: d_m holds e4m3 codes of m / s and d_v of
 * sqrt(v) / s, where s = d_m_scale[b], d_v_scale[b] is a power of two for each 256 values; a value between two codes goes
 * to either by a hash of its place and t, so that it is right on the mean: with beta2 = 0.999 a step moves sqrt(v) by
 * 1/2000 of itself, which rounding to nearest would lose every time.  A second moment that overflows is kept as an infinity
 * (the value then stands still) with 32 bits and becomes NaN, as the value does one step later, with 8.
 *
 * d_tensors: n descriptors in device memory; d_tiles: for each STAG_ADAMW_TILE values of each tensor (the last tile
 * of a tensor may be shorter) its tensor and its number in the tensor.  d_step: STAG_ADAMW_STEP_WORDS words, t and then
 * zeros, which the call leaves zero.  Two steps that share any of these buffers have to run one after the other.
 */
#define STAG_ADAMW_BLOCK 256
#define STAG_ADAMW_TILE 1024
#define STAG_ADAMW_STEP_WORDS 1088
typedef struct {
    void *param;
    const void *grad;
    int64_t count;
    int64_t state_at;
    float weight_decay;
    float l1;
    int32_t param_type;
    int32_t grad_type;
} stag_adamw_tensor_t;

typedef struct {
    int32_t tensor;
    int32_t tile;
} stag_adamw_tile_t;

int stag_adamw_dev(const stag_adamw_tensor_t *d_tensors, const stag_adamw_tile_t *d_tiles, int64_t n_tiles, int32_t state_bits,
                   void *d_m, void *d_v, float *d_m_scale, float *d_v_scale, int32_t *d_step, double lr, double beta1,
                   double beta2, double eps, void *stream);

#ifdef __cplusplus
}
#endif
#endif /* STAG_TRAIN_H */
