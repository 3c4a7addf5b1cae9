/*
 * lfm_ops.h -- C ABI of liblfm_ops.so: operators on DEVICE memory (MI355X, gfx950).
 *
 * Where lfm_hip.h takes host buffers and keeps its state in sessions, these entry points work on arrays that
 * already live on the GPU (a torch tensor's data pointer, for instance) and on the caller's stream:
 *
 *   - every pointer is a device pointer unless it is called a host pointer;
 *   - `stream` is a hipStream_t (NULL = the default stream) of the current device; everything is enqueued on it and
 *     nothing is waited for, copied to the host or allocated, so every call can be recorded into a HIP graph;
 *   - scratch memory is the caller's: lfm_ops_*_workspace says how many bytes a call needs (256-byte aligned);
 *     a workspace belongs to one call at a time and carries nothing from one call to the next;
 *   - the return value is LFM_OK or a negative LFM_E* code of lfm_hip.h, lfm_ops_last_error() its description
 *     (thread-local).  All checks of sizes happen on the host before anything is launched.
 *
 * Ids (targets, embedding ids) live on the device and cannot be checked on the host: an id outside [0, vocab) is
 * never followed -- it has no loss, contributes a zero row and receives no gradient.  -1 is the padding id.
 */
#ifndef LFM_OPS_H
#define LFM_OPS_H

#include <stdint.h>

#include "lfm_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

#define LFM_F32 0
#define LFM_BF16 1
#define LFM_F16 2

const char *lfm_ops_last_error(void);

/* Softmax cross entropy of `rows` hidden vectors against every row of `table` (the catalogue is the vocabulary):
 *   s[n, v] = <hidden[n], table[v]> + bias[v],  lse[n] = log sum_v exp s[n, v],
 *   loss[n] = weights[n] * (lse[n] - s[n, targets[n]])            (0 for a row without a target),
 * and, for lfm_ops_softmax_loss_grad, the gradients of sum_n loss[n]:
 *   q[n, v] = weights[n] * (exp(s[n, v] - lse[n]) - [v == targets[n]])     (0 for a row without a target),
 *   d_hidden = q table,  d_table = q^T hidden,  d_bias[v] = sum_n q[n, v].
 * The logits are never written to memory.  bias / weights may be NULL (0 / 1); d_bias may be NULL.  A bias of -inf
 * removes an item: its row of the table is not looked at, whatever it holds, and has a zero gradient.  As the target of row n
 * its loss is infinite and the gradients are the formula's with a probability of 0: -weights[n] table[v] in d_hidden[n]
 * (elements of that row that are not finite count as 0), -weights[n] hidden[n] in d_table[v], -weights[n] in d_bias[v].
 * Rows of hidden and table are contiguous, `*_stride` elements apart; the gradients are dense.
 * A bias may be a large negative number instead, as masks are.  Biases beyond +-2^67 (float32 operands; +-2^127 in half
 * precision) may be cut there: below, the probability is 0 beside any other score, and the loss of a target so masked is the
 * uncut score's; in a row where nothing else is left, cut scores count as equal and lse is float32's lowest value.
 * float32 operands keep 22 bits and a floor of 2^-39 of the largest magnitude of hidden (rows with a target; all rows where none
 * has one) or table (items not removed); the terms q of d_table keep 22 bits and an absolute error of 2^-38 of the largest weight,
 * the terms of d_hidden 22 bits and 2^-32 of the row's largest.  In half precision the terms of both are rounded to the operands'
 * type before they are summed (in float32).  At most 2^27 rows and 2^30 items. */
typedef struct lfm_softmax_args {
    const void *hidden, *table; /* [rows, d], [vocab, d] of `dtype` */
    const void *targets;        /* [rows] int32 or int64 */
    const float *bias;          /* [vocab] or NULL */
    const float *weights;       /* [rows] or NULL */
    float *loss, *lse;          /* [rows] */
    void *d_hidden, *d_table;   /* like hidden / table */
    float *d_bias;              /* [vocab] or NULL */
    int64_t rows, vocab;
    int64_t hidden_stride, table_stride;
    int32_t d, dtype;           /* 1 <= d <= LFM_MAX_COMPONENTS */
    int32_t id_bytes;           /* 4 or 8: width of targets */
    int32_t reserved;
} lfm_softmax_args;

int lfm_ops_softmax_workspace(int64_t rows, int64_t vocab, int32_t d, int32_t dtype, int32_t grad, int64_t *bytes);
int lfm_ops_softmax_loss(const lfm_softmax_args *args, void *workspace, int64_t workspace_bytes, void *stream);
int lfm_ops_softmax_loss_grad(const lfm_softmax_args *args, void *workspace, int64_t workspace_bytes, void *stream);

/* out[r] = scale * sum_{j in bag r} values[j] * table[ids[j]]; without indptr bag r is the single id ids[r] (then
 * nnz == rows), without values every value is 1.  Sums are float32 in the order of the bag. */
typedef struct lfm_lookup_args {
    const void *table;          /* lookup: [vocab, d], rows table_stride apart; gradient: unused */
    const void *ids;            /* [nnz] int32 or int64 */
    const void *indptr;         /* [rows + 1], the type of ids, or NULL */
    const float *values;        /* [nnz] or NULL */
    void *out;                  /* lookup: [rows, d] dense; gradient: d_table, [vocab, d] dense */
    const void *d_out;          /* gradient: [rows, d], rows d_out_stride apart */
    int64_t rows, vocab, nnz;
    int64_t table_stride, d_out_stride;
    int32_t d, dtype, id_bytes;
    float scale;
} lfm_lookup_args;

int lfm_ops_embedding_lookup(const lfm_lookup_args *args, void *stream);
/* d_table[v] = scale * sum_{(r, j): ids[j] == v} values[j] * d_out[r]: the ids are sorted (stable), every row of
 * d_table is summed in float32 in the order of the ids' positions -- no float atomics, the same bits every time. */
int lfm_ops_embedding_grad_workspace(int64_t rows, int64_t vocab, int64_t nnz, int32_t d, int32_t bags, int64_t *bytes);
int lfm_ops_embedding_lookup_grad(const lfm_lookup_args *args, void *workspace, int64_t workspace_bytes, void *stream);

/* norm = sqrt(sum of squares over all tensors), summed in float64; out[i] = x[i] * min(1, max_norm / norm).
 * `x`, `out`, `counts`, `dtypes` are HOST arrays of n_tensors entries; out[i] may be x[i] and overlaps nothing else (a
 * tensor that is listed twice cannot be scaled: LFM_EINVAL); out NULL computes the norm alone.  Where an element is not
 * finite the norm is not either and the values are left unscaled; a finite norm beyond float32 is reported as infinite, and
 * the values are scaled by it. */
int lfm_ops_clip_workspace(int64_t n_tensors, const int64_t *counts, int64_t *bytes);
int lfm_ops_clip_global_norm(int64_t n_tensors, const void *const *x, void *const *out, const int64_t *counts,
                             const int32_t *dtypes, double max_norm, float *norm, void *workspace,
                             int64_t workspace_bytes, void *stream);

#ifdef __cplusplus
}
#endif
#endif /* LFM_OPS_H */
