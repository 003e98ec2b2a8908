/*
 * mlxc_train — C ABI of the operators that train node embeddings on walks
 * (libmlxc.so): the step after the walks and windows of mlxc.h.
 *
 * The conventions are those of mlxc.h: d_* are device pointers on the current
 * device, every call is asynchronous on `stream` (a hipStream_t), the caller
 * allocates every buffer, a call returns MLXC_OK or a negative MLXC_ERR_* code
 * with the message in mlxc_last_error().  None of it has a counterpart in the
 * reference, which stops at the walks
 * (/root/reference/random_walks/BiasedRandomWalk.cpp:96).
 *
 * Tables and gradients are row-major with `dim` values a row, of one of the
 * MLXC_FLOAT* types; every sum is made in 32 bits or more and rounded once, to
 * the type that it is written in.  Node arrays are MLXC_OUT_INT64 or
 * MLXC_OUT_INT32.  A node of -1 is no node (the walks' edge ids hold -1 where
 * a walk stayed): its row reads as zeros and takes no gradient.  Any other
 * node outside [0, num_rows) is treated the same and reported as
 * MLXC_STATUS_BAD_NODE where the call takes a status word.
 *
 * Results do not depend on the order in which blocks run: the same call gives
 * the same bits every time.
 */
#ifndef MLXC_TRAIN_H
#define MLXC_TRAIN_H

#include "mlxc.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Element types. */
#define MLXC_FLOAT32 0
#define MLXC_BFLOAT16 1
#define MLXC_FLOAT16 2

/* flags of the gradients. */
#define MLXC_GRAD_SPARSE 1 /* coalesced: ids and their rows instead of the whole table's */

/* flags of mlxc_preference_loss. */
#define MLXC_PREFERENCE_NORMALIZE 1 /* a log ratio is the mean over its values, not the sum */
#define MLXC_PREFERENCE_SUM 2       /* the loss is the sum over the pairs, not the mean */

/*
 * Embedding lookup with scaling:
 *   d_out[i, :] = scale * d_weight[d_nodes[i], :]   (zeros where there is no node)
 *
 * d_weight   [num_rows, dim] of dtype, rows row_stride values apart (>= dim)
 * d_nodes    [count] of node_type
 * d_out      [count, dim] of dtype
 * d_status   one int64 for MLXC_STATUS_* bits, or NULL
 * num_rows in [0, 2^31), dim in [1, 65536].
 */
int mlxc_embedding(const void* d_weight, int64_t num_rows, int32_t dim, int64_t row_stride,
                   int32_t dtype, const void* d_nodes, int64_t count, int32_t node_type,
                   float scale, void* d_out, int64_t* d_status, void* stream);

/* Workspace bytes of mlxc_embedding_grad (0: sizes out of range). */
size_t mlxc_embedding_grad_workspace_bytes(int64_t num_rows, int32_t dim, int64_t count,
                                           int32_t flags);

/*
 * Gradient of mlxc_embedding by sorted nodes:
 *   G[v, :] = scale * sum over i with d_nodes[i] = v of d_grad[i, :]
 *
 * d_grad     [count, dim] of dtype
 * d_out      dense: [num_rows, dim] of out_dtype, every row written.  With
 *            MLXC_GRAD_SPARSE: [min(count, num_rows), dim], row u the gradient
 *            of node d_ids[u]
 * d_ids      MLXC_GRAD_SPARSE: int64 [min(count, num_rows)], the nodes that
 *            occur, ascending, then -1 (whose rows are zeros); else NULL
 * d_workspace 16-byte aligned, of the size the query returns; word 0 holds the
 *            MLXC_STATUS_* bits once the call has completed.
 * count in [0, 2^31 - 1).  The order of a node's sum is fixed by the places
 * at which it occurs.
 */
int mlxc_embedding_grad(const void* d_grad, int32_t dim, int32_t dtype, const void* d_nodes,
                        int64_t count, int32_t node_type, int64_t num_rows, float scale,
                        int32_t flags, int64_t* d_ids, void* d_out, int32_t out_dtype,
                        void* d_workspace, size_t workspace_bytes, void* stream);

/*
 * Scores of the skip-gram windows of walks: with W = walk_nodes -
 * context_size + 1 windows a walk,
 *   d_scores[(n * W + j) * (C - 1) + k - 1] =
 *       scale * <row of node j of walk n, row of node j + k>,   1 <= k < C
 * (0 where either is no node), i.e. a window's first node against the nodes
 * after it.  The same numbers as for mlxc_context_windows' windows, walk by
 * walk instead of window-major, without writing the windows; windows made
 * elsewhere are walks of context_size nodes.
 *
 * d_walks    [num_walks, walk_nodes] of node_type
 * d_scores   float32 [num_walks, W, C - 1]
 * context_size in [2, min(32, walk_nodes)]; the rest as in mlxc_embedding.
 * num_walks * walk_nodes below 2^31 - 1.
 */
int mlxc_window_scores(const void* d_weight, int64_t num_rows, int32_t dim, int64_t row_stride,
                       int32_t dtype, const void* d_walks, int64_t num_walks, int32_t walk_nodes,
                       int32_t context_size, int32_t node_type, float scale, float* d_scores,
                       int64_t* d_status, void* stream);

/* Workspace bytes of mlxc_window_scores_grad (0: sizes out of range). */
size_t mlxc_window_scores_grad_workspace_bytes(int64_t num_rows, int32_t dim, int64_t num_walks,
                                               int32_t walk_nodes, int32_t context_size,
                                               int32_t flags);

/*
 * Gradient of mlxc_window_scores with respect to the table:
 *   G = scale * sum over n, j, k of d_grad[n, j, k - 1] *
 *       (e(u) (x) row(v) + e(v) (x) row(u)),  u, v = nodes j, j + k of walk n,
 * dense or coalesced as in mlxc_embedding_grad (count = num_walks *
 * walk_nodes).  Values of d_grad at pairs with no node are not read as
 * numbers: they may be anything.
 */
int mlxc_window_scores_grad(const float* d_grad, const void* d_weight, int64_t num_rows,
                            int32_t dim, int64_t row_stride, int32_t dtype, const void* d_walks,
                            int64_t num_walks, int32_t walk_nodes, int32_t context_size,
                            int32_t node_type, float scale, int32_t flags, int64_t* d_ids,
                            void* d_out, int32_t out_dtype, void* d_workspace,
                            size_t workspace_bytes, void* stream);

/* One side of the pairs of mlxc_preference_loss: `length` values a pair. */
typedef struct mlxc_preference_side {
    const void* values;    /* [pairs, length] log-probabilities or scores */
    const void* reference; /* [pairs, length] of the reference model, or NULL (zeros) */
    const uint8_t* mask;   /* [pairs, length], 0 leaves a value out, or NULL (none left out) */
    int64_t length;        /* [0, 2^30) */
    void* grad;            /* [pairs, length] of dtype, or NULL (not wanted) */
} mlxc_preference_side;

/* Workspace bytes of mlxc_preference_loss. */
size_t mlxc_preference_loss_workspace_bytes(int64_t pairs);

/*
 * Preference loss of paired log ratios.  With r a side's sum (or mean, with
 * MLXC_PREFERENCE_NORMALIZE; 0 if nothing is left) of values - reference over
 * the places that its mask leaves, and z = beta * (r_chosen - r_rejected):
 *   loss = mean (or sum) over the pairs of
 *          (1 - label_smoothing) * log(1 + e^-z) + label_smoothing * log(1 + e^z)
 *
 * Both sides' values and references are of dtype; the references take no
 * gradient; what stands in masked places is not used.  A side's grad, where
 * given, receives the loss's gradient (0 in masked places).  Of no pairs the
 * loss is 0.
 *
 * d_loss     one float32
 * d_rewards  float32 [2, pairs]: beta * r_chosen, beta * r_rejected, or NULL
 * d_slopes   float32 [2, pairs]: the loss's derivative by each value of a
 *            pair's chosen and rejected side (mlxc_preference_grad), or NULL
 * beta finite, label_smoothing in [0, 1].
 */
int mlxc_preference_loss(const mlxc_preference_side* chosen, const mlxc_preference_side* rejected,
                         int64_t pairs, int32_t dtype, float beta, float label_smoothing,
                         int32_t flags, float* d_loss, float* d_rewards, float* d_slopes,
                         void* d_workspace, size_t workspace_bytes, void* stream);

/*
 * The gradients of mlxc_preference_loss from its d_slopes, times *d_upstream
 * (a float32 on the device, or NULL: 1): sides' grad [p, t] = upstream *
 * slope[p] where the mask leaves t, else 0.  values and reference are not
 * read; a side whose grad is NULL is left out.
 */
int mlxc_preference_grad(const mlxc_preference_side* chosen, const mlxc_preference_side* rejected,
                         int64_t pairs, int32_t dtype, const float* d_slopes,
                         const float* d_upstream, void* stream);

/* Host twins: host pointers, on the calling thread, no workspace.  The same
 * formulas with 64-bit sums, so equal to the device's up to rounding. */
int mlxc_embedding_cpu(const void* weight, int64_t num_rows, int32_t dim, int64_t row_stride,
                       int32_t dtype, const void* nodes, int64_t count, int32_t node_type,
                       float scale, void* out, int64_t* status);
int mlxc_embedding_grad_cpu(const void* grad, int32_t dim, int32_t dtype, const void* nodes,
                            int64_t count, int32_t node_type, int64_t num_rows, float scale,
                            int32_t flags, int64_t* ids, void* out, int32_t out_dtype,
                            int64_t* status);
int mlxc_window_scores_cpu(const void* weight, int64_t num_rows, int32_t dim, int64_t row_stride,
                           int32_t dtype, const void* walks, int64_t num_walks,
                           int32_t walk_nodes, int32_t context_size, int32_t node_type,
                           float scale, float* scores, int64_t* status);
int mlxc_window_scores_grad_cpu(const float* grad, const void* weight, int64_t num_rows,
                                int32_t dim, int64_t row_stride, int32_t dtype, const void* walks,
                                int64_t num_walks, int32_t walk_nodes, int32_t context_size,
                                int32_t node_type, float scale, int32_t flags, int64_t* ids,
                                void* out, int32_t out_dtype, int64_t* status);
int mlxc_preference_loss_cpu(const mlxc_preference_side* chosen,
                             const mlxc_preference_side* rejected, int64_t pairs, int32_t dtype,
                             float beta, float label_smoothing, int32_t flags, float* loss,
                             float* rewards, float* slopes);
int mlxc_preference_grad_cpu(const mlxc_preference_side* chosen,
                             const mlxc_preference_side* rejected, int64_t pairs, int32_t dtype,
                             const float* slopes, const float* upstream);

#ifdef __cplusplus
}
#endif
#endif
