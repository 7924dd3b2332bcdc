/* vs_learn.h -- learning the vectors an index serves: rows of a table read by number, the softmax loss of queries over ALL rows of a
 * table (or all members of an index), and the gradients of both (libvs_learn.so, on top of libvs_hnsw.so).
 *
 *   lookup   out[t]  = scale * rows[id[t]]                                (ids outside [0, rows): a row of zeros)
 *   loss     loss[i] = log(sum_j exp z[i][j]) - z[i][label[i]],           z[i][j] = scale * <query i, row j>   (VS_METRIC_IP)
 *                                                                                   scale * cos(query i, row j) (VS_METRIC_COS)
 *
 * vs_softmax_loss_* is vs_hnsw_exact_search_batch_device with a log-sum-exp in place of the top-k: the scores of every query against
 * every row, which never exist in memory as a whole (training needs them twice: the backward call computes them again).
 *
 * Conventions (as include/vs_hnsw.h, and):
 *  - Every pointer named d_* is device memory of the current device (of the index's device where `rows.index` is set), `stream` a
 *    hipStream_t of it.  Nothing is synchronised and nothing is allocated: a call only enqueues kernels on `stream`, so it can be captured
 *    into a graph.  Scratch comes from the caller (`d_work`, at least the bytes the matching _work function names, 256-byte aligned); two
 *    calls that may run at the same time need two of them.
 *  - Matrices are row-major with a row stride in ELEMENTS (>= the row's length); any stride and alignment of whole elements will do
 *    (16-byte aligned rows of a multiple of 8 elements are read in place, others are re-laid in d_work first).
 *  - Scalars: VS_SCALAR_F32, VS_SCALAR_F16, VS_SCALAR_BF16.  Sums are kept in f32.  Two calls with the same inputs give the same bits.
 *  - Rows, and queries with a label, hold finite numbers (an infinity or NaN among them reaches every loss and gradient), their inner
 *    products are finite in f32 before the scale is applied, and so are the gradients.  Under
 *    VS_METRIC_COS a vector's length lies between 1e-18 and 1e18 (its square is an f32; zero vectors are fine: their scores and gradients
 *    are 0), of bf16 vectors also a query's length times a row's between 1e-36 and 1e36.
 *  - Ids and labels: int32 (id_bytes 4) or int64 (8).
 *  - Outputs must not overlap inputs.
 */
#ifndef VS_LEARN_H
#define VS_LEARN_H

#include "vs_hnsw.h"

#ifdef __cplusplus
extern "C" {
#endif

/* The rows: a table in device memory, or -- `index` set, the other fields ignored -- the members of an index by SLOT number
 * (vs_hnsw_slots; rows = vs_hnsw_graph_info.slots): f32 / f16 / bf16 storage as stored.  Removed members are read as zeros by a lookup,
 * take no part in a loss and get a gradient of zero; a label that names one is ignored.  The metric of a loss must be the index's.
 * As for a search, adds / removes / reserves must not overlap the call's work on the stream, and a captured graph stays valid only until
 * the next one. */
typedef struct vs_rows {
    vs_hnsw* index;
    const void* d_data;
    int scalar;
    size_t rows, dim, stride;
} vs_rows;

/* out: n x dim of out_scalar. */
VS_API int vs_lookup_device(const vs_rows* rows, const void* d_ids, size_t id_bytes, size_t n, float scale, void* d_out, int out_scalar,
                            size_t out_stride, void* stream);

/* out[v] = scale * sum of grad[t] over the t with id[t] == v, in the order of t: all `rows` rows of `out` are written (rows nobody read
 * become zero), or, with accumulate != 0, the sums are added to the rows somebody read and the others are left as they are. */
VS_API size_t vs_lookup_grad_work(size_t n, size_t rows, size_t dim);
VS_API int vs_lookup_grad_device(const void* d_grad, int grad_scalar, size_t grad_stride, const void* d_ids, size_t id_bytes, size_t n,
                                 size_t rows, size_t dim, float scale, int accumulate, void* d_out, int out_scalar, size_t out_stride,
                                 void* d_work, size_t work_bytes, void* stream);

/* The queries of a loss and what they are labelled with.  A label outside [0, rows) marks a row of padding: its loss is 0, its gradient 0,
 * and whatever its query holds reaches no other row (its lse is computed like any other). */
typedef struct vs_softmax {
    const void* d_queries;
    int scalar;
    size_t n, stride;
    const void* d_labels;
    size_t label_bytes; /* 4 or 8 */
    float scale;
    int metric; /* VS_METRIC_IP or VS_METRIC_COS */
} vs_softmax;

/* loss: n floats; lse: n floats (log-sum-exp of the row's scores: what the backward call needs; -inf where there is no row at all). */
VS_API size_t vs_softmax_loss_work(const vs_rows* rows, const vs_softmax* q);
VS_API int vs_softmax_loss_device(const vs_rows* rows, const vs_softmax* q, float* d_loss, float* d_lse, void* d_work, size_t work_bytes,
                                  void* stream);

/* Gradients of sum_i grad_loss[i] * loss[i]: of the queries (n x dim, the queries' scalar) and of the rows (rows x dim, the rows' scalar);
 * either may be NULL.  Under VS_METRIC_COS the gradient goes through the normalisation. */
VS_API size_t vs_softmax_loss_grad_work(const vs_rows* rows, const vs_softmax* q, int queries, int table);
VS_API int vs_softmax_loss_grad_device(const vs_rows* rows, const vs_softmax* q, const float* d_lse, const float* d_grad_loss,
                                       void* d_grad_queries, size_t grad_queries_stride, void* d_grad_rows, size_t grad_rows_stride,
                                       void* d_work, size_t work_bytes, void* stream);

VS_API const char* vs_learn_last_error(void);

#ifdef __cplusplus
}
#endif
#endif /* VS_LEARN_H */
