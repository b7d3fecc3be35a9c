/* Compute operators of a rank's training or serving step, beside the collectives: plain C.
 *
 *   gradients   the global norm of many tensors, and clipping by it
 *   norms       layer norm and RMS norm, forward and backward
 *   embedding   lookup with scaling, and its gradient by sorted tokens
 *   experts     tokens sorted by expert and back, with weights, and the gradients
 *
 * Every call enqueues work on `stream` of the CURRENT device and returns 0, or non-zero for bad
 * arguments or a failed launch (bcclGetLastError() says which); nothing synchronises, allocates
 * device memory or keeps state between calls, so calls may be captured into CUDA graphs and may
 * run at the same time on different streams. Scratch memory is the caller's: a call that takes a
 * `workspace` needs bccl<Op>Workspace() bytes, 16-byte aligned, that no other call uses until
 * this one has finished on its stream. Pointers are device memory of the current device unless
 * the name says host. dtype codes are those of bccl::DataType: 0 f32, 4 bf16, 5 f16; index
 * types: 2 int32, 3 int64. Row strides are in elements; the elements of a row are adjacent.
 * Sums, means and norms are kept in 32 bits or more and outputs are rounded once.
 */
#ifndef BCCL_OPS_H_
#define BCCL_OPS_H_

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* ---- Gradients. Global norm: sqrt(sum over tensors and elements of g^2).
 * bcclGradSquares writes (accumulate == 0) the sum of the squares to *sum or adds it (accumulate != 0: lists of
 * another type); ranks that hold shards of the parameters may AllReduce (SUM) it before it is used. The
 * sum does not depend on timing. The pointer and count arrays are host memory, read before the call
 * returns. workspace_bytes of BCCL_GRAD_WORKSPACE(total elements, n) are always enough.
 * bcclGradClip: norm = sqrt(*sum), c = min(1, max_norm / (norm + eps)), NaN kept; outs[i] = c * grads[i]
 * (outs[i] == grads[i] with one type: in place, and nothing is moved when c == 1). Outputs must not
 * otherwise overlap tensors of the list. norm (one float, may be NULL) receives the norm. n may be 0. */
#define BCCL_GRAD_WORKSPACE(elements, n) (((size_t)(elements) / 8192 + 2 * (size_t)(n) + 1) * sizeof(double))
int bcclGradSquares(const void* const* grads_host, const size_t* counts_host, int n, int dtype, int accumulate,
                    double* sum, void* workspace, size_t workspace_bytes, void* stream);
int bcclGradClip(const void* const* grads_host, void* const* outs_host, const size_t* counts_host, int n, int dtype,
                 int out_dtype, const double* sum, float max_norm, float eps, float* norm, void* stream);

/* ---- Norms over the last dimension: y = (x - mean) * rstd * weight + bias, with
 * rstd = 1 / sqrt(var + eps) and var the mean of (x - mean)^2; kind 0 layer norm, kind 1 RMS norm (mean = 0, no bias).
 * x, y [rows, h] of dtype; weight, bias [h] of wdtype (dtype or f32), each may be NULL; mean (layer norm) and
 * rstd [rows] f32. Backward: dx = rstd * (g - mean(g) - xh * mean(g * xh)), g = dy * weight (RMS norm without the
 * first mean); dweight = sum over rows of dy * xh and dbias = sum of dy in wdtype, each may be NULL. */
int bcclNormForward(int kind, const void* x, int64_t x_stride, const void* weight, const void* bias, void* y,
                    int64_t y_stride, float* mean, float* rstd, int64_t rows, int64_t h, float eps, int dtype, int wdtype,
                    void* stream);
size_t bcclNormBackwardWorkspace(int kind, int64_t rows, int64_t h, int dtype);
int bcclNormBackward(int kind, const void* dy, int64_t dy_stride, const void* x, int64_t x_stride, const float* mean,
                     const float* rstd, const void* weight, void* dx, int64_t dx_stride, void* dweight, void* dbias,
                     int64_t rows, int64_t h, int dtype, int wdtype, void* workspace, size_t workspace_bytes,
                     void* stream);

/* ---- Embedding. out[i] = scale * table[ids[i] - first_row]; ids outside [first_row, first_row + rows) (tokens
 * of other ranks' shards) give rows of zeros.
 * Gradient: dtable[v] = scale * sum of dy[i] over the i with ids[i] == first_row + v, summed in a fixed order;
 * ids outside the shard and skip_id (has_skip != 0) add nothing. accumulate == 0 writes all rows of dtable
 * (zeros for absent tokens), else rows of present tokens are added to. dtable: out_dtype (dtype or f32), dense. */
int bcclEmbeddingForward(const void* ids, int ids_dtype, int64_t n, const void* table, int64_t table_stride, int64_t rows,
                         int64_t h, int64_t first_row, float scale, void* out, int64_t out_stride, int dtype, void* stream);
size_t bcclEmbeddingBackwardWorkspace(int64_t n, int64_t rows, int64_t h);
int bcclEmbeddingBackward(const void* dy, int64_t dy_stride, const void* ids, int ids_dtype, int64_t n, void* dtable,
                          int64_t rows, int64_t h, int64_t first_row, float scale, int64_t skip_id, int has_skip,
                          int accumulate, int dtype, int out_dtype, void* workspace, size_t workspace_bytes,
                          void* stream);

/* ---- Experts. Assignment a = t * top + j sends token t to expert ids[a]; ids outside [0, experts) are dropped.
 * bcclExpertSort orders the kept assignments by expert, those of one expert by a: sources[s] = a of sorted row
 * s (-1 behind the last), slots[a] = s (-1: dropped), offsets[e] = first row of expert e, offsets[experts] =
 * kept rows. experts <= BCCL_MAX_EXPERTS, tokens * top < 2^31. top <= BCCL_MAX_TOP.
 * Dispatch: rows[slots[a]] = x[t]; rows behind the last kept one are zeros.
 * Combine: y[t] = sum over j of weights[a] * rows[slots[a]] (weights NULL: 1).
 * Combine backward: drows[slots[a]] = weights[a] * dy[t], zeros behind the last; dweights[a] = <dy[t], rows[slots[a]]>
 * (0: dropped). The gradient of dispatch is a combine without weights. */
#define BCCL_MAX_EXPERTS 1023
#define BCCL_MAX_TOP 64
size_t bcclExpertSortWorkspace(int64_t tokens, int top);
int bcclExpertSort(const void* ids, int ids_dtype, int64_t tokens, int top, int experts, int32_t* slots, int32_t* sources,
                   int32_t* offsets, void* workspace, size_t workspace_bytes, void* stream);
int bcclExpertDispatch(const void* x, int64_t x_stride, const int32_t* slots, const int32_t* offsets, int64_t tokens,
                       int top, int experts, int64_t h, void* rows, int dtype, void* stream);
int bcclExpertCombine(const void* rows, const int32_t* slots, const void* weights, int wdtype, int64_t tokens, int top,
                      int64_t h, void* y, int64_t y_stride, int dtype, void* stream);
int bcclExpertCombineBackward(const void* dy, int64_t dy_stride, const void* rows, const int32_t* slots,
                              const int32_t* offsets, const void* weights, int wdtype, int64_t tokens, int top, int experts,
                              int64_t h, void* drows, void* dweights, int dtype, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* BCCL_OPS_H_ */
