// Host launchers of the compute operators; arguments as in bccl/ops.h, checked by the C interface.
#pragma once

#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace bccl {

size_t GradSquaresWorkspace(const void* const* grads, const size_t* counts, int n, int dtype);
cudaError_t LaunchGradSquares(const void* const* grads, const size_t* counts, int n, int dtype, bool accumulate,
                              double* sum, void* workspace, cudaStream_t stream);
cudaError_t LaunchGradClip(const void* const* grads, void* const* outs, const size_t* counts, int n, int dtype,
                           int out_dtype, const double* sum, float max_norm, float eps, float* norm, cudaStream_t stream);

struct NormForwardArgs {
    const void* x;
    long long x_stride;
    const void* w;
    const void* b;
    void* y;
    long long y_stride;
    float* mean;
    float* rstd;
    long long rows, h;
    float eps;
};
cudaError_t LaunchNormForward(bool layer, const NormForwardArgs& a, int dtype, int wdtype, cudaStream_t stream);

struct NormBackwardArgs {
    const void* dy;
    long long dy_stride;
    const void* x;
    long long x_stride;
    const float* mean;
    const float* rstd;
    const void* w;
    void* dx;
    long long dx_stride;
    void* dw;
    void* db;
    float* partials;  // [2][blocks][h]: dw, then db
    long long rows, h;
};
size_t NormBackwardWorkspace(bool layer, long long rows, long long h, int dtype);
cudaError_t LaunchNormBackward(bool layer, NormBackwardArgs a, int dtype, int wdtype, cudaStream_t stream);

struct EmbeddingArgs {
    const void* ids;
    int ids64;
    long long n;
    long long rows, h, first;
};
cudaError_t LaunchEmbeddingForward(const EmbeddingArgs& a, const void* table, long long table_stride, float scale,
                                   void* out, long long out_stride, int dtype, cudaStream_t stream);
size_t EmbeddingBackwardWorkspace(long long n, long long h);
cudaError_t LaunchEmbeddingBackward(const EmbeddingArgs& a, const void* dy, long long dy_stride, void* dtable,
                                    float scale, long long skip, bool has_skip, bool accumulate, int dtype,
                                    int out_dtype, void* workspace, cudaStream_t stream);

size_t ExpertSortWorkspace(long long n);
cudaError_t LaunchExpertSort(const void* ids, int ids64, long long n, int experts, int* slots, int* sources,
                             int* offsets, void* workspace, cudaStream_t stream);
cudaError_t LaunchExpertDispatch(const void* x, long long x_stride, const int* slots, const int* offsets,
                                 long long tokens, int top, int experts, long long h, void* rows, int dtype,
                                 cudaStream_t stream);
cudaError_t LaunchExpertCombine(const void* rows, const int* slots, const void* weights, int wdtype, long long tokens,
                                int top, long long h, void* y, long long y_stride, int dtype, cudaStream_t stream);
cudaError_t LaunchExpertCombineBackward(const void* dy, long long dy_stride, const void* rows, const int* slots,
                                        const int* offsets, const void* weights, int wdtype, long long tokens, int top,
                                        int experts, long long h, void* drows, void* dweights, int dtype,
                                        cudaStream_t stream);

}  // namespace bccl
