// C interface of the compute operators (see bccl/ops.h): argument checks, then the launchers.
#include "bccl/ops.h"

#include "core/logger.h"
#include "kernels/ops.h"

namespace {

constexpr int kF32 = 0, kI32 = 2, kI64 = 3, kBF16 = 4, kF16 = 5;
constexpr int64_t kMaxWidth = 1 << 23;       // elements of a row
constexpr int64_t kMaxRows = int64_t{1} << 40;  // rows of an operand: offsets stay within 64 bits

bool FloatType(int d) { return d == kF32 || d == kBF16 || d == kF16; }
bool SameOrF32(int w, int d) { return w == d || w == kF32; }
bool IndexType(int d) { return d == kI32 || d == kI64; }
size_t SizeOf(int d) { return d == kF32 || d == kI32 ? 4 : d == kI64 ? 8 : 2; }
bool Aligned(const void* p, size_t size) { return (reinterpret_cast<uintptr_t>(p) & (size - 1)) == 0; }

// A 2-D operand: there unless it is empty, elements aligned, rows not overlapping when written.
bool Rows(const void* p, int64_t rows, int64_t h, int64_t stride, int dtype, bool written) {
    if (rows == 0) return true;
    return p != nullptr && Aligned(p, SizeOf(dtype)) && stride >= 0 && stride < kMaxRows &&
           (!written || rows == 1 || stride >= h);
}

int Bad(const char* op, const char* what) {
    LOG_ERROR("%s: %s", op, what);
    return 1;
}
int Launched(const char* op, cudaError_t e) {
    if (e == cudaSuccess) return 0;
    LOG_ERROR("%s: launch failed: %s", op, cudaGetErrorString(e));
    return 1;
}
cudaStream_t Stream(void* s) { return static_cast<cudaStream_t>(s); }

}  // namespace

extern "C" {

int bcclGradSquares(const void* const* grads, const size_t* counts, int n, int dtype, int accumulate, double* sum,
                    void* workspace, size_t workspace_bytes, void* stream) {
    const char* op = "grad squares";
    if (n < 0 || (n > 0 && (grads == nullptr || counts == nullptr))) return Bad(op, "invalid tensor list");
    if (!FloatType(dtype)) return Bad(op, "invalid dtype (f32, bf16, f16)");
    if (sum == nullptr || !Aligned(sum, 8)) return Bad(op, "sum must be a double");
    for (int i = 0; i < n; ++i)
        if (counts[i] > 0 && (grads[i] == nullptr || !Aligned(grads[i], SizeOf(dtype))))
            return Bad(op, "null or misaligned tensor");
    if (workspace == nullptr || !Aligned(workspace, 16) ||
        workspace_bytes < bccl::GradSquaresWorkspace(grads, counts, n, dtype))
        return Bad(op, "workspace too small or misaligned");
    return Launched(op, bccl::LaunchGradSquares(grads, counts, n, dtype, accumulate != 0, sum, workspace, Stream(stream)));
}

int bcclGradClip(const void* const* grads, void* const* outs, const size_t* counts, int n, int dtype, int out_dtype,
                 const double* sum, float max_norm, float eps, float* norm, void* stream) {
    const char* op = "grad clip";
    if (n < 0 || (n > 0 && (grads == nullptr || outs == nullptr || counts == nullptr)))
        return Bad(op, "invalid tensor list");
    if (!FloatType(dtype) || !SameOrF32(out_dtype, dtype)) return Bad(op, "invalid dtypes (out: the gradients' or f32)");
    if (sum == nullptr || !Aligned(sum, 8)) return Bad(op, "sum must be a double");
    if (!(max_norm >= 0.0f) || !(eps >= 0.0f)) return Bad(op, "max_norm and eps must not be negative or NaN");
    for (int i = 0; i < n; ++i) {
        if (counts[i] == 0) continue;
        if (grads[i] == nullptr || outs[i] == nullptr || !Aligned(grads[i], SizeOf(dtype)) ||
            !Aligned(outs[i], SizeOf(out_dtype)))
            return Bad(op, "null or misaligned tensor");
        if (grads[i] == outs[i] && dtype != out_dtype) return Bad(op, "in place needs one dtype");
    }
    return Launched(op, bccl::LaunchGradClip(grads, outs, counts, n, dtype, out_dtype, sum, max_norm, eps, norm,
                                             Stream(stream)));
}

int bcclNormForward(int kind, const void* x, int64_t x_stride, const void* weight, const void* bias, void* y,
                    int64_t y_stride, float* mean, float* rstd, int64_t rows, int64_t h, float eps, int dtype, int wdtype,
                    void* stream) {
    const char* op = kind == 0 ? "layer norm" : "rms norm";
    if (kind != 0 && kind != 1) return Bad("norm", "kind is 0 (layer norm) or 1 (rms norm)");
    if (!FloatType(dtype) || !SameOrF32(wdtype, dtype)) return Bad(op, "invalid dtypes (weight: the input's or f32)");
    if (rows < 0 || rows > kMaxRows || h < 1 || h > kMaxWidth) return Bad(op, "invalid shape");
    if (!(eps >= 0.0f)) return Bad(op, "eps must not be negative or NaN");
    if (!Rows(x, rows, h, x_stride, dtype, false) || !Rows(y, rows, h, y_stride, dtype, true))
        return Bad(op, "invalid input or output");
    if ((kind == 1 && bias != nullptr) || !Aligned(weight, SizeOf(wdtype)) || !Aligned(bias, SizeOf(wdtype)))
        return Bad(op, "invalid weight or bias");
    if (rows > 0 && (rstd == nullptr || (kind == 0 && mean == nullptr))) return Bad(op, "statistics are missing");
    const bccl::NormForwardArgs a{x, x_stride, weight, bias, y, y_stride, mean, rstd, rows, h, eps};
    return Launched(op, bccl::LaunchNormForward(kind == 0, a, dtype, wdtype, Stream(stream)));
}

size_t bcclNormBackwardWorkspace(int kind, int64_t rows, int64_t h, int dtype) {
    if (rows < 1 || rows > kMaxRows || h < 1 || h > kMaxWidth || !FloatType(dtype)) return 0;
    return bccl::NormBackwardWorkspace(kind == 0, rows, h, dtype);
}

int bcclNormBackward(int kind, const void* dy, int64_t dy_stride, const void* x, int64_t x_stride, const float* mean,
                     const float* rstd, const void* weight, void* dx, int64_t dx_stride, void* dweight, void* dbias,
                     int64_t rows, int64_t h, int dtype, int wdtype, void* workspace, size_t workspace_bytes,
                     void* stream) {
    const char* op = kind == 0 ? "layer norm backward" : "rms norm backward";
    if (kind != 0 && kind != 1) return Bad("norm backward", "kind is 0 (layer norm) or 1 (rms norm)");
    if (!FloatType(dtype) || !SameOrF32(wdtype, dtype)) return Bad(op, "invalid dtypes (weight: the input's or f32)");
    if (rows < 0 || rows > kMaxRows || h < 1 || h > kMaxWidth) return Bad(op, "invalid shape");
    if (!Rows(x, rows, h, x_stride, dtype, false) || !Rows(dy, rows, h, dy_stride, dtype, false) ||
        !Rows(dx, rows, h, dx_stride, dtype, true))
        return Bad(op, "invalid input or output");
    if ((kind == 1 && dbias != nullptr) || !Aligned(weight, SizeOf(wdtype)) || !Aligned(dweight, SizeOf(wdtype)) ||
        !Aligned(dbias, SizeOf(wdtype)))
        return Bad(op, "invalid weight or weight gradient");
    if (rows > 0 && (rstd == nullptr || (kind == 0 && mean == nullptr))) return Bad(op, "statistics are missing");
    if ((dweight != nullptr || dbias != nullptr) && rows > 0 &&
        (workspace == nullptr || !Aligned(workspace, 16) ||
         workspace_bytes < bccl::NormBackwardWorkspace(kind == 0, rows, h, dtype)))
        return Bad(op, "workspace too small or misaligned");
    bccl::NormBackwardArgs a{dy, dy_stride, x, x_stride, mean, rstd, weight, dx, dx_stride, dweight, dbias,
                             static_cast<float*>(workspace), rows, h};
    return Launched(op, bccl::LaunchNormBackward(kind == 0, a, dtype, wdtype, Stream(stream)));
}

int bcclEmbeddingForward(const void* ids, int ids_dtype, int64_t n, const void* table, int64_t table_stride, int64_t rows,
                         int64_t h, int64_t first_row, float scale, void* out, int64_t out_stride, int dtype,
                         void* stream) {
    const char* op = "embedding";
    if (!FloatType(dtype) || !IndexType(ids_dtype)) return Bad(op, "invalid dtypes");
    if (n < 0 || n > INT32_MAX || rows < 0 || rows > INT32_MAX - 1 || h < 1 || h > kMaxWidth || first_row < 0)
        return Bad(op, "invalid shape");
    if (n > 0 && (ids == nullptr || !Aligned(ids, SizeOf(ids_dtype)))) return Bad(op, "invalid ids");
    if (!Rows(table, rows, h, table_stride, dtype, false) || !Rows(out, n, h, out_stride, dtype, true))
        return Bad(op, "invalid table or output");
    const bccl::EmbeddingArgs a{ids, ids_dtype == kI64, n, rows, h, first_row};
    return Launched(op, bccl::LaunchEmbeddingForward(a, table, table_stride, scale, out, out_stride, dtype,
                                                     Stream(stream)));
}

size_t bcclEmbeddingBackwardWorkspace(int64_t n, int64_t rows, int64_t h) {
    if (n < 1 || n > INT32_MAX || rows < 0 || rows > INT32_MAX - 1 || h < 1 || h > kMaxWidth) return 0;
    return bccl::EmbeddingBackwardWorkspace(n, h);
}

int bcclEmbeddingBackward(const void* dy, int64_t dy_stride, const void* ids, int ids_dtype, int64_t n, void* dtable,
                          int64_t rows, int64_t h, int64_t first_row, float scale, int64_t skip_id, int has_skip,
                          int accumulate, int dtype, int out_dtype, void* workspace, size_t workspace_bytes,
                          void* stream) {
    const char* op = "embedding backward";
    if (!FloatType(dtype) || !SameOrF32(out_dtype, dtype) || !IndexType(ids_dtype)) return Bad(op, "invalid dtypes");
    if (n < 0 || n > INT32_MAX || rows < 0 || rows > INT32_MAX - 1 || h < 1 || h > kMaxWidth || first_row < 0)
        return Bad(op, "invalid shape");
    if (n > 0 && (ids == nullptr || !Aligned(ids, SizeOf(ids_dtype)))) return Bad(op, "invalid ids");
    if (!Rows(dy, n, h, dy_stride, dtype, false) || !Rows(dtable, rows, h, h, out_dtype, true))
        return Bad(op, "invalid gradient");
    if (n > 0 && rows > 0 &&
        (workspace == nullptr || !Aligned(workspace, 16) ||
         workspace_bytes < bccl::EmbeddingBackwardWorkspace(n, h)))
        return Bad(op, "workspace too small or misaligned");
    const bccl::EmbeddingArgs a{ids, ids_dtype == kI64, n, rows, h, first_row};
    return Launched(op, bccl::LaunchEmbeddingBackward(a, dy, dy_stride, dtable, scale, skip_id, has_skip != 0,
                                                      accumulate != 0, dtype, out_dtype, workspace, Stream(stream)));
}

namespace {
bool ExpertShape(int64_t tokens, int top) {
    return tokens >= 0 && top >= 1 && top <= BCCL_MAX_TOP && tokens <= INT32_MAX / top;
}
bool Experts(int experts) { return experts >= 1 && experts <= BCCL_MAX_EXPERTS; }
}  // namespace

size_t bcclExpertSortWorkspace(int64_t tokens, int top) {
    return ExpertShape(tokens, top) ? bccl::ExpertSortWorkspace(tokens * top) : 0;
}

int bcclExpertSort(const void* ids, int ids_dtype, int64_t tokens, int top, int experts, int32_t* slots, int32_t* sources,
                   int32_t* offsets, void* workspace, size_t workspace_bytes, void* stream) {
    const char* op = "expert sort";
    if (!IndexType(ids_dtype)) return Bad(op, "ids are int32 or int64");
    if (!ExpertShape(tokens, top) || !Experts(experts)) return Bad(op, "invalid shape (top <= 64, experts <= 1023)");
    if (offsets == nullptr || (tokens > 0 && (ids == nullptr || slots == nullptr || sources == nullptr ||
                                              !Aligned(ids, SizeOf(ids_dtype)))))
        return Bad(op, "null or misaligned array");
    const size_t need = bccl::ExpertSortWorkspace(tokens * top);
    if (need > 0 && (workspace == nullptr || !Aligned(workspace, 16) || workspace_bytes < need))
        return Bad(op, "workspace too small or misaligned");
    return Launched(op, bccl::LaunchExpertSort(ids, ids_dtype == kI64, tokens * top, experts, slots, sources, offsets,
                                               workspace, Stream(stream)));
}

int bcclExpertDispatch(const void* x, int64_t x_stride, const int32_t* slots, const int32_t* offsets, int64_t tokens,
                       int top, int experts, int64_t h, void* rows, int dtype, void* stream) {
    const char* op = "expert dispatch";
    if (!FloatType(dtype)) return Bad(op, "invalid dtype");
    if (!ExpertShape(tokens, top) || !Experts(experts) || h < 1 || h > kMaxWidth) return Bad(op, "invalid shape");
    if (!Rows(x, tokens, h, x_stride, dtype, false) || !Rows(rows, tokens * top, h, h, dtype, true) ||
        (tokens > 0 && (slots == nullptr || offsets == nullptr)))
        return Bad(op, "null or misaligned array");
    return Launched(op, bccl::LaunchExpertDispatch(x, x_stride, slots, offsets, tokens, top, experts, h, rows, dtype,
                                                   Stream(stream)));
}

int bcclExpertCombine(const void* rows, const int32_t* slots, const void* weights, int wdtype, int64_t tokens, int top,
                      int64_t h, void* y, int64_t y_stride, int dtype, void* stream) {
    const char* op = "expert combine";
    if (!FloatType(dtype) || !SameOrF32(wdtype, dtype)) return Bad(op, "invalid dtypes (weights: the rows' or f32)");
    if (!ExpertShape(tokens, top) || h < 1 || h > kMaxWidth) return Bad(op, "invalid shape");
    if (!Rows(rows, tokens * top, h, h, dtype, false) || !Rows(y, tokens, h, y_stride, dtype, true) ||
        (tokens > 0 && slots == nullptr) || !Aligned(weights, SizeOf(wdtype)))
        return Bad(op, "null or misaligned array");
    return Launched(op, bccl::LaunchExpertCombine(rows, slots, weights, wdtype, tokens, top, h, y, y_stride, dtype,
                                                  Stream(stream)));
}

int bcclExpertCombineBackward(const void* dy, int64_t dy_stride, const void* rows, const int32_t* slots,
                              const int32_t* offsets, const void* weights, int wdtype, int64_t tokens, int top, int experts,
                              int64_t h, void* drows, void* dweights, int dtype, void* stream) {
    const char* op = "expert combine backward";
    if (!FloatType(dtype) || !SameOrF32(wdtype, dtype)) return Bad(op, "invalid dtypes (weights: the rows' or f32)");
    if (!ExpertShape(tokens, top) || !Experts(experts) || h < 1 || h > kMaxWidth) return Bad(op, "invalid shape");
    if (!Rows(dy, tokens, h, dy_stride, dtype, false) ||
        (drows != nullptr && !Rows(drows, tokens * top, h, h, dtype, true)) ||
        (dweights != nullptr && !Rows(rows, tokens * top, h, h, dtype, false)) ||
        (tokens > 0 && (slots == nullptr || offsets == nullptr)) || !Aligned(weights, SizeOf(wdtype)) ||
        !Aligned(dweights, SizeOf(wdtype)))
        return Bad(op, "null or misaligned array");
    if (drows == nullptr && dweights == nullptr) return 0;
    return Launched(op, bccl::LaunchExpertCombineBackward(dy, dy_stride, rows, slots, offsets, weights, wdtype, tokens, top,
                                                          experts, h, drows, dweights, dtype, Stream(stream)));
}

}  // extern "C"
