// nk_head.h -- kernel launchers of the operators at the model's end
// (include/noetic/head.h).  Arguments are checked by the callers in
// head_api.cu; strides are in elements.
#pragma once

#include <cstdint>
#include <cuda_runtime.h>

namespace nk {

struct LogprobsArgs {
    const void *logits;
    int64_t rows, stride;
    int vocab;
    const uint32_t *targets;  // nullable
    float scale;              // log2(e) / temperature
    float inv_t;              // 1 / temperature
    int top;
    float *logprob, *entropy, *stats;  // each nullable
    uint32_t *top_ids;                 // nullable
    float *top_logprobs;               // nullable
};
cudaError_t token_logprobs(const LogprobsArgs &a, int dtype, cudaStream_t st);

struct LogprobsGradArgs {
    const void *logits;
    void *dlogits;
    int64_t rows, stride, dstride;
    int vocab;
    const uint32_t *targets;  // nullable
    float scale, inv_t;
    const float *stats, *entropy, *g_logprob, *g_entropy;
};
cudaError_t token_logprobs_backward(const LogprobsGradArgs &a, int dtype, cudaStream_t st);

struct DistillArgs {
    const void *logits;
    void *dlogits;  // nullable
    int64_t rows, stride, dstride;
    int vocab;
    const uint32_t *ids;  // [rows][n]
    const void *teacher;  // [rows][n]
    int teacher_dtype, n;
    float scale, inv_t, temperature;
    float *loss;              // nullable
    const float *row_weight;  // nullable
    float grad_scale;
};
cudaError_t distill(const DistillArgs &a, int dtype, cudaStream_t st);

struct NormArgs {
    const void *x;
    void *y;
    int64_t rows, x_stride, y_stride;
    int width;
    const float *gain, *bias;  // each nullable
    float eps;
    int rms;
    float *mean, *rstd;  // each nullable
};
cudaError_t norm_rows(const NormArgs &a, int dtype, cudaStream_t st);

struct NormGradArgs {
    const void *x, *dy;
    void *dx;  // nullable
    int64_t rows, x_stride, dy_stride, dx_stride;
    int width;
    const float *gain, *mean, *rstd;  // gain nullable; mean null for rms
    int rms;
    float *dgain, *dbias;  // each nullable
    int accumulate;
    float *workspace;
};
cudaError_t norm_backward(const NormGradArgs &a, int dtype, cudaStream_t st);
size_t norm_backward_workspace_bytes(int64_t rows, int width);

}  // namespace nk
