// nk_train.h -- kernel launchers of the operators at a training step's end
// (include/noetic/train.h).  Arguments are checked by the callers in
// train_api.cu; strides are in elements.
#pragma once

#include <cstddef>
#include <cstdint>
#include <cuda_runtime.h>

#include "../../include/noetic/train.h"
#include "nk_kernels.h"

namespace nk {

// ---- AdamW over many tensors (adamw_many.cu)
// Part of a tensor: a model's chunks (10 to 20 thousand of a large one) are walked by a
// persistent grid, so one launch serves tensors of any number and size.
struct AdamwChunk {
    uint32_t tensor, n;  // n <= the plan's chunk size
    uint64_t first;      // element, a multiple of NK_ADAMW_BLOCK
};

struct AdamwMany {
    const nk_adamw_tensor *tensors;  // device
    const AdamwChunk *chunks;        // device: [0, n_chunks32) of 32-bit moments, then those of 8-bit ones
    uint32_t n_chunks, n_chunks32;
    double *partial;   // device [adamw_partials]: sums of squares
    uint32_t *ticket;  // device, 0 between calls
    float *clip;       // device [2]: the factor of the gradients; 0 or 1: whether the step runs
};
// How many elements a chunk should have, of `total` with moments of `bits`, and how
// many partial sums the norm leaves at most.
uint32_t adamw_chunk_elements(uint64_t total, int sms, int bits);
uint32_t adamw_partials(int sms);
// clip[0] = grad_scale * min(1, max_norm / norm), with the norm also to *norm (nullable).
cudaError_t adamw_many_norm(const AdamwMany &p, float grad_scale, float max_norm, float *norm, uint32_t *bad,
                            int sms, cudaStream_t st);
// with_clip: the factor and the decision come from p.clip; else the factor is grad_scale.
// t: the step's counter, for what is rounded by chance.
cudaError_t adamw_many_step(const AdamwMany &p, const AdamwParams &a, uint32_t t, float grad_scale, bool with_clip, uint32_t *bad,
                            int sms, cudaStream_t st);

// ---- cross entropy from hidden rows (linear_ce.cu)
struct LinearCeArgs {
    const void *x, *w;
    int dtype;
    int64_t rows, x_stride, w_stride;
    int width, vocab;
    const uint32_t *targets;
    // forward
    float *loss, *stats;  // each nullable
    // backward
    const float *in_stats, *row_weight;  // row_weight nullable
    float grad_scale;
    void *dx, *dw;  // each nullable
    int64_t dx_stride, dw_stride;
    int dw_dtype, accumulate;
    void *workspace;
    bool copy_lines;
};
// copy_lines: with room for a copy of a w that is not on 128-byte lines, where one pays.
size_t linear_ce_workspace_bytes(int dtype, int64_t rows, int width, int vocab, const void *w, int64_t w_stride,
                                 bool backward, bool copy_lines);
void linear_ce_withhold(int product);  // nk_linear_ce_withhold
// What calls of up to `rows` rows take at most.
size_t linear_ce_most_workspace_bytes(int dtype, int64_t rows, int width, int vocab, const void *w, int64_t w_stride,
                                      bool backward);
cudaError_t linear_ce(const LinearCeArgs &a, int sms, cudaStream_t st);
cudaError_t linear_ce_backward(const LinearCeArgs &a, int sms, cudaStream_t st);

}  // namespace nk
