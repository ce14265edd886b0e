/*
 * noetic/train.h -- the end of a training step: cross entropy straight from
 * hidden rows and the vocabulary matrix, its gradients, and AdamW over all of a
 * model's tensors at once.
 *
 * These go beyond the reference crate, whose nearest parts are named beside
 * each.  Implemented by the same libnoetic_gpu.so; the status codes and
 * nk_last_error() of noetic_gpu.h apply, and so do the conventions of
 * noetic/head.h: devices and streams of the _device calls, nk_dtype, row
 * strides, token ids (0xFFFFFFFF: no token), results that do not depend on
 * scheduling, and refusals (NK_ERR_INVALID).  Calls that overlap on the GPU,
 * replays of captured graphs among them, need a workspace each, and a
 * nk_adamw_many each.
 */
#ifndef NOETIC_TRAIN_H
#define NOETIC_TRAIN_H

#include "head.h"

#ifdef __cplusplus
extern "C" {
#endif

#if defined(__GNUC__)
#pragma GCC visibility push(default)
#endif

/* Cross entropy of logits z = x w^T that are not kept (the logits product and
 * softmax_ce of Lm::loss, model.rs:209-234, autograd.rs:579-624): x [rows,
 * width], w [vocab, width] (the tied embedding), both of type `dtype`;
 *   loss[r]      log sum_j exp(z_j) - z[targets[r]]
 *   stats[r][2]  the row's maximum m and log sum_j exp(z_j - m): what the
 *                backward call needs
 * each nullable, not both.  A row whose target is no token is not read; its loss
 * and stats are 0.  A NaN or an infinity in a row of x makes the row's numbers
 * NaN; one in w those of every row, unless it makes a logit -infinity, which can
 * count as one of a token that is never chosen.  Products of 16-bit elements are
 * exact and their sums f32; f32 elements count with 22 bits at least, relative to
 * the largest of their row (for the gradients, of their matrix).  (-infinity cannot
 * mask a token here: a logit comes from w.)
 * workspace: nk_linear_ce_workspace bytes, 256-byte aligned.  Should a wait
 * between parts of the kernel ever run out (it has a limit of seconds, for a
 * broken device), the loss is NaN. */
nk_status nk_linear_ce_device(const void *x, int dtype, uint64_t rows, uint64_t width, uint64_t x_stride,
                              const void *w, uint64_t vocab, uint64_t w_stride, const uint32_t *targets, float *loss,
                              float *stats, void *workspace, uint64_t workspace_bytes, void *stream);
nk_status nk_linear_ce(const void *x, int dtype, uint64_t rows, uint64_t width, const void *w, uint64_t vocab,
                       const uint32_t *targets, float *loss, float *stats, int device);

/* The workspace of the call above (backward == 0) or below, with any number of rows up
 * to `rows`.  w: where the
 * matrix will be; what counts is its place within 128 bytes and its stride.  One
 * that does not start its rows on 16-byte boundaries is copied, and so is an f32
 * one, as two 16-bit parts.  One of 16 bits whose rows start on 16-byte but not on
 * 128-byte boundaries is copied from 1024 rows on (2048 without gradients), if the
 * workspace has the room that is asked for here; the size for a place on 128 bytes
 * (256, say) does for it too, and the call is up to 30% slower then, with the same
 * results. */
nk_status nk_linear_ce_workspace(int dtype, uint64_t rows, uint64_t width, uint64_t vocab, const void *w,
                                 uint64_t w_stride, int backward, uint64_t *bytes);

/* Its gradients: with p = exp(z - m - log sum) and
 *   G[r][j] = grad_scale row_weight[r] (p_j - [j = targets[r]]),
 *   dx = G w,  dw = G^T x,
 * those of grad_scale sum_r row_weight[r] loss[r].  stats is the forward call's;
 * row_weight null: 1.  The logits are computed again, a piece of the vocabulary
 * at a time.  dx (type of x) and dw (type of w, or f32: dw_dtype) are each
 * nullable, not both; accumulate != 0 adds to dw (dx is set).  Rows whose target
 * is no token, or whose weight is 0, are not read, have dx = 0 and add nothing
 * to dw.  Each element of G is rounded once to the type of x (f32: 22 bits) relative
 * to the largest finite weight (f16 and f32: floor 2^-38 of it); sums are f32, and an
 * f32 dw holds them.  A weight that is not finite breaks its row of dx, and dw.  After
 * a wait that ran out, what is not right is NaN.  dx and dw must not overlap x, w or
 * each other. */
nk_status nk_linear_ce_backward_device(const void *x, int dtype, uint64_t rows, uint64_t width, uint64_t x_stride,
                                       const void *w, uint64_t vocab, uint64_t w_stride, const uint32_t *targets,
                                       const float *stats, const float *row_weight, float grad_scale, void *dx,
                                       uint64_t dx_stride, void *dw, int dw_dtype, uint64_t dw_stride, int accumulate,
                                       void *workspace, uint64_t workspace_bytes, void *stream);
nk_status nk_linear_ce_backward(const void *x, int dtype, uint64_t rows, uint64_t width, const void *w, uint64_t vocab,
                                const uint32_t *targets, const float *stats, const float *row_weight, float grad_scale,
                                void *dx, void *dw, int dw_dtype, int accumulate, int device);

/* Test control of the failure path, for the calls that this host thread makes from
 * now on: in the product of the loss (1), of G (2) or of dx and dw (3) one copy is
 * left out (0: none, the default), so that the waits for it run out, which are
 * bounded at 2 ms then.  The call's loss, or what its gradients have from there on, is
 * NaN, never a sum that lacks a product; the next call is as any other.  (Calls of few
 * rows have no such product.) */
nk_status nk_linear_ce_withhold(int product);

/* Elements of a tensor that share a scale of the 8-bit moments. */
#define NK_ADAMW_BLOCK 256u

/* One parameter tensor of an AdamW step.  val: f32.  grad: grad_dtype.
 * state_bits 32: m and v are f32, the scales null.  state_bits 8: m and v hold a
 * byte for each element, m_scale and v_scale one f32 for each NK_ADAMW_BLOCK
 * elements (the last block can be short); a byte is an e4m3 number (4 exponent
 * and 3 fraction bits, at most 448) and stands for byte * scale: m itself, and
 * the square root of v.  All zero is the start of training in both.  copy
 * (nullable): receives val rounded to copy_dtype (NK_F16 or NK_BF16).  decay !=
 * 0: the weight decay applies (Param::decay). */
typedef struct nk_adamw_tensor {
    float *val;
    const void *grad;
    void *m, *v;
    float *m_scale, *v_scale;
    void *copy;
    uint64_t n;
    int grad_dtype, copy_dtype, state_bits, decay;
} nk_adamw_tensor;

/* The tensors of a model, registered once (device arrays of one device, which
 * stay where they are until the free; a tensor may be empty).  Outputs must not
 * overlap each other or a gradient.  Synchronous. */
typedef struct nk_adamw_many nk_adamw_many;
nk_status nk_adamw_many_create(const nk_adamw_tensor *tensors, uint64_t count, nk_adamw_many **out);
void nk_adamw_many_free(nk_adamw_many *many);

/* AdamW::step (optim.rs:33-72) of all of them in one launch, with gradients g =
 * grad c:  c = grad_scale, or, where max_norm > 0 and the norm of all grad_scale
 * grad is larger, grad_scale max_norm / norm.  With f32 gradients and moments
 * and c = 1 a tensor's result is nk_adamw_step's, bit for bit.  cfg->decay is not
 * read (each tensor has its own).  8-bit moments are read, stepped in f32 (with
 * a few roundings of 2^-23), used for this step's val, and rounded afterwards with a
 * new scale for the block; a v of 2^-126 or more does not become 0 (a smaller one
 * counts as 0), and |m| is kept up to 2^100.  A moment whose factor (b1, b2) is at most 0.95 is rounded to nearest; what
 * it forgets in a step is then about half a step of the grid, and it follows its
 * gradients as far as these, or the scale of its block, move it by more.  Above 0.95 it
 * is rounded up or down in proportion to where it lies, so that the mean of m, or of v,
 * is the formula's; which of the two goes by the element's number, val, g and cfg->t
 * alone, so the same call on the same arrays gives the same bytes.
 * norm (nullable, device): receives the norm.  bad (nullable, device): becomes 1
 * where an element's g, value or 8-bit moment is not finite; that element's val and
 * moments stay (8-bit moments: as far as the block's new scale holds them).
 * A norm that is not finite, with max_norm > 0: nothing changes, bad becomes 1.
 * A captured call repeats its cfg, grad_scale and max_norm in each replay. */
nk_status nk_adamw_many_step_device(nk_adamw_many *many, const nk_adamw_cfg *cfg, float grad_scale, float max_norm,
                                    float *norm, uint32_t *bad, void *stream);

/* The same for host arrays, once (norm nullable).  An element that is not finite
 * returns NK_ERR_INVALID with that element untouched and the others updated. */
nk_status nk_adamw_many_step(const nk_adamw_tensor *tensors, uint64_t count, const nk_adamw_cfg *cfg, float grad_scale,
                             float max_norm, float *norm, int device);

#if defined(__GNUC__)
#pragma GCC visibility pop
#endif

#ifdef __cplusplus
}
#endif
#endif /* NOETIC_TRAIN_H */
