/*
 * noetic/head.h -- operators at the model's end: log probabilities of given
 * tokens, the distillation loss, layer norm and RMSNorm, with gradients.
 *
 * These go beyond the reference crate, whose nearest parts are named beside
 * each: they score texts, train a student on a teacher's top logits and carry
 * the gradient back through the norm before the logits.  Implemented by the
 * same libnoetic_gpu.so; the status codes and nk_last_error() of
 * noetic_gpu.h apply.
 *
 * Conventions
 *   - Entry points whose name ends in _device take device pointers and a CUDA
 *     stream (cudaStream_t, NULL for the legacy default stream), do not
 *     synchronise or allocate, and can be captured into a CUDA graph after a
 *     first call on that device.  They run on the device that owns their arrays,
 *     whichever is current (managed memory alone: the current one); the stream
 *     has to belong to it.
 *     The others take contiguous host arrays and run on `device`.
 *   - dtype is an nk_dtype.  Sums, maxima and statistics are f32 at least;
 *     results are rounded once, on the way out.
 *   - Matrices are row-major with a row stride in elements (>= the width); an
 *     array only has to be aligned to its element.  Rows that start on 16-byte
 *     boundaries are read fastest.  Matrices of one call (logits and dlogits; x
 *     and y; x, dy and dx) should start their rows at the same places of 16
 *     bytes: equal strides, or strides that differ by multiples of 16 bytes.
 *     Otherwise 16-bit gradients take three times as long, and the norm's
 *     gradient, where dy starts elsewhere than x, five to nine times.  What lies
 *     between the rows is not touched.
 *   - A token id is a u32.  0xFFFFFFFF means "no token"; so does, on the device,
 *     every id that is not below the vocabulary size (the host forms refuse
 *     those).
 *   - Results do not depend on scheduling: the same call gives the same bits.
 *     How a row's sum is split goes by the number of rows, their strides and
 *     places and what is asked for, so the same row in another call can differ in
 *     its last bits.
 *   - NK_ERR_INVALID: a null array with a non-zero size, a pointer that is not
 *     device memory or not on the same device as the others, a misaligned one, a
 *     stride below the width, a size beyond the limits (rows <= 2^26, vocab and
 *     width <= 2^30, rows * stride <= 2^37), a temperature outside [1e-30, 1e30],
 *     an eps that is negative or not finite; on the device also an output that
 *     overlaps an input, other than as said below, or another output.
 */
#ifndef NOETIC_HEAD_H
#define NOETIC_HEAD_H

#include "../noetic_gpu.h"

#ifdef __cplusplus
extern "C" {
#endif

#if defined(__GNUC__)
#pragma GCC visibility push(default)
#endif

typedef enum nk_dtype { NK_F32 = 0, NK_F16 = 1, NK_BF16 = 2 } nk_dtype;

/* The most alternatives that one row can be asked for. */
#define NK_MAX_TOP 128u
/* The most entries that a teacher's row can have. */
#define NK_MAX_TEACHER 256u

/* Log probabilities of given tokens (the per-position form of softmax_ce,
 * autograd.rs:579-624), with p = softmax(logits / temperature) over `vocab`
 * columns of `rows` rows:
 *   logprob[r]     log p[targets[r]]
 *   entropy[r]     -sum_j p_j log p_j, in nats
 *   stats[r][2]    the row's maximum and log sum_j exp((z_j - maximum) /
 *                  temperature): what the backward call needs
 *   top_ids[r][top], top_logprobs[r][top]
 *                  the `top` (<= NK_MAX_TOP) most probable tokens, most
 *                  probable first, equal logits in the order of their ids
 * Any of the outputs can be null; targets can be null when logprob is.
 * A row whose target is no token is not read: its logprob, entropy and stats
 * are 0 and it has no alternatives (id 0xFFFFFFFF, -infinity), which is also
 * what fills the places beyond a row's logits above -infinity.  Masked logits
 * are -infinity.  In a row that has nothing else, logprob and stats are
 * -infinity and entropy is 0.  A NaN or +infinity makes the row's numbers NaN;
 * a NaN is no alternative.
 * In calls of up to 148 rows a sure token's log probability (near 0) keeps its
 * digits; beyond, log p is good to about 2^-24 of 1, as the sum 1 + rest is. */
nk_status nk_token_logprobs_device(const void *logits, int dtype, uint64_t rows, uint64_t vocab, uint64_t row_stride,
                                   const uint32_t *targets, float temperature, uint32_t top, float *logprob,
                                   float *entropy, float *stats, uint32_t *top_ids, float *top_logprobs,
                                   void *stream);
nk_status nk_token_logprobs(const void *logits, int dtype, uint64_t rows, uint64_t vocab, const uint32_t *targets,
                            float temperature, uint32_t top, float *logprob, float *entropy, float *stats,
                            uint32_t *top_ids, float *top_logprobs, int device);

/* The gradient of sum_r g_logprob[r] logprob[r] + g_entropy[r] entropy[r]:
 *   dlogits[r][j] = (g_logprob[r] ([j = targets[r]] - p_j)
 *                    - g_entropy[r] p_j (log p_j + entropy[r])) / temperature
 * stats and entropy are the forward call's.  g_logprob or g_entropy can be null
 * (not both); targets, g_logprob null: every row counts; entropy is read only
 * with g_entropy.  The gradient of softmax_ce's mean is g_logprob[r] = -1 / n.
 * Rows whose target is no token, and rows without a logit above -infinity, get
 * zeros.  dlogits has the type of the logits and can be the same array with the
 * same stride; it must not overlap them otherwise. */
nk_status nk_token_logprobs_backward_device(const void *logits, int dtype, uint64_t rows, uint64_t vocab,
                                            uint64_t row_stride, const uint32_t *targets, float temperature,
                                            const float *stats, const float *entropy, const float *g_logprob,
                                            const float *g_entropy, void *dlogits, uint64_t dlogits_stride,
                                            void *stream);
nk_status nk_token_logprobs_backward(const void *logits, int dtype, uint64_t rows, uint64_t vocab,
                                     const uint32_t *targets, float temperature, const float *stats,
                                     const float *entropy, const float *g_logprob, const float *g_entropy,
                                     void *dlogits, int device);

/* Distillation from a teacher's top logits.  A row of the teacher is n_teacher
 * (<= NK_MAX_TEACHER) ids and their logits or log probabilities (they are
 * normalised here: q = softmax(teacher / temperature) over the row's entries;
 * an id that is no token, or a logit of -infinity, is no entry).  With p the
 * student's softmax(logits / temperature) over the vocabulary,
 *   loss[r] = temperature^2 sum_i q_i (log q_i - log p[id_i])
 *   dlogits[r][j] = grad_scale row_weight[r] temperature (p_j - sum_{i: id_i = j} q_i)
 * which is the gradient of grad_scale sum_r row_weight[r] loss[r].  row_weight
 * null: 1.  dlogits null: the loss alone (summed in another order in long rows,
 * so its last bits can differ); loss null: the gradient alone.  The logits are
 * read once for both.  A row without entries is not read: its loss
 * and gradient are 0.  A row of weight 0 has gradient 0.  Where the student has
 * no logit above -infinity the loss is infinity and the gradient 0.  An id may
 * stand in a row more than once (its shares add up).  dlogits has the type of
 * the logits and can be the same array with the same stride.  The temperature is
 * limited to [1e-4, 1e4] (the loss comes with an error of about 1e-7 temperature^2). */
nk_status nk_distill_device(const void *logits, int dtype, uint64_t rows, uint64_t vocab, uint64_t row_stride,
                            const uint32_t *teacher_ids, const void *teacher_logits, int teacher_dtype,
                            uint32_t n_teacher, float temperature, float *loss, const float *row_weight,
                            float grad_scale, void *dlogits, uint64_t dlogits_stride, void *stream);
nk_status nk_distill(const void *logits, int dtype, uint64_t rows, uint64_t vocab, const uint32_t *teacher_ids,
                     const void *teacher_logits, int teacher_dtype, uint32_t n_teacher, float temperature,
                     float *loss, const float *row_weight, float grad_scale, void *dlogits, int device);

/* Layer norm of each row, or with rms != 0 the model's RMSNorm (rms_norm_vec,
 * tensor.rs:298-312):
 *   y = (x - mean) rstd gain + bias,  rstd = 1 / sqrt(mean((x - mean)^2) + eps)
 * rms: mean is 0 and `mean` and `bias` must be null.  gain (null: 1) and bias
 * (null: 0) are f32.  y has the type of x and can be the same array with the
 * same stride.  mean and rstd (each nullable) are what the backward call needs. */
nk_status nk_layer_norm_device(const void *x, int dtype, uint64_t rows, uint64_t width, uint64_t x_stride,
                               const float *gain, const float *bias, float eps, int rms, void *y, uint64_t y_stride,
                               float *mean, float *rstd, void *stream);
nk_status nk_layer_norm(const void *x, int dtype, uint64_t rows, uint64_t width, const float *gain, const float *bias,
                        float eps, int rms, void *y, float *mean, float *rstd, int device);

/* Its gradients: with c = dy gain and n = (x - mean) rstd,
 *   dx = rstd (c - mean(c) - n mean(c n))   (rms: without mean(c))
 *   dgain = sum over rows of dy n,  dbias = sum over rows of dy
 * dx, dgain and dbias are each nullable; dx can be the same array as dy, with
 * the same stride; accumulate != 0 adds to dgain and dbias instead of setting
 * them (dx is set).  The sums over rows, in f32 (a term passes through at most
 * rows / 32 + 64 additions), are split and joined in a fixed order through
 * `workspace` (of nk_layer_norm_backward_workspace bytes, 16-byte aligned; not
 * needed without dgain and dbias): calls that overlap on the GPU, replays of
 * captured graphs among them, need a workspace each. */
nk_status nk_layer_norm_backward_workspace(uint64_t rows, uint64_t width, uint64_t *bytes);
nk_status nk_layer_norm_backward_device(const void *x, int dtype, uint64_t rows, uint64_t width, uint64_t x_stride,
                                        const float *gain, const float *mean, const float *rstd, int rms,
                                        const void *dy, uint64_t dy_stride, void *dx, uint64_t dx_stride,
                                        float *dgain, float *dbias, int accumulate, void *workspace,
                                        uint64_t workspace_bytes, void *stream);
nk_status nk_layer_norm_backward(const void *x, int dtype, uint64_t rows, uint64_t width, const float *gain,
                                 const float *mean, const float *rstd, int rms, const void *dy, void *dx,
                                 float *dgain, float *dbias, int accumulate, int device);

/* The scores of whole texts: the forward of nk_model_loss (model.rs:209-226)
 * over `batch` sequences of `t` tokens, then nk_token_logprobs of its logits at
 * temperature 1.  ids and targets: host [batch * t], sequence-major; logprob,
 * entropy [batch * t], top_ids and top_logprobs [batch * t, top]: host, each
 * nullable.  Positions whose target is 0xFFFFFFFF have no scores, as above.
 * A text's scores beside other texts, or cut elsewhere, can differ in the last
 * digits (see nk_token_logprobs; the logits' product, too, goes by its rows).
 * Runs on a scratch decoder, as nk_model_loss does. */
nk_status nk_model_score(nk_model *model, const uint32_t *ids, const uint32_t *targets, uint32_t batch, uint32_t t,
                         uint32_t top, float *logprob, float *entropy, uint32_t *top_ids, float *top_logprobs);

#if defined(__GNUC__)
#pragma GCC visibility pop
#endif

#ifdef __cplusplus
}
#endif
#endif /* NOETIC_HEAD_H */
