// head_api.cu -- the C ABI of the operators at the model's end
// (include/noetic/head.h): argument checks, the device of the call, and the
// host-array forms.

#include <cmath>

#include "../../include/noetic/head.h"
#include "nk_api.h"
#include "nk_head.h"

namespace {

// Its reciprocal has to be a normal f32 too.
void check_temperature(float t) { need(t >= 1e-30f && t <= 1e30f, "temperature must be within [1e-30, 1e30]"); }

constexpr double LOG2E_D = 1.4426950408889634074;

// ---------------------------------------------------------------- argument checks
void check_logits(const void *logits, int dtype, uint64_t rows, uint64_t vocab, uint64_t stride, float temperature) {
    check_dtype(dtype);
    check_temperature(temperature);
    need(vocab > 0, "an empty vocabulary");
    check_matrix(rows, vocab, stride, "logits");
    need(rows == 0 || logits, "null logits");
    check_aligned(logits, elem_size(dtype), "logits");
}

void check_logprobs(uint64_t rows, const uint32_t *targets, uint32_t top, const float *logprob, const float *entropy,
                    const float *stats, const uint32_t *top_ids, const float *top_logprobs) {
    need(top <= NK_MAX_TOP, "top is limited to NK_MAX_TOP");
    need(rows == 0 || !logprob || targets, "logprob needs targets");
    need(top > 0 || (!top_ids && !top_logprobs), "top is 0 and its arrays are not null");
    check_f32({targets, logprob, entropy, stats, top_ids, top_logprobs});
}

void check_logprobs_grad(uint64_t rows, const uint32_t *targets, const float *stats, const float *entropy,
                         const float *g_logprob, const float *g_entropy, const void *dlogits) {
    if (rows == 0) return;
    need(stats && dlogits, "null stats or dlogits");
    need(g_logprob || g_entropy, "g_logprob and g_entropy are both null");
    need(!g_logprob || targets, "g_logprob needs targets");
    need(!g_entropy || entropy, "g_entropy needs entropy");
    check_f32({targets, stats, entropy, g_logprob, g_entropy});
}

void check_distill(uint64_t rows, const uint32_t *ids, const void *teacher, int teacher_dtype, uint32_t n,
                   float temperature, const float *loss, const float *row_weight, float grad_scale, const void *dlogits) {
    check_dtype(teacher_dtype);
    need(n <= NK_MAX_TEACHER, "n_teacher is limited to NK_MAX_TEACHER");
    need(std::isfinite(grad_scale), "grad_scale must be finite");
    // Beyond these temperature^2 leaves the loss no digits of an f32.
    need(temperature >= 1e-4f && temperature <= 1e4f, "temperature must be within [1e-4, 1e4]");
    if (rows == 0) return;
    need(n == 0 || (ids && teacher), "null teacher arrays");
    need(loss || dlogits, "loss and dlogits are both null");
    check_aligned(teacher, elem_size(teacher_dtype), "teacher_logits");
    check_f32({ids, loss, row_weight});
}

void check_norm(int dtype, uint64_t rows, uint64_t width, float eps, int rms, const void *x, const void *y,
                const float *gain, const float *bias, const float *mean, const float *rstd) {
    check_dtype(dtype);
    need(width > 0, "an empty row");
    need(std::isfinite(eps) && eps >= 0.0f, "eps must be finite and not negative");
    need(!rms || (!bias && !mean), "RMSNorm has no mean and no bias");
    need(rows == 0 || (x && y), "null argument");
    check_aligned(x, elem_size(dtype), "x");
    check_aligned(y, elem_size(dtype), "y");
    check_f32({gain, bias, mean, rstd});
}

void check_norm_grad(int dtype, uint64_t rows, uint64_t width, int rms, const void *x, const void *dy, const void *dx,
                     const float *gain, const float *mean, const float *rstd, const float *dgain, const float *dbias) {
    check_dtype(dtype);
    need(width > 0, "an empty row");
    need(!rms || (!mean && !dbias), "RMSNorm has no mean and no bias");
    if (rows != 0) {
        need(x && dy && rstd && (rms || mean), "null argument");
        check_aligned(x, elem_size(dtype), "x");
        check_aligned(dy, elem_size(dtype), "dy");
        check_aligned(dx, elem_size(dtype), "dx");
    }
    check_f32({gain, mean, rstd, dgain, dbias});
}

}  // namespace

extern "C" {

nk_status nk_token_logprobs_device(const void *logits, int dtype, uint64_t rows, uint64_t vocab, uint64_t row_stride,
                                   const uint32_t *targets, float temperature, uint32_t top, float *logprob,
                                   float *entropy, float *stats, uint32_t *top_ids, float *top_logprobs,
                                   void *stream) {
    return guard("nk_token_logprobs", [&] {
        check_logits(logits, dtype, rows, vocab, row_stride, temperature);
        check_logprobs(rows, targets, top, logprob, entropy, stats, top_ids, top_logprobs);
        if (rows == 0 || !(logprob || entropy || stats || top_ids || top_logprobs)) return;
        check_apart({{logprob, rows * 4}, {entropy, rows * 4}, {stats, rows * 8}, {top_ids, rows * top * 4}, {top_logprobs, rows * top * 4}},
                    {matrix_span(logits, rows, vocab, row_stride, elem_size(dtype)), {targets, rows * 4}});
        OnDevice on({logits, targets, logprob, entropy, stats, top_ids, top_logprobs});
        nk::LogprobsArgs a{};
        a.logits = logits;
        a.rows = (int64_t)rows;
        a.stride = (int64_t)row_stride;
        a.vocab = (int)vocab;
        a.targets = targets;
        a.scale = (float)(LOG2E_D / temperature);
        a.inv_t = 1.0f / temperature;
        a.top = top_ids || top_logprobs ? (int)top : 0;
        a.logprob = logprob;
        a.entropy = entropy;
        a.stats = stats;
        a.top_ids = top_ids;
        a.top_logprobs = top_logprobs;
        cuda_check(nk::token_logprobs(a, dtype, (cudaStream_t)stream), "launch");
    });
}

nk_status nk_token_logprobs(const void *logits, int dtype, uint64_t rows, uint64_t vocab, const uint32_t *targets,
                            float temperature, uint32_t top, float *logprob, float *entropy, float *stats,
                            uint32_t *top_ids, float *top_logprobs, int device) {
    return guard("nk_token_logprobs", [&] {
        check_logits(logits, dtype, rows, vocab, vocab, temperature);
        check_logprobs(rows, targets, top, logprob, entropy, stats, top_ids, top_logprobs);
        if (rows == 0) return;
        if (targets) check_ids(targets, rows, vocab);
        HostCall h(device);
        const auto *dz = h.up(logits, rows * vocab * elem_size(dtype));
        const auto *dt = h.up(targets, rows * 4);
        auto *lp = h.room<float>(rows * 4, logprob), *en = h.room<float>(rows * 4, entropy);
        auto *st = h.room<float>(rows * 8, stats), *tl = h.room<float>(rows * top * 4, top_logprobs);
        auto *ti = h.room<uint32_t>(rows * top * 4, top_ids);
        nested(nk_token_logprobs_device(dz, dtype, rows, vocab, vocab, dt, temperature, top, lp, en, st, ti, tl, nullptr));
        h.down(logprob, lp, rows * 4);
        h.down(entropy, en, rows * 4);
        h.down(stats, st, rows * 8);
        h.down(top_ids, ti, rows * top * 4);
        h.down(top_logprobs, tl, rows * top * 4);
    });
}

nk_status nk_token_logprobs_backward_device(const void *logits, int dtype, uint64_t rows, uint64_t vocab,
                                            uint64_t row_stride, const uint32_t *targets, float temperature,
                                            const float *stats, const float *entropy, const float *g_logprob,
                                            const float *g_entropy, void *dlogits, uint64_t dlogits_stride,
                                            void *stream) {
    return guard("nk_token_logprobs_backward", [&] {
        check_logits(logits, dtype, rows, vocab, row_stride, temperature);
        check_logprobs_grad(rows, targets, stats, entropy, g_logprob, g_entropy, dlogits);
        if (rows == 0) return;
        check_matrix(rows, vocab, dlogits_stride, "dlogits");
        check_aligned(dlogits, elem_size(dtype), "dlogits");
        need(!overlap(logits, row_stride, dlogits, dlogits_stride, rows, vocab, elem_size(dtype)),
             "dlogits overlaps the logits");
        check_apart({matrix_span(dlogits, rows, vocab, dlogits_stride, elem_size(dtype))},
                    {{targets, rows * 4}, {stats, rows * 8}, {entropy, rows * 4}, {g_logprob, rows * 4}, {g_entropy, rows * 4}});
        OnDevice on({logits, targets, stats, entropy, g_logprob, g_entropy, dlogits});
        nk::LogprobsGradArgs a{};
        a.logits = logits;
        a.dlogits = dlogits;
        a.rows = (int64_t)rows;
        a.stride = (int64_t)row_stride;
        a.dstride = (int64_t)dlogits_stride;
        a.vocab = (int)vocab;
        a.targets = targets;
        a.scale = (float)(LOG2E_D / temperature);
        a.inv_t = 1.0f / temperature;
        a.stats = stats;
        a.entropy = entropy;
        a.g_logprob = g_logprob;
        a.g_entropy = g_entropy;
        cuda_check(nk::token_logprobs_backward(a, dtype, (cudaStream_t)stream), "launch");
    });
}

nk_status nk_token_logprobs_backward(const void *logits, int dtype, uint64_t rows, uint64_t vocab,
                                     const uint32_t *targets, float temperature, const float *stats,
                                     const float *entropy, const float *g_logprob, const float *g_entropy,
                                     void *dlogits, int device) {
    return guard("nk_token_logprobs_backward", [&] {
        check_logits(logits, dtype, rows, vocab, vocab, temperature);
        check_logprobs_grad(rows, targets, stats, entropy, g_logprob, g_entropy, dlogits);
        if (rows == 0) return;
        if (targets) check_ids(targets, rows, vocab);
        HostCall h(device);
        const size_t bytes = rows * vocab * elem_size(dtype);
        void *dz = (void *)h.up(logits, bytes);
        const auto *dt = h.up(targets, rows * 4);
        const auto *st = h.up(stats, rows * 8), *en = h.up(entropy, rows * 4);
        const auto *gl = h.up(g_logprob, rows * 4), *ge = h.up(g_entropy, rows * 4);
        nested(nk_token_logprobs_backward_device(dz, dtype, rows, vocab, vocab, dt, temperature, st, en, gl, ge, dz,
                                                 vocab, nullptr));
        h.down(dlogits, dz, bytes);
    });
}

nk_status nk_distill_device(const void *logits, int dtype, uint64_t rows, uint64_t vocab, uint64_t row_stride,
                            const uint32_t *teacher_ids, const void *teacher_logits, int teacher_dtype,
                            uint32_t n_teacher, float temperature, float *loss, const float *row_weight,
                            float grad_scale, void *dlogits, uint64_t dlogits_stride, void *stream) {
    return guard("nk_distill", [&] {
        check_logits(logits, dtype, rows, vocab, row_stride, temperature);
        check_distill(rows, teacher_ids, teacher_logits, teacher_dtype, n_teacher, temperature, loss, row_weight, grad_scale, dlogits);
        if (rows == 0) return;
        if (dlogits) {
            check_matrix(rows, vocab, dlogits_stride, "dlogits");
            check_aligned(dlogits, elem_size(dtype), "dlogits");
            need(!overlap(logits, row_stride, dlogits, dlogits_stride, rows, vocab, elem_size(dtype)),
                 "dlogits overlaps the logits");
        }
        const Span z = matrix_span(logits, rows, vocab, row_stride, elem_size(dtype));
        const Span ids{teacher_ids, rows * n_teacher * 4}, q{teacher_logits, rows * n_teacher * elem_size(teacher_dtype)};
        check_apart({{loss, rows * 4}}, {z});
        check_apart({{loss, rows * 4}, matrix_span(dlogits, rows, vocab, dlogits_stride, elem_size(dtype))},
                    {ids, q, {row_weight, rows * 4}});
        OnDevice on({logits, n_teacher ? teacher_ids : nullptr, n_teacher ? teacher_logits : nullptr, loss, row_weight, dlogits});
        nk::DistillArgs a{};
        a.logits = logits;
        a.dlogits = dlogits;
        a.rows = (int64_t)rows;
        a.stride = (int64_t)row_stride;
        a.dstride = (int64_t)dlogits_stride;
        a.vocab = (int)vocab;
        a.ids = teacher_ids;
        a.teacher = teacher_logits;
        a.teacher_dtype = teacher_dtype;
        a.n = (int)n_teacher;
        a.scale = (float)(LOG2E_D / temperature);
        a.inv_t = 1.0f / temperature;
        a.temperature = temperature;
        a.loss = loss;
        a.row_weight = row_weight;
        a.grad_scale = grad_scale;
        cuda_check(nk::distill(a, dtype, (cudaStream_t)stream), "launch");
    });
}

nk_status nk_distill(const void *logits, int dtype, uint64_t rows, uint64_t vocab, const uint32_t *teacher_ids,
                     const void *teacher_logits, int teacher_dtype, uint32_t n_teacher, float temperature,
                     float *loss, const float *row_weight, float grad_scale, void *dlogits, int device) {
    return guard("nk_distill", [&] {
        check_logits(logits, dtype, rows, vocab, vocab, temperature);
        check_distill(rows, teacher_ids, teacher_logits, teacher_dtype, n_teacher, temperature, loss, row_weight, grad_scale, dlogits);
        if (rows == 0) return;
        check_ids(teacher_ids, rows * n_teacher, vocab);
        HostCall h(device);
        const size_t bytes = rows * vocab * elem_size(dtype);
        void *dz = (void *)h.up(logits, bytes);
        const auto *ids = n_teacher ? h.up(teacher_ids, rows * n_teacher * 4) : nullptr;
        const auto *tl = n_teacher ? h.up(teacher_logits, rows * n_teacher * elem_size(teacher_dtype)) : nullptr;
        const auto *w = h.up(row_weight, rows * 4);
        auto *dl = h.room<float>(rows * 4, loss);
        nested(nk_distill_device(dz, dtype, rows, vocab, vocab, ids, tl, teacher_dtype, n_teacher, temperature, dl, w,
                                 grad_scale, dlogits ? dz : nullptr, vocab, nullptr));
        h.down(loss, dl, rows * 4);
        h.down(dlogits, dz, bytes);
    });
}

nk_status nk_layer_norm_device(const void *x, int dtype, uint64_t rows, uint64_t width, uint64_t x_stride,
                               const float *gain, const float *bias, float eps, int rms, void *y, uint64_t y_stride,
                               float *mean, float *rstd, void *stream) {
    return guard("nk_layer_norm", [&] {
        check_norm(dtype, rows, width, eps, rms, x, y, gain, bias, mean, rstd);
        check_matrix(rows, width, x_stride, "x");
        check_matrix(rows, width, y_stride, "y");
        if (rows == 0) return;
        need(!overlap(x, x_stride, y, y_stride, rows, width, elem_size(dtype)), "y overlaps x");
        const int es = elem_size(dtype);
        check_apart({{mean, rows * 4}, {rstd, rows * 4}}, {matrix_span(x, rows, width, x_stride, es)});
        check_apart({{mean, rows * 4}, {rstd, rows * 4}, matrix_span(y, rows, width, y_stride, es)}, {{gain, width * 4}, {bias, width * 4}});
        OnDevice on({x, gain, bias, y, mean, rstd});
        nk::NormArgs a{};
        a.x = x;
        a.y = y;
        a.rows = (int64_t)rows;
        a.x_stride = (int64_t)x_stride;
        a.y_stride = (int64_t)y_stride;
        a.width = (int)width;
        a.gain = gain;
        a.bias = bias;
        a.eps = eps;
        a.rms = rms != 0;
        a.mean = mean;
        a.rstd = rstd;
        cuda_check(nk::norm_rows(a, dtype, (cudaStream_t)stream), "launch");
    });
}

nk_status nk_layer_norm(const void *x, int dtype, uint64_t rows, uint64_t width, const float *gain, const float *bias,
                        float eps, int rms, void *y, float *mean, float *rstd, int device) {
    return guard("nk_layer_norm", [&] {
        check_norm(dtype, rows, width, eps, rms, x, y, gain, bias, mean, rstd);
        check_matrix(rows, width, width, "x");
        if (rows == 0) return;
        HostCall h(device);
        const size_t bytes = rows * width * elem_size(dtype);
        void *dx = (void *)h.up(x, bytes);
        const auto *g = h.up(gain, width * 4), *b = h.up(bias, width * 4);
        auto *dm = h.room<float>(rows * 4, mean), *dr = h.room<float>(rows * 4, rstd);
        nested(nk_layer_norm_device(dx, dtype, rows, width, width, g, b, eps, rms, dx, width, dm, dr, nullptr));
        h.down(y, dx, bytes);
        h.down(mean, dm, rows * 4);
        h.down(rstd, dr, rows * 4);
    });
}

nk_status nk_layer_norm_backward_workspace(uint64_t rows, uint64_t width, uint64_t *bytes) {
    return guard("nk_layer_norm_backward_workspace", [&] {
        need(bytes, "null argument");
        *bytes = 0;
        check_matrix(rows, width, width, "x");
        *bytes = nk::norm_backward_workspace_bytes((int64_t)rows, (int)width);
    });
}

nk_status nk_layer_norm_backward_device(const void *x, int dtype, uint64_t rows, uint64_t width, uint64_t x_stride,
                                        const float *gain, const float *mean, const float *rstd, int rms,
                                        const void *dy, uint64_t dy_stride, void *dx, uint64_t dx_stride,
                                        float *dgain, float *dbias, int accumulate, void *workspace,
                                        uint64_t workspace_bytes, void *stream) {
    return guard("nk_layer_norm_backward", [&] {
        check_norm_grad(dtype, rows, width, rms, x, dy, dx, gain, mean, rstd, dgain, dbias);
        check_matrix(rows, width, x_stride, "x");
        check_matrix(rows, width, dy_stride, "dy");
        if (dx) check_matrix(rows, width, dx_stride, "dx");
        if (!dx && !dgain && !dbias) return;
        if (dgain || dbias) {
            need(workspace, "dgain and dbias need a workspace");
            check_aligned(workspace, 16, "workspace");
            need(workspace_bytes >= nk::norm_backward_workspace_bytes((int64_t)rows, (int)width),
                 "the workspace is smaller than nk_layer_norm_backward_workspace says");
        }
        if (rows == 0 && !dgain && !dbias) return;
        if (rows && dx) {
            need(!overlap(dy, dy_stride, dx, dx_stride, rows, width, elem_size(dtype)), "dx overlaps dy");
            need(dx != x && !overlap(x, x_stride, dx, dx_stride, rows, width, elem_size(dtype)), "dx overlaps x");
        }
        const int es = elem_size(dtype);
        const Span dg{dgain, width * 4}, db{dbias, width * 4}, ws{dgain || dbias ? workspace : nullptr, nk::norm_backward_workspace_bytes((int64_t)rows, (int)width)};
        check_apart({dg, db, ws}, {matrix_span(x, rows, width, x_stride, es), matrix_span(dy, rows, width, dy_stride, es)});
        check_apart({dg, db, ws, matrix_span(dx, rows, width, dx_stride, es)}, {{gain, width * 4}, {mean, rows * 4}, {rstd, rows * 4}});
        const bool some = rows != 0;
        OnDevice on({some ? x : nullptr, some ? gain : nullptr, some ? mean : nullptr, some ? rstd : nullptr, some ? dy : nullptr,
                     some ? dx : nullptr, ws.p, dgain, dbias});
        nk::NormGradArgs a{};
        a.x = x;
        a.dy = dy;
        a.dx = dx;
        a.rows = (int64_t)rows;
        a.x_stride = (int64_t)x_stride;
        a.dy_stride = (int64_t)dy_stride;
        a.dx_stride = (int64_t)dx_stride;
        a.width = (int)width;
        a.gain = gain;
        a.mean = mean;
        a.rstd = rstd;
        a.rms = rms != 0;
        a.dgain = dgain;
        a.dbias = dbias;
        a.accumulate = accumulate != 0;
        a.workspace = (float *)workspace;
        cuda_check(nk::norm_backward(a, dtype, (cudaStream_t)stream), "launch");
    });
}

nk_status nk_layer_norm_backward(const void *x, int dtype, uint64_t rows, uint64_t width, const float *gain,
                                 const float *mean, const float *rstd, int rms, const void *dy, void *dx,
                                 float *dgain, float *dbias, int accumulate, int device) {
    return guard("nk_layer_norm_backward", [&] {
        check_norm_grad(dtype, rows, width, rms, x, dy, dx, gain, mean, rstd, dgain, dbias);
        check_matrix(rows, width, width, "x");
        if (!dx && !dgain && !dbias) return;
        HostCall h(device);
        const size_t bytes = rows * width * elem_size(dtype);
        const void *px = h.up(x, bytes);
        void *pdy = (void *)h.up(dy, bytes);
        const auto *g = h.up(gain, width * 4), *m = h.up(mean, rows * 4), *rs = h.up(rstd, rows * 4);
        auto *dg = h.up(dgain, width * 4), *db = h.up(dbias, width * 4);
        const size_t ws = nk::norm_backward_workspace_bytes((int64_t)rows, (int)width);
        nested(nk_layer_norm_backward_device(px, dtype, rows, width, width, g, m, rs, rms, pdy, width,
                                             dx ? pdy : nullptr, width, dg, db, accumulate,
                                             h.room<void>(ws, dg || db), ws, nullptr));
        if (rows) h.down(dx, pdy, bytes);
        h.down(dgain, dg, width * 4);
        h.down(dbias, db, width * 4);
    });
}

}  // extern "C"
