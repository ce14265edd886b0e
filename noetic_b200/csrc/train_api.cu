// train_api.cu -- the C ABI of the operators at a training step's end
// (include/noetic/train.h): argument checks, the device of the call, and the
// host-array forms.

#include <algorithm>
#include <cmath>
#include <memory>

#include "../../include/noetic/train.h"
#include "nk_api.h"
#include "nk_train.h"

struct nk_adamw_many {
    nk::AdamwMany plan{};
    void *room = nullptr;  // device: all of the plan's arrays
    int device = -1, sms = 1;
};

namespace {

int sm_count() {
    int dev = 0, n = 0;
    cuda_check(cudaGetDevice(&dev), "cudaGetDevice");
    cuda_check(cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev), "cudaDeviceGetAttribute");
    return n > 0 ? n : 1;
}

// ---------------------------------------------------------------- cross entropy
void check_linear_ce(int dtype, uint64_t rows, uint64_t width, uint64_t x_stride, uint64_t vocab, uint64_t w_stride,
                     const void *x, const void *w, const uint32_t *targets) {
    check_dtype(dtype);
    need(width > 0, "an empty row");
    need(vocab > 0, "an empty vocabulary");
    check_matrix(rows, width, x_stride, "x");
    // (The vocabulary is a number of rows here, and a width in head.h: the smaller limit.)
    check_matrix(vocab, width, w_stride, "w");
    need(width <= (1u << 24), "the width is limited to 2^24");
    uint64_t n = 0;
    need(nk::checked_mul(rows, vocab, n), "rows * vocab is limited to 2^37");
    need(w, "null w");
    need(rows == 0 || (x && targets), "null x or targets");
    check_aligned(x, elem_size(dtype), "x");
    check_aligned(w, elem_size(dtype), "w");
    check_f32({targets});
}

// The bytes that a call takes of its workspace.  One without room for a copy of w that only
// makes the call faster will do: the sizes for a w on 128-byte lines serve any on 16 bytes.
uint64_t check_workspace(int dtype, uint64_t rows, uint64_t width, uint64_t vocab, const void *w, uint64_t w_stride, bool backward,
                         const void *workspace, uint64_t have, bool &copy_lines) {
    need(workspace, "null workspace");
    check_aligned(workspace, 256, "workspace");
    uint64_t bytes = 0;
    for (const bool lines : {true, false}) {
        copy_lines = lines;
        bytes = nk::linear_ce_workspace_bytes(dtype, (int64_t)rows, (int)width, (int)vocab, w, (int64_t)w_stride, backward, lines);
        if (have >= bytes) return bytes;
    }
    fail(NK_ERR_INVALID, "the workspace is smaller than nk_linear_ce_workspace says");
}

// ---------------------------------------------------------------- AdamW
// AdamW::step's checks and bias corrections (optim.rs:35-47), on the host.
nk::AdamwParams adamw_params(const nk_adamw_cfg *cfg, float grad_scale, float max_norm) {
    need(cfg, "null AdamW configuration");
    const nk_adamw_cfg &c = *cfg;
    need(std::isfinite(c.lr) && c.lr >= 0.0f, "the learning rate must be finite and non-negative");
    need(std::isfinite(c.b1) && c.b1 >= 0.0f && c.b1 < 1.0f, "beta1 must be in [0, 1)");
    need(std::isfinite(c.b2) && c.b2 >= 0.0f && c.b2 < 1.0f, "beta2 must be in [0, 1)");
    need(std::isfinite(c.eps) && c.eps > 0.0f, "epsilon must be finite and positive");
    need(std::isfinite(c.wd) && c.wd >= 0.0f, "the weight decay must be finite and non-negative");
    need(c.t > 0, "the step counter must be at least 1");
    need(std::isfinite(grad_scale), "grad_scale must be finite");
    need(std::isfinite(max_norm) && max_norm >= 0.0f, "max_norm must be finite and non-negative");
    const float tf = (float)c.t;
    const float bc1 = 1.0f - powf(c.b1, tf), bc2 = 1.0f - powf(c.b2, tf);
    return nk::AdamwParams{c.lr, c.b1, c.b2, c.eps, c.wd, 1.0f / bc1, 1.0f / bc2, 1};
}

uint64_t blocks_of(uint64_t n) { return (n + NK_ADAMW_BLOCK - 1) / NK_ADAMW_BLOCK; }

void check_tensors(const nk_adamw_tensor *tensors, uint64_t count) {
    need(count == 0 || tensors, "null tensors");
    need(count <= (1u << 24), "the number of tensors is limited to 2^24");
    uint64_t total = 0;
    for (uint64_t i = 0; i < count; ++i) {
        const nk_adamw_tensor &t = tensors[i];
        need(t.n <= nk::MAX_ELEMENTS - total, "the tensors are limited to 2^37 elements together");
        total += t.n;
        check_dtype(t.grad_dtype);
        need(t.state_bits == 8 || t.state_bits == 32, "state_bits must be 8 or 32");
        need(!t.copy || t.copy_dtype == NK_F16 || t.copy_dtype == NK_BF16, "copy_dtype must be NK_F16 or NK_BF16");
        if (t.n == 0) continue;
        need(t.val && t.grad && t.m && t.v, "null val, grad, m or v");
        if (t.state_bits == 8)
            need(t.m_scale && t.v_scale, "8-bit moments need m_scale and v_scale");
        else
            need(!t.m_scale && !t.v_scale, "32-bit moments have no scales");
        check_f32({t.val, t.m_scale, t.v_scale});
        if (t.state_bits == 32) check_f32({t.m, t.v});
        check_aligned(t.grad, elem_size(t.grad_dtype), "grad");
        if (t.copy) check_aligned(t.copy, 2, "copy");
    }
}

// No output shares a byte with another output or a gradient (gradients may share).
void check_tensors_apart(const nk_adamw_tensor *tensors, uint64_t count) {
    struct Range {
        uintptr_t from, to;
        bool out;
    };
    std::vector<Range> all;
    auto add = [&](const void *p, uint64_t bytes, bool out) {
        if (p && bytes) all.push_back({(uintptr_t)p, (uintptr_t)p + bytes, out});
    };
    for (uint64_t i = 0; i < count; ++i) {
        const nk_adamw_tensor &t = tensors[i];
        const uint64_t state = t.state_bits == 8 ? 1 : 4;
        add(t.val, t.n * 4, true);
        add(t.m, t.n * state, true);
        add(t.v, t.n * state, true);
        add(t.m_scale, blocks_of(t.n) * 4, true);
        add(t.v_scale, blocks_of(t.n) * 4, true);
        add(t.copy, t.n * 2, true);
        add(t.grad, t.n * elem_size(t.grad_dtype), false);
    }
    std::sort(all.begin(), all.end(), [](const Range &a, const Range &b) { return a.from < b.from; });
    uintptr_t out_end = 0, end = 0;  // the furthest ends so far: of outputs, of anything
    for (const Range &r : all) {
        need(r.from >= out_end && (!r.out || r.from >= end), "an output overlaps another array");
        end = std::max(end, r.to);
        if (r.out) out_end = std::max(out_end, r.to);
    }
}

// The one device of all the tensors' arrays (managed memory: any), else `now`.
int device_of(const nk_adamw_tensor *tensors, uint64_t count, int now) {
    int device = -1;
    for (uint64_t i = 0; i < count; ++i) {
        const nk_adamw_tensor &t = tensors[i];
        if (t.n == 0) continue;
        for (const void *p : {(const void *)t.val, t.grad, (const void *)t.m, (const void *)t.v, (const void *)t.m_scale,
                              (const void *)t.v_scale, (const void *)t.copy}) {
            if (!p) continue;
            cudaPointerAttributes at{};
            cuda_check(cudaPointerGetAttributes(&at, p), "cudaPointerGetAttributes");
            if (at.type == cudaMemoryTypeManaged) continue;
            need(at.type == cudaMemoryTypeDevice, "the arrays must be in device memory");
            if (device < 0) device = at.device;
            need(device == at.device, "the arrays are on different devices");
        }
    }
    return device < 0 ? now : device;
}

// `device` current until the end of the scope.
struct Current {
    int before = 0;
    explicit Current(int device) {
        cuda_check(cudaGetDevice(&before), "cudaGetDevice");
        if (device != before)
            cuda_check(cudaSetDevice(device), "cudaSetDevice");
        else
            before = -1;
    }
    ~Current() {
        if (before >= 0) cudaSetDevice(before);
    }
};

}  // namespace

extern "C" {

nk_status nk_linear_ce_workspace(int dtype, uint64_t rows, uint64_t width, uint64_t vocab, const void *w,
                                 uint64_t w_stride, int backward, uint64_t *bytes) {
    return guard("nk_linear_ce_workspace", [&] {
        need(bytes, "null argument");
        *bytes = 0;
        const uint32_t some = 0;
        check_linear_ce(dtype, rows, width, width, vocab, w_stride, &some, w, &some);
        *bytes = nk::linear_ce_most_workspace_bytes(dtype, (int64_t)rows, (int)width, (int)vocab, w, (int64_t)w_stride, backward != 0);
    });
}

nk_status nk_linear_ce_device(const void *x, int dtype, uint64_t rows, uint64_t width, uint64_t x_stride,
                              const void *w, uint64_t vocab, uint64_t w_stride, const uint32_t *targets, float *loss,
                              float *stats, void *workspace, uint64_t workspace_bytes, void *stream) {
    return guard("nk_linear_ce", [&] {
        check_linear_ce(dtype, rows, width, x_stride, vocab, w_stride, x, w, targets);
        check_f32({loss, stats});
        if (rows == 0) return;
        need(loss || stats, "loss and stats are both null");
        bool copy_lines = true;
        const uint64_t bytes = check_workspace(dtype, rows, width, vocab, w, w_stride, false, workspace, workspace_bytes, copy_lines);
        const int es = elem_size(dtype);
        check_apart({{loss, rows * 4}, {stats, rows * 8}, {workspace, bytes}},
                    {matrix_span(x, rows, width, x_stride, es), matrix_span(w, vocab, width, w_stride, es), {targets, rows * 4}});
        OnDevice on({x, w, targets, loss, stats, workspace});
        nk::LinearCeArgs a{};
        a.x = x;
        a.w = w;
        a.dtype = dtype;
        a.rows = (int64_t)rows;
        a.x_stride = (int64_t)x_stride;
        a.w_stride = (int64_t)w_stride;
        a.width = (int)width;
        a.vocab = (int)vocab;
        a.targets = targets;
        a.loss = loss;
        a.stats = stats;
        a.workspace = workspace;
        a.copy_lines = copy_lines;
        cuda_check(nk::linear_ce(a, sm_count(), (cudaStream_t)stream), "launch");
    });
}

nk_status nk_linear_ce(const void *x, int dtype, uint64_t rows, uint64_t width, const void *w, uint64_t vocab,
                       const uint32_t *targets, float *loss, float *stats, int device) {
    return guard("nk_linear_ce", [&] {
        check_linear_ce(dtype, rows, width, width, vocab, width, x, w, targets);
        if (rows == 0) return;
        need(loss || stats, "loss and stats are both null");
        check_ids(targets, rows, vocab);
        HostCall h(device);
        const int es = elem_size(dtype);
        const void *dx = h.up((const char *)x, rows * width * es), *dw = h.up((const char *)w, vocab * width * es);
        const auto *dt = h.up(targets, rows * 4);
        auto *dl = h.room<float>(rows * 4, loss), *ds = h.room<float>(rows * 8, stats);
        uint64_t bytes = 0;
        nested(nk_linear_ce_workspace(dtype, rows, width, vocab, dw, width, 0, &bytes));
        nested(nk_linear_ce_device(dx, dtype, rows, width, width, dw, vocab, width, dt, dl, ds, h.room<void>(bytes), bytes, nullptr));
        h.down(loss, dl, rows * 4);
        h.down(stats, ds, rows * 8);
    });
}

nk_status nk_linear_ce_backward_device(const void *x, int dtype, uint64_t rows, uint64_t width, uint64_t x_stride,
                                       const void *w, uint64_t vocab, uint64_t w_stride, const uint32_t *targets,
                                       const float *stats, const float *row_weight, float grad_scale, void *dx,
                                       uint64_t dx_stride, void *dw, int dw_dtype, uint64_t dw_stride, int accumulate,
                                       void *workspace, uint64_t workspace_bytes, void *stream) {
    return guard("nk_linear_ce_backward", [&] {
        check_linear_ce(dtype, rows, width, x_stride, vocab, w_stride, x, w, targets);
        need(rows == 0 || stats, "null stats");
        need(std::isfinite(grad_scale), "grad_scale must be finite");
        need(dx || dw, "dx and dw are both null");
        check_f32({stats, row_weight});
        const int es = elem_size(dtype);
        if (dx) {
            check_matrix(rows, width, dx_stride, "dx");
            check_aligned(dx, es, "dx");
        }
        if (dw) {
            need(dw_dtype == dtype || dw_dtype == NK_F32, "dw_dtype must be that of w or NK_F32");
            check_matrix(vocab, width, dw_stride, "dw");
            check_aligned(dw, elem_size(dw_dtype), "dw");
        }
        if (rows == 0 && (!dw || accumulate)) return;
        bool copy_lines = true;
        const uint64_t bytes = check_workspace(dtype, rows, width, vocab, w, w_stride, true, workspace, workspace_bytes, copy_lines);
        const Span sx = matrix_span(x, rows, width, x_stride, es), sw = matrix_span(w, vocab, width, w_stride, es);
        check_apart({matrix_span(dx, rows, width, dx_stride, es), matrix_span(dw, vocab, width, dw_stride, dw ? elem_size(dw_dtype) : 0), {workspace, bytes}},
                    {sx, sw, {targets, rows * 4}, {stats, rows * 8}, {row_weight, rows * 4}});
        const bool some = rows != 0;
        OnDevice on({some ? x : nullptr, w, some ? targets : nullptr, some ? stats : nullptr, some ? row_weight : nullptr,
                     some ? dx : nullptr, dw, workspace});
        nk::LinearCeArgs a{};
        a.x = x;
        a.w = w;
        a.dtype = dtype;
        a.rows = (int64_t)rows;
        a.x_stride = (int64_t)x_stride;
        a.w_stride = (int64_t)w_stride;
        a.width = (int)width;
        a.vocab = (int)vocab;
        a.targets = targets;
        a.in_stats = stats;
        a.row_weight = row_weight;
        a.grad_scale = grad_scale;
        a.dx = some ? dx : nullptr;
        a.dw = dw;
        a.dx_stride = (int64_t)dx_stride;
        a.dw_stride = (int64_t)dw_stride;
        a.dw_dtype = dw_dtype;
        a.accumulate = accumulate != 0;
        a.workspace = workspace;
        a.copy_lines = copy_lines;
        cuda_check(nk::linear_ce_backward(a, sm_count(), (cudaStream_t)stream), "launch");
    });
}

nk_status nk_linear_ce_backward(const void *x, int dtype, uint64_t rows, uint64_t width, const void *w, uint64_t vocab,
                                const uint32_t *targets, const float *stats, const float *row_weight, float grad_scale,
                                void *dx, void *dw, int dw_dtype, int accumulate, int device) {
    return guard("nk_linear_ce_backward", [&] {
        check_linear_ce(dtype, rows, width, width, vocab, width, x, w, targets);
        need(rows == 0 || stats, "null stats");
        need(std::isfinite(grad_scale), "grad_scale must be finite");
        need(dx || dw, "dx and dw are both null");
        need(!dw || dw_dtype == dtype || dw_dtype == NK_F32, "dw_dtype must be that of w or NK_F32");
        if (rows) check_ids(targets, rows, vocab);
        HostCall h(device);
        const int es = elem_size(dtype);
        const size_t xb = rows * width * es, wb = vocab * width * es, gb = dw ? vocab * width * elem_size(dw_dtype) : 0;
        const void *px = h.up((const char *)x, xb), *pw = h.up((const char *)w, wb);
        const auto *dt = h.up(targets, rows * 4);
        const auto *ds = h.up(stats, rows * 8), *rw = h.up(row_weight, rows * 4);
        void *gx = h.room<void>(xb, dx), *gw = dw && accumulate ? (void *)h.up((const char *)dw, gb) : h.room<void>(gb, dw);
        uint64_t bytes = 0;
        nested(nk_linear_ce_workspace(dtype, rows, width, vocab, pw, width, 1, &bytes));
        nested(nk_linear_ce_backward_device(px, dtype, rows, width, width, pw, vocab, width, dt, ds, rw, grad_scale, gx,
                                            width, gw, dw_dtype, width, accumulate, h.room<void>(bytes), bytes, nullptr));
        h.down(dx, gx, xb);
        h.down(dw, gw, gb);
    });
}

nk_status nk_linear_ce_withhold(int product) {
    return guard("nk_linear_ce_withhold", [&] {
        need(product >= 0 && product <= 3, "product must be 0 to 3");
        nk::linear_ce_withhold(product);
    });
}

nk_status nk_adamw_many_create(const nk_adamw_tensor *tensors, uint64_t count, nk_adamw_many **out) {
    return guard("nk_adamw_many_create", [&] {
        need(out, "null argument");
        *out = nullptr;
        check_tensors(tensors, count);
        check_tensors_apart(tensors, count);
        int now = 0;
        cuda_check(cudaGetDevice(&now), "cudaGetDevice");
        const int device = device_of(tensors, count, now);
        Current current(device);
        const int sms = sm_count();
        std::vector<nk::AdamwChunk> chunks;
        uint32_t n32 = 0;
        for (const int bits : {32, 8}) {
            uint64_t total = 0;
            for (uint64_t i = 0; i < count; ++i) total += tensors[i].state_bits == bits ? tensors[i].n : 0;
            const uint32_t size = nk::adamw_chunk_elements(total, sms, bits);
            for (uint64_t i = 0; i < count; ++i) {
                if (tensors[i].state_bits != bits) continue;
                for (uint64_t at = 0; at < tensors[i].n; at += size)
                    chunks.push_back({(uint32_t)i, (uint32_t)std::min<uint64_t>(size, tensors[i].n - at), at});
            }
            // Whole chunks first: the last round of a grid is then one of short ones.
            std::stable_partition(chunks.begin() + (bits == 32 ? 0 : n32), chunks.end(), [&](const nk::AdamwChunk &c) { return c.n == size; });
            if (bits == 32) n32 = (uint32_t)chunks.size();
        }
        // One allocation: the tables, the partial sums, the ticket and the factor.
        auto round = [](size_t n) { return (n + 255) / 256 * 256; };
        const size_t tb = round(count * sizeof(nk_adamw_tensor)), cb = round(chunks.size() * sizeof(nk::AdamwChunk)),
                     pb = round(nk::adamw_partials(sms) * sizeof(double));
        std::unique_ptr<nk_adamw_many, void (*)(nk_adamw_many *)> many(new nk_adamw_many, nk_adamw_many_free);
        many->device = device;
        many->sms = sms;
        cuda_check(cudaMalloc(&many->room, tb + cb + pb + 256), "cudaMalloc");
        char *room = (char *)many->room;
        if (count) cuda_check(cudaMemcpy(room, tensors, count * sizeof(nk_adamw_tensor), cudaMemcpyHostToDevice), "upload");
        if (!chunks.empty())
            cuda_check(cudaMemcpy(room + tb, chunks.data(), chunks.size() * sizeof(nk::AdamwChunk), cudaMemcpyHostToDevice), "upload");
        cuda_check(cudaMemset(room + tb + cb + pb, 0, 256), "memset");
        cuda_check(cudaStreamSynchronize(nullptr), "synchronize");
        many->plan.tensors = (const nk_adamw_tensor *)room;
        many->plan.chunks = (const nk::AdamwChunk *)(room + tb);
        many->plan.n_chunks = (uint32_t)chunks.size();
        many->plan.n_chunks32 = n32;
        many->plan.partial = (double *)(room + tb + cb);
        many->plan.clip = (float *)(room + tb + cb + pb);
        many->plan.ticket = (uint32_t *)(room + tb + cb + pb + 64);
        *out = many.release();
    });
}

void nk_adamw_many_free(nk_adamw_many *many) {
    if (!many) return;
    if (many->room) {
        int now = 0;
        if (cudaGetDevice(&now) == cudaSuccess && cudaSetDevice(many->device) == cudaSuccess) {
            cudaFree(many->room);
            cudaSetDevice(now);
        }
    }
    delete many;
}

nk_status nk_adamw_many_step_device(nk_adamw_many *many, const nk_adamw_cfg *cfg, float grad_scale, float max_norm,
                                    float *norm, uint32_t *bad, void *stream) {
    return guard("nk_adamw_many_step", [&] {
        need(many, "null argument");
        const nk::AdamwParams a = adamw_params(cfg, grad_scale, max_norm);
        check_f32({norm, bad});
        check_apart({{norm, 4}, {bad, 4}}, {});
        {
            OnDevice on({norm, bad, many->room});
        }
        Current current(many->device);
        if (norm || max_norm > 0.0f)
            cuda_check(nk::adamw_many_norm(many->plan, grad_scale, max_norm, norm, bad, many->sms, (cudaStream_t)stream), "launch");
        cuda_check(nk::adamw_many_step(many->plan, a, (uint32_t)cfg->t, grad_scale, max_norm > 0.0f, bad, many->sms, (cudaStream_t)stream), "launch");
    });
}

nk_status nk_adamw_many_step(const nk_adamw_tensor *tensors, uint64_t count, const nk_adamw_cfg *cfg, float grad_scale,
                             float max_norm, float *norm, int device) {
    return guard("nk_adamw_many_step", [&] {
        adamw_params(cfg, grad_scale, max_norm);
        check_tensors(tensors, count);
        check_tensors_apart(tensors, count);
        HostCall h(device);
        std::vector<nk_adamw_tensor> dev(tensors, tensors + count);
        for (uint64_t i = 0; i < count; ++i) {
            const nk_adamw_tensor &t = tensors[i];
            nk_adamw_tensor &d = dev[i];
            if (t.n == 0) continue;
            const uint64_t state = t.n * (t.state_bits == 8 ? 1 : 4), scales = blocks_of(t.n) * 4;
            d.val = h.up(t.val, t.n * 4);
            d.grad = h.up((const char *)t.grad, t.n * elem_size(t.grad_dtype));
            d.m = h.up((const char *)t.m, state) ? h.own.back() : nullptr;
            d.v = h.up((const char *)t.v, state) ? h.own.back() : nullptr;
            d.m_scale = h.up(t.m_scale, scales);
            d.v_scale = h.up(t.v_scale, scales);
            // (With what is there: a norm that is not finite leaves it.)
            d.copy = h.up((const char *)t.copy, t.n * 2) ? h.own.back() : nullptr;
        }
        auto *flags = h.room<char>(8);
        cuda_check(cudaMemset(flags, 0, 8), "memset");
        nk_adamw_many *raw = nullptr;
        nested(nk_adamw_many_create(dev.data(), count, &raw));
        std::unique_ptr<nk_adamw_many, void (*)(nk_adamw_many *)> many(raw, nk_adamw_many_free);
        nested(nk_adamw_many_step_device(raw, cfg, grad_scale, max_norm, norm ? (float *)flags : nullptr, (uint32_t *)(flags + 4), nullptr));
        for (uint64_t i = 0; i < count; ++i) {
            const nk_adamw_tensor &t = tensors[i], &d = dev[i];
            if (t.n == 0) continue;
            const uint64_t state = t.n * (t.state_bits == 8 ? 1 : 4), scales = blocks_of(t.n) * 4;
            h.down(t.val, d.val, t.n * 4);
            h.down(t.m, d.m, state);
            h.down(t.v, d.v, state);
            h.down(t.m_scale, d.m_scale, scales);
            h.down(t.v_scale, d.v_scale, scales);
            h.down(t.copy, d.copy, t.n * 2);
        }
        h.down(norm, flags, 4);
        uint32_t bad = 0;
        h.down(&bad, flags + 4, 4);
        need(bad == 0, "a gradient or parameter, or their clipped norm, is not finite");
    });
}

}  // extern "C"
