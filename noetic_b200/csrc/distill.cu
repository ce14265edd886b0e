// distill.cu -- the distillation loss from a teacher's top logits with its
// gradient (include/noetic/head.h).

#include "nk_head.cuh"
#include "nk_head.h"

namespace nk {

namespace {

constexpr int DS_NT = 256;
constexpr int TEACHER_MAX = 256;

__device__ __forceinline__ float teacher_value(const void *p, int dtype, int64_t i) {
    return dtype == 0   ? ((const float *)p)[i]
           : dtype == 1 ? to_f32(((const __half *)p)[i])
                        : to_f32(((const __nv_bfloat16 *)p)[i]);
}

template <class T>
__global__ void __launch_bounds__(DS_NT) distill_k(DistillArgs a) {
    __shared__ float red[32];
    __shared__ uint32_t id[TEACHER_MAX];
    __shared__ float q[TEACHER_MAX], zt[TEACHER_MAX];
    const int64_t r = blockIdx.x;
    const int tid = threadIdx.x;
    const T *row = (const T *)a.logits + r * a.stride;
    T *out = a.dlogits ? (T *)a.dlogits + r * a.dstride : nullptr;

    // The teacher's entry of this thread: q = softmax(teacher / temperature).
    const uint32_t my = tid < a.n ? a.ids[r * a.n + tid] : NO_TOKEN;
    const float t = my < (uint32_t)a.vocab ? teacher_value(a.teacher, a.teacher_dtype, r * a.n + tid) : -INFINITY;
    const bool live = t != -INFINITY;
    const float tm = block_max(t, red);
    const float ty = (t - tm) * a.inv_t;
    const float te = live ? expf(ty) : 0.0f;
    const float ts = block_sum(te, red);
    const bool any = __syncthreads_or(live);
    const float w = a.row_weight ? a.row_weight[r] : 1.0f;
    if (!any) {
        if (tid == 0 && a.loss) a.loss[r] = 0.0f;
        if (out)
            for (int e = tid; e < a.vocab; e += DS_NT) out[e] = from_f32<T>(0.0f);
        return;
    }
    const float my_q = ts == 0.0f ? 0.0f : te / ts;
    if (tid < a.n) {
        id[tid] = live ? my : NO_TOKEN;
        q[tid] = my_q;
        zt[tid] = live ? to_f32(row[my]) : 0.0f;
    }
    SoftSums sums;
    for (int e = tid; e < a.vocab; e += DS_NT) {
        const float z = to_f32(row[e]);
        sums.raise(z, a.scale);
        sums.add(z, sums.base(), a.scale);
    }
    sums = block_join(sums, a.scale, red);
    const float log_s = logf(sums.s);
    float part = 0.0f;
    if (live && my_q != 0.0f) part = my_q * ((ty - logf(ts)) - ((zt[tid] - sums.m) * a.inv_t - log_s));
    const float kl = block_sum(part, red);
    if (tid == 0 && a.loss) a.loss[r] = a.temperature * a.temperature * kl;
    if (!out) return;
    if (w == 0.0f) {
        for (int e = tid; e < a.vocab; e += DS_NT) out[e] = from_f32<T>(0.0f);
        return;
    }
    const float g = a.grad_scale * w * a.temperature, log2_s = log_s * LOG2E;
    for (int e = tid; e < a.vocab; e += DS_NT)
        out[e] = from_f32<T>(g * ex2(fmaf(to_f32(row[e]) - sums.m, a.scale, -log2_s)));
    __syncthreads();
    // The entries' own places, from the first of each id.
    if (live) {
        float share = 0.0f;
        bool first = true;
        for (int i = 0; i < a.n; ++i)
            if (id[i] == my) {
                share += q[i];
                first = first && i >= tid;
            }
        if (first) out[my] = from_f32<T>(g * (ex2(fmaf(zt[tid] - sums.m, a.scale, -log2_s)) - share));
    }
}

}  // namespace

cudaError_t distill(const DistillArgs &a, int dtype, cudaStream_t st) {
    const unsigned grid = (unsigned)a.rows;
    switch (dtype) {
        case 0: distill_k<float><<<grid, DS_NT, 0, st>>>(a); break;
        case 1: distill_k<__half><<<grid, DS_NT, 0, st>>>(a); break;
        default: distill_k<__nv_bfloat16><<<grid, DS_NT, 0, st>>>(a); break;
    }
    return cudaGetLastError();
}

}  // namespace nk
