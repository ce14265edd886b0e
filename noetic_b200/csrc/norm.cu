// norm.cu -- layer norm and RMSNorm of rows, and their gradients
// (include/noetic/head.h).

#include <algorithm>

#include "nk_head.cuh"
#include "nk_head.h"

namespace nk {

namespace {

constexpr int NM_NT = 256;
constexpr int PARTIAL_ROWS = 512;  // most partial sums of dgain and dbias

template <class T>
__global__ void __launch_bounds__(NM_NT) norm_rows_k(NormArgs a) {
    __shared__ float red[32];
    const int64_t r = blockIdx.x;
    const T *x = (const T *)a.x + r * a.x_stride;
    T *y = (T *)a.y + r * a.y_stride;
    const float n = (float)a.width;
    float mean = 0.0f;
    if (!a.rms) {
        float s = 0.0f;
        for (int e = threadIdx.x; e < a.width; e += NM_NT) s += to_f32(x[e]);
        mean = block_sum(s, red) / n;
    }
    float v = 0.0f;
    for (int e = threadIdx.x; e < a.width; e += NM_NT) {
        const float d = to_f32(x[e]) - mean;
        v = fmaf(d, d, v);
    }
    const float rstd = 1.0f / sqrtf(block_sum(v, red) / n + a.eps);
    for (int e = threadIdx.x; e < a.width; e += NM_NT) {
        const float h = (to_f32(x[e]) - mean) * rstd;
        y[e] = from_f32<T>(fmaf(h, a.gain ? a.gain[e] : 1.0f, a.bias ? a.bias[e] : 0.0f));
    }
    if (threadIdx.x == 0) {
        if (a.mean) a.mean[r] = mean;
        if (a.rstd) a.rstd[r] = rstd;
    }
}

template <class T>
__global__ void __launch_bounds__(NM_NT) norm_dx_k(NormGradArgs a) {
    __shared__ float red[32];
    const int64_t r = blockIdx.x;
    const T *x = (const T *)a.x + r * a.x_stride, *dy = (const T *)a.dy + r * a.dy_stride;
    T *dx = (T *)a.dx + r * a.dx_stride;
    const float n = (float)a.width, mean = a.rms ? 0.0f : a.mean[r], rstd = a.rstd[r];
    float sc = 0.0f, sch = 0.0f;
    for (int e = threadIdx.x; e < a.width; e += NM_NT) {
        const float c = to_f32(dy[e]) * (a.gain ? a.gain[e] : 1.0f), h = (to_f32(x[e]) - mean) * rstd;
        sc += c;
        sch = fmaf(c, h, sch);
    }
    sc = a.rms ? 0.0f : block_sum(sc, red) / n;
    sch = block_sum(sch, red) / n;
    for (int e = threadIdx.x; e < a.width; e += NM_NT) {
        const float c = to_f32(dy[e]) * (a.gain ? a.gain[e] : 1.0f), h = (to_f32(x[e]) - mean) * rstd;
        dx[e] = from_f32<T>(rstd * (c - sc - h * sch));
    }
}

// Partial sums over the rows p, p + P, ... of one column per thread.
template <class T>
__global__ void __launch_bounds__(NM_NT) norm_param_k(NormGradArgs a) {
    const int e = blockIdx.x * NM_NT + threadIdx.x;
    if (e >= a.width) return;
    float dg = 0.0f, db = 0.0f;
    for (int64_t r = blockIdx.y; r < a.rows; r += gridDim.y) {
        const float dy = to_f32(((const T *)a.dy)[r * a.dy_stride + e]);
        const float h = (to_f32(((const T *)a.x)[r * a.x_stride + e]) - (a.rms ? 0.0f : a.mean[r])) * a.rstd[r];
        dg = fmaf(dy, h, dg);
        db += dy;
    }
    float *w = a.workspace + (int64_t)blockIdx.y * 2 * a.width;
    w[e] = dg;
    w[a.width + e] = db;
}

__global__ void __launch_bounds__(NM_NT) norm_param_sum_k(NormGradArgs a, int parts) {
    const int e = blockIdx.x * NM_NT + threadIdx.x;
    if (e >= a.width) return;
    float dg = 0.0f, db = 0.0f;
    for (int p = 0; p < parts; ++p) {
        dg += a.workspace[(int64_t)p * 2 * a.width + e];
        db += a.workspace[(int64_t)p * 2 * a.width + a.width + e];
    }
    if (a.dgain) a.dgain[e] = a.accumulate ? a.dgain[e] + dg : dg;
    if (a.dbias) a.dbias[e] = a.accumulate ? a.dbias[e] + db : db;
}

int partial_rows(int64_t rows) { return (int)std::min<int64_t>(std::max<int64_t>(rows, 1), PARTIAL_ROWS); }

template <class T>
cudaError_t backward(const NormGradArgs &a, cudaStream_t st) {
    // The parameters' sums first: dx may be the array of dy.
    if (a.dgain || a.dbias) {
        const unsigned cols = (unsigned)((a.width + NM_NT - 1) / NM_NT);
        const int parts = partial_rows(a.rows);
        norm_param_k<T><<<dim3(cols, parts), NM_NT, 0, st>>>(a);
        if (cudaError_t e = cudaGetLastError()) return e;
        norm_param_sum_k<<<cols, NM_NT, 0, st>>>(a, parts);
        if (cudaError_t e = cudaGetLastError()) return e;
    }
    if (a.dx && a.rows) norm_dx_k<T><<<(unsigned)a.rows, NM_NT, 0, st>>>(a);
    return cudaGetLastError();
}

}  // namespace

cudaError_t norm_rows(const NormArgs &a, int dtype, cudaStream_t st) {
    const unsigned grid = (unsigned)a.rows;
    switch (dtype) {
        case 0: norm_rows_k<float><<<grid, NM_NT, 0, st>>>(a); break;
        case 1: norm_rows_k<__half><<<grid, NM_NT, 0, st>>>(a); break;
        default: norm_rows_k<__nv_bfloat16><<<grid, NM_NT, 0, st>>>(a); break;
    }
    return cudaGetLastError();
}

size_t norm_backward_workspace_bytes(int64_t rows, int width) {
    return (size_t)partial_rows(rows) * 2 * (size_t)width * sizeof(float);
}

cudaError_t norm_backward(const NormGradArgs &a, int dtype, cudaStream_t st) {
    switch (dtype) {
        case 0: return backward<float>(a, st);
        case 1: return backward<__half>(a, st);
        default: return backward<__nv_bfloat16>(a, st);
    }
}

}  // namespace nk
