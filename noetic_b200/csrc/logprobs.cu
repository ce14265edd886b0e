// logprobs.cu -- log probabilities of given tokens with the row's entropy and
// most probable alternatives, and their gradient (include/noetic/head.h).

#include "nk_head.cuh"
#include "nk_head.h"

namespace nk {

namespace {

constexpr int LP_NT = 256;
constexpr int TOP_MAX = 128;

// The `top` largest of row[e0, e1) above -infinity, equal values by index:
// keys (order_key << 32 | ~index) in descending order in out[0, top), 0 behind
// the last.  A radix select finds the last value kept; one ordered walk then
// takes what lies above it and the first of those equal to it.
struct TopScratch {
    uint32_t hist[256];
    uint32_t warp_count[32];
    uint64_t kept[TOP_MAX];
    uint32_t prefix, above, n_kept;
};

template <class T>
__device__ void exact_top(const T *__restrict__ row, int e0, int e1, int top, TopScratch &sc, uint64_t *out) {
    const int tid = threadIdx.x, nt = blockDim.x, lane = tid & 31, warp = tid >> 5;
    if (tid == 0) sc.prefix = sc.above = 0;
    __syncthreads();
    for (int shift = 24; shift >= 0; shift -= 8) {
        for (int i = tid; i < 256; i += nt) sc.hist[i] = 0;
        __syncthreads();
        const uint32_t prefix = sc.prefix;
        for (int e = e0 + tid; e < e1; e += nt) {
            const float z = to_f32(row[e]);
            if (!(z > -INFINITY)) continue;
            const uint32_t k = order_key(z);
            if (shift == 24 || (k >> (shift + 8)) == (prefix >> (shift + 8))) atomicAdd(&sc.hist[(k >> shift) & 255], 1u);
        }
        __syncthreads();
        if (tid == 0) {
            uint32_t above = sc.above;
            int b = 255;
            while (b > 0 && above + sc.hist[b] < (uint32_t)top) above += sc.hist[b--];
            sc.above = above;
            sc.prefix = prefix | ((uint32_t)b << shift);
        }
        __syncthreads();
    }
    const uint32_t last = sc.prefix, above = sc.above;
    uint32_t equal = 0;  // seen so far, the same in every thread
    if (tid == 0) sc.n_kept = 0;
    __syncthreads();
    for (int b = e0; b < e1; b += nt) {
        const int e = b + tid;
        const float z = e < e1 ? to_f32(row[e]) : -INFINITY;
        const bool real = z > -INFINITY;
        const uint32_t k = order_key(z);
        const uint64_t key = ((uint64_t)k << 32) | (uint32_t)~(uint32_t)e;
        if (real && k > last) sc.kept[atomicAdd(&sc.n_kept, 1u)] = key;
        const bool eq = real && k == last;
        const uint32_t votes = __ballot_sync(0xffffffffu, eq);
        if (lane == 0) sc.warp_count[warp] = __popc(votes);
        __syncthreads();
        uint32_t before = equal, total = 0;
        for (int w = 0; w < (nt >> 5); ++w) {
            if (w < warp) before += sc.warp_count[w];
            total += sc.warp_count[w];
        }
        before += __popc(votes & ((1u << lane) - 1u));
        if (eq && above + before < (uint32_t)top) sc.kept[above + before] = key;
        equal += total;
        __syncthreads();
    }
    const int n = min((uint32_t)top, above + equal);
    for (int i = tid; i < top; i += nt) {
        if (i < n) {
            int rank = 0;
            for (int j = 0; j < n; ++j) rank += sc.kept[j] > sc.kept[i];
            out[rank] = sc.kept[i];
        } else {
            out[i] = 0;
        }
    }
    __syncthreads();
}

template <class T>
__global__ void __launch_bounds__(LP_NT) token_logprobs_k(LogprobsArgs a) {
    __shared__ float red[32];
    __shared__ TopScratch sc;
    __shared__ uint64_t best[TOP_MAX];
    const int64_t r = blockIdx.x;
    const T *row = (const T *)a.logits + r * a.stride;
    const uint32_t target = a.targets ? a.targets[r] : NO_TOKEN;
    if (a.targets && target >= (uint32_t)a.vocab) {
        if (threadIdx.x == 0) {
            if (a.logprob) a.logprob[r] = 0.0f;
            if (a.entropy) a.entropy[r] = 0.0f;
            if (a.stats) a.stats[2 * r] = a.stats[2 * r + 1] = 0.0f;
        }
        for (int i = threadIdx.x; i < a.top; i += LP_NT) {
            if (a.top_ids) a.top_ids[r * a.top + i] = NO_TOKEN;
            if (a.top_logprobs) a.top_logprobs[r * a.top + i] = -INFINITY;
        }
        return;
    }
    SoftSums sums;
    for (int e = threadIdx.x; e < a.vocab; e += LP_NT) {
        const float z = to_f32(row[e]);
        sums.raise(z, a.scale);
        sums.add(z, sums.base(), a.scale);
    }
    sums = block_join(sums, a.scale, red);
    const float log_s = logf(sums.s);
    const bool empty = sums.m == -INFINITY && sums.s == 0.0f;
    if (threadIdx.x == 0) {
        if (a.logprob) a.logprob[r] = empty ? -INFINITY : (to_f32(row[target]) - sums.m) * a.inv_t - log_s;
        if (a.entropy) {
            const float h = log_s - LN2 * (sums.t / sums.s);
            a.entropy[r] = empty || h < 0.0f ? 0.0f : h;
        }
        if (a.stats) {
            a.stats[2 * r] = sums.m;
            a.stats[2 * r + 1] = log_s;
        }
    }
    if (a.top) {
        exact_top(row, 0, a.vocab, a.top, sc, best);
        for (int i = threadIdx.x; i < a.top; i += LP_NT) {
            const uint64_t k = best[i];
            if (a.top_ids) a.top_ids[r * a.top + i] = k ? ~(uint32_t)k : NO_TOKEN;
            if (a.top_logprobs)
                a.top_logprobs[r * a.top + i] =
                    k ? (key_value((uint32_t)(k >> 32)) - sums.m) * a.inv_t - log_s : -INFINITY;
        }
    }
}

template <class T>
__global__ void __launch_bounds__(LP_NT) token_logprobs_backward_k(LogprobsGradArgs a) {
    const int64_t r = blockIdx.x;
    const T *row = (const T *)a.logits + r * a.stride;
    T *out = (T *)a.dlogits + r * a.dstride;
    const uint32_t target = a.targets ? a.targets[r] : NO_TOKEN;
    const float m = a.stats[2 * r], log_s = a.stats[2 * r + 1];
    if ((a.targets && target >= (uint32_t)a.vocab) || (m == -INFINITY && log_s == -INFINITY)) {
        for (int e = threadIdx.x; e < a.vocab; e += LP_NT) out[e] = from_f32<T>(0.0f);
        return;
    }
    const float gl = a.g_logprob ? a.g_logprob[r] : 0.0f, ge = a.g_entropy ? a.g_entropy[r] : 0.0f;
    const float ca = -(gl + (a.g_entropy ? ge * a.entropy[r] : 0.0f)) * a.inv_t, cb = -ge * LN2 * a.inv_t;
    const float log2_s = log_s * LOG2E;
    for (int e = threadIdx.x; e < a.vocab; e += LP_NT) {
        const float y = fmaf(to_f32(row[e]) - m, a.scale, -log2_s);
        float dz = ex2(y) * fmaf(cb, fmaxf(y, -256.0f), ca);
        if ((uint32_t)e == target) dz = fmaf(gl, a.inv_t, dz);
        out[e] = from_f32<T>(dz);
    }
}

}  // namespace

cudaError_t token_logprobs(const LogprobsArgs &a, int dtype, cudaStream_t st) {
    const unsigned grid = (unsigned)a.rows;
    switch (dtype) {
        case 0: token_logprobs_k<float><<<grid, LP_NT, 0, st>>>(a); break;
        case 1: token_logprobs_k<__half><<<grid, LP_NT, 0, st>>>(a); break;
        default: token_logprobs_k<__nv_bfloat16><<<grid, LP_NT, 0, st>>>(a); break;
    }
    return cudaGetLastError();
}

cudaError_t token_logprobs_backward(const LogprobsGradArgs &a, int dtype, cudaStream_t st) {
    const unsigned grid = (unsigned)a.rows;
    switch (dtype) {
        case 0: token_logprobs_backward_k<float><<<grid, LP_NT, 0, st>>>(a); break;
        case 1: token_logprobs_backward_k<__half><<<grid, LP_NT, 0, st>>>(a); break;
        default: token_logprobs_backward_k<__nv_bfloat16><<<grid, LP_NT, 0, st>>>(a); break;
    }
    return cudaGetLastError();
}

}  // namespace nk
