// logprobs.cu -- log probabilities of given tokens with the row's entropy and
// most probable alternatives, and their gradient (include/noetic/head.h).

#include <cooperative_groups.h>

#include <algorithm>

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

// One row by a cluster of `cs` CTAs (one, when there are rows enough to fill
// the GPU), each with a contiguous part of it.  The row is read once: a thread
// takes four 16-byte vectors at a time, raises its running maximum by theirs
// and adds their exponentials.  What bounds it: HBM; 16-bit logits need one
// exponential per two bytes, 16 of which an SM's special-function unit makes
// per clock, 1.4 times what HBM delivers.
//
// Alternatives.  Every thread keeps the maximum of each group of its vectors
// in shared memory.  The top-th largest of the threads' own maxima bounds the
// top-th logit from below (top distinct elements reach it), and only the few
// groups that reach this bound are read again, from L2, for their elements
// above it: about `top` candidates, ranked by counting.  Rows that leave more
// candidates than fit (many equal logits, an order that gives one thread all
// the large ones) go to exact_top.
constexpr int LP_U = 4;
constexpr int LP_SLOTS = 32;        // groups per thread
constexpr int CANDIDATES = 1024;    // at least 8 CTAs' TOP_MAX
constexpr int MAX_CLUSTER = 8;

struct LogprobsShared {
    float red[32];
    float sums[3];
    uint32_t bound, n_cand;
    uint64_t cand[CANDIDATES];
    uint64_t best[TOP_MAX];
    float thread_max[LP_NT];
};

// How many of list[0, n) (descending) are above key.
__device__ __forceinline__ int count_above(const uint64_t *list, int n, uint64_t key) {
    int lo = 0, hi = n;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (list[mid] > key)
            lo = mid + 1;
        else
            hi = mid;
    }
    return lo;
}

template <class T>
__global__ void __launch_bounds__(LP_NT) token_logprobs_k(LogprobsArgs a, int cs, int slot_shift) {
    extern __shared__ float group_max[];
    __shared__ LogprobsShared sh;
    __shared__ TopScratch sc;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int64_t r = blockIdx.x / cs;
    const int rank = blockIdx.x % cs;
    const T *row = (const T *)a.logits + r * a.stride;
    const uint32_t target = a.targets ? a.targets[r] : NO_TOKEN;
    if (a.targets && target >= (uint32_t)a.vocab) {
        if (rank == 0) {
            if (tid == 0) {
                if (a.logprob) a.logprob[r] = 0.0f;
                if (a.entropy) a.entropy[r] = 0.0f;
                if (a.stats) a.stats[2 * r] = a.stats[2 * r + 1] = 0.0f;
            }
            for (int i = tid; i < a.top; i += LP_NT) {
                if (a.top_ids) a.top_ids[r * a.top + i] = NO_TOKEN;
                if (a.top_logprobs) a.top_logprobs[r * a.top + i] = -INFINITY;
            }
        }
        return;  // the whole cluster
    }
    const float z_target = a.targets && rank == 0 && tid == 0 ? to_f32(row[target]) : 0.0f;

    constexpr int N = Vec<T>::N;
    const RowSpan span = row_span(row, a.vocab);
    const T *body = row + span.head;
    const int v0 = (int)((int64_t)span.n_vec * rank / cs), v1 = (int)((int64_t)span.n_vec * (rank + 1) / cs);
    const int n_head = rank == 0 ? span.head : 0, n_tail = rank == cs - 1 ? span.tail : 0;
    const float scale = a.scale;
    SoftSums sums;
    float tmax = -INFINITY, gmax = -INFINITY;
    const int batch = stream_sums<T, LP_NT, LP_U>(body, v0, v1, scale, sums, [&](int b, float bm) {
        if (a.top) {
            gmax = (b & ((1 << slot_shift) - 1)) == 0 ? bm : fmaxf(gmax, bm);
            group_max[(b >> slot_shift) * LP_NT + tid] = gmax;
            tmax = fmaxf(tmax, bm);
        }
    });
    // The ends that no vector covers, one element per thread and end.
    auto single = [&](int e) {
        const float z = to_f32(row[e]);
        sums.raise(z, scale);
        sums.add(z, scale);
        tmax = fmaxf(tmax, z);
    };
    if (tid < n_head) single(tid);
    if (tid < n_tail) single(a.vocab - span.tail + tid);
    sums = block_join(sums, scale, sh.red);

    if (a.top) {
        sh.thread_max[tid] = tmax;
        if (tid == 0) sh.n_cand = 0;
        __syncthreads();
        if (warp == 0) {
            // The upper half of the top-th largest key, bit by bit.
            uint32_t k[LP_NT / 32], p = 0;
#pragma unroll
            for (int i = 0; i < LP_NT / 32; ++i) k[i] = order_key(sh.thread_max[i * 32 + lane]);
            for (uint32_t bit = 1u << 31; bit >= 1u << 16; bit >>= 1) {
                int n = 0;
#pragma unroll
                for (int i = 0; i < LP_NT / 32; ++i) n += k[i] >= (p | bit);
                if ((int)__reduce_add_sync(0xffffffffu, (unsigned)n) >= a.top) p |= bit;
            }
            if (lane == 0) sh.bound = p;
        }
        __syncthreads();
        const uint32_t bound = sh.bound;
        auto offer = [&](float z, int e) {
            const uint32_t k = order_key(z);
            if (z > -INFINITY && k >= bound) {
                const uint32_t at = atomicAdd(&sh.n_cand, 1u);
                if (at < CANDIDATES) sh.cand[at] = ((uint64_t)k << 32) | (uint32_t)~(uint32_t)e;
            }
        };
        if (tmax > -INFINITY && order_key(tmax) >= bound) {
            const int groups = (batch + (1 << slot_shift) - 1) >> slot_shift;
            for (int g = 0; g < groups; ++g) {
                if (order_key(group_max[g * LP_NT + tid]) < bound) continue;
                const int end = min(batch, (g + 1) << slot_shift);
                for (int b = g << slot_shift; b < end; ++b) {
#pragma unroll
                    for (int u = 0; u < LP_U; ++u) {
                        const int v = v0 + tid + (b * LP_U + u) * LP_NT;
                        if (v >= v1) continue;
                        float x[N];
                        unpack<T>(load16(body + (int64_t)v * N), x);
#pragma unroll
                        for (int i = 0; i < N; ++i) offer(x[i], span.head + v * N + i);
                    }
                }
            }
            if (tid < n_head) offer(to_f32(row[tid]), tid);
            if (tid < n_tail) offer(to_f32(row[a.vocab - span.tail + tid]), a.vocab - span.tail + tid);
        }
        __syncthreads();
        const int n = (int)sh.n_cand;
        if (n > CANDIDATES) {
            exact_top(row, rank == 0 ? 0 : span.head + v0 * N, rank == cs - 1 ? a.vocab : span.head + v1 * N, a.top, sc,
                      sh.best);
        } else {
            for (int i = n + tid; i < a.top; i += LP_NT) sh.best[i] = 0;
            for (int i = tid; i < n; i += LP_NT) {
                const uint64_t key = sh.cand[i];
                int rk = 0;
                for (int j = 0; j < n; ++j) rk += sh.cand[j] > key;
                if (rk < a.top) sh.best[rk] = key;
            }
            __syncthreads();
        }
    }

    if (cs > 1) {
        namespace cg = cooperative_groups;
        cg::cluster_group cluster = cg::this_cluster();
        if (tid == 0) {
            sh.sums[0] = sums.m;
            sh.sums[1] = sums.s;
            sh.sums[2] = sums.t;
        }
        cluster.sync();
        if (rank == 0) {
            // The parts in their order.
            SoftSums all;
            for (int c = 0; c < cs; ++c) all.m = fmaxf(all.m, cluster.map_shared_rank(sh.sums, c)[0]);
            for (int c = 0; c < cs; ++c) {
                const float *p = cluster.map_shared_rank(sh.sums, c);
                SoftSums part;
                part.m = p[0];
                part.s = p[1];
                part.t = p[2];
                if (part.m != -INFINITY) part.raise(all.m, scale);
                all.s += part.s;
                all.t += part.t;
            }
            sums = all;
            if (a.top) {
                for (int i = tid; i < cs * a.top; i += LP_NT)
                    sh.cand[i] = cluster.map_shared_rank(sh.best, i / a.top)[i % a.top];
                __syncthreads();
                for (int i = tid; i < a.top; i += LP_NT) sh.best[i] = 0;
                __syncthreads();
                for (int i = tid; i < cs * a.top; i += LP_NT) {
                    const uint64_t key = sh.cand[i];
                    if (key == 0) continue;
                    int rk = 0;
                    for (int c = 0; c < cs; ++c) rk += count_above(sh.cand + c * a.top, a.top, key);
                    if (rk < a.top) sh.best[rk] = key;
                }
                __syncthreads();
            }
        }
        cluster.sync();  // the others' shared memory is read until here
        if (rank != 0) return;
    }

    const float log_s = logf(sums.s);
    const bool empty = sums.m == -INFINITY && sums.s == 0.0f;
    if (tid == 0) {
        if (a.logprob) a.logprob[r] = empty ? -INFINITY : (z_target - sums.m) * a.inv_t - log_s;
        if (a.entropy) {
            const float h = log_s - LN2 * (sums.t / sums.s);
            a.entropy[r] = empty || h < 0.0f ? 0.0f : h;
        }
        if (a.stats) {
            a.stats[2 * r] = sums.m;
            a.stats[2 * r + 1] = log_s;
        }
    }
    for (int i = tid; i < a.top; i += LP_NT) {
        const uint64_t k = sh.best[i];
        if (a.top_ids) a.top_ids[r * a.top + i] = k ? ~(uint32_t)k : NO_TOKEN;
        if (a.top_logprobs)
            a.top_logprobs[r * a.top + i] = k ? (key_value((uint32_t)(k >> 32)) - sums.m) * a.inv_t - log_s : -INFINITY;
    }
}

// The gradient, element by element: a CTA takes LP_NT * LP_U vectors of one
// row, read once and written once.  Bound by HBM.
template <class T>
__global__ void __launch_bounds__(LP_NT) token_logprobs_backward_k(LogprobsGradArgs a, int chunks) {
    constexpr int N = Vec<T>::N;
    const int tid = threadIdx.x;
    const int64_t r = blockIdx.x / chunks;
    const int c = blockIdx.x % chunks;
    const T *row = (const T *)a.logits + r * a.stride;
    T *out = (T *)a.dlogits + r * a.dstride;
    const RowSpan span = row_span(row, a.vocab);
    const T *body = row + span.head;
    T *obody = out + span.head;
    const bool wide = ((uintptr_t)obody & 15) == 0;
    const int v0 = c * LP_NT * LP_U + tid;
    const uint32_t target = a.targets ? a.targets[r] : NO_TOKEN;
    const bool gone = a.targets && target >= (uint32_t)a.vocab;
    uint4 raw[LP_U];
    if (!gone) {
#pragma unroll
        for (int u = 0; u < LP_U; ++u)
            if (v0 + u * LP_NT < span.n_vec) raw[u] = load16_rw(body + (int64_t)(v0 + u * LP_NT) * N);
    }
    const float m = a.stats[2 * r], log_s = a.stats[2 * r + 1];
    const bool zero = gone || (m == -INFINITY && log_s == -INFINITY);
    const float gl = a.g_logprob ? a.g_logprob[r] : 0.0f, ge = a.g_entropy ? a.g_entropy[r] : 0.0f;
    const float ca = -(gl + (a.g_entropy ? ge * a.entropy[r] : 0.0f)) * a.inv_t, cb = -ge * LN2 * a.inv_t;
    const float log2_s = log_s * LOG2E;
    auto grad = [&](float z, int e) {
        const float y = fmaf(z - m, a.scale, -log2_s);
        float dz = ex2(y) * fmaf(cb, fmaxf(y, -256.0f), ca);
        if ((uint32_t)e == target) dz = fmaf(gl, a.inv_t, dz);
        return zero ? 0.0f : dz;
    };
#pragma unroll
    for (int u = 0; u < LP_U; ++u) {
        const int v = v0 + u * LP_NT;
        if (v >= span.n_vec) break;
        float x[N];
        if (zero) raw[u] = make_uint4(0, 0, 0, 0);
        unpack<T>(raw[u], x);
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = grad(x[i], span.head + v * N + i);
        if (wide) {
            store16(obody + (int64_t)v * N, pack<T>(x));
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) obody[(int64_t)v * N + i] = from_f32<T>(x[i]);
        }
    }
    auto single = [&](int e) { out[e] = from_f32<T>(zero ? 0.0f : grad(to_f32(row[e]), e)); };
    if (c == 0 && tid < span.head) single(tid);
    if (c == chunks - 1 && tid < span.tail) single(a.vocab - span.tail + tid);
}

}  // namespace

template <class T>
cudaError_t launch_logprobs(const LogprobsArgs &a, cudaStream_t st) {
    constexpr int N = Vec<T>::N;
    const int64_t n_vec = a.vocab / N;
    // A row is split while the rows alone do not fill the GPU and every thread
    // keeps a vector.
    int cs = 1;
    while (cs < MAX_CLUSTER && a.rows * cs < 148 * 4 && n_vec / (2 * cs) >= LP_NT) cs *= 2;
    const int64_t batches = ((n_vec + cs - 1) / cs + LP_NT * LP_U - 1) / (LP_NT * LP_U);
    int shift = 0;
    while ((batches >> shift) >= LP_SLOTS) ++shift;
    const size_t smem = a.top ? ((batches >> shift) + 1) * LP_NT * sizeof(float) : 0;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(a.rows * cs));
    cfg.blockDim = dim3(LP_NT);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cs;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cs > 1 ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, token_logprobs_k<T>, a, cs, shift);
}

template <class T>
cudaError_t launch_backward(const LogprobsGradArgs &a, cudaStream_t st) {
    constexpr int N = Vec<T>::N;
    const int64_t chunks = std::max<int64_t>(1, (a.vocab / N + LP_NT * LP_U - 1) / (LP_NT * LP_U));
    // One grid dimension holds 2^31 - 1 CTAs: more rows than that go in parts.
    const int64_t most = std::max<int64_t>(1, ((1ll << 31) - 1) / chunks);
    for (int64_t r = 0; r < a.rows; r += most) {
        LogprobsGradArgs b = a;
        b.rows = std::min(most, a.rows - r);
        b.logits = (const T *)a.logits + r * a.stride;
        b.dlogits = (T *)a.dlogits + r * a.dstride;
        b.stats = a.stats + 2 * r;
        if (a.targets) b.targets = a.targets + r;
        if (a.entropy) b.entropy = a.entropy + r;
        if (a.g_logprob) b.g_logprob = a.g_logprob + r;
        if (a.g_entropy) b.g_entropy = a.g_entropy + r;
        token_logprobs_backward_k<T><<<(unsigned)(b.rows * chunks), LP_NT, 0, st>>>(b, (int)chunks);
        if (cudaError_t e = cudaGetLastError()) return e;
    }
    return cudaSuccess;
}

cudaError_t token_logprobs(const LogprobsArgs &a, int dtype, cudaStream_t st) {
    switch (dtype) {
        case 0: return launch_logprobs<float>(a, st);
        case 1: return launch_logprobs<__half>(a, st);
        default: return launch_logprobs<__nv_bfloat16>(a, st);
    }
}

cudaError_t token_logprobs_backward(const LogprobsGradArgs &a, int dtype, cudaStream_t st) {
    switch (dtype) {
        case 0: return launch_backward<float>(a, st);
        case 1: return launch_backward<__half>(a, st);
        default: return launch_backward<__nv_bfloat16>(a, st);
    }
}

}  // namespace nk
