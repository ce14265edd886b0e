// distill.cu -- the distillation loss from a teacher's top logits with its
// gradient (include/noetic/head.h).

#include <cooperative_groups.h>

#include <algorithm>

#include "nk_head.cuh"
#include "nk_head.h"

namespace nk {

namespace {

constexpr int DS_NT = 256;
constexpr int TEACHER_MAX = 256;  // one entry per thread
constexpr int DS_U = 4;
constexpr int DS_DEPTH = 4;
constexpr int DS_CLUSTER = 8;
constexpr int DS_PART = 68 << 10;   // bytes of a part: three to an SM
constexpr int DS_MOST = 216 << 10;  // the most that a CTA keeps

__device__ __forceinline__ float teacher_value(const void *p, int dtype, int64_t i) {
    return dtype == 0   ? ((const float *)p)[i]
           : dtype == 1 ? to_f32(((const __half *)p)[i])
                        : to_f32(((const __nv_bfloat16 *)p)[i]);
}

// One row by a cluster of `cs` CTAs, each with a contiguous part of it that
// stays in shared memory between the two passes: the logits are read from HBM
// once, for the softmax sums, and the gradient is made from the copy.  A
// thread keeps the vectors that it loaded itself, so the copy needs no
// barrier.  Bound by HBM (one read, one write).
//
// The teacher's entries lie one per thread; each CTA answers for the entries
// whose ids are in its part: their terms of the loss, and their places in the
// gradient, which it writes after a barrier over the dense gradient's values.
template <class T>
__global__ void __launch_bounds__(DS_NT) distill_k(DistillArgs a, int cs, int keep) {
    namespace cg = cooperative_groups;
    extern __shared__ uint4 kept[];  // keep vectors
    __shared__ float red[32], sums_out[2], kl_part[DS_CLUSTER];
    __shared__ uint32_t id[TEACHER_MAX];
    __shared__ float q[TEACHER_MAX];
    constexpr int N = Vec<T>::N;
    const int tid = threadIdx.x;
    const int64_t r = blockIdx.x / cs;
    const int rank = blockIdx.x % cs;
    const T *row = (const T *)a.logits + r * a.stride;
    T *out = a.dlogits ? (T *)a.dlogits + r * a.dstride : nullptr;
    const RowSpan span = row_span(row, a.vocab);
    const T *body = row + span.head;
    T *obody = out + span.head;
    const bool wide = ((uintptr_t)obody & 15) == 0;
    const int v0 = (int)((int64_t)span.n_vec * rank / cs), v1 = (int)((int64_t)span.n_vec * (rank + 1) / cs);
    const int n_head = rank == 0 ? span.head : 0, n_tail = rank == cs - 1 ? span.tail : 0;
    // The elements of this part.
    const int e0 = rank == 0 ? 0 : span.head + v0 * N, e1 = rank == cs - 1 ? a.vocab : span.head + v1 * N;
    const float scale = a.scale;

    auto put = [&](int v, float (&x)[N]) {
        if (wide) {
            store16(obody + (int64_t)v * N, pack<T>(x));
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) obody[(int64_t)v * N + i] = from_f32<T>(x[i]);
        }
    };
    auto zeros = [&] {
        float x[N] = {};
        for (int v = v0 + tid; v < v1; v += DS_NT) put(v, x);
        if (tid < n_head) out[tid] = from_f32<T>(0.0f);
        if (tid < n_tail) out[a.vocab - span.tail + tid] = from_f32<T>(0.0f);
    };

    // The teacher's entry of this thread: q = softmax(teacher / temperature).
    const uint32_t my = tid < a.n ? a.ids[r * a.n + tid] : NO_TOKEN;
    const float t = my < (uint32_t)a.vocab ? teacher_value(a.teacher, a.teacher_dtype, r * a.n + tid) : -INFINITY;
    const float w = a.row_weight ? a.row_weight[r] : 1.0f;
    const bool live = t != -INFINITY;
    if (!__syncthreads_or(live)) {  // no entries: the row is not read, in no CTA of the cluster
        if (rank == 0 && tid == 0 && a.loss) a.loss[r] = 0.0f;
        if (out) zeros();
        return;
    }
    const bool mine = live && (int)my >= e0 && (int)my < e1;
    const float z_my = mine ? to_f32(row[my]) : 0.0f;

    SoftSums sums;
    if (out) {
        // Groups of DS_U vectors per thread, DS_DEPTH groups on their way.
        constexpr int STEP = DS_NT * DS_U;
        auto fetch = [&](int v) {
#pragma unroll
            for (int u = 0; u < DS_U; ++u)
                if (v + u * DS_NT < keep && v0 + v + u * DS_NT < v1)
                    copy_async16(&kept[v + u * DS_NT], body + (int64_t)(v0 + v + u * DS_NT) * N);
            copy_commit();
        };
#pragma unroll
        for (int g = 0; g < DS_DEPTH; ++g) fetch(tid + g * STEP);
        const int n_kept = min(keep, v1 - v0);
        for (int v = tid; v < n_kept; v += STEP) {
            copy_wait<DS_DEPTH - 1>();
            uint4 raw[DS_U];
#pragma unroll
            for (int u = 0; u < DS_U; ++u) raw[u] = v + u * DS_NT < n_kept ? kept[v + u * DS_NT] : masked16<T>();
            fetch(v + DS_DEPTH * STEP);
            add_batch<T, DS_U>(raw, sums, scale);
        }
        copy_wait<0>();
        if (v0 + keep < v1) stream_sums<T, DS_NT, DS_U>(body, v0 + keep, v1, scale, sums, [](int, float) {});
    } else {
        stream_sums<T, DS_NT, DS_U>(body, v0, v1, scale, sums, [](int, float) {});
    }
    float z_head = 0.0f, z_tail = 0.0f;
    if (tid < n_head) {
        z_head = to_f32(row[tid]);
        sums.raise(z_head, scale);
        sums.add(z_head, scale);
    }
    if (tid < n_tail) {
        z_tail = to_f32(row[a.vocab - span.tail + tid]);
        sums.raise(z_tail, scale);
        sums.add(z_tail, scale);
    }

    const float tm = block_max(t, red);
    const float ty = (t - tm) * a.inv_t;
    const float te = live ? expf(ty) : 0.0f;
    const float ts = block_sum(te, red);
    const float my_q = te / ts;
    if (tid < a.n) {
        id[tid] = live ? my : NO_TOKEN;
        q[tid] = my_q;
    }
    sums = block_join(sums, scale, red);
    if (cs > 1) {
        cg::cluster_group cluster = cg::this_cluster();
        if (tid == 0) {
            sums_out[0] = sums.m;
            sums_out[1] = sums.s;
        }
        cluster.sync();
        // The parts in their order, the same in every CTA.
        SoftSums all;
        for (int c = 0; c < cs; ++c) all.m = fmaxf(all.m, cluster.map_shared_rank(sums_out, c)[0]);
        for (int c = 0; c < cs; ++c) {
            SoftSums part;
            part.m = cluster.map_shared_rank(sums_out, c)[0];
            part.s = cluster.map_shared_rank(sums_out, c)[1];
            if (part.m != -INFINITY) part.raise(all.m, scale);
            all.s += part.s;
        }
        sums = all;
    }
    const float log_s = logf(sums.s);
    const bool empty = sums.m == -INFINITY && sums.s == 0.0f;  // a student that can say nothing
    float part = 0.0f;
    if (mine && my_q != 0.0f)
        part = empty ? INFINITY : my_q * ((ty - logf(ts)) - ((z_my - sums.m) * a.inv_t - log_s));
    const float kl = block_sum(part, red);
    if (cs > 1) {
        cg::cluster_group cluster = cg::this_cluster();
        if (tid == 0) cluster.map_shared_rank(kl_part, 0)[rank] = kl;
        cluster.barrier_arrive();
    }

    if (out && (w == 0.0f || empty)) {
        zeros();
    } else if (out) {
        const float g = a.grad_scale * w * a.temperature, log2_s = log_s * LOG2E;
        auto grad = [&](float z) { return g * ex2(fmaf(z - sums.m, scale, -log2_s)); };
        for (int v = v0 + tid; v < v1; v += DS_NT) {
            float x[N];
            unpack<T>(v - v0 < keep ? kept[v - v0] : load16_rw(body + (int64_t)v * N), x);
#pragma unroll
            for (int i = 0; i < N; ++i) x[i] = grad(x[i]);
            put(v, x);
        }
        if (tid < n_head) out[tid] = from_f32<T>(grad(z_head));
        if (tid < n_tail) out[a.vocab - span.tail + tid] = from_f32<T>(grad(z_tail));
        __syncthreads();
        // The entries' own places, from the first of each id.
        if (mine) {
            float share = 0.0f;
            bool first = true;
            for (int i = 0; i < a.n; ++i)
                if (id[i] == my) {
                    share += q[i];
                    first = first && i >= tid;
                }
            if (first) out[my] = from_f32<T>(g * (ex2(fmaf(z_my - sums.m, scale, -log2_s)) - share));
        }
    }
    if (cs > 1) {
        cg::this_cluster().barrier_wait();
        if (rank == 0 && tid == 0 && a.loss) {
            float all = 0.0f;
            for (int c = 0; c < cs; ++c) all += kl_part[c];
            a.loss[r] = a.temperature * a.temperature * all;
        }
    } else if (tid == 0 && a.loss) {
        a.loss[r] = a.temperature * a.temperature * kl;
    }
}

template <class T>
cudaError_t launch_distill(const DistillArgs &a, cudaStream_t st) {
    constexpr int N = Vec<T>::N;
    const int64_t n_vec = a.vocab / N;
    // A row is split until a part and those of two more CTAs fit an SM's shared
    // memory, and while the rows alone do not fill the GPU and every thread keeps a vector.
    int cs = 1;
    while (cs < DS_CLUSTER && ((a.dlogits && (n_vec + cs - 1) / cs * 16 > DS_PART) ||
                               (a.rows * cs < 148 * 2 && n_vec / (2 * cs) >= DS_NT)))
        cs *= 2;
    const int64_t keep = a.dlogits ? std::min<int64_t>((n_vec + cs - 1) / cs, DS_MOST / 16) : 0;
    auto kern = distill_k<T>;
    if (keep * 16 > 32768) {
        cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, DS_MOST);
        if (e != cudaSuccess) return e;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(a.rows * cs));
    cfg.blockDim = dim3(DS_NT);
    cfg.dynamicSmemBytes = (size_t)keep * 16;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cs;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cs > 1 ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kern, a, cs, (int)keep);
}

}  // namespace

cudaError_t distill(const DistillArgs &a, int dtype, cudaStream_t st) {
    switch (dtype) {
        case 0: return launch_distill<float>(a, st);
        case 1: return launch_distill<__half>(a, st);
        default: return launch_distill<__nv_bfloat16>(a, st);
    }
}

}  // namespace nk
