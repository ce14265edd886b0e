// logprobs.cu -- log probabilities of given tokens with the row's entropy and
// most probable alternatives, and their gradient (include/noetic/head.h).

#include <cooperative_groups.h>

#include <algorithm>
#include <cfloat>

#include "nk_head.cuh"
#include "nk_head.h"

namespace nk {

namespace {

constexpr int LP_NT = 256, LP_U = 4;  // the gradient: threads of a CTA, vectors of each
constexpr int TOP_MAX = 128;
constexpr int MAX_CLUSTER = 8;
constexpr int MAXIMA = 256;  // that a warp takes the bound on the alternatives from

// The threads that share a row: a warp or a block.
template <int NT>
__device__ __forceinline__ void team_sync() {
    if constexpr (NT == 32)
        __syncwarp();
    else
        __syncthreads();
}

// Shared memory of a team that looks for alternatives.  `cand` holds keys:
// order_key << 32 | ~index, so that the larger key is the better alternative
// and equal logits go to the lower index.
struct TopScratch {
    uint32_t hist[256];
    uint32_t warp_count[32];
    uint64_t kept[TOP_MAX];
};
struct TopTeam {
    uint64_t *cand;    // [cand_cap], shared with sc
    uint64_t *best;    // [top]
    float *group_max;  // [slots][team size]
    float *thread_max; // [team size], a block's
    uint32_t *hits;    // [hit_cap]
    TopScratch *sc;
    uint32_t *word;    // [4]: candidates, hits, prefix, above
    int cand_cap, hit_cap;
};

// The `top` largest of row[e0, e1) above -infinity, equal values by index, in
// descending order in out[0, top), 0 behind the last: a radix select finds the
// last value kept; one ordered walk then takes what lies above it and the
// first of those equal to it.
template <class T, int NT>
__device__ __noinline__ void exact_top(const T *row, int e0, int e1, int top, TopScratch *sc, uint32_t *word, uint64_t *out) {
    const int tid = threadIdx.x % NT, lane = tid & 31, warp = tid >> 5;
    team_sync<NT>();
    if (tid == 0) word[2] = word[3] = 0;
    team_sync<NT>();
    for (int shift = 24; shift >= 0; shift -= 8) {
        for (int i = tid; i < 256; i += NT) sc->hist[i] = 0;
        team_sync<NT>();
        const uint32_t prefix = word[2];
        for (int e = e0 + tid; e < e1; e += NT) {
            const float z = to_f32(row[e]);
            if (!(z > -INFINITY)) continue;
            const uint32_t k = order_key(z);
            if (shift == 24 || (k >> (shift + 8)) == (prefix >> (shift + 8))) atomicAdd(&sc->hist[(k >> shift) & 255], 1u);
        }
        team_sync<NT>();
        if (tid == 0) {
            uint32_t above = word[3];
            int b = 255;
            while (b > 0 && above + sc->hist[b] < (uint32_t)top) above += sc->hist[b--];
            word[3] = above;
            word[2] = prefix | ((uint32_t)b << shift);
        }
        team_sync<NT>();
    }
    const uint32_t last = word[2], above = word[3];
    uint32_t equal = 0;  // seen so far, the same in every thread
    team_sync<NT>();
    if (tid == 0) word[0] = 0;
    team_sync<NT>();
    for (int b = e0; b < e1; b += NT) {
        const int e = b + tid;
        const float z = e < e1 ? to_f32(row[e]) : -INFINITY;
        const bool real = z > -INFINITY;
        const uint32_t k = order_key(z);
        const uint64_t key = ((uint64_t)k << 32) | (uint32_t)~(uint32_t)e;
        if (real && k > last) sc->kept[atomicAdd(&word[0], 1u)] = key;
        const bool eq = real && k == last;
        const uint32_t votes = __ballot_sync(0xffffffffu, eq);
        uint32_t before = equal;
        if constexpr (NT == 32) {
            equal += __popc(votes);
        } else {
            if (lane == 0) sc->warp_count[warp] = __popc(votes);
            __syncthreads();
            for (int w = 0; w < NT / 32; ++w) {
                if (w < warp) before += sc->warp_count[w];
                equal += sc->warp_count[w];
            }
            __syncthreads();
        }
        before += __popc(votes & ((1u << lane) - 1u));
        if (eq && above + before < (uint32_t)top) sc->kept[above + before] = key;
    }
    team_sync<NT>();
    const int n = min((uint32_t)top, above + equal);
    for (int i = tid; i < top; i += NT) {
        if (i < n) {
            int rank = 0;
            for (int j = 0; j < n; ++j) rank += sc->kept[j] > sc->kept[i];
            out[rank] = sc->kept[i];
        } else {
            out[i] = 0;
        }
    }
    team_sync<NT>();
}

// Vectors (log2) that a thread of a team takes at a time.
template <int NT>
constexpr int log_batch() {
    return NT == 32 ? 2 : 3;
}

// One team's part of one row: the softmax sums, and with a.top its best
// alternatives in w.best.  The part is read once: a thread takes a batch of
// 16-byte vectors at a time, raises its running maximum by theirs and adds
// their exponentials.
//
// Alternatives.  Threads keep the maximum of each group of their vectors in
// shared memory.  The top-th largest of MAXIMA of these (a block: of its
// threads' own maxima; a warp: of eight groups per lane) bounds the top-th
// logit from below, since as many distinct elements reach it.  Only the few
// groups that reach the bound are read again, from L2, a vector to a thread
// and all at once, for the elements that reach it: about `top` candidates,
// ranked by counting.  Where more groups or candidates reach it than fit (many
// equal logits, an order that gives one thread all the large ones), exact_top
// takes over.
template <class T, int NT, bool FINE>
__device__ __forceinline__ SoftSums logprobs_part(const LogprobsArgs &a, const T *row, RowSpan span, int v0, int v1, bool first,
                                                  bool last, int slot_shift, const TopTeam &w) {
    constexpr int N = Vec<T>::N;
    const int tid = threadIdx.x % NT, lane = tid & 31;
    const T *body = row + span.head;
    const int n_head = first ? span.head : 0, n_tail = last ? span.tail : 0;
    const float scale = a.scale;
    SoftSums sums;
    float tmax = -INFINITY, gmax = -INFINITY;
    const int batches = stream_sums<T, NT, 1 << log_batch<NT>(), true, false, FINE>(body, v0, v1, tid, scale, sums, [&](int b, float bm) {
        if (a.top) {
            gmax = (b & ((1 << slot_shift) - 1)) == 0 ? bm : fmaxf(gmax, bm);
            w.group_max[(b >> slot_shift) * NT + tid] = gmax;
            tmax = fmaxf(tmax, bm);
        }
    });
    // The ends that no vector covers, one element per thread and end.
    auto single = [&](int e) {
        const float z = to_f32(row[e]);
        sums.raise(z, scale);
        sums.template add<FINE>(z, scale);
        tmax = fmaxf(tmax, z);
    };
    if (tid < n_head) single(tid);
    if (tid < n_tail) single(a.vocab - span.tail + tid);
    if (!a.top) return sums;

    const int groups = (batches + (1 << slot_shift) - 1) >> slot_shift;
    if (tid == 0) w.word[0] = w.word[1] = 0;
    if constexpr (NT == 32) {
        for (int g = groups; g < MAXIMA / 32; ++g) w.group_max[g * 32 + lane] = -INFINITY;
    } else {
        w.thread_max[tid] = tmax;
    }
    team_sync<NT>();
    if (tid < 32) {
        // A key that at least `top` of the maxima reach, and few more: halving
        // the range between the least and the greatest of them, sixteen times at
        // most.
        const float *maxima = NT == 32 ? w.group_max : w.thread_max;
        constexpr int PER_LANE = (NT == 32 ? MAXIMA : NT) / 32;
        uint32_t k[PER_LANE], lo = 0xFFFFFFFFu, hi = 0;
#pragma unroll
        for (int i = 0; i < PER_LANE; ++i) {
            k[i] = order_key(maxima[i * 32 + lane]);
            lo = min(lo, k[i]);
            hi = max(hi, k[i]);
        }
        lo = __reduce_min_sync(0xffffffffu, lo);
        hi = __reduce_max_sync(0xffffffffu, hi) + 1;
        const int enough = a.top + (a.top >> 2);
        for (int i = 0; i < 16 && hi - lo > 1; ++i) {
            const uint32_t mid = lo + (hi - lo) / 2;
            int n = 0;
#pragma unroll
            for (int j = 0; j < PER_LANE; ++j) n += k[j] >= mid;
            n = (int)__reduce_add_sync(0xffffffffu, (unsigned)n);
            if (n < a.top) {
                hi = mid;
            } else {
                lo = mid;
                if (n <= enough) break;
            }
        }
        if (lane == 0) w.word[2] = lo;
    }
    team_sync<NT>();
    // As a value; nothing above -infinity is below the lowest one.
    const float bound = w.word[2] > 0x00800000u ? key_value(w.word[2]) : -FLT_MAX;
    auto offer = [&](float z, int e) {
        if (z >= bound) {
            const uint32_t at = atomicAdd(&w.word[0], 1u);
            if (at < (uint32_t)w.cand_cap) w.cand[at] = ((uint64_t)order_key(z) << 32) | (uint32_t)~(uint32_t)e;
        }
    };
    if (tmax >= bound) {
        for (int g = 0; g < groups; ++g)
            if (w.group_max[g * NT + tid] >= bound) {
                const uint32_t at = atomicAdd(&w.word[1], 1u);
                if (at < (uint32_t)w.hit_cap) w.hits[at] = (uint32_t)(g * NT + tid);
            }
        if (tid < n_head) offer(to_f32(row[tid]), tid);
        if (tid < n_tail) offer(to_f32(row[a.vocab - span.tail + tid]), a.vocab - span.tail + tid);
    }
    team_sync<NT>();
    const int log_group = log_batch<NT>() + slot_shift, n_hits = (int)w.word[1];
    if (n_hits <= w.hit_cap) {
        for (int i = tid; i < (n_hits << log_group); i += NT) {
            const uint32_t hit = w.hits[i >> log_group];
            const int in_group = i & ((1 << log_group) - 1);
            const int v = v0 + (int)(hit % NT) + ((int)(hit / NT << log_group) + in_group) * NT;
            if (v >= v1) continue;
            float x[N];
            unpack<T>(load16(body + (int64_t)v * N), x);
#pragma unroll
            for (int k = 0; k < N; ++k) offer(x[k], span.head + v * N + k);
        }
    }
    team_sync<NT>();
    const int n = (int)w.word[0];
    if (n > w.cand_cap || n_hits > w.hit_cap) {
        exact_top<T, NT>(row, first ? 0 : span.head + v0 * N, last ? a.vocab : span.head + v1 * N, a.top, w.sc, w.word, w.best);
    } else {
        for (int i = n + tid; i < a.top; i += NT) w.best[i] = 0;
        for (int i = tid; i < n; i += NT) {
            const uint64_t key = w.cand[i];
            int rk = 0;
            for (int j = 0; j < n; ++j) rk += w.cand[j] > key;
            if (rk < a.top) w.best[rk] = key;
        }
        team_sync<NT>();
    }
    return sums;
}

// What a row without a token gets.
template <int NT>
__device__ __forceinline__ void no_token_row(const LogprobsArgs &a, int64_t r) {
    const int tid = threadIdx.x % NT;
    if (tid == 0) {
        if (a.logprob) a.logprob[r] = 0.0f;
        if (a.entropy) a.entropy[r] = 0.0f;
        if (a.stats) a.stats[2 * r] = a.stats[2 * r + 1] = 0.0f;
    }
    for (int i = tid; i < a.top; i += NT) {
        if (a.top_ids) a.top_ids[r * a.top + i] = NO_TOKEN;
        if (a.top_logprobs) a.top_logprobs[r * a.top + i] = -INFINITY;
    }
}

// The row's results from its whole sums and its best keys.
template <int NT, bool FINE>
__device__ __forceinline__ void write_row(const LogprobsArgs &a, int64_t r, const SoftSums &sums, float z_target,
                                          const uint64_t *best) {
    const int tid = threadIdx.x % NT;
    const float log_s = sums.log_sum<FINE>(), total = sums.s + sums.n;
    const bool empty = sums.m == -INFINITY && sums.s == 0.0f;
    if (tid == 0) {
        if (a.logprob) a.logprob[r] = empty ? -INFINITY : (z_target - sums.m) * a.inv_t - log_s;
        if (a.entropy) {
            const float h = log_s - LN2 * (sums.t / total);
            a.entropy[r] = empty || h < 0.0f ? 0.0f : h;
        }
        if (a.stats) {
            a.stats[2 * r] = sums.m;
            a.stats[2 * r + 1] = log_s;
        }
    }
    for (int i = tid; i < a.top; i += NT) {
        const uint64_t k = best[i];
        if (a.top_ids) a.top_ids[r * a.top + i] = k ? ~(uint32_t)k : NO_TOKEN;
        if (a.top_logprobs)
            a.top_logprobs[r * a.top + i] = k ? (key_value((uint32_t)(k >> 32)) - sums.m) * a.inv_t - log_s : -INFINITY;
    }
}

// ---------------------------------------------------------------- short rows: a warp each
// No barrier but the warp's own, so that 32 rows are in the air per SM and one
// row's search overlaps the others' loads.  16384 rows of 8192 bf16 with 20
// alternatives take 78 us (3.5 TB/s) and without 52 (5.2 TB/s): a short row waits
// for the search, that is for the warps' issue slots.
constexpr int WARP_ROWS = 8;

// Places for candidates and for hits per warp; more than these are rare.
__host__ __device__ inline int warp_cand_cap(int top) { return 3 * top + 64; }
__host__ __device__ inline int warp_hit_cap(int top) { return 2 * top + 64; }
// Bytes of one warp's TopTeam (a multiple of 16).
__host__ __device__ inline int warp_team_bytes(int top) {
    if (top == 0) return 0;
    const int cand = warp_cand_cap(top) * 8, sc = (int)sizeof(TopScratch);
    return ((cand > sc ? cand : sc) + top * 8 + MAXIMA * 4 + warp_hit_cap(top) * 4 + 16 + 15) & ~15;
}

template <class T>
__global__ void __launch_bounds__(32 * WARP_ROWS, 4) token_logprobs_warp_k(LogprobsArgs a, int slot_shift) {
    extern __shared__ __align__(16) unsigned char shared[];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t r = (int64_t)blockIdx.x * WARP_ROWS + warp;
    if (r >= a.rows) return;
    const T *row = (const T *)a.logits + r * a.stride;
    const uint32_t target = a.targets ? a.targets[r] : NO_TOKEN;
    if (a.targets && target >= (uint32_t)a.vocab) {
        no_token_row<32>(a, r);
        return;
    }
    const float z_target = a.targets && lane == 0 ? to_f32(row[target]) : 0.0f;
    TopTeam w = {};
    if (a.top) {
        unsigned char *p = shared + warp * warp_team_bytes(a.top);
        w.cand_cap = warp_cand_cap(a.top);
        w.hit_cap = warp_hit_cap(a.top);
        w.cand = (uint64_t *)p;
        w.sc = (TopScratch *)p;
        p += max(w.cand_cap * 8, (int)sizeof(TopScratch));
        w.best = (uint64_t *)p;
        w.group_max = (float *)(p + a.top * 8);
        w.hits = (uint32_t *)(w.group_max + MAXIMA);
        w.word = w.hits + w.hit_cap;
    }
    const RowSpan span = row_span(row, a.vocab);
    SoftSums sums = logprobs_part<T, 32, false>(a, row, span, 0, span.n_vec, true, true, slot_shift, w);
    write_row<32, false>(a, r, warp_join<true>(sums, a.scale), z_target, w.best);
}

// ---------------------------------------------------------------- long rows: a block or a cluster each
// One row by a cluster of `cs` CTAs (one, when there are rows enough to fill
// the GPU), each with a contiguous part of it.  What bounds it: HBM; 16-bit
// logits need one exponential per two bytes, 16 of which an SM's
// special-function unit makes per clock, 1.4 times what HBM delivers.  4096 rows
// of 131072 bf16 take 180 us with 20 alternatives (6.0 TB/s, 0.91 of the copy rate)
// and 159 without (as fast as it only reads, 1.03), 2048 of f32 170 with them (0.97):
// two sets of inputs in turn.  Among passes over other inputs the first takes 195 to
// 207.
constexpr int LP_SLOTS = 32;      // groups per thread
constexpr int HITS = 512;
constexpr int CANDIDATES = 1024;  // at least MAX_CLUSTER * TOP_MAX

template <int NT>
struct LogprobsShared {
    float4 warps[NT / 32 > MAX_CLUSTER ? NT / 32 : MAX_CLUSTER], part;
    uint32_t word[4], hits[HITS];
    uint64_t cand[CANDIDATES];
    uint64_t best[TOP_MAX];
    float thread_max[NT];
};
static_assert(sizeof(TopScratch) <= CANDIDATES * 8 && CANDIDATES >= MAX_CLUSTER * TOP_MAX, "");

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

template <class T, int NT, bool FINE>
__global__ void __launch_bounds__(NT, 1024 / NT) token_logprobs_k(LogprobsArgs a, int log_cs, int slot_shift) {
    extern __shared__ float group_max[];
    __shared__ LogprobsShared<NT> sh;
    const int tid = threadIdx.x;
    const int cs = 1 << log_cs;
    const int64_t r = blockIdx.x >> log_cs;
    const int rank = blockIdx.x & (cs - 1);
    const T *row = (const T *)a.logits + r * a.stride;
    const uint32_t target = a.targets ? a.targets[r] : NO_TOKEN;
    if (a.targets && target >= (uint32_t)a.vocab) {
        if (rank == 0) no_token_row<NT>(a, r);
        return;  // the whole cluster
    }
    const float z_target = a.targets && rank == 0 && tid == 0 ? to_f32(row[target]) : 0.0f;
    TopTeam w;
    w.cand = sh.cand;
    w.best = sh.best;
    w.group_max = group_max;
    w.thread_max = sh.thread_max;
    w.hits = sh.hits;
    w.sc = (TopScratch *)sh.cand;
    w.word = sh.word;
    w.cand_cap = CANDIDATES;
    w.hit_cap = HITS;
    const RowSpan span = row_span(row, a.vocab);
    const int v0 = (int)((int64_t)span.n_vec * rank >> log_cs), v1 = (int)((int64_t)span.n_vec * (rank + 1) >> log_cs);
    SoftSums sums = logprobs_part<T, NT, FINE>(a, row, span, v0, v1, rank == 0, rank == cs - 1, slot_shift, w);
    sums = block_join<NT, FINE>(sums, a.scale, sh.warps);

    if (cs > 1) {
        namespace cg = cooperative_groups;
        cg::cluster_group cluster = cg::this_cluster();
        if (tid == 0) sh.part = make_float4(sums.m, sums.s, sums.t, sums.n);
        cluster.sync();
        if (rank == 0) {
            // The parts in their order.
            if (tid < cs) sh.warps[tid] = *cluster.map_shared_rank(&sh.part, tid);
            __syncthreads();
            sums = join_places<true, FINE>(sh.warps, cs, a.scale);
            if (a.top) {
                for (int i = tid; i < cs * a.top; i += NT)
                    sh.cand[i] = cluster.map_shared_rank(sh.best, i / a.top)[i % a.top];
                __syncthreads();
                for (int i = tid; i < a.top; i += NT) sh.best[i] = 0;
                __syncthreads();
                for (int i = tid; i < cs * a.top; i += NT) {
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
    write_row<NT, FINE>(a, r, sums, z_target, sh.best);
}

// The gradient, element by element: a CTA takes LP_NT * LP_U vectors of one
// row, read once and written once.  Bound by HBM: 4096 rows of 32768 f32, an
// eighth of them without a target (not read), take 152 us (6.6 TB/s), 2048 rows of
// 65537 bf16, read and written in vectors that start at the same places, 93 us (5.8
// TB/s).  Where the gradient's rows start elsewhere than the logits' it is stored
// element by element: these rows of stride 65544 into dense ones 337 us, f32 rows,
// whose stores still fill their sectors, 165 as dense.
template <class T>
__global__ void __launch_bounds__(LP_NT) token_logprobs_backward_k(LogprobsGradArgs a, int chunks) {
    // (A 32-bit division: rows * chunks is below 2^31.)
    constexpr int N = Vec<T>::N;
    const int tid = threadIdx.x;
    const int64_t r = blockIdx.x / (unsigned)chunks;
    const int c = blockIdx.x % (unsigned)chunks;
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

template <class T, int NT, bool FINE>
cudaError_t launch_blocks(const LogprobsArgs &a, cudaStream_t st) {
    const int64_t n_vec = a.vocab / Vec<T>::N;
    // A row is split over a cluster while the rows alone leave SMs idle and
    // every thread keeps a vector: 16 rows of 131072 f32 13 us and unsplit 23, 120 rows
    // 23 and 28.  Not further: to a split of two, 200 such rows take 34 us instead
    // of 28, 120 rows in splits of eight 31.
    int log_cs = 0;
    while ((1 << log_cs) < MAX_CLUSTER && a.rows << log_cs < 148 && n_vec >> (log_cs + 1) >= NT) ++log_cs;
    const int cs = 1 << log_cs;
    constexpr int step = NT << log_batch<NT>();
    const int64_t batches = ((n_vec + cs - 1) / cs + step - 1) / step;
    int shift = 0;
    while ((batches >> shift) >= LP_SLOTS) ++shift;
    const size_t smem = a.top ? ((batches >> shift) + 1) * NT * sizeof(float) : 0;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(a.rows * cs));
    cfg.blockDim = dim3(NT);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cs;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cs > 1 ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, token_logprobs_k<T, NT, FINE>, a, log_cs, shift);
}

template <class T>
cudaError_t launch_logprobs(const LogprobsArgs &a, cudaStream_t st) {
    constexpr int N = Vec<T>::N;
    const int64_t n_vec = a.vocab / N;
    // A warp per row for rows of up to 32 KB, when there are enough to fill the
    // GPU with warps.  Measured with 20 alternatives, a warp against a block per
    // row: 16384 rows of 4 KB 45 and 127 us, of 16 KB 81 and 133, of 32 KB 127 and
    // 160, of 64 KB 257 and 216; 1024 rows of 32 KB 27 and 22.
    if (n_vec <= 2048 && a.rows >= std::max<int64_t>(512, n_vec)) {
        int shift = 0;
        constexpr int step = 32 << log_batch<32>();
        while (((n_vec + step - 1) / step + (1 << shift) - 1) >> shift > MAXIMA / 32) ++shift;
        const int smem = WARP_ROWS * warp_team_bytes(a.top);
        auto kern = token_logprobs_warp_k<T>;
        if (smem > 48 << 10) {
            cudaError_t e = allow_shared(kern, WARP_ROWS * warp_team_bytes(TOP_MAX));
            if (e != cudaSuccess) return e;
        }
        kern<<<(unsigned)((a.rows + WARP_ROWS - 1) / WARP_ROWS), 32 * WARP_ROWS, smem, st>>>(a, shift);
        return cudaGetLastError();
    }
    // A block of 128 threads, eight to an SM, or of 256, four: the smaller one
    // where the larger would need a second round for few rows, and for rows of up to 128
    // KB, whose search is a larger share.  Measured with 20 alternatives, 128
    // against 256: 700 rows of 40 KB 16 and 23 us, of 256 KB 47 and 57; 3000 rows of
    // 100 KB 74 and 82; but 1500 rows of 256 KB 96 and 86, 450 rows of 100 KB 23 and 20.
    // With more than 64 alternatives 128 threads' maxima bound them loosely.
    const bool small = a.rows > 592 && a.top <= 64 && (a.rows <= 1184 || n_vec <= 8192);
    if (small) return launch_blocks<T, 128, false>(a, st);
    // With few rows the SMs wait for memory, and a single row's log probability
    // may be all that is looked at: fine sums (one row of 32768 f32 10 us with and
    // without, 120 of 131072 23 and 21; but 4096 of 131072 bf16 243 and 192, one after
    // the other on one GPU).
    return a.rows <= 148 ? launch_blocks<T, 256, true>(a, st) : launch_blocks<T, 256, false>(a, st);
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
