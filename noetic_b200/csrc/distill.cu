// distill.cu -- the distillation loss from a teacher's top logits with its
// gradient (include/noetic/head.h).

#include <cooperative_groups.h>

#include <algorithm>

#include "nk_head.cuh"
#include "nk_head.h"

namespace nk {

namespace {

constexpr int TEACHER_MAX = 256;
constexpr int DS_U = 4;       // vectors of a thread at a time
constexpr int DS_NT = 192;    // streaming threads of a CTA
constexpr int DS_CLUSTER = 8;
constexpr int DUP_BITS = 16384, WARP_DUP_BITS = 8192;
constexpr int DS_PART = 68 << 10;  // bytes of a part
constexpr int DS_MOST = (208 << 10) / (DS_NT * DS_U * 16) * (DS_NT * DS_U * 16);  // the most that a CTA keeps, in whole batches
constexpr int DS_ROWS = 4;         // rows of a cluster, at most

__device__ __forceinline__ float teacher_value(const void *p, int dtype, int64_t i) {
    return dtype == 0   ? ((const float *)p)[i]
           : dtype == 1 ? to_f32(((const __half *)p)[i])
                        : to_f32(((const __nv_bfloat16 *)p)[i]);
}

// Waits until at most n of this thread's groups of copies are on their way
// (from 8 on: until at most 7 are).
__device__ __forceinline__ void copy_wait_for(int n) {
    switch (n) {
        case 0: copy_wait<0>(); break;
        case 1: copy_wait<1>(); break;
        case 2: copy_wait<2>(); break;
        case 3: copy_wait<3>(); break;
        case 4: copy_wait<4>(); break;
        case 5: copy_wait<5>(); break;
        case 6: copy_wait<6>(); break;
        default: copy_wait<7>(); break;
    }
}

// The entries of one row in the lanes of a warp, lane l with l, l + 32, ...;
// an entry that does not count has no token.  q holds the teacher's logits, then
// the shares.  ENTRIES is 2 for teachers of up to 64 entries, else 8: these
// registers are every warp's.
template <int ENTRIES>
struct Entries {
    uint32_t id[ENTRIES];
    float q[ENTRIES];

    __device__ __forceinline__ void load(const DistillArgs &a, int64_t r, int lane) {
#pragma unroll
        for (int k = 0; k < ENTRIES; ++k) {
            const int i = k * 32 + lane;
            id[k] = i < a.n ? a.ids[r * a.n + i] : NO_TOKEN;
            q[k] = i < a.n ? teacher_value(a.teacher, a.teacher_dtype, r * a.n + i) : -INFINITY;
        }
    }
    // Drops what does not count; whether anything is left.
    __device__ __forceinline__ bool settle(const DistillArgs &a) {
        bool any = false;
#pragma unroll
        for (int k = 0; k < ENTRIES; ++k) {
            if (id[k] >= (uint32_t)a.vocab) q[k] = -INFINITY;
            if (q[k] == -INFINITY) id[k] = NO_TOKEN;
            any |= id[k] != NO_TOKEN;
        }
        return __any_sync(0xffffffffu, any);
    }
    // q = softmax(q / temperature); returns the maximum and the logarithm of the sum that log q takes.
    __device__ __forceinline__ void share(float inv_t, int n, float (&log_q)[ENTRIES]) {
        float m = -INFINITY, s = 0.0f;
#pragma unroll
        for (int k = 0; k < ENTRIES; ++k) m = fmaxf(m, q[k]);
        m = warp_max1(m);
#pragma unroll
        for (int k = 0; k < ENTRIES; ++k) {
            log_q[k] = (q[k] - m) * inv_t;
            q[k] = k * 32 < n && id[k] != NO_TOKEN ? expf(log_q[k]) : 0.0f;
            s += q[k];
        }
        s = warp_sum(s);
        const float log_s = logf(s), inv_s = 1.0f / s;
#pragma unroll
        for (int k = 0; k < ENTRIES; ++k) {
            log_q[k] -= log_s;
            q[k] *= inv_s;
        }
    }
};

// temperature q (log q - log p) of an entry, p = exp((z - m) / temperature - log_s).
// Not divided by the temperature, so that a student's logit of f32's lowest value
// stays in range at temperatures below 1.
__device__ __forceinline__ float loss_term(float q, float log_q, float z, float m, float log_s, float temperature) {
    return q * fmaf(temperature, log_q + log_s, m - z);
}

// Whether two of a warp's entries have the same id, by a bitmap of DUP_BITS bits
// in shared memory that is clear before and after; ids that far apart may pass
// for the same one.  Walking all pairs costs a row more than its other teacher
// work together, and ids are nearly always distinct.
template <int DUP_BITS, int ENTRIES>
__device__ __forceinline__ bool perhaps_twice(const uint32_t (&id)[ENTRIES], uint32_t *bits) {
    bool twice = false;
    __syncwarp();
#pragma unroll
    for (int k = 0; k < ENTRIES; ++k)
        if (id[k] != NO_TOKEN) {
            const uint32_t at = id[k] & (DUP_BITS - 1), bit = 1u << (at & 31);
            twice |= atomicOr(&bits[at >> 5], bit) & bit;
        }
    __syncwarp();
#pragma unroll
    for (int k = 0; k < ENTRIES; ++k)
        if (id[k] != NO_TOKEN) bits[(id[k] & (DUP_BITS - 1)) >> 5] = 0;
    return __any_sync(0xffffffffu, twice);
}

// The shares of this lane's ids, over all entries that have them.
template <int ENTRIES>
__device__ __forceinline__ void total_shares(const Entries<ENTRIES> &e, int n, uint32_t *id, float *q, float (&share)[ENTRIES]) {
    const int lane = threadIdx.x & 31;
    __syncwarp();
#pragma unroll
    for (int k = 0; k < ENTRIES; ++k)
        if (k * 32 + lane < n) {
            id[k * 32 + lane] = e.id[k];
            q[k * 32 + lane] = e.q[k];
        }
    __syncwarp();
#pragma unroll
    for (int k = 0; k < ENTRIES; ++k) {
        share[k] = 0.0f;
        for (int j = 0; j < n; ++j) share[k] += id[j] == e.id[k] ? q[j] : 0.0f;
    }
    __syncwarp();
}

// Rows by a cluster of CTAs, each with a contiguous part of every row that
// stays in shared memory between the two passes over it: the logits are read
// from HBM once, for the softmax sums, and the gradient is made from the copy.
// A thread keeps the vectors that it copied itself, so the copy needs no
// barrier; as it takes a vector for the gradient it sends for the same vector
// of the cluster's next row, so that reads and writes run side by side.
//
// What a row costs beside its elements is kept off the NT threads that stream
// it.  They meet once per row, to join their sums.  A warp of its own sees to
// the teacher: it reads the next row's entries a row ahead, softmaxes this
// row's while the logits stream in, exchanges the sums with the cluster's other
// CTAs, and after the streaming threads have passed (they do not wait for it)
// puts the gradient's values in the entries' places.  Each CTA answers for the
// entries in its part.
//
// 4096 rows of 16384 f32 with 32 entries take 90 us (5.6 TB/s, 0.86 of HBM's copy
// rate), 8192 of 131072 bf16 with 64 take 932 us (4.6 TB/s, 0.70; 980 on the GPU of what
// follows).  16-bit rows cost the special-function unit two exponentials per element,
// one for the sum and one for the gradient, about 480 us of its time, and their
// instructions issue in turns with the copies: without the exponentials the same rows
// measured 770 us, without the cluster's exchange, which every row waits for, 872,
// without both 725.  Taking the exponentials of half of the elements by a polynomial
// instead gained nothing, reading the row a second time from L2 in place of shared
// memory cost 1084 us.  The loss alone keeps nothing and reads in vectors (stream_rest):
// 8192 of 131072 bf16 475 us (0.69).  Where the gradient's rows start elsewhere than the
// logits' it is stored element by element: 8192 rows of 65537 bf16, stride 65544, into
// dense ones 1130 us where equal strides take 436; f32 rows of 16384 106 and 87.
// The streaming threads' mark and the teacher warp's wait for it.
template <int THREADS>
__device__ __forceinline__ void mark_arrive() {
    asm volatile("bar.arrive 1, %0;" ::"n"(THREADS) : "memory");
}
template <int THREADS>
__device__ __forceinline__ void mark_wait() {
    asm volatile("bar.sync 1, %0;" ::"n"(THREADS) : "memory");
}

// What the two sides of a CTA share, by a row's or a turn's parity (a turn is a
// row that is read).
template <int NT>
struct DistillShared {
    float4 warps[2][NT / 32];    // the streaming warps' sums
    float4 parts[2][DS_CLUSTER]; // the cluster's CTAs'
    float kl[2][DS_CLUSTER];     // their terms of the loss (rank 0's)
    float weight[2];
    int any[2];  // whether the row has entries
    uint32_t id[TEACHER_MAX], bits[DUP_BITS / 32];
    float q[TEACHER_MAX];
};

// A part of one row.
template <class T>
struct RowOfPart {
    const T *row;
    const uint4 *from;  // the part's first vector
    int head, v0, n_vec, tail;
    __device__ __forceinline__ RowOfPart(const DistillArgs &a, int64_t r, int rank, int log_cs) {
        row = (const T *)a.logits + r * a.stride;
        const RowSpan span = row_span(row, a.vocab);
        // (At most 2^28 vectors times 8.)
        v0 = (int)((uint32_t)span.n_vec * (uint32_t)rank >> log_cs);
        n_vec = (int)((uint32_t)span.n_vec * (uint32_t)(rank + 1) >> log_cs) - v0;
        from = (const uint4 *)(row + span.head) + v0;
        head = span.head;
        tail = span.tail;
    }
};

// The sums of the whole row from a CTA's warps, through the cluster; the
// teacher warp (`speaks`) carries the exchange, and does `meanwhile` while it waits.
template <int NT, class F>
__device__ __forceinline__ SoftSums row_sums(DistillShared<NT> &sh, int turn, int log_cs, int rank, float scale, bool speaks,
                                             F &&meanwhile) {
    namespace cg = cooperative_groups;
    const int lane = threadIdx.x & 31, cs = 1 << log_cs;
    SoftSums sums;
    if (log_cs == 0 || speaks) sums = join_places<false>(sh.warps[turn & 1], NT / 32, scale);
    if (log_cs) {
        if (speaks) {
            if (lane < cs)
                *cg::this_cluster().map_shared_rank(&sh.parts[turn & 1][rank], lane) = make_float4(sums.m, sums.s, 0.0f, 0.0f);
            cluster_arrive();
        } else {
            cluster_arrive_relaxed();
        }
        meanwhile();
        cluster_wait();
        sums = join_places<false>(sh.parts[turn & 1], cs, scale);
    } else {
        meanwhile();
    }
    return sums;
}

// What does not fit the part's shared memory, from global memory.
template <class T, int NT>
__device__ __noinline__ SoftSums stream_rest(const uint4 *from, int v0, int v1, float scale, SoftSums sums) {
    stream_sums<T, NT, DS_U, false, true>((const T *)from, v0, v1, threadIdx.x, scale, sums, [](int, float) {});
    return sums;
}

template <class T, int NT, int ENTRIES>
__global__ void __launch_bounds__(NT + 32, 3) distill_k(DistillArgs a, int log_cs, int keep, int rows_per) {
    namespace cg = cooperative_groups;
    extern __shared__ uint4 kept[];  // [keep]
    __shared__ DistillShared<NT> sh;
    constexpr int N = Vec<T>::N, STEP = NT * DS_U;
    const int tid = threadIdx.x, lane = tid & 31;
    const int cs = 1 << log_cs, rank = blockIdx.x & (cs - 1);
    const int64_t r0 = (int64_t)(blockIdx.x >> log_cs) * rows_per;
    const int n_rows = (int)min((int64_t)rows_per, a.rows - r0);
    const float scale = a.scale;
    int turn = 0;
    if (log_cs) {  // every CTA has to run before its shared memory is written
        cluster_arrive_relaxed();
        cluster_wait();
    }

    if (tid >= NT) {
        // ---- the teacher
        Entries<ENTRIES> now, next;
        float next_weight = 1.0f;
        auto read_ahead = [&](int i) {
            next.load(a, r0 + i, lane);
            if (a.row_weight) next_weight = a.row_weight[r0 + i];
        };
        auto tell = [&](int i) {
            const bool some = next.settle(a);
            if (lane == 0) {
                sh.any[i & 1] = some;
                sh.weight[i & 1] = next_weight;
            }
            return some;
        };
        int64_t loss_row = -1;  // whose terms the cluster's next barrier brings
        auto write_loss = [&](int t) {
            if (loss_row >= 0 && rank == 0 && lane == 0 && a.loss) {
                float all = 0.0f;
                for (int c = 0; c < cs; ++c) all += sh.kl[t & 1][c];
                a.loss[loss_row] = a.temperature * all;
            }
        };
        for (int i = lane; i < DUP_BITS / 32; i += 32) sh.bits[i] = 0;
        read_ahead(0);
        bool any = tell(0);
        __syncthreads();
        for (int i = 0; i < n_rows; ++i) {
            const int64_t r = r0 + i;
            const bool more = i + 1 < n_rows, live = any;
            const float w = next_weight;
            now = next;
            if (more) read_ahead(i + 1);
            float z[ENTRIES], log_q[ENTRIES];
            uint32_t mine = 0;  // which of this lane's entries are in the part
            if (live) {
                const RowOfPart<T> here(a, r, rank, log_cs);
                const int e0 = rank == 0 ? 0 : here.head + here.v0 * N;
                const int e1 = rank == cs - 1 ? a.vocab : here.head + (here.v0 + here.n_vec) * N;
#pragma unroll
                for (int k = 0; k < ENTRIES; ++k) {
                    z[k] = 0.0f;
                    if (now.id[k] != NO_TOKEN && (int)now.id[k] >= e0 && (int)now.id[k] < e1) {
                        mine |= 1u << k;
                        z[k] = to_f32(here.row[now.id[k]]);
                    }
                }
            }
            any = more && tell(i + 1);
            __syncthreads();
            if (!live) {
                if (rank == 0 && lane == 0 && a.loss) a.loss[r] = 0.0f;
                continue;
            }
            const SoftSums sums = row_sums<NT>(sh, turn, log_cs, rank, scale, true, [&] { now.share(a.inv_t, a.n, log_q); });
            if (log_cs) write_loss(turn - 1);
            const float log_s = logf(sums.s), log2_s = log_s * LOG2E;
            const bool empty = sums.m == -INFINITY && sums.s == 0.0f;  // a student that can say nothing
            float kl = 0.0f;
#pragma unroll
            for (int k = 0; k < ENTRIES; ++k)
                if ((mine >> k & 1) && now.q[k] != 0.0f)
                    kl += empty ? INFINITY : loss_term(now.q[k], log_q[k], z[k], sums.m, log_s, a.temperature);
            kl = warp_sum(kl);
            if (log_cs) {
                if (lane == 0) cg::this_cluster().map_shared_rank(&sh.kl[turn & 1][0], 0)[rank] = kl;
            } else if (lane == 0 && a.loss) {
                a.loss[r] = a.temperature * kl;
            }
            loss_row = r;
            ++turn;
            if (!a.dlogits || w == 0.0f || empty) continue;
            // What stands at an entry: p less the shares of its id.
            const float gs = a.grad_scale * w * a.temperature;
            float share[ENTRIES];
#pragma unroll
            for (int k = 0; k < ENTRIES; ++k) share[k] = now.q[k];
            if (perhaps_twice<DUP_BITS>(now.id, sh.bits)) total_shares(now, a.n, sh.id, sh.q, share);
#pragma unroll
            for (int k = 0; k < ENTRIES; ++k)
                if (mine >> k & 1) z[k] = gs * (ex2(fmaf(z[k] - sums.m, scale, -log2_s)) - share[k]);
            mark_wait<NT + 32>();
            // (An id that stands here more than once gets the same value each time.)
            T *out = (T *)a.dlogits + r * a.dstride;
#pragma unroll
            for (int k = 0; k < ENTRIES; ++k)
                if (mine >> k & 1) out[now.id[k]] = from_f32<T>(z[k]);
        }
        if (log_cs) {
            cluster_arrive();
            cluster_wait();
            write_loss(turn - 1);
        }
        return;
    }

    // ---- the stream
    const int groups = (keep + STEP - 1) / STEP;
    auto fetch = [&](const RowOfPart<T> &p, int g) {  // group g of this thread's vectors
        const int v = g * STEP + tid, n = min(keep, p.n_vec);
        const uint4 *from = p.from + v;
        uint4 *to = kept + v;
        if ((g + 1) * STEP <= n) {
#pragma unroll
            for (int u = 0; u < DS_U; ++u) copy_async16(to + u * NT, from + u * NT);
        } else {
#pragma unroll
            for (int u = 0; u < DS_U; ++u)
                if (v + u * NT < n) copy_async16(to + u * NT, from + u * NT);
        }
        copy_commit();
    };
    auto fetch_all = [&](const RowOfPart<T> &p) {
        for (int g = 0; g < groups; ++g) fetch(p, g);
    };
    RowOfPart<T> part(a, r0, rank, log_cs);
    __syncthreads();
    // A row without entries is not read, in no CTA of the cluster.
    bool any = sh.any[0];
    if (any) fetch_all(part);
    for (int i = 0; i < n_rows; ++i) {
        const int64_t r = r0 + i;
        const RowOfPart<T> here = part;
        const bool more = i + 1 < n_rows, live = any;
        const float w = sh.weight[i & 1];
        if (more) part = RowOfPart<T>(a, r + 1, rank, log_cs);
        const int n_kept = min(keep, here.n_vec);
        const int n_head = rank == 0 ? here.head : 0, n_tail = rank == cs - 1 ? here.tail : 0;
        const int e_tail = a.vocab - here.tail + tid;

        SoftSums sums;
        float z_head = 0.0f, z_tail = 0.0f;
        if (live) {
            for (int g = 0; g < groups; ++g) {
                copy_wait_for(groups - 1 - g);
                const int v = tid + g * STEP;
                uint4 raw[DS_U];
                if ((g + 1) * STEP <= n_kept) {
#pragma unroll
                    for (int u = 0; u < DS_U; ++u) raw[u] = kept[v + u * NT];
                } else {
#pragma unroll
                    for (int u = 0; u < DS_U; ++u) raw[u] = v + u * NT < n_kept ? kept[v + u * NT] : masked16<T>();
                }
                add_batch<T, DS_U, false>(raw, sums, scale);
            }
            if (n_kept < here.n_vec) sums = stream_rest<T, NT>(here.from, n_kept, here.n_vec, scale, sums);
            if (tid < n_head) {
                z_head = to_f32(here.row[tid]);
                sums.raise(z_head, scale);
                sums.add(z_head, scale);
            }
            if (tid < n_tail) {
                z_tail = to_f32(here.row[e_tail]);
                sums.raise(z_tail, scale);
                sums.add(z_tail, scale);
            }
            sums = warp_join<false>(sums, scale);
            if (lane == 0) sh.warps[turn & 1][tid >> 5] = make_float4(sums.m, sums.s, 0.0f, 0.0f);
        }
        __syncthreads();
        any = more && sh.any[(i + 1) & 1];
        bool nothing = !live || w == 0.0f;
        if (live) {
            sums = row_sums<NT>(sh, turn, log_cs, rank, scale, false, [] {});
            ++turn;
            nothing |= sums.m == -INFINITY && sums.s == 0.0f;
        }
        if (!a.dlogits) {
            if (any) fetch_all(part);
            continue;
        }
        T *out = (T *)a.dlogits + r * a.dstride;
        uint4 *to = (uint4 *)(out + here.head) + here.v0;  // the part's first vector
        const bool wide = ((uintptr_t)to & 15) == 0;
        auto put = [&](int v, float (&x)[N]) {
            if (wide) {
                store16(to + v, pack<T>(x));
            } else {
#pragma unroll
                for (int k = 0; k < N; ++k) ((T *)(to + v))[k] = from_f32<T>(x[k]);
            }
        };
        if (nothing) {
            float x[N] = {};
            for (int v = tid; v < here.n_vec; v += NT) put(v, x);
            if (tid < n_head) out[tid] = from_f32<T>(0.0f);
            if (tid < n_tail) out[e_tail] = from_f32<T>(0.0f);
            if (any) fetch_all(part);
            continue;
        }
        const float gs = a.grad_scale * w * a.temperature, log2_s = logf(sums.s) * LOG2E;
        const float2 nm = make_float2(-sums.m, -sums.m), sc2 = make_float2(scale, scale), nl = make_float2(-log2_s, -log2_s),
                     g2 = make_float2(gs, gs);
        auto dense = [&](float z) { return gs * ex2(fmaf(z - sums.m, scale, -log2_s)); };
        auto vec = [&](int v, uint4 raw) {
            float x[N];
            unpack<T>(raw, x);
#pragma unroll
            for (int k = 0; k < N; k += 2) {
                const float2 y = fma2(add2(make_float2(x[k], x[k + 1]), nm), sc2, nl);
                const float2 p = mul2(make_float2(ex2(y.x), ex2(y.y)), g2);
                x[k] = p.x;
                x[k + 1] = p.y;
            }
            put(v, x);
        };
        for (int g = 0; g < groups; ++g) {
            const int v = tid + g * STEP;
            uint4 raw[DS_U];
            if ((g + 1) * STEP <= n_kept) {
#pragma unroll
                for (int u = 0; u < DS_U; ++u) raw[u] = kept[v + u * NT];
#pragma unroll
                for (int u = 0; u < DS_U; ++u) vec(v + u * NT, raw[u]);
            } else {
                for (int u = 0; u < DS_U; ++u)
                    if (v + u * NT < n_kept) vec(v + u * NT, kept[v + u * NT]);
            }
            if (any) fetch(part, g);
        }
        for (int v = n_kept + tid; v < here.n_vec; v += NT) vec(v, load16_rw(here.from + v));
        if (tid < n_head) out[tid] = from_f32<T>(dense(z_head));
        if (tid < n_tail) out[e_tail] = from_f32<T>(dense(z_tail));
        mark_arrive<NT + 32>();
    }
    if (log_cs) {  // the others' shared memory is written until here
        cluster_arrive_relaxed();
        cluster_wait();
    }
}

// ---------------------------------------------------------------- short rows: a warp each
// The same in a warp, without a barrier but its own: 12 rows of 16 KB in the air
// per SM.  16384 rows of 1024 f32 take 31 us (4.3 TB/s, 0.68): a warp's loads, sums
// and stores follow one another, and no other row's are fetched meanwhile.
constexpr int WARP_ROWS = 4;
constexpr int WARP_VECTORS = 1024;  // of a row, at most

// 16-byte units of shared memory of one warp that makes a gradient: `keep` vectors
// (none in rows shorter than a vector), ids and shares, the bitmap.
__host__ __device__ inline int warp_vectors(int keep, int n) { return keep + (2 * n + 3) / 4 + WARP_DUP_BITS / 128; }

template <class T, int ENTRIES>
__global__ void __launch_bounds__(32 * WARP_ROWS) distill_warp_k(DistillArgs a, int keep) {
    extern __shared__ uint4 shared[];  // WARP_ROWS of: [keep] vectors, [n] ids, [n] shares, the bitmap
    constexpr int N = Vec<T>::N;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t r = (int64_t)blockIdx.x * WARP_ROWS + warp;
    if (r >= a.rows) return;
    uint4 *kept = shared + warp * warp_vectors(keep, a.n);
    uint32_t *id = (uint32_t *)(kept + keep);
    float *q = (float *)(id + a.n);
    uint32_t *bits = (uint32_t *)(kept + warp_vectors(keep, a.n)) - WARP_DUP_BITS / 32;
    const T *row = (const T *)a.logits + r * a.stride;
    const RowSpan span = row_span(row, a.vocab);
    const uint4 *body = (const uint4 *)(row + span.head);
    const int n_vec = span.n_vec, e_tail = a.vocab - span.tail + lane;
    const float scale = a.scale;
    T *out = a.dlogits ? (T *)a.dlogits + r * a.dstride : nullptr;
    T *obody = out + span.head;
    const bool wide = ((uintptr_t)obody & 15) == 0;
    auto put = [&](int v, float (&x)[N]) {
        T *to = obody + (int64_t)v * N;
        if (wide) {
            store16(to, pack<T>(x));
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) to[i] = from_f32<T>(x[i]);
        }
    };
    auto zeros = [&] {
        float x[N] = {};
        for (int v = lane; v < n_vec; v += 32) put(v, x);
        if (lane < span.head) out[lane] = from_f32<T>(0.0f);
        if (lane < span.tail) out[e_tail] = from_f32<T>(0.0f);
    };

    Entries<ENTRIES> now;
    now.load(a, r, lane);
    const bool any = now.settle(a);
    const float w = a.row_weight ? a.row_weight[r] : 1.0f;
    if (!any) {
        if (lane == 0 && a.loss) a.loss[r] = 0.0f;
        if (out) zeros();
        return;
    }
    float z_entry[ENTRIES];
    auto entry_logits = [&] {
#pragma unroll
        for (int k = 0; k < ENTRIES; ++k) z_entry[k] = now.id[k] != NO_TOKEN ? to_f32(row[now.id[k]]) : 0.0f;
    };
    SoftSums sums;
    if (out) {
        const int half = n_vec / (64 * DS_U) * (32 * DS_U);  // in two groups, of whole batches
        for (int v = lane; v < half; v += 32) copy_async16(&kept[v], body + v);
        copy_commit();
        for (int v = half + lane; v < n_vec; v += 32) copy_async16(&kept[v], body + v);
        copy_commit();
        entry_logits();
        for (int i = lane; i < WARP_DUP_BITS / 32; i += 32) bits[i] = 0;
        auto add = [&](int from, int to) {
            for (int v = from + lane; v < to; v += 32 * DS_U) {
                uint4 raw[DS_U];
#pragma unroll
                for (int u = 0; u < DS_U; ++u)
                    if (v + u * 32 < to) raw[u] = kept[v + u * 32];
                if (v + (DS_U - 1) * 32 < to)
                    add_batch<T, DS_U, false>(raw, sums, scale);
                else
                    add_some<T, 32, DS_U, false>(raw, v, to, sums, scale);
            }
        };
        copy_wait<1>();
        add(0, half);
        copy_wait<0>();
        add(half, n_vec);
    } else {
        entry_logits();
        stream_sums<T, 32, DS_U, false>(row + span.head, 0, n_vec, lane, scale, sums, [](int, float) {});
    }
    float z_head = 0.0f, z_tail = 0.0f;
    if (lane < span.head) {
        z_head = to_f32(row[lane]);
        sums.raise(z_head, scale);
        sums.add(z_head, scale);
    }
    if (lane < span.tail) {
        z_tail = to_f32(row[e_tail]);
        sums.raise(z_tail, scale);
        sums.add(z_tail, scale);
    }
    const SoftSums all = warp_join<false>(sums, scale);
    const float log_s = logf(all.s), log2_s = log_s * LOG2E;
    const bool empty = all.m == -INFINITY && all.s == 0.0f;  // a student that can say nothing
    float log_q[ENTRIES], kl = 0.0f;
    now.share(a.inv_t, a.n, log_q);
#pragma unroll
    for (int k = 0; k < ENTRIES; ++k)
        if (now.id[k] != NO_TOKEN && now.q[k] != 0.0f)
            kl += empty ? INFINITY : loss_term(now.q[k], log_q[k], z_entry[k], all.m, log_s, a.temperature);
    kl = warp_sum(kl);
    if (lane == 0 && a.loss) a.loss[r] = a.temperature * kl;
    if (!out) return;
    if (w == 0.0f || empty) {
        zeros();
        return;
    }
    const float gs = a.grad_scale * w * a.temperature;
    auto dense = [&](float z) { return gs * ex2(fmaf(z - all.m, scale, -log2_s)); };
    const float2 nm = make_float2(-all.m, -all.m), sc2 = make_float2(scale, scale), nl = make_float2(-log2_s, -log2_s),
                 g2 = make_float2(gs, gs);
    float share[ENTRIES];
#pragma unroll
    for (int k = 0; k < ENTRIES; ++k) share[k] = now.q[k];
    if (perhaps_twice<WARP_DUP_BITS>(now.id, bits)) total_shares(now, a.n, id, q, share);
    __syncwarp();
    for (int v = lane; v < n_vec; v += 32) {
        float x[N];
        unpack<T>(kept[v], x);
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            const float2 y = fma2(add2(make_float2(x[i], x[i + 1]), nm), sc2, nl);
            const float2 p = mul2(make_float2(ex2(y.x), ex2(y.y)), g2);
            x[i] = p.x;
            x[i + 1] = p.y;
        }
        put(v, x);
    }
    if (lane < span.head) out[lane] = from_f32<T>(dense(z_head));
    if (lane < span.tail) out[e_tail] = from_f32<T>(dense(z_tail));
    __syncwarp();
    // What stands at an entry: p less the shares of its id.  (An id that stands
    // here more than once gets the same value each time.)
#pragma unroll
    for (int k = 0; k < ENTRIES; ++k)
        if (now.id[k] != NO_TOKEN) out[now.id[k]] = from_f32<T>(gs * (ex2(fmaf(z_entry[k] - all.m, scale, -log2_s)) - share[k]));
}

template <class T>
cudaError_t launch_distill(const DistillArgs &a, cudaStream_t st) {
    constexpr int N = Vec<T>::N;
    const int64_t n_vec = a.vocab / N;
    // A warp per row for rows of up to 16 KB, when there are enough to fill the GPU.
    // Measured, a warp against a cluster's CTA per row: 16384 rows of 4 KB 31 and
    // 217 us, 8192 of 16 KB 74 and 175, 1000 of 16 KB 16 and 25; but 8192 rows of 32 KB
    // 230 and 135 (few fit an SM), 256 rows of 4 KB 14 and 12.
    if (n_vec <= WARP_VECTORS && a.rows >= 512) {
        const int keep = (int)n_vec;
        const int smem = a.dlogits ? WARP_ROWS * warp_vectors(keep, a.n) * 16 : 0;
        auto kern = a.n <= 64 ? distill_warp_k<T, 2> : distill_warp_k<T, TEACHER_MAX / 32>;
        if (smem > 48 << 10) {
            cudaError_t e = allow_shared(kern, WARP_ROWS * warp_vectors(WARP_VECTORS, TEACHER_MAX) * 16);
            if (e != cudaSuccess) return e;
        }
        kern<<<(unsigned)((a.rows + WARP_ROWS - 1) / WARP_ROWS), 32 * WARP_ROWS, smem, st>>>(a, keep);
        return cudaGetLastError();
    }
    // A row is split until a part and those of two more CTAs fit an SM's shared
    // memory, and while the rows alone leave SMs idle and every thread keeps a vector.
    // (8192 rows of 131072 bf16: parts of at most 68 KB 982 us, of 36 KB 1225, of 104 KB
    // 954; 4096 rows of 16384 f32 93, 112 and 92; 1500 rows of 50000 bf16 80, 99 and 80:
    // with larger parts two CTAs share an SM, which then differs little, and leaves it
    // idle where rows end unevenly.  192 threads against 128 and 256: 982, 983 and 945 us;
    // 93, 97 and 96; 80, 74 and 78.)
    int log_cs = 0;
    while ((1 << log_cs) < DS_CLUSTER && ((a.dlogits && (n_vec >> log_cs) * 16 > DS_PART) ||
                                          (a.rows << log_cs < 148 && n_vec >> (log_cs + 1) >= DS_NT)))
        ++log_cs;
    const int cs = 1 << log_cs;
    const int64_t keep = a.dlogits ? std::min<int64_t>((n_vec + cs - 1) / cs, DS_MOST / 16) : 0;
    // Several rows to a cluster, as long as there are some turns of clusters left to
    // even out.  (8192 rows of 131072 bf16: four 982 us, one 1072, sixteen 995.)
    const int64_t rows_per = std::max<int64_t>(1, std::min<int64_t>(DS_ROWS, a.rows * cs / (148 * 3 * 4)));
    const int64_t clusters = (a.rows + rows_per - 1) / rows_per;
    auto kern = a.n <= 64 ? distill_k<T, DS_NT, 2> : distill_k<T, DS_NT, TEACHER_MAX / 32>;
    if (keep * 16 > 32768) {
        cudaError_t e = allow_shared(kern, DS_MOST);
        if (e != cudaSuccess) return e;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(clusters * cs));
    cfg.blockDim = dim3(DS_NT + 32);
    cfg.dynamicSmemBytes = (size_t)keep * 16;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cs;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cs > 1 ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kern, a, log_cs, (int)keep, (int)rows_per);
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
