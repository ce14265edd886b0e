// norm.cu -- layer norm and RMSNorm of rows, and their gradients
// (include/noetic/head.h).
//
// Rows are taken by groups of G threads (a warp to 512 threads), VALS elements to
// a thread, which stay on the SM from the one load of the row to its one
// store: the mean and then the sum of squared differences from it are two
// reductions over registers, not two passes over memory.  A block walks rows
// blockIdx, blockIdx + gridDim, ..., so that the gain, the bias and (backward)
// the sums for dgain and dbias stay in registers too, and the next rows are on
// their way while the present one is worked on.  All of it is bound by HBM,
// as long as a row costs its threads few instructions beside its elements:
// hence the f32 operations in pairs, and 64 bytes of a row to a thread where it
// has them.  Rows too wide for that are shared by a cluster of CTAs in the same
// way; wider ones still, or wide ones that start anywhere, take a block per row
// that reads them again from L2.
//
// Rows that do not start on 16-byte boundaries (an odd width) are read in the
// same 16-byte units of memory.  Where a row starts in its first unit repeats
// every 8 rows at most, so a group that steps by a multiple of 8 rows sees
// every row start at the same place, and each thread's columns stay the same.
//
// Times below are of calls back to back on inputs beyond L2, HBM's copy rate
// being 6.55 TB/s.

#include <cooperative_groups.h>

#include <algorithm>

#include "nk_head.cuh"
#include "nk_head.h"

namespace nk {

namespace {

constexpr int NM_NT = 256;
constexpr int BWD_VALS = 16;  // elements of a thread
constexpr int FWD_DEPTH = 4;  // rows on their way to each group
constexpr int BWD_DEPTH = 3;

// ---------------------------------------------------------------- groups of threads
// Sum over the G threads of a group, the same in all of them, in a fixed
// order.  Groups beyond a warp go through `red` (one float per warp of the
// block), which the caller changes from one reduction to the next so that one
// barrier is enough; every thread of the block calls it.
template <int G>
__device__ __forceinline__ float group_sum(float v, float *red) {
    v = warp_sum(v);
    if constexpr (G > 32) {
        constexpr int W = G / 32;
        const int warp = threadIdx.x >> 5;
        if ((threadIdx.x & 31) == 0) red[warp] = v;
        __syncthreads();
        const float *mine = red + warp / W * W;
        v = 0.0f;
#pragma unroll
        for (int i = 0; i < W; ++i) v += mine[i];
    }
    return v;
}
__device__ __forceinline__ float2 warp_sum2(float2 v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
        v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
    }
    return v;
}
template <int G>
__device__ __forceinline__ float2 group_sum2(float2 v, float2 *red) {
    v = warp_sum2(v);
    if constexpr (G > 32) {
        constexpr int W = G / 32;
        const int warp = threadIdx.x >> 5;
        if ((threadIdx.x & 31) == 0) red[warp] = v;
        __syncthreads();
        const float2 *mine = red + warp / W * W;
        v = make_float2(0.0f, 0.0f);
#pragma unroll
        for (int i = 0; i < W; ++i) {
            v.x += mine[i].x;
            v.y += mine[i].y;
        }
    }
    return v;
}

// Where a group's elements lie: 16-byte units of N elements, unit base + l * G +
// lane the l-th of a thread, up to `end`.  With EDGE the row starts `shift` elements
// into unit 0 and may end inside the last one.  A row that a cluster shares (CL,
// without EDGE) is cut into even parts.
template <class T, int G, int VALS, bool EDGE, bool CL>
struct Place {
    static constexpr int N = Vec<T>::N, LOADS = VALS / N, H = VALS / 2, C = N / 2;  // pairs in all, in a unit
    static constexpr bool whole = !EDGE;
    int lane, width, shift, units, base, end, last;  // last: the load that holds the part's last unit

    __device__ __forceinline__ Place(const void *row, int lane_, int width_, int rank = 0, int cs = 1) : lane(lane_), width(width_) {
        shift = EDGE ? (int)((uintptr_t)row & 15) / (int)sizeof(T) : 0;
        units = (shift + width + N - 1) / N;
        const int share = CL ? (units + cs - 1) / cs : units;
        base = CL ? min(units, rank * share) : 0;
        end = CL ? min(units, base + share) : units;
        last = (end - base - 1) / G;
    }
    __device__ __forceinline__ int unit(int l) const { return base + l * G + lane; }
    __device__ __forceinline__ int column(int l) const { return unit(l) * N - shift; }
    __device__ __forceinline__ bool has(int l) const { return unit(l) < end; }
    // Whether one of the group's units of load l may reach out of the row; whether
    // this thread's does.
    __device__ __forceinline__ bool edgy(int l) const { return EDGE && (l == 0 || l == last); }
    __device__ __forceinline__ bool on_edge(int l) const { return edgy(l) && (unit(l) == 0 || unit(l) == units - 1); }
    __device__ __forceinline__ bool inside(int col) const { return (unsigned)col < (unsigned)width; }
    // Elements of a part (of a row without EDGE).
    __device__ __forceinline__ int count() const { return (end - base) * N; }
    // A pair of elements, 0 where it is not in the row.
    __device__ __forceinline__ float2 keep(int l, int i, float2 v) const {
        if (!has(l)) return make_float2(0.0f, 0.0f);
        if (edgy(l)) v = make_float2(inside(column(l) + i) ? v.x : 0.0f, inside(column(l) + i + 1) ? v.y : 0.0f);
        return v;
    }
};

// The rows that a thread will work on next, ARRAYS of them at a time: its units
// in its own places of a ring in shared memory, DEPTH rows on their way by
// asynchronous copies (no barrier: a thread reads only what it copied).
template <class T, class P, bool EDGE, int NT, int DEPTH, int ARRAYS>
struct RowQueue {
    static constexpr int BYTES = DEPTH * ARRAYS * P::LOADS * NT * 16;
    uint4 *ring;  // [DEPTH][ARRAYS][LOADS][NT], from this thread's place on
    int slot = 0;

    __device__ __forceinline__ uint4 *place(int at, int k) const { return ring + (at * ARRAYS + k) * P::LOADS * NT; }
    // Sends for one row of each array (for nothing, if it is not `real`).
    __device__ __forceinline__ void push(const P &p, const T *const (&rows)[ARRAYS], int at, bool real, bool first_row) {
#pragma unroll
        for (int k = 0; k < ARRAYS; ++k)
#pragma unroll
            for (int l = 0; l < P::LOADS; ++l) {
                if (!real || !p.has(l)) continue;
                uint4 *to = place(at, k) + l * NT;
                const T *from = rows[k] + p.column(l);
                if (!EDGE) {
                    copy_async16(to, from);
                } else if (p.unit(l) > 0 || p.shift == 0) {
                    copy_async16_part(to, from, min(16, (p.width - p.column(l)) * (int)sizeof(T)));
                } else if (p.units > 1 && !first_row) {
                    // The unit that the row starts inside: by words, of which the first
                    // may begin with the element before (there is one, but for the first row).
#pragma unroll
                    for (int w = 0; w < 4; ++w)
                        if ((w + 1) * 4 > p.shift * (int)sizeof(T)) copy_async4((char *)to + 4 * w, (const char *)from + 4 * w);
                } else {
                    for (int i = p.shift; i < min(P::N, p.shift + p.width); ++i) ((T *)to)[i] = from[i];
                }
            }
        copy_commit();
    }
    // Waits until the first n rows that were pushed, from the present one on, are there.
    template <int n = 1>
    __device__ __forceinline__ void wait() const {
        copy_wait<DEPTH - n>();
    }
    // Done with it: the next push goes to its slot.
    __device__ __forceinline__ void pop() { slot = ahead(1); }
    // The slot of the k-th row behind the present one.
    __device__ __forceinline__ int ahead(int k) const { return slot + k < DEPTH ? slot + k : slot + k - DEPTH; }
    // Load l of the row in a slot, in pairs; zeros outside the row.
    __device__ __forceinline__ void get(const P &p, int at, int k, int l, bool real, float2 (&x)[P::C]) const {
        float v[P::N];
        unpack<T>(real && p.has(l) ? place(at, k)[l * NT] : make_uint4(0, 0, 0, 0), v);
        if (EDGE && l == 0) {
#pragma unroll
            for (int i = 0; i < P::N; ++i) v[i] = p.inside(p.column(0) + i) ? v[i] : 0.0f;
        }
#pragma unroll
        for (int i = 0; i < P::C; ++i) x[i] = make_float2(v[2 * i], v[2 * i + 1]);
    }
};

template <class P, class T>
__device__ __forceinline__ void store_unit(const P &p, T *row, int col, bool whole, uint4 v) {
    if (whole) {
        store16(row + col, v);
    } else {
        const T *x = (const T *)&v;
#pragma unroll
        for (int i = 0; i < P::N; ++i)
            if (p.inside(col + i)) row[col + i] = x[i];
    }
}

// The 16 bytes that start d elements into a, b.
template <class T>
__device__ __forceinline__ uint4 shifted(uint4 a, uint4 b, int d) {
    uint32_t o[5];
    switch (d * (int)sizeof(T) / 4) {
        case 0: o[0] = a.x, o[1] = a.y, o[2] = a.z, o[3] = a.w, o[4] = b.x; break;
        case 1: o[0] = a.y, o[1] = a.z, o[2] = a.w, o[3] = b.x, o[4] = b.y; break;
        case 2: o[0] = a.z, o[1] = a.w, o[2] = b.x, o[3] = b.y, o[4] = b.z; break;
        default: o[0] = a.w, o[1] = b.x, o[2] = b.y, o[3] = b.z, o[4] = b.w; break;
    }
    if (sizeof(T) == 2 && (d & 1)) {
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = __funnelshift_r(o[i], o[i + 1], 16);
    }
    return make_uint4(o[0], o[1], o[2], o[3]);
}

// A thread's part x(l) of a row that starts at `row`.  `same`: in the same place
// of a unit as the rows read (without EDGE always).  Otherwise the group hands the units over in
// `stage` ([LOADS][NT] units, from the group's place on), where each thread
// reads the two that its unit of the row written is cut from.  (Groups of several
// warps: the barriers of the caller's reductions keep one row's stage from the next.)
template <int G, int NT, class P, class T, class F>
__device__ __forceinline__ void store_row(const P &p, T *row, bool same, uint4 *stage, F &&x) {
    if (P::whole || same) {
#pragma unroll
        for (int l = 0; l < P::LOADS; ++l)
            if (p.has(l)) store_unit(p, row, p.column(l), !p.on_edge(l), x(l));
        return;
    }
    if (G == 32) __syncwarp();
#pragma unroll
    for (int l = 0; l < P::LOADS; ++l)
        if (p.has(l)) stage[l * NT + p.lane] = x(l);
    if constexpr (G == 32)
        __syncwarp();
    else
        asm volatile("bar.sync %0, %1;" ::"r"(1 + (int)threadIdx.x / G), "n"(G) : "memory");
    const int shift = (int)((uintptr_t)row & 15) / (int)sizeof(T), d = p.shift - shift;
    const int units = (shift + p.width + P::N - 1) / P::N, first = d < 0 ? -1 : 0;
    auto staged = [&](int u) {
        return u >= 0 && u < p.units ? stage[u / G * NT + u % G] : make_uint4(0, 0, 0, 0);
    };
#pragma unroll
    for (int l = 0; l < P::LOADS; ++l) {
        const int u = p.unit(l);
        if (u < units)
            store_unit(p, row, u * P::N - shift, u > 0 && u < units - 1,
                       shifted<T>(staged(u + first), staged(u + first + 1), d < 0 ? d + P::N : d));
    }
}

template <class T, int C>
__device__ __forceinline__ uint4 pack_pairs(const float2 (&x)[C]) {
    float v[2 * C];
#pragma unroll
    for (int i = 0; i < C; ++i) {
        v[2 * i] = x[i].x;
        v[2 * i + 1] = x[i].y;
    }
    return pack<T>(v);
}

// A thread's part of an f32 vector of the width (null: `other`); 0 outside it.
template <class P>
__device__ __forceinline__ void column_part(const P &p, const float *v, float other, float2 (&x)[P::H]) {
    auto one = [&](int j) {
        const int e = p.column(j / P::N) + j % P::N;
        return p.has(j / P::N) && p.inside(e) ? (v ? v[e] : other) : 0.0f;
    };
#pragma unroll
    for (int j = 0; j < P::H; ++j) x[j] = make_float2(one(2 * j), one(2 * j + 1));
}

__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }

// ---------------------------------------------------------------- forward
// 16384 rows of 4096 bf16 in 49 to 52 us (5.3 TB/s, 0.81 of the copy rate); 8192 rows of
// 8192 the same.  Four rows on their way to each group, since a block's own
// reductions leave memory idle otherwise.  Rows of 64 x 1024 f32 cost their launch.
template <class T, int G, int VALS, bool EDGE>
__global__ void __launch_bounds__(G > NM_NT ? G : NM_NT, G > NM_NT ? 1 : 2) norm_rows_k(NormArgs a, int same) {
    constexpr int NT = G > NM_NT ? G : NM_NT, GROUPS = NT / G;
    using P = Place<T, G, VALS, EDGE, false>;
    constexpr int C = P::C;
    __shared__ float red[2][32];
    extern __shared__ uint4 ring[];
    const int group = threadIdx.x / G;
    const float inv_n = 1.0f / (float)a.width;
    float2 gain[P::H], bias[P::H];
    RowQueue<T, P, EDGE, NT, FWD_DEPTH, 1> queue;
    queue.ring = ring + threadIdx.x;
    uint4 *stage = ring + queue.BYTES / 16 + group * G;
    const int64_t step = (int64_t)gridDim.x * GROUPS;
    int64_t r = (int64_t)blockIdx.x * GROUPS + group;
    const P p((const T *)a.x + r * a.x_stride, threadIdx.x % G, a.width);
    auto push = [&](int64_t q, int at) {
        const T *const rows[1] = {(const T *)a.x + q * a.x_stride};
        queue.push(p, rows, at, q < a.rows, q == 0);
    };
    for (int k = 0; k < FWD_DEPTH; ++k) push(r + k * step, k);
    column_part(p, a.gain, 1.0f, gain);
    column_part(p, a.bias, 0.0f, bias);
    // Every group takes the same number of turns: the reductions hold barriers.
    const int turns = (int)((a.rows - (int64_t)blockIdx.x * GROUPS + step - 1) / step);
    for (int i = 0; i < turns; ++i, r += step) {
        const bool real = r < a.rows;
        float2 x[P::H];
        queue.wait();
#pragma unroll
        for (int l = 0; l < P::LOADS; ++l) {
            float2 v[C];
            queue.get(p, queue.slot, 0, l, real, v);
#pragma unroll
            for (int j = 0; j < C; ++j) x[l * C + j] = v[j];
        }
        push(r + FWD_DEPTH * step, queue.slot);
        queue.pop();
        float mean = 0.0f;
        if (!a.rms) {
            float2 s = x[0];
#pragma unroll
            for (int j = 1; j < P::H; ++j) s = add2(s, x[j]);
            mean = group_sum<G>(s.x + s.y, red[0]) * inv_n;
        }
        float2 v = both(0.0f);
#pragma unroll
        for (int j = 0; j < P::H; ++j) {
            x[j] = p.keep(j / C, 2 * (j % C), add2(x[j], both(-mean)));
            v = fma2(x[j], x[j], v);
        }
        const float rstd = 1.0f / sqrtf(fmaf(group_sum<G>(v.x + v.y, red[1]), inv_n, a.eps));
        if (G > 32 && a.rms) __syncthreads();  // red[1] again in the next turn
        if (!real) continue;
        store_row<G, NT>(p, (T *)a.y + r * a.y_stride, same, stage, [&](int l) {
            float2 z[C];
#pragma unroll
            for (int j = 0; j < C; ++j) z[j] = fma2(mul2(x[l * C + j], both(rstd)), gain[l * C + j], bias[l * C + j]);
            return pack_pairs<T>(z);
        });
        if (p.lane == 0) {
            if (a.mean) a.mean[r] = mean;
            if (a.rstd) a.rstd[r] = rstd;
        }
    }
}

template <class T>
constexpr int fwd_vals() {
    return 64 / (int)sizeof(T);
}

// ---------------------------------------------------------------- rows that a cluster shares
// Of R rows at a time (a turn), which share an exchange.  What a cluster's CTAs
// tell each other: the NM_NT streaming threads leave two sums per warp and row in
// `warps`; a warp of its own, the speaker, joins these, writes them to every CTA of
// the cluster and carries the barrier's release: the streaming threads' arrival
// promises nothing, or it would wait for their stores to the rows before.  They
// send the next turn's sums off before they finish the present one's rows, which
// covers the exchange.  (Two turns' places, by parity.)  Bound by that exchange, about
// 2 us a turn with two CTAs to an SM, where the parts are small: 2048 rows of 32768
// bf16 84 us (3.2 TB/s; 96 with one row to a turn, 161 by a block per row), 4096 of
// 16384 f32 107 (124, 132).
constexpr int CL_MOST = 8;  // CTAs of a cluster
template <int R>
struct RowExchange {
    float2 warps[2][R][NM_NT / 32], parts[2][R][CL_MOST];
    float counts[NM_NT / 32];  // elements of a warp

    // The streaming threads' side: a warp's sums for a turn; after the exchange the
    // parts', one to a lane.
    __device__ __forceinline__ void send(const float2 (&v)[R], int turn) {
        if ((threadIdx.x & 31) == 0) {
#pragma unroll
            for (int k = 0; k < R; ++k) warps[turn & 1][k][threadIdx.x >> 5] = v[k];
        }
        __syncthreads();
        cluster_arrive_relaxed();
    }
    __device__ __forceinline__ void receive(float2 (&v)[R], int turn, int cs) const {
        cluster_wait();
        const int lane = threadIdx.x & 31;
#pragma unroll
        for (int k = 0; k < R; ++k) v[k] = lane < cs ? parts[turn & 1][k][lane] : make_float2(0.0f, 0.0f);
    }
    // The speaker's; join(a warp's sums in each lane) gives the CTA's in all.
    template <class F>
    __device__ __forceinline__ void speak(int turns, int rank, int cs, F &&join) {
        namespace cg = cooperative_groups;
        const int lane = threadIdx.x & 31;
        for (int i = 0; i < turns; ++i) {
            __syncthreads();
#pragma unroll
            for (int k = 0; k < R; ++k) {
                const float2 all = join(lane < NM_NT / 32 ? warps[i & 1][k][lane] : make_float2(0.0f, 0.0f));
                if (lane < cs) *cg::this_cluster().map_shared_rank(&parts[i & 1][k][rank], lane) = all;
            }
            cluster_arrive();
            cluster_wait();
        }
    }
};

// Sums (of elements; of squared differences from the own mean) over parts of n
// elements each, one part to a lane, joined.
__device__ __forceinline__ float2 join_moments(float2 v, float n, float inv_all) {
    const float s = warp_sum(v.x), off = (n > 0.0f ? v.x / n : 0.0f) - s * inv_all;
    return make_float2(s, warp_sum(fmaf(n * off, off, v.y)));
}

constexpr int CL_FWD_ROWS = 2;
template <class T>
__global__ void __launch_bounds__(NM_NT + 32, 2) norm_cluster_rows_k(NormArgs a, int cs) {
    constexpr int R = CL_FWD_ROWS;
    using P = Place<T, NM_NT, fwd_vals<T>(), false, true>;
    constexpr int C = P::C;
    __shared__ RowExchange<R> ex;
    extern __shared__ uint4 ring[];
    const int rank = blockIdx.x % cs, lane = threadIdx.x & 31;
    const int64_t step = gridDim.x / cs;
    int64_t r = blockIdx.x / cs;
    const int turns = (int)((a.rows - r + R * step - 1) / (R * step));
    const T *row = (const T *)a.x + r * a.x_stride;
    const float inv_n = 1.0f / (float)a.width;
    cluster_arrive_relaxed();  // every CTA has to run before its shared memory is written
    cluster_wait();
    if (threadIdx.x >= NM_NT) {
        const P p(row, 0, a.width, rank, cs);
        const float inv_part = 1.0f / (float)max(1, p.count());
        ex.speak(turns, rank, cs, [&](float2 v) { return join_moments(v, lane < NM_NT / 32 ? ex.counts[lane] : 0.0f, inv_part); });
        return;
    }
    float2 gain[P::H], bias[P::H];
    RowQueue<T, P, false, NM_NT, 3 * R, 1> queue;
    queue.ring = ring + threadIdx.x;
    const P p(row, threadIdx.x, a.width, rank, cs);
    auto push = [&](int64_t q, int at) {
        const T *const rows[1] = {(const T *)a.x + q * a.x_stride};
        queue.push(p, rows, at, q < a.rows, q == 0);
    };
    for (int k = 0; k < 3 * R; ++k) push(r + k * step, k);
    column_part(p, a.gain, 1.0f, gain);
    column_part(p, a.bias, 0.0f, bias);
    float count = 0.0f;
#pragma unroll
    for (int l = 0; l < P::LOADS; ++l) count += p.has(l) ? P::N : 0.0f;
    count = warp_sum(count);
    if (lane == 0) ex.counts[threadIdx.x >> 5] = count;
    const float inv_count = count > 0.0f ? 1.0f / count : 0.0f;
    const P of(row, 0, a.width, min(lane, cs - 1), cs);  // the part that this lane receives
    const float n_part = lane < cs ? (float)of.count() : 0.0f;
    // A turn's sums, of the rows that start at q, `first` slots on.
    auto send = [&](int turn, int first, int64_t q) {
        queue.template wait<2 * R>();
        float2 own[R], v[R];  // the warp's means; the sums
#pragma unroll
        for (int k = 0; k < R; ++k) {
            own[k] = v[k] = both(0.0f);
            if (a.rms) continue;
            float2 s = both(0.0f), x[C];
#pragma unroll
            for (int l = 0; l < P::LOADS; ++l) {
                queue.get(p, queue.ahead(first + k), 0, l, q + k * step < a.rows, x);
#pragma unroll
                for (int j = 0; j < C; ++j) s = add2(s, x[j]);
            }
            v[k].x = s.x + s.y;
        }
        if (!a.rms) {
#pragma unroll
            for (int k = 0; k < R; ++k) {
                v[k].x = warp_sum(v[k].x);
                own[k] = both(-v[k].x * inv_count);
            }
        }
#pragma unroll
        for (int k = 0; k < R; ++k) {
            float2 s = both(0.0f), x[C];
#pragma unroll
            for (int l = 0; l < P::LOADS; ++l) {
                queue.get(p, queue.ahead(first + k), 0, l, q + k * step < a.rows, x);
#pragma unroll
                for (int j = 0; j < C; ++j) {
                    x[j] = p.keep(l, 2 * j, add2(x[j], own[k]));
                    s = fma2(x[j], x[j], s);
                }
            }
            v[k].y = s.x + s.y;
        }
#pragma unroll
        for (int k = 0; k < R; ++k) v[k].y = warp_sum(v[k].y);
        ex.send(v, turn);
    };
    send(0, 0, r);
    for (int i = 0; i < turns; ++i) {
        float2 all[R];
        ex.receive(all, i, cs);
        if (i + 1 < turns) send(i + 1, R, r + R * step);
#pragma unroll
        for (int k = 0; k < R; ++k) all[k] = join_moments(all[k], n_part, inv_n);
#pragma unroll
        for (int k = 0; k < R; ++k) {
            if (r < a.rows) {
                const float mean = all[k].x * inv_n, rstd = 1.0f / sqrtf(fmaf(all[k].y, inv_n, a.eps));
                store_row<NM_NT, NM_NT>(p, (T *)a.y + r * a.y_stride, true, nullptr, [&](int l) {
                    float2 x[C];
                    queue.get(p, queue.slot, 0, l, true, x);
#pragma unroll
                    for (int j = 0; j < C; ++j) x[j] = fma2(mul2(add2(x[j], both(-mean)), both(rstd)), gain[l * C + j], bias[l * C + j]);
                    return pack_pairs<T>(x);
                });
                if (rank == 0 && threadIdx.x == 0) {
                    if (a.mean) a.mean[r] = mean;
                    if (a.rstd) a.rstd[r] = rstd;
                }
            }
            push(r + 3 * R * step, queue.slot);
            queue.pop();
            r += step;
        }
    }
}

// ---------------------------------------------------------------- wider rows
// A block each, in 16-byte vectors (VEC) or element by element, read again from L2
// for each pass over them (kept in shared memory instead, fewer blocks share an SM:
// 2048 rows of 40000 bf16 205 us with 64 KB of each kept, 193 so).  The f32 gain
// and bias, read once per row, are most of what passes L2: 4096 rows of 16381 bf16
// take 124 us, a third of HBM's rate.
constexpr int WIDE_NT = 512;

// f(v, the elements of unit v) over a thread's part of a row, whose units are 16 bytes
// of N elements (VEC) or one element, as `at(v)` gives them.
template <class T, bool VEC, class At, class F>
__device__ __forceinline__ void wide_each(int width, At &&at, F &&f) {
    if constexpr (VEC) {
        constexpr int N = Vec<T>::N;
#pragma unroll 4
        for (int v = threadIdx.x; v < width / N; v += WIDE_NT) {
            float x[N];
            unpack<T>(at(v), x);
            f(v, x);
        }
    } else {
#pragma unroll 4
        for (int v = threadIdx.x; v < width; v += WIDE_NT) {
            float x[1] = {to_f32(at(v))};
            f(v, x);
        }
    }
}

template <class T, bool VEC>
__global__ void __launch_bounds__(WIDE_NT) norm_wide_rows_k(NormArgs a) {
    __shared__ float red[32];
    constexpr int N = VEC ? Vec<T>::N : 1;
    const int64_t r = blockIdx.x;
    const T *x = (const T *)a.x + r * a.x_stride;
    T *y = (T *)a.y + r * a.y_stride;
    auto at = [&](int v) {
        if constexpr (VEC)
            return load16_rw(x + (int64_t)v * N);
        else
            return x[v];
    };
    const float n = (float)a.width;
    float mean = 0.0f;
    if (!a.rms) {
        float s = 0.0f;
        wide_each<T, VEC>(a.width, at, [&](int, float (&z)[N]) {
#pragma unroll
            for (int i = 0; i < N; ++i) s += z[i];
        });
        mean = block_sum(s, red) / n;
    }
    float v = 0.0f;
    wide_each<T, VEC>(a.width, at, [&](int, float (&z)[N]) {
#pragma unroll
        for (int i = 0; i < N; ++i) v = fmaf(z[i] - mean, z[i] - mean, v);
    });
    const float rstd = 1.0f / sqrtf(block_sum(v, red) / n + a.eps);
    wide_each<T, VEC>(a.width, at, [&](int w, float (&z)[N]) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int e = w * N + i;
            z[i] = fmaf((z[i] - mean) * rstd, a.gain ? a.gain[e] : 1.0f, a.bias ? a.bias[e] : 0.0f);
        }
        if constexpr (VEC)
            store16(y + (int64_t)w * N, pack<T>(z));
        else
            y[w] = from_f32<T>(z[0]);
    });
    if (threadIdx.x == 0) {
        if (a.mean) a.mean[r] = mean;
        if (a.rstd) a.rstd[r] = rstd;
    }
}

// ---------------------------------------------------------------- backward
// dx of the rows, and with PARAMS this block's sums for dgain and dbias: its
// groups' registers joined in shared memory in their order, one row of the
// workspace per block.  The row is unpacked twice, once for the sums and once
// for dx: it waits in shared memory, not in registers.  65536 rows of 1024 bf16 with
// the parameters' sums in 76 us (5.3 TB/s); then the instructions per element
// (about 10, two unpackings) are near to binding.  With EDGE 65536 x 1001 bf16 105 us
// (0.58 of the copy rate) and f32 141 (0.85); into rows that start elsewhere, by way of
// the stage, 65536 x 1024 bf16 of stride 1025 into dense rows 203.
template <class T, int G, int VALS, bool EDGE, bool PARAMS>
__global__ void __launch_bounds__(G > NM_NT ? G : NM_NT, G > NM_NT ? 1 : 2) norm_backward_k(NormGradArgs a, int same) {
    constexpr int NT = G > NM_NT ? G : NM_NT, GROUPS = NT / G;
    using P = Place<T, G, VALS, EDGE, false>;
    constexpr int C = P::C;
    __shared__ float2 red[2][32];
    extern __shared__ uint4 ring[];
    float *joined = (float *)ring;  // [GROUPS][2][width], when the rows are done
    const int group = threadIdx.x / G;
    const float inv_n = 1.0f / (float)a.width;
    float2 gain[P::H], dg[P::H], db[P::H];
#pragma unroll
    for (int j = 0; j < P::H; ++j) dg[j] = db[j] = both(0.0f);
    RowQueue<T, P, EDGE, NT, BWD_DEPTH, 2> queue;
    queue.ring = ring + threadIdx.x;
    uint4 *stage = ring + queue.BYTES / 16 + group * G;
    const int64_t step = (int64_t)gridDim.x * GROUPS;
    int64_t r = (int64_t)blockIdx.x * GROUPS + group;
    const P p((const T *)a.x + r * a.x_stride, threadIdx.x % G, a.width);
    auto push = [&](int64_t q, int at) {
        const T *const rows[2] = {(const T *)a.x + q * a.x_stride, (const T *)a.dy + q * a.dy_stride};
        queue.push(p, rows, at, q < a.rows, q == 0);
    };
    float next_mean, next_rstd;
    auto stats = [&](int64_t q) {
        next_mean = q < a.rows && !a.rms ? a.mean[q] : 0.0f;
        next_rstd = q < a.rows ? a.rstd[q] : 0.0f;
    };
    for (int k = 0; k < BWD_DEPTH; ++k) push(r + k * step, k);
    stats(r);
    column_part(p, a.gain, 1.0f, gain);
    if (PARAMS) pdl_trigger();  // norm_param_sum_k comes up, and waits for this grid's end
    const int turns = (int)((a.rows - (int64_t)blockIdx.x * GROUPS + step - 1) / step);
    for (int i = 0; i < turns; ++i, r += step) {
        const bool real = r < a.rows;
        const float mean = next_mean, rstd = next_rstd;
        queue.wait();
        stats(r + step);
        float2 sc = both(0.0f), sch = sc;
        // Outside the row dy and the gain are 0, and h does not count.
#pragma unroll
        for (int l = 0; l < P::LOADS; ++l) {
            float2 h[C], c[C];
            queue.get(p, queue.slot, 0, l, real, h);
            queue.get(p, queue.slot, 1, l, real, c);
#pragma unroll
            for (int j = 0; j < C; ++j) {
                h[j] = mul2(add2(h[j], both(-mean)), both(rstd));
                if (PARAMS) {
                    dg[l * C + j] = fma2(c[j], h[j], dg[l * C + j]);
                    db[l * C + j] = add2(db[l * C + j], c[j]);
                }
                c[j] = mul2(c[j], gain[l * C + j]);
                sc = add2(sc, c[j]);
                sch = fma2(c[j], h[j], sch);
            }
        }
        if (a.dx) {
            const float2 s = group_sum2<G>(make_float2(sc.x + sc.y, sch.x + sch.y), red[i & 1]);
            const float mc = a.rms ? 0.0f : s.x * inv_n, mch = s.y * inv_n;
            if (real)
                store_row<G, NT>(p, (T *)a.dx + r * a.dx_stride, same, stage, [&](int l) {
                    float2 h[C], c[C];
                    queue.get(p, queue.slot, 0, l, real, h);
                    queue.get(p, queue.slot, 1, l, real, c);
#pragma unroll
                    for (int j = 0; j < C; ++j) {
                        h[j] = mul2(add2(h[j], both(-mean)), both(rstd));
                        c[j] = fma2(c[j], gain[l * C + j], both(-mc));
                        h[j] = mul2(both(rstd), fma2(h[j], both(-mch), c[j]));
                    }
                    return pack_pairs<T>(h);
                });
        }
        push(r + BWD_DEPTH * step, queue.slot);
        queue.pop();
    }
    if constexpr (PARAMS) {
        float *w = a.workspace + (int64_t)blockIdx.x * 2 * a.width;
        float *to = GROUPS > 1 ? joined + group * 2 * a.width : w;
        if (GROUPS > 1) __syncthreads();
#pragma unroll
        for (int j = 0; j < VALS; ++j) {
            const int e = p.column(j / P::N) + j % P::N;
            if (!p.inside(e)) continue;
            to[e] = j & 1 ? dg[j / 2].y : dg[j / 2].x;
            to[a.width + e] = j & 1 ? db[j / 2].y : db[j / 2].x;
        }
        if (GROUPS > 1) {
            __syncthreads();
            for (int e = threadIdx.x; e < 2 * a.width; e += NT) {
                float sum = joined[e];
#pragma unroll
                for (int g = 1; g < GROUPS; ++g) sum += joined[g * 2 * a.width + e];
                w[e] = sum;
            }
        }
    }
}

// Rows of a turn: f32 rows leave shared memory for two CTAs with one only.  4096 rows
// of 16384 bf16 with the parameters' sums: 133 us, 141 with one row to a turn, 231 by
// the kernels for wider rows, which read everything twice; f32 168 and 311.
template <class T>
constexpr int cl_bwd_rows() {
    return sizeof(T) == 4 ? 1 : 2;
}
template <class T, bool PARAMS>
__global__ void __launch_bounds__(NM_NT + 32, 2) norm_cluster_backward_k(NormGradArgs a, int cs) {
    constexpr int R = cl_bwd_rows<T>();
    using P = Place<T, NM_NT, BWD_VALS, false, true>;
    constexpr int C = P::C;
    __shared__ RowExchange<R> ex;
    extern __shared__ uint4 ring[];
    const int rank = blockIdx.x % cs;
    const int64_t step = gridDim.x / cs;
    int64_t r = blockIdx.x / cs;
    const int turns = (int)((a.rows - r + R * step - 1) / (R * step));
    const float inv_n = 1.0f / (float)a.width;
    if (PARAMS) pdl_trigger();  // norm_param_sum_k comes up, and waits for this grid's end
    cluster_arrive_relaxed();   // every CTA has to run before its shared memory is written
    cluster_wait();
    if (threadIdx.x >= NM_NT) {
        if (a.dx) ex.speak(turns, rank, cs, [](float2 v) { return warp_sum2(v); });
        return;
    }
    float2 gain[P::H], dg[P::H], db[P::H];
#pragma unroll
    for (int j = 0; j < P::H; ++j) dg[j] = db[j] = both(0.0f);
    RowQueue<T, P, false, NM_NT, 3 * R, 2> queue;
    queue.ring = ring + threadIdx.x;
    const P p((const T *)a.x + r * a.x_stride, threadIdx.x, a.width, rank, cs);
    auto push = [&](int64_t q, int at) {
        const T *const rows[2] = {(const T *)a.x + q * a.x_stride, (const T *)a.dy + q * a.dy_stride};
        queue.push(p, rows, at, q < a.rows, q == 0);
    };
    for (int k = 0; k < 3 * R; ++k) push(r + k * step, k);
    column_part(p, a.gain, 1.0f, gain);
    float next_mean[R], next_rstd[R];  // of the rows that are sent next
    auto stats = [&](int64_t q) {
#pragma unroll
        for (int k = 0; k < R; ++k, q += step) {
            next_mean[k] = q < a.rows && !a.rms ? a.mean[q] : 0.0f;
            next_rstd[k] = q < a.rows ? a.rstd[q] : 0.0f;
        }
    };
    stats(r);
    // A turn's share in the parameters' sums, and its rows' own sums.
    auto send = [&](int turn, int first, int64_t q) {
        queue.template wait<2 * R>();
        float2 v[R];
#pragma unroll
        for (int k = 0; k < R; ++k) {
            const bool real = q + k * step < a.rows;
            float2 sc = both(0.0f), sch = sc;
#pragma unroll
            for (int l = 0; l < P::LOADS; ++l) {
                float2 h[C], c[C];
                queue.get(p, queue.ahead(first + k), 0, l, real, h);
                queue.get(p, queue.ahead(first + k), 1, l, real, c);
#pragma unroll
                for (int j = 0; j < C; ++j) {
                    h[j] = mul2(add2(h[j], both(-next_mean[k])), both(next_rstd[k]));
                    if (PARAMS) {
                        dg[l * C + j] = fma2(c[j], h[j], dg[l * C + j]);
                        db[l * C + j] = add2(db[l * C + j], c[j]);
                    }
                    c[j] = mul2(c[j], gain[l * C + j]);
                    sc = add2(sc, c[j]);
                    sch = fma2(c[j], h[j], sch);
                }
            }
            v[k] = make_float2(sc.x + sc.y, sch.x + sch.y);
        }
        if (!a.dx) return;
#pragma unroll
        for (int k = 0; k < R; ++k) v[k] = warp_sum2(v[k]);
        ex.send(v, turn);
    };
    send(0, 0, r);
    for (int i = 0; i < turns; ++i) {
        float mean[R], rstd[R];
        float2 s[R];
#pragma unroll
        for (int k = 0; k < R; ++k) {
            mean[k] = next_mean[k];
            rstd[k] = next_rstd[k];
        }
        if (a.dx) ex.receive(s, i, cs);
        stats(r + R * step);
        if (i + 1 < turns) send(i + 1, R, r + R * step);
#pragma unroll
        for (int k = 0; k < R; ++k) {
            if (a.dx && r < a.rows) {
                const float2 all = warp_sum2(s[k]);
                const float mc = a.rms ? 0.0f : all.x * inv_n, mch = all.y * inv_n;
                store_row<NM_NT, NM_NT>(p, (T *)a.dx + r * a.dx_stride, true, nullptr, [&](int l) {
                    float2 h[C], c[C];
                    queue.get(p, queue.slot, 0, l, true, h);
                    queue.get(p, queue.slot, 1, l, true, c);
#pragma unroll
                    for (int j = 0; j < C; ++j) {
                        h[j] = mul2(add2(h[j], both(-mean[k])), both(rstd[k]));
                        c[j] = fma2(c[j], gain[l * C + j], both(-mc));
                        h[j] = mul2(both(rstd[k]), fma2(h[j], both(-mch), c[j]));
                    }
                    return pack_pairs<T>(h);
                });
            }
            push(r + 3 * R * step, queue.slot);
            queue.pop();
            r += step;
        }
    }
    if constexpr (PARAMS) {
        float *w = a.workspace + (int64_t)(blockIdx.x / cs) * 2 * a.width;
#pragma unroll
        for (int j = 0; j < BWD_VALS; ++j) {
            const int e = p.column(j / P::N) + j % P::N;
            if (!p.has(j / P::N) || !p.inside(e)) continue;
            w[e] = j & 1 ? dg[j / 2].y : dg[j / 2].x;
            w[a.width + e] = j & 1 ? db[j / 2].y : db[j / 2].x;
        }
    }
}

// Rows too wide for the kernels above, and those of which x and dy (VEC: dx too) start at
// different places of a 16-byte unit, at any width: 65536 x 1024 bf16 with dy of stride
// 1025 take 658 us, nine times what equal strides do (f32 625 us, five times).
template <class T, bool VEC>
__global__ void __launch_bounds__(WIDE_NT) norm_wide_dx_k(NormGradArgs a) {
    __shared__ float red[32];
    constexpr int N = VEC ? Vec<T>::N : 1;
    const int64_t r = blockIdx.x;
    const T *x = (const T *)a.x + r * a.x_stride, *dy = (const T *)a.dy + r * a.dy_stride;
    T *dx = (T *)a.dx + r * a.dx_stride;
    // The gradient's vector (element) v beside x's.
    auto x_at = [&](int v) {
        if constexpr (VEC)
            return load16_rw(x + (int64_t)v * N);
        else
            return x[v];
    };
    const float n = (float)a.width, mean = a.rms ? 0.0f : a.mean[r], rstd = a.rstd[r];
    auto both_of = [&](int v, float (&h)[N], float (&c)[N]) {
        if constexpr (VEC)
            unpack<T>(load16_rw(dy + (int64_t)v * N), c);
        else
            c[0] = to_f32(dy[v]);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            c[i] *= a.gain ? a.gain[v * N + i] : 1.0f;
            h[i] = (h[i] - mean) * rstd;
        }
    };
    float sc = 0.0f, sch = 0.0f;
    wide_each<T, VEC>(a.width, x_at, [&](int v, float (&h)[N]) {
        float c[N];
        both_of(v, h, c);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            sc += c[i];
            sch = fmaf(c[i], h[i], sch);
        }
    });
    sc = a.rms ? 0.0f : block_sum(sc, red) / n;
    sch = block_sum(sch, red) / n;
    wide_each<T, VEC>(a.width, x_at, [&](int v, float (&h)[N]) {
        float c[N];
        both_of(v, h, c);
#pragma unroll
        for (int i = 0; i < N; ++i) h[i] = rstd * (c[i] - sc - h[i] * sch);
        if constexpr (VEC)
            store16(dx + (int64_t)v * N, pack<T>(h));
        else
            dx[v] = from_f32<T>(h[0]);
    });
}

// Partial sums over the rows p, p + P, ... of N columns (one without VEC) per
// thread; of PARAM_ROWS at a time, joined in the workspace, so that with millions of
// rows a term still passes through few additions (2^20 rows: 64 + 256 in place of
// 16384).  (Two rows at once, four of single f32: 65536 rows of 1024 f32, dx included, 625
// us, with two 816; of bf16, element by element, 658 and with four 1053.)
constexpr int PARAM_ROWS = 64;
template <class T, bool VEC>
__global__ void __launch_bounds__(NM_NT) norm_wide_param_k(NormGradArgs a) {
    constexpr int N = VEC ? Vec<T>::N : 1;
    const int e = (blockIdx.x * NM_NT + threadIdx.x) * N;
    if (e >= a.width) return;
    float *w = a.workspace + (int64_t)blockIdx.y * 2 * a.width;
    const T *x = (const T *)a.x + blockIdx.y * a.x_stride + e, *dy = (const T *)a.dy + blockIdx.y * a.dy_stride + e;
    const int64_t x_step = gridDim.y * a.x_stride, dy_step = gridDim.y * a.dy_stride;
    const int n = (int)((a.rows - blockIdx.y + gridDim.y - 1) / gridDim.y);
    int r = blockIdx.y;
    for (int done = 0; done < n; done += PARAM_ROWS) {
        const int m = min(n - done, PARAM_ROWS);
        float dg[N] = {}, db[N] = {};
#pragma unroll (sizeof(T) == 4 && !VEC ? 4 : 2)
        for (int k = 0; k < m; ++k, r += gridDim.y, x += x_step, dy += dy_step) {
            const float mean = a.rms ? 0.0f : a.mean[r], rstd = a.rstd[r];
            float h[N], c[N];
            if constexpr (VEC) {
                unpack<T>(load16_rw(x), h);
                unpack<T>(load16_rw(dy), c);
            } else {
                h[0] = to_f32(*x);
                c[0] = to_f32(*dy);
            }
#pragma unroll
            for (int i = 0; i < N; ++i) {
                dg[i] = fmaf(c[i], (h[i] - mean) * rstd, dg[i]);
                db[i] += c[i];
            }
        }
#pragma unroll
        for (int i = 0; i < N; ++i) {
            w[e + i] = done == 0 ? dg[i] : w[e + i] + dg[i];
            w[a.width + e + i] = done == 0 ? db[i] : w[a.width + e + i] + db[i];
        }
    }
}

// The partial rows' sum, from L2 (it starts while the rows' kernel ends): 32 columns to a block, SUM_LANES threads to a column,
// each over every SUM_LANES-th row; their sums are added in order.
constexpr int SUM_LANES = 16;
__global__ void __launch_bounds__(32 * SUM_LANES) norm_param_sum_k(NormGradArgs a, int parts) {
    __shared__ float sums[SUM_LANES][32];
    pdl_wait();
    const int col = threadIdx.x & 31, w = threadIdx.x >> 5;
    const int64_t e = (int64_t)blockIdx.x * 32 + col, n = 2 * (int64_t)a.width;
    float s = 0.0f;
    if (e < n) {
#pragma unroll 8
        for (int p = w; p < parts; p += SUM_LANES) s += a.workspace[p * n + e];
    }
    sums[w][col] = s;
    __syncthreads();
    if (w || e >= n) return;
#pragma unroll
    for (int i = 1; i < SUM_LANES; ++i) s += sums[i][col];
    float *to = e < a.width ? a.dgain : a.dbias;
    if (!to) return;
    const int64_t at = e < a.width ? e : e - a.width;
    to[at] = a.accumulate ? to[at] + s : s;
}

// ---------------------------------------------------------------- launches
bool aligned16(const void *p, int64_t stride, int es) { return ((uintptr_t)p & 15) == 0 && stride * es % 16 == 0; }
// Whether every row of b starts at the same place of a 16-byte unit as that of a.
bool same_place(const void *a, int64_t a_stride, const void *b, int64_t b_stride, int es) {
    return (((uintptr_t)a ^ (uintptr_t)b) & 15) == 0 && (a_stride - b_stride) * es % 16 == 0;
}

// Blocks (or clusters) that the GPU holds at once, at most one per turn of
// rows; a multiple of 8 where rows that start anywhere take several turns.
// (More clusters than fit would run all their turns after the others.)
constexpr int MOST_CLUSTERS[] = {0, 2 * 148, 148, 92, 68, 55, 44, 36, 32};  // of that many CTAs, two to an SM
int64_t blocks(int64_t rows, int groups, int most, bool edge) {
    return std::max<int64_t>(1, std::min<int64_t>((rows + groups - 1) / groups, edge ? most / 8 * 8 : most));
}

// With `smem` bytes of shared memory of the `most` that any call of this kernel takes.
template <class... Params, class... Args>
cudaError_t launch(void (*kern)(Params...), int64_t grid, int nt, int smem, int most, int cs, cudaStream_t st, Args... args) {
    if (smem > 40000) {
        cudaError_t e = allow_shared(kern, most);
        if (e != cudaSuccess) return e;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(grid * cs));
    cfg.blockDim = dim3(nt);
    cfg.dynamicSmemBytes = (size_t)smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)cs;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cs > 1 ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kern, static_cast<Params>(args)...);
}

// The group and the elements per thread for a number of 16-byte units: as few
// threads as hold it with MOST elements each, a warp at least; three quarters of
// them where that is enough (16384 rows of 2560 bf16 34 us, with the unused places 41).
// Forward MOST is 64 bytes (16384 rows of 4096 bf16 cold: 45 us, with 32 bytes 49);
// backward 16 elements, whose gain and sums take 48 registers (65536 rows of 1024
// bf16 cold: 73 us, with 32 elements 95).
template <class T, int MOST, class F>
cudaError_t with_group(int units, F &&f) {
    constexpr int N = Vec<T>::N, L = MOST / N;
    using std::integral_constant;
    if (units <= 32) return f(integral_constant<int, 32>(), integral_constant<int, N>());
    if (2 < L && units <= 64) return f(integral_constant<int, 32>(), integral_constant<int, 2 * N>());
    integral_constant<int, MOST> vals;
    integral_constant<int, (L > 3 ? 3 * N : MOST)> fewer;
    if (units <= 32 * L) return f(integral_constant<int, 32>(), vals);
    if (L > 3 && units <= 64 * 3) return f(integral_constant<int, 64>(), fewer);
    if (units <= 64 * L) return f(integral_constant<int, 64>(), vals);
    if (L > 3 && units <= 128 * 3) return f(integral_constant<int, 128>(), fewer);
    if (units <= 128 * L) return f(integral_constant<int, 128>(), vals);
    if (L > 3 && units <= 256 * 3) return f(integral_constant<int, 256>(), fewer);
    if (units <= 256 * L) return f(integral_constant<int, 256>(), vals);
    return f(integral_constant<int, 512>(), vals);
}
// The most units of a part of a row that a cluster shares, and its CTAs: as few as hold it.
template <class T, int MOST>
constexpr int part_units() {
    return NM_NT * MOST / Vec<T>::N;
}
template <class T, int MOST>
int cluster_of(int units) {
    return (units + part_units<T, MOST>() - 1) / part_units<T, MOST>();
}
// The units that a row can cover.
template <class T, bool EDGE>
int units_of(int width) {
    return (width + (EDGE ? 2 : 1) * (Vec<T>::N - 1)) / Vec<T>::N;
}

template <class T, bool EDGE>
cudaError_t forward_g(const NormArgs &a, int same, cudaStream_t st) {
    return with_group<T, fwd_vals<T>()>(units_of<T, EDGE>(a.width), [&](auto g, auto vals) {
        constexpr int G = decltype(g)::value, VALS = decltype(vals)::value, NT = G > NM_NT ? G : NM_NT;
        constexpr int queue = RowQueue<T, Place<T, G, VALS, EDGE, false>, EDGE, NT, FWD_DEPTH, 1>::BYTES, stage = NT * VALS * (int)sizeof(T);
        return launch(norm_rows_k<T, G, VALS, EDGE>, blocks(a.rows, NT / G, NT > NM_NT ? 148 : 2 * 148, EDGE), NT, queue + (same ? 0 : stage),
                      queue + (EDGE ? stage : 0), 1, st, a, same);
    });
}
template <class T>
cudaError_t forward(const NormArgs &a, cudaStream_t st) {
    constexpr int N = Vec<T>::N, ES = sizeof(T), MOST = fwd_vals<T>(), most = 512 * MOST / N;
    const bool same = same_place(a.x, a.x_stride, a.y, a.y_stride, ES);
    const bool whole = same && a.width % N == 0 && aligned16(a.x, a.x_stride, ES);
    const int units = a.width / N;
    if (whole && units <= most) return forward_g<T, false>(a, 1, st);
    if (units_of<T, true>(a.width) <= most) return forward_g<T, true>(a, same, st);
    if (whole && units <= CL_MOST * part_units<T, MOST>()) {
        const int cs = cluster_of<T, MOST>(units), smem = RowQueue<T, Place<T, NM_NT, MOST, false, true>, false, NM_NT, 3 * CL_FWD_ROWS, 1>::BYTES;
        return launch(norm_cluster_rows_k<T>, blocks(a.rows, 1, MOST_CLUSTERS[cs], false), NM_NT + 32, smem, smem, cs, st, a, cs);
    }
    if (whole)
        norm_wide_rows_k<T, true><<<(unsigned)a.rows, WIDE_NT, 0, st>>>(a);
    else
        norm_wide_rows_k<T, false><<<(unsigned)a.rows, WIDE_NT, 0, st>>>(a);
    return cudaGetLastError();
}

// The partial rows of dgain and dbias, at most: what `blocks` gives, or in rows
// that are too wide for any group WIDE_PARTS.
constexpr int WIDE_PARTS = 64;
int partial_rows(int64_t rows, int width) {
    return (int)std::min<int64_t>(std::max<int64_t>(rows, 1), width > CL_MOST * NM_NT * BWD_VALS ? WIDE_PARTS : 2 * 148);
}

template <class T, bool EDGE>
cudaError_t backward_g(const NormGradArgs &a, int same, bool params, int64_t &parts, cudaStream_t st) {
    return with_group<T, BWD_VALS>(units_of<T, EDGE>(a.width), [&](auto g, auto vals) {
        constexpr int G = decltype(g)::value, VALS = decltype(vals)::value, NT = G > NM_NT ? G : NM_NT, GROUPS = NT / G;
        parts = blocks(a.rows, GROUPS, NT > NM_NT ? 148 : 2 * 148, EDGE);
        // (Where the parameters' sums are joined the rows were: two f32 for each of their elements.)
        constexpr int queue = RowQueue<T, Place<T, G, VALS, EDGE, false>, EDGE, NT, BWD_DEPTH, 2>::BYTES, stage = NT * VALS * (int)sizeof(T);
        static_assert(GROUPS == 1 || queue >= NT * VALS * 2 * (int)sizeof(float), "");
        const int smem = queue + (same ? 0 : stage), most = queue + (EDGE ? stage : 0);
        return params ? launch(norm_backward_k<T, G, VALS, EDGE, true>, parts, NT, smem, most, 1, st, a, same)
                      : launch(norm_backward_k<T, G, VALS, EDGE, false>, parts, NT, smem, most, 1, st, a, same);
    });
}

template <class T>
cudaError_t backward(const NormGradArgs &a, cudaStream_t st) {
    constexpr int N = Vec<T>::N, ES = sizeof(T), most = 512 * BWD_VALS / N;
    const bool params = a.dgain || a.dbias;
    int64_t parts = 0;
    const bool like = same_place(a.x, a.x_stride, a.dy, a.dy_stride, ES);
    const bool same = !a.dx || same_place(a.x, a.x_stride, a.dx, a.dx_stride, ES);
    const bool vec = like && same && a.width % N == 0 && aligned16(a.x, a.x_stride, ES);
    const int units = a.width / N;
    if (a.rows && vec && units <= most) {
        if (cudaError_t e = backward_g<T, false>(a, 1, params, parts, st)) return e;
    } else if (a.rows && like && units_of<T, true>(a.width) <= most) {
        if (cudaError_t e = backward_g<T, true>(a, same, params, parts, st)) return e;
    } else if (a.rows && vec && units <= CL_MOST * part_units<T, BWD_VALS>()) {
        const int cs = cluster_of<T, BWD_VALS>(units);
        const int smem = RowQueue<T, Place<T, NM_NT, BWD_VALS, false, true>, false, NM_NT, 3 * cl_bwd_rows<T>(), 2>::BYTES;
        parts = blocks(a.rows, 1, MOST_CLUSTERS[cs], false);
        cudaError_t e = params ? launch(norm_cluster_backward_k<T, true>, parts, NM_NT + 32, smem, smem, cs, st, a, cs)
                               : launch(norm_cluster_backward_k<T, false>, parts, NM_NT + 32, smem, smem, cs, st, a, cs);
        if (e) return e;
    } else if (a.rows) {
        // The parameters' sums first: dx may be the array of dy.
        if (params) {
            parts = std::min<int64_t>(a.rows, WIDE_PARTS);
            const unsigned cols = (unsigned)((a.width / (vec ? N : 1) + NM_NT - 1) / NM_NT);
            if (vec)
                norm_wide_param_k<T, true><<<dim3(cols, (unsigned)parts), NM_NT, 0, st>>>(a);
            else
                norm_wide_param_k<T, false><<<dim3(cols, (unsigned)parts), NM_NT, 0, st>>>(a);
            if (cudaError_t e = cudaGetLastError()) return e;
        }
        if (a.dx) {
            if (vec)
                norm_wide_dx_k<T, true><<<(unsigned)a.rows, WIDE_NT, 0, st>>>(a);
            else
                norm_wide_dx_k<T, false><<<(unsigned)a.rows, WIDE_NT, 0, st>>>(a);
            if (cudaError_t e = cudaGetLastError()) return e;
        }
    }
    if (params) {
        return pdl_launch(norm_param_sum_k, dim3((unsigned)((2 * (int64_t)a.width + 31) / 32)), dim3(32 * SUM_LANES), 0, st, a, (int)parts);
    }
    return cudaSuccess;
}

}  // namespace

cudaError_t norm_rows(const NormArgs &a, int dtype, cudaStream_t st) {
    switch (dtype) {
        case 0: return forward<float>(a, st);
        case 1: return forward<__half>(a, st);
        default: return forward<__nv_bfloat16>(a, st);
    }
}

size_t norm_backward_workspace_bytes(int64_t rows, int width) {
    return (size_t)partial_rows(rows, width) * 2 * (size_t)width * sizeof(float);
}

cudaError_t norm_backward(const NormGradArgs &a, int dtype, cudaStream_t st) {
    switch (dtype) {
        case 0: return backward<float>(a, st);
        case 1: return backward<__half>(a, st);
        default: return backward<__nv_bfloat16>(a, st);
    }
}

}  // namespace nk
