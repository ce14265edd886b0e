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
// hence the f32 operations in pairs, and 64 bytes of a row to a thread where it has them.
// Rows too wide for that take one block per row and read it again from L2.

#include <algorithm>

#include "nk_head.cuh"
#include "nk_head.h"

namespace nk {

namespace {

constexpr int NM_NT = 256;
constexpr int ONE_VALS = 16;  // of a thread, backward and where no vectors fit
constexpr int FWD_DEPTH = 4;  // rows on their way to each group
constexpr int BWD_DEPTH = 3;
constexpr int PARTIAL_ROWS = 1024;  // most partial sums of dgain and dbias

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
template <int G>
__device__ __forceinline__ float2 group_sum2(float2 v, float2 *red) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
        v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
    }
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

// Where a thread's elements lie: with VEC, VALS / N vectors of N elements, G
// vectors apart; else single elements, G apart.
template <class T, int G, int VALS, bool VEC>
struct Place {
    static constexpr int N = VEC ? Vec<T>::N : 1;
    static constexpr int LOADS = VALS / N;
    static __device__ __forceinline__ int at(int lane, int l) { return (l * G + lane) * N; }
};

// The rows that a thread will work on next, ARRAYS of them at a time: with VEC
// in its own places of a ring in shared memory, DEPTH rows on their way by
// asynchronous copies (no barrier: a thread reads only what it copied); else
// one row in registers, which the next push overwrites.
template <class T, int G, int VALS, bool VEC, int NT, int DEPTH, int ARRAYS>
struct RowQueue {
    using P = Place<T, G, VALS, VEC>;
    static constexpr int AHEAD = VEC ? DEPTH : 1;
    static constexpr int BYTES = VEC ? DEPTH * ARRAYS * P::LOADS * NT * 16 : 0;
    T next[ARRAYS][VEC ? 1 : VALS];
    uint4 *ring;  // [DEPTH][ARRAYS][LOADS][NT], from this thread's place on
    int slot = 0;

    __device__ __forceinline__ uint4 *place(int at, int k) const { return ring + (at * ARRAYS + k) * P::LOADS * NT; }
    __device__ __forceinline__ void push(const T *const (&rows)[ARRAYS], int at, int lane, int width, bool real) {
#pragma unroll
        for (int k = 0; k < ARRAYS; ++k) {
            const T *row = rows[k] + lane * P::N;
#pragma unroll
            for (int l = 0; l < P::LOADS; ++l) {
                const bool in = real && P::at(lane, l) < width;
                if constexpr (VEC) {
                    if (in) copy_async16(place(at, k) + l * NT, row + l * G * P::N);
                } else {
                    next[k][l] = in ? row[l * G] : from_f32<T>(0.0f);
                }
            }
        }
        if constexpr (VEC) copy_commit();
    }
    // Waits for the row pushed first, which is then the present one.
    __device__ __forceinline__ void wait() const {
        if constexpr (VEC) copy_wait<DEPTH - 1>();
    }
    // Done with it: the next push goes to its slot.
    __device__ __forceinline__ void pop() { slot = slot + 1 == AHEAD ? 0 : slot + 1; }
    // Chunk c of the present row: a vector's elements (VEC) or two of the single
    // ones, in pairs; zeros beyond the width.
    static constexpr int CHUNK = VEC ? P::N / 2 : 1;
    __device__ __forceinline__ void get(int k, int c, int lane, int width, bool real, float2 (&x)[CHUNK]) const {
        if constexpr (VEC) {
            float v[P::N];
            unpack<T>(real && P::at(lane, c) < width ? place(slot, k)[c * NT] : make_uint4(0, 0, 0, 0), v);
#pragma unroll
            for (int i = 0; i < CHUNK; ++i) x[i] = make_float2(v[2 * i], v[2 * i + 1]);
        } else {
            x[0] = make_float2(to_f32(next[k][2 * c]), to_f32(next[k][2 * c + 1]));
        }
    }
    // A pair of chunk c, 0 where it is beyond the width.
    static __device__ __forceinline__ float2 keep(int c, int lane, int width, float2 v) {
        if constexpr (VEC) return P::at(lane, c) < width ? v : make_float2(0.0f, 0.0f);
        return make_float2(P::at(lane, 2 * c) < width ? v.x : 0.0f, P::at(lane, 2 * c + 1) < width ? v.y : 0.0f);
    }
};

// Chunk c of a thread's part of a row, as RowQueue::get has it.
template <class T, int G, int VALS, bool VEC, int CHUNK>
__device__ __forceinline__ void store_chunk(T *row, int c, int lane, int width, const float2 (&x)[CHUNK]) {
    using P = Place<T, G, VALS, VEC>;
    if constexpr (VEC) {
        if (P::at(lane, c) >= width) return;
        float v[P::N];
#pragma unroll
        for (int i = 0; i < CHUNK; ++i) {
            v[2 * i] = x[i].x;
            v[2 * i + 1] = x[i].y;
        }
        store16(row + P::at(lane, c), pack<T>(v));
    } else {
        if (P::at(lane, 2 * c) < width) row[P::at(lane, 2 * c)] = from_f32<T>(x[0].x);
        if (P::at(lane, 2 * c + 1) < width) row[P::at(lane, 2 * c + 1)] = from_f32<T>(x[0].y);
    }
}

// A thread's part of an f32 vector of the width (null: `other`); 0 beyond it.
template <class T, int G, int VALS, bool VEC>
__device__ __forceinline__ void column_part(const float *p, float other, int lane, int width, float2 (&x)[VALS / 2]) {
    using P = Place<T, G, VALS, VEC>;
    auto one = [&](int k) {
        const int e = P::at(lane, k / P::N) + k % P::N;
        return e < width ? (p ? p[e] : other) : 0.0f;
    };
#pragma unroll
    for (int k = 0; k < VALS / 2; ++k) x[k] = make_float2(one(2 * k), one(2 * k + 1));
}

// Elements e and e + step of a row, 0 beyond the width.
template <class T>
__device__ __forceinline__ float2 pair_of(const T *row, int e, int step, int width) {
    return make_float2(e < width ? to_f32(row[e]) : 0.0f, e + step < width ? to_f32(row[e + step]) : 0.0f);
}

__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }

// ---------------------------------------------------------------- forward
template <class T, int G, int VALS, bool VEC>
__global__ void __launch_bounds__(G > NM_NT ? G : NM_NT, G > NM_NT ? 1 : 2) norm_rows_k(NormArgs a) {
    constexpr int NT = G > NM_NT ? G : NM_NT, GROUPS = NT / G, H = VALS / 2;
    using Queue = RowQueue<T, G, VALS, VEC, NT, FWD_DEPTH, 1>;
    constexpr int C = Queue::CHUNK;
    __shared__ float red[2][32];
    extern __shared__ uint4 ring[];
    const int lane = threadIdx.x % G, group = threadIdx.x / G;
    const float inv_n = 1.0f / (float)a.width;
    float2 gain[H], bias[H];
    Queue queue;
    queue.ring = ring + threadIdx.x;
    const int64_t step = (int64_t)gridDim.x * GROUPS;
    int64_t r = (int64_t)blockIdx.x * GROUPS + group;
    auto push = [&](int64_t q, int at) {
        const T *const rows[1] = {(const T *)a.x + q * a.x_stride};
        queue.push(rows, at, lane, a.width, q < a.rows);
    };
    for (int k = 0; k < Queue::AHEAD; ++k) push(r + k * step, k);
    if constexpr (VEC) {
        column_part<T, G, VALS, VEC>(a.gain, 1.0f, lane, a.width, gain);
        column_part<T, G, VALS, VEC>(a.bias, 0.0f, lane, a.width, bias);
    }
    // Every group takes the same number of turns: the reductions hold barriers.
    const int turns = (int)((a.rows - (int64_t)blockIdx.x * GROUPS + step - 1) / step);
    for (int i = 0; i < turns; ++i, r += step) {
        const bool real = r < a.rows;
        float2 x[H];
        queue.wait();
#pragma unroll
        for (int c = 0; c < H / C; ++c) {
            float2 v[C];
            queue.get(0, c, lane, a.width, real, v);
#pragma unroll
            for (int j = 0; j < C; ++j) x[c * C + j] = v[j];
        }
        push(r + Queue::AHEAD * step, queue.slot);
        queue.pop();
        float mean = 0.0f;
        if (!a.rms) {
            float2 s = x[0];
#pragma unroll
            for (int j = 1; j < H; ++j) s = add2(s, x[j]);
            mean = group_sum<G>(s.x + s.y, red[0]) * inv_n;
        }
        float2 v = both(0.0f);
#pragma unroll
        for (int j = 0; j < H; ++j) {
            x[j] = Queue::keep(j / C, lane, a.width, add2(x[j], both(-mean)));
            v = fma2(x[j], x[j], v);
        }
        const float rstd = 1.0f / sqrtf(fmaf(group_sum<G>(v.x + v.y, red[1]), inv_n, a.eps));
        if (G > 32 && a.rms) __syncthreads();  // red[1] again in the next turn
        if (!real) continue;
        if constexpr (!VEC) {  // from L1 for every row: the loads' sixteen registers are taken
            column_part<T, G, VALS, VEC>(a.gain, 1.0f, lane, a.width, gain);
            column_part<T, G, VALS, VEC>(a.bias, 0.0f, lane, a.width, bias);
        }
#pragma unroll
        for (int c = 0; c < H / C; ++c) {
            float2 v[C];
#pragma unroll
            for (int j = 0; j < C; ++j) v[j] = fma2(mul2(x[c * C + j], both(rstd)), gain[c * C + j], bias[c * C + j]);
            store_chunk<T, G, VALS, VEC>((T *)a.y + r * a.y_stride, c, lane, a.width, v);
        }
        if (lane == 0) {
            if (a.mean) a.mean[r] = mean;
            if (a.rstd) a.rstd[r] = rstd;
        }
    }
}

// Rows that are too wide for a group: a block each, the first `keep` vectors
// (16 bytes with VEC) waiting in shared memory, the others read again from L2.
constexpr int WIDE_NT = 512;
constexpr int WIDE_KEEP = 64 << 10;  // bytes: three blocks to an SM

// f(pair of elements, index of the first) over a thread's part of a row, which
// `at(v)` gives as 16 bytes of N elements (VEC) or one element.
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
__global__ void __launch_bounds__(WIDE_NT) norm_wide_rows_k(NormArgs a, int keep) {
    __shared__ float red[32];
    extern __shared__ uint4 kept[];
    constexpr int N = VEC ? Vec<T>::N : 1;
    const int64_t r = blockIdx.x;
    const T *x = (const T *)a.x + r * a.x_stride;
    T *y = (T *)a.y + r * a.y_stride;
    if constexpr (VEC) {
        for (int v = threadIdx.x; v < min(keep, a.width / N); v += WIDE_NT) copy_async16(&kept[v], x + v * N);
        copy_commit();
        copy_wait<0>();
    }
    auto at = [&](int v) {
        if constexpr (VEC)
            return v < keep ? kept[v] : load16_rw(x + (int64_t)v * N);
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
// groups' registers joined in shared memory in their order, one row of
// the workspace per block.  The row is unpacked twice, once for the sums and
// once for dx: it waits in shared memory (without VEC in L1), not in registers.
template <class T, int G, int VALS, bool VEC, bool PARAMS>
__global__ void __launch_bounds__(G > NM_NT ? G : NM_NT, G > NM_NT ? 1 : 2) norm_backward_k(NormGradArgs a) {
    using P = Place<T, G, VALS, VEC>;
    constexpr int NT = G > NM_NT ? G : NM_NT, GROUPS = NT / G, H = VALS / 2;
    using Queue = RowQueue<T, G, VALS, VEC, NT, BWD_DEPTH, 2>;
    constexpr int C = Queue::CHUNK;
    __shared__ float2 red[2][32];
    extern __shared__ uint4 ring[];
    float *joined = (float *)ring;  // [GROUPS][2][width], when the rows are done
    const int lane = threadIdx.x % G, group = threadIdx.x / G;
    const float inv_n = 1.0f / (float)a.width;
    float2 gain[H], dg[H], db[H];
#pragma unroll
    for (int j = 0; j < H; ++j) dg[j] = db[j] = both(0.0f);
    Queue queue;
    queue.ring = ring + threadIdx.x;
    const int64_t step = (int64_t)gridDim.x * GROUPS;
    int64_t r = (int64_t)blockIdx.x * GROUPS + group;
    auto push = [&](int64_t q, int at) {
        const T *const rows[2] = {(const T *)a.x + q * a.x_stride, (const T *)a.dy + q * a.dy_stride};
        queue.push(rows, at, lane, a.width, q < a.rows);
    };
    float next_mean, next_rstd;
    auto stats = [&](int64_t q) {
        next_mean = q < a.rows && !a.rms ? a.mean[q] : 0.0f;
        next_rstd = q < a.rows ? a.rstd[q] : 0.0f;
    };
    for (int k = 0; k < Queue::AHEAD; ++k) push(r + k * step, k);
    stats(r);
    if constexpr (VEC) column_part<T, G, VALS, VEC>(a.gain, 1.0f, lane, a.width, gain);
    const int turns = (int)((a.rows - (int64_t)blockIdx.x * GROUPS + step - 1) / step);
    for (int i = 0; i < turns; ++i, r += step) {
        const bool real = r < a.rows;
        const float mean = next_mean, rstd = next_rstd;
        queue.wait();
        if constexpr (!VEC) column_part<T, G, VALS, VEC>(a.gain, 1.0f, lane, a.width, gain);
        stats(r + step);
        float2 sc = both(0.0f), sch = sc;
        // Beyond the width dy and the gain are 0, and h does not count.
#pragma unroll
        for (int q = 0; q < H / C; ++q) {
            float2 h[C], c[C];
            queue.get(0, q, lane, a.width, real, h);
            queue.get(1, q, lane, a.width, real, c);
#pragma unroll
            for (int j = 0; j < C; ++j) {
                h[j] = mul2(add2(h[j], both(-mean)), both(rstd));
                if (PARAMS) {
                    dg[q * C + j] = fma2(c[j], h[j], dg[q * C + j]);
                    db[q * C + j] = add2(db[q * C + j], c[j]);
                }
                c[j] = mul2(c[j], gain[q * C + j]);
                sc = add2(sc, c[j]);
                sch = fma2(c[j], h[j], sch);
            }
        }
        if constexpr (!VEC) push(r + step, 0);
        if (a.dx) {
            const float2 s = group_sum2<G>(make_float2(sc.x + sc.y, sch.x + sch.y), red[i & 1]);
            const float mc = a.rms ? 0.0f : s.x * inv_n, mch = s.y * inv_n;
            T *to = (T *)a.dx + r * a.dx_stride;
            if (real) {
#pragma unroll
                for (int q = 0; q < H / C; ++q) {
                    float2 h[C], c[C];
                    if constexpr (VEC) {
                        queue.get(0, q, lane, a.width, real, h);
                        queue.get(1, q, lane, a.width, real, c);
                    } else {  // from L1
                        h[0] = pair_of((const T *)a.x + r * a.x_stride, P::at(lane, 2 * q), G, a.width);
                        c[0] = pair_of((const T *)a.dy + r * a.dy_stride, P::at(lane, 2 * q), G, a.width);
                    }
#pragma unroll
                    for (int j = 0; j < C; ++j) {
                        h[j] = mul2(add2(h[j], both(-mean)), both(rstd));
                        c[j] = fma2(c[j], gain[q * C + j], both(-mc));
                        h[j] = mul2(both(rstd), fma2(h[j], both(-mch), c[j]));
                    }
                    store_chunk<T, G, VALS, VEC>(to, q, lane, a.width, h);
                }
            }
        }
        if constexpr (VEC) {
            push(r + Queue::AHEAD * step, queue.slot);
            queue.pop();
        }
    }
    if constexpr (PARAMS) {
        float *w = a.workspace + (int64_t)blockIdx.x * 2 * a.width;
        float *to = GROUPS > 1 ? joined + group * 2 * a.width : w;
        if (GROUPS > 1) __syncthreads();
#pragma unroll
        for (int j = 0; j < VALS; ++j) {
            const int e = P::at(lane, j / P::N) + j % P::N;
            if (e >= a.width) continue;
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

template <class T, bool VEC>
__global__ void __launch_bounds__(WIDE_NT) norm_wide_dx_k(NormGradArgs a, int keep) {
    __shared__ float red[32];
    extern __shared__ uint4 kept[];  // [keep] of x, [keep] of dy
    constexpr int N = VEC ? Vec<T>::N : 1;
    const int64_t r = blockIdx.x;
    const T *x = (const T *)a.x + r * a.x_stride, *dy = (const T *)a.dy + r * a.dy_stride;
    T *dx = (T *)a.dx + r * a.dx_stride;
    if constexpr (VEC) {
        for (int v = threadIdx.x; v < min(keep, a.width / N); v += WIDE_NT) {
            copy_async16(&kept[v], x + v * N);
            copy_async16(&kept[keep + v], dy + v * N);
        }
        copy_commit();
        copy_wait<0>();
    }
    // The gradient's vector (element) v beside x's.
    auto x_at = [&](int v) {
        if constexpr (VEC)
            return v < keep ? kept[v] : load16_rw(x + (int64_t)v * N);
        else
            return x[v];
    };
    const float n = (float)a.width, mean = a.rms ? 0.0f : a.mean[r], rstd = a.rstd[r];
    auto both_of = [&](int v, float (&h)[N], float (&c)[N]) {
        if constexpr (VEC)
            unpack<T>(v < keep ? kept[keep + v] : load16_rw(dy + (int64_t)v * N), c);
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
// thread.
template <class T, bool VEC>
__global__ void __launch_bounds__(NM_NT) norm_wide_param_k(NormGradArgs a) {
    constexpr int N = VEC ? Vec<T>::N : 1;
    const int e = (blockIdx.x * NM_NT + threadIdx.x) * N;
    if (e >= a.width) return;
    float dg[N] = {}, db[N] = {};
#pragma unroll 2
    for (int64_t r = blockIdx.y; r < a.rows; r += gridDim.y) {
        const T *x = (const T *)a.x + r * a.x_stride + e, *dy = (const T *)a.dy + r * a.dy_stride + e;
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
    float *w = a.workspace + (int64_t)blockIdx.y * 2 * a.width;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        w[e + i] = dg[i];
        w[a.width + e + i] = db[i];
    }
}

// The partial rows' sum: 32 columns to a block, SUM_LANES threads to a column,
// each over every SUM_LANES-th row; their sums are added in order.
constexpr int SUM_LANES = 16;
__global__ void __launch_bounds__(32 * SUM_LANES) norm_param_sum_k(NormGradArgs a, int parts) {
    __shared__ float sums[SUM_LANES][32];
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

// Blocks that the GPU holds at once, at most one per turn of rows.
int64_t blocks(int64_t rows, int groups, int per_sm) {
    return std::max<int64_t>(1, std::min<int64_t>((rows + groups - 1) / groups, 148 * per_sm));
}

template <class Args, class... More>
cudaError_t launch(void (*kern)(Args, More...), const Args &a, int64_t grid, int nt, int smem, cudaStream_t st, More... more) {
    if (smem > 40000) {
        cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (e != cudaSuccess) return e;
    }
    kern<<<(unsigned)grid, nt, smem, st>>>(a, more...);
    return cudaGetLastError();
}

// The group and the elements per thread for a width: as few threads as hold it
// with MOST elements each, a warp at least.  Forward MOST is 64 bytes with VEC
// (16384 x 4096 bf16: 45 us, with 32 bytes 49); backward 16 elements, whose
// gain and sums take 48 registers (65536 x 1024 bf16: 32 elements take 95 us, 16 73).
template <class T>
constexpr int forward_vals(bool vec) {
    return vec ? 64 / (int)sizeof(T) : ONE_VALS;
}
template <class T, bool VEC, int MOST, class F>
cudaError_t with_group(int width, F &&f) {
    constexpr int N = Vec<T>::N;
    using std::integral_constant;
    auto go = [&](auto g, auto vals) { return f(g, vals); };
    if constexpr (VEC) {
        if (width <= 32 * N) return go(integral_constant<int, 32>(), integral_constant<int, N>());
        if (2 * N < MOST && width <= 64 * N) return go(integral_constant<int, 32>(), integral_constant<int, 2 * N>());
    }
    integral_constant<int, MOST> vals;
    if (width <= 32 * MOST) return go(integral_constant<int, 32>(), vals);
    if (width <= 64 * MOST) return go(integral_constant<int, 64>(), vals);
    if (width <= 128 * MOST) return go(integral_constant<int, 128>(), vals);
    if (width <= 256 * MOST) return go(integral_constant<int, 256>(), vals);
    return go(integral_constant<int, 512>(), vals);
}

template <class T, bool VEC>
cudaError_t forward_v(const NormArgs &a, cudaStream_t st) {
    return with_group<T, VEC, forward_vals<T>(VEC)>(a.width, [&](auto g, auto vals) {
        constexpr int G = decltype(g)::value, VALS = decltype(vals)::value, NT = G > NM_NT ? G : NM_NT;
        constexpr int smem = RowQueue<T, G, VALS, VEC, NT, FWD_DEPTH, 1>::BYTES;
        return launch(norm_rows_k<T, G, VALS, VEC>, a, blocks(a.rows, NT / G, NT > NM_NT ? 1 : 2), NT, smem, st);
    });
}
template <class T>
cudaError_t forward(const NormArgs &a, cudaStream_t st) {
    const bool vec = a.width % Vec<T>::N == 0 && aligned16(a.x, a.x_stride, sizeof(T)) && aligned16(a.y, a.y_stride, sizeof(T));
    if (a.width > 512 * forward_vals<T>(vec)) {
        if (!vec) {
            norm_wide_rows_k<T, false><<<(unsigned)a.rows, WIDE_NT, 0, st>>>(a, 0);
            return cudaGetLastError();
        }
        const int keep = std::min(a.width / Vec<T>::N, WIDE_KEEP / 16);
        return launch(norm_wide_rows_k<T, true>, a, a.rows, WIDE_NT, keep * 16, st, keep);
    }
    return vec ? forward_v<T, true>(a, st) : forward_v<T, false>(a, st);
}

// The partial rows of dgain and dbias: what `blocks` gives at most.
int partial_rows(int64_t rows) { return (int)std::min<int64_t>(std::max<int64_t>(rows, 1), PARTIAL_ROWS); }

template <class T, bool VEC>
cudaError_t backward_v(const NormGradArgs &a, bool params, int64_t &parts, cudaStream_t st) {
    return with_group<T, VEC, ONE_VALS>(a.width, [&](auto g, auto vals) {
        constexpr int G = decltype(g)::value, VALS = decltype(vals)::value, NT = G > NM_NT ? G : NM_NT, GROUPS = NT / G;
        parts = blocks(a.rows, GROUPS, NT > NM_NT ? 1 : 2);
        const int join = params && GROUPS > 1 ? GROUPS * 2 * a.width * (int)sizeof(float) : 0;
        const int smem = std::max(join, RowQueue<T, G, VALS, VEC, NT, BWD_DEPTH, 2>::BYTES);
        return params ? launch(norm_backward_k<T, G, VALS, VEC, true>, a, parts, NT, smem, st)
                      : launch(norm_backward_k<T, G, VALS, VEC, false>, a, parts, NT, smem, st);
    });
}

template <class T>
cudaError_t backward(const NormGradArgs &a, cudaStream_t st) {
    const bool params = a.dgain || a.dbias;
    int64_t parts = 0;
    const bool vec = a.width % Vec<T>::N == 0 && aligned16(a.x, a.x_stride, sizeof(T)) &&
                       aligned16(a.dy, a.dy_stride, sizeof(T)) && (!a.dx || aligned16(a.dx, a.dx_stride, sizeof(T)));
    if (a.rows && a.width <= 512 * ONE_VALS) {
        cudaError_t e = vec ? backward_v<T, true>(a, params, parts, st) : backward_v<T, false>(a, params, parts, st);
        if (e != cudaSuccess) return e;
    } else if (a.rows) {
        // The parameters' sums first: dx may be the array of dy.
        if (params) {
            parts = std::min<int64_t>(a.rows, 64);
            const unsigned cols = (unsigned)((a.width / (vec ? Vec<T>::N : 1) + NM_NT - 1) / NM_NT);
            if (vec)
                norm_wide_param_k<T, true><<<dim3(cols, (unsigned)parts), NM_NT, 0, st>>>(a);
            else
                norm_wide_param_k<T, false><<<dim3(cols, (unsigned)parts), NM_NT, 0, st>>>(a);
            if (cudaError_t e = cudaGetLastError()) return e;
        }
        if (a.dx && vec) {
            const int keep = std::min(a.width / Vec<T>::N, WIDE_KEEP / 16);
            if (cudaError_t e = launch(norm_wide_dx_k<T, true>, a, a.rows, WIDE_NT, 2 * keep * 16, st, keep)) return e;
        } else if (a.dx) {
            norm_wide_dx_k<T, false><<<(unsigned)a.rows, WIDE_NT, 0, st>>>(a, 0);
            if (cudaError_t e = cudaGetLastError()) return e;
        }
    }
    if (params) {
        norm_param_sum_k<<<(unsigned)((2 * (int64_t)a.width + 31) / 32), 32 * SUM_LANES, 0, st>>>(a, (int)parts);
        return cudaGetLastError();
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
