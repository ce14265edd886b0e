// norm.cu -- layer norm and RMSNorm of rows, and their gradients
// (include/noetic/head.h).
//
// Rows of up to NM_WIDE elements are taken by groups of G threads (a warp to
// 512 threads), NM_VALS elements to a thread, which stay in registers from the
// one load of the row to its one store: the mean and then the sum of squared
// differences from it are two reductions over registers, not two passes over
// memory.  A block walks rows blockIdx, blockIdx + gridDim, ... so that the
// gain, the bias and (backward) the sums for dgain and dbias stay in registers
// too, and the next row is on its way while the present one is worked on.  All
// of it is bound by HBM.  Wider rows take one block per row and read it again
// from L2.

#include <algorithm>

#include "nk_head.cuh"
#include "nk_head.h"

namespace nk {

namespace {

constexpr int NM_NT = 256;
constexpr int NM_VALS = 16;
constexpr int NM_WIDE = 8192;
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

// Where a thread's elements lie: with VEC, NM_VALS / N vectors of N elements, G
// vectors apart; else single elements, G apart.
template <class T, int G, bool VEC>
struct Place {
    static constexpr int N = VEC ? Vec<T>::N : 1;
    static constexpr int LOADS = NM_VALS / N;
    static __device__ __forceinline__ int at(int lane, int l) { return (l * G + lane) * N; }
};

// A thread's part of one row as it lies in memory.
template <class T, int G, bool VEC>
struct RowPart {
    using P = Place<T, G, VEC>;
    uint4 raw[VEC ? P::LOADS : 1];
    T one[VEC ? 1 : P::LOADS];

    __device__ __forceinline__ void load(const T *row, int lane, int width, bool real) {
#pragma unroll
        for (int l = 0; l < P::LOADS; ++l) {
            const int e = P::at(lane, l);
            if constexpr (VEC)
                raw[l] = real && e < width ? load16_rw(row + e) : make_uint4(0, 0, 0, 0);
            else
                one[l] = real && e < width ? row[e] : from_f32<T>(0.0f);
        }
    }
    __device__ __forceinline__ void get(float (&x)[NM_VALS]) const {
#pragma unroll
        for (int l = 0; l < P::LOADS; ++l) {
            if constexpr (VEC) {
                float v[P::N];
                unpack<T>(raw[l], v);
#pragma unroll
                for (int i = 0; i < P::N; ++i) x[l * P::N + i] = v[i];
            } else {
                x[l] = to_f32(one[l]);
            }
        }
    }
    static __device__ __forceinline__ void store(T *row, int lane, int width, const float (&x)[NM_VALS]) {
#pragma unroll
        for (int l = 0; l < P::LOADS; ++l) {
            const int e = P::at(lane, l);
            if (e >= width) continue;
            if constexpr (VEC) {
                float v[P::N];
#pragma unroll
                for (int i = 0; i < P::N; ++i) v[i] = x[l * P::N + i];
                store16(row + e, pack<T>(v));
            } else {
                row[e] = from_f32<T>(x[l]);
            }
        }
    }
};

// The rows that a thread will work on next: with VEC in its own places of a
// ring in shared memory, DEPTH rows on their way by asynchronous copies (no
// barrier: a thread reads only what it copied); else one row in registers.
template <class T, int G, bool VEC, int NT, int DEPTH, int ARRAYS>
struct RowQueue {
    using P = Place<T, G, VEC>;
    static constexpr int BYTES = VEC ? DEPTH * ARRAYS * P::LOADS * NT * 16 : 0;
    RowPart<T, G, VEC> next[ARRAYS];
    uint4 *ring;  // [DEPTH][ARRAYS][LOADS][NT]
    int at = 0;

    __device__ __forceinline__ void push(const T *const (&rows)[ARRAYS], int slot, int lane, int width, bool real) {
#pragma unroll
        for (int k = 0; k < ARRAYS; ++k) {
            if constexpr (VEC) {
#pragma unroll
                for (int l = 0; l < P::LOADS; ++l)
                    if (real && P::at(lane, l) < width)
                        copy_async16(ring + ((slot * ARRAYS + k) * P::LOADS + l) * NT + threadIdx.x, rows[k] + P::at(lane, l));
            } else {
                next[k].load(rows[k], lane, width, real);
            }
        }
        if constexpr (VEC) copy_commit();
    }
    // The row pushed DEPTH pushes ago (VEC) or last.
    __device__ __forceinline__ void front(int k, int lane, int width, bool real, float (&x)[NM_VALS]) {
        if constexpr (VEC) {
#pragma unroll
            for (int l = 0; l < P::LOADS; ++l) {
                float v[P::N];
                unpack<T>(real && P::at(lane, l) < width ? ring[((at * ARRAYS + k) * P::LOADS + l) * NT + threadIdx.x]
                                                         : make_uint4(0, 0, 0, 0), v);
#pragma unroll
                for (int i = 0; i < P::N; ++i) x[l * P::N + i] = v[i];
            }
        } else {
            next[k].get(x);
        }
    }
};

// A thread's part of an f32 vector of the width (null: `other`).
template <class T, int G, bool VEC>
__device__ __forceinline__ void column_part(const float *p, float other, int lane, int width, float (&x)[NM_VALS]) {
    using P = Place<T, G, VEC>;
#pragma unroll
    for (int l = 0; l < P::LOADS; ++l) {
        const int e = P::at(lane, l);
#pragma unroll
        for (int i = 0; i < P::N; ++i) x[l * P::N + i] = e < width ? (p ? p[e + i] : other) : 0.0f;
    }
}

// ---------------------------------------------------------------- forward
template <class T, int G, bool VEC>
__global__ void __launch_bounds__(G > NM_NT ? G : NM_NT, G > NM_NT ? 1 : 3) norm_rows_k(NormArgs a) {
    using P = Place<T, G, VEC>;
    constexpr int NT = G > NM_NT ? G : NM_NT, GROUPS = NT / G;
    __shared__ float red[2][32];
    const int lane = threadIdx.x % G, group = threadIdx.x / G;
    const float inv_n = 1.0f / (float)a.width;
    float gain[NM_VALS], bias[NM_VALS];
    extern __shared__ uint4 ring[];
    RowQueue<T, G, VEC, NT, FWD_DEPTH, 1> queue;
    queue.ring = ring;
    constexpr int AHEAD = VEC ? FWD_DEPTH : 1;
    const int64_t step = (int64_t)gridDim.x * GROUPS;
    int64_t r = (int64_t)blockIdx.x * GROUPS + group;
    auto push = [&](int64_t q, int slot) {
        const T *const rows[1] = {(const T *)a.x + q * a.x_stride};
        queue.push(rows, slot, lane, a.width, q < a.rows);
    };
    for (int k = 0; k < AHEAD; ++k) push(r + k * step, k);
    if constexpr (VEC) {
        column_part<T, G, VEC>(a.gain, 1.0f, lane, a.width, gain);
        column_part<T, G, VEC>(a.bias, 0.0f, lane, a.width, bias);
    }
    // Every group takes the same number of turns: the reductions hold barriers.
    const int64_t turns = (a.rows - (int64_t)blockIdx.x * GROUPS + step - 1) / step;
    for (int64_t i = 0; i < turns; ++i, r += step) {
        const bool real = r < a.rows;
        float x[NM_VALS];
        if constexpr (VEC) copy_wait<FWD_DEPTH - 1>();
        queue.front(0, lane, a.width, real, x);
        push(r + AHEAD * step, queue.at);
        queue.at = queue.at + 1 == AHEAD ? 0 : queue.at + 1;
        float mean = 0.0f;
        if (!a.rms) {
            float s = 0.0f;
#pragma unroll
            for (int j = 0; j < NM_VALS; ++j) s += x[j];
            mean = group_sum<G>(s, red[0]) * inv_n;
        }
        float v = 0.0f;
#pragma unroll
        for (int l = 0; l < P::LOADS; ++l)
            if (P::at(lane, l) < a.width) {
#pragma unroll
                for (int j = 0; j < P::N; ++j) {
                    float &d = x[l * P::N + j];
                    d -= mean;
                    v = fmaf(d, d, v);
                }
            }
        const float rstd = 1.0f / sqrtf(fmaf(group_sum<G>(v, red[1]), inv_n, a.eps));
        if (G > 32 && a.rms) __syncthreads();  // red[1] again in the next turn
        if (!real) continue;
        if constexpr (!VEC) {  // from L1 for every row: the loads' sixteen registers are taken
            column_part<T, G, VEC>(a.gain, 1.0f, lane, a.width, gain);
            column_part<T, G, VEC>(a.bias, 0.0f, lane, a.width, bias);
        }
#pragma unroll
        for (int j = 0; j < NM_VALS; ++j) x[j] = fmaf(x[j] * rstd, gain[j], bias[j]);
        RowPart<T, G, VEC>::store((T *)a.y + r * a.y_stride, lane, a.width, x);
        if (lane == 0) {
            if (a.mean) a.mean[r] = mean;
            if (a.rstd) a.rstd[r] = rstd;
        }
    }
}

// Rows wider than NM_WIDE.
template <class T>
__global__ void __launch_bounds__(NM_NT) norm_wide_rows_k(NormArgs a) {
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

// ---------------------------------------------------------------- backward
// dx of the rows, and with PARAMS this block's sums for dgain and dbias: its
// groups' registers joined in shared memory in their order, then one row of
// the workspace per block.
template <class T, int G, bool VEC, bool PARAMS>
__global__ void __launch_bounds__(G > NM_NT ? G : NM_NT, G > NM_NT ? 1 : 2) norm_backward_k(NormGradArgs a) {
    using P = Place<T, G, VEC>;
    constexpr int NT = G > NM_NT ? G : NM_NT, GROUPS = NT / G;
    __shared__ float2 red[2][32];
    extern __shared__ uint4 ring[];
    float *joined = (float *)ring;  // [2][width], when the rows are done
    const int lane = threadIdx.x % G, group = threadIdx.x / G;
    const float inv_n = 1.0f / (float)a.width;
    float gain[NM_VALS], dg[NM_VALS], db[NM_VALS];
#pragma unroll
    for (int j = 0; j < NM_VALS; ++j) dg[j] = db[j] = 0.0f;
    RowQueue<T, G, VEC, NT, BWD_DEPTH, 2> queue;
    queue.ring = ring;
    constexpr int AHEAD = VEC ? BWD_DEPTH : 1;
    const int64_t step = (int64_t)gridDim.x * GROUPS;
    int64_t r = (int64_t)blockIdx.x * GROUPS + group;
    auto push = [&](int64_t q, int slot) {
        const T *const rows[2] = {(const T *)a.x + q * a.x_stride, (const T *)a.dy + q * a.dy_stride};
        queue.push(rows, slot, lane, a.width, q < a.rows);
    };
    float next_mean, next_rstd;
    auto stats = [&](int64_t q) {
        next_mean = q < a.rows && !a.rms ? a.mean[q] : 0.0f;
        next_rstd = q < a.rows ? a.rstd[q] : 0.0f;
    };
    for (int k = 0; k < AHEAD; ++k) push(r + k * step, k);
    stats(r);
    if constexpr (VEC) column_part<T, G, VEC>(a.gain, 1.0f, lane, a.width, gain);
    const int64_t turns = (a.rows - (int64_t)blockIdx.x * GROUPS + step - 1) / step;
    for (int64_t i = 0; i < turns; ++i, r += step) {
        float h[NM_VALS], c[NM_VALS];
        if constexpr (VEC) copy_wait<BWD_DEPTH - 1>();
        queue.front(0, lane, a.width, r < a.rows, h);
        queue.front(1, lane, a.width, r < a.rows, c);
        const float mean = next_mean, rstd = next_rstd;
        push(r + AHEAD * step, queue.at);
        queue.at = queue.at + 1 == AHEAD ? 0 : queue.at + 1;
        stats(r + step);
        if constexpr (!VEC) column_part<T, G, VEC>(a.gain, 1.0f, lane, a.width, gain);
        float2 s = make_float2(0.0f, 0.0f);
#pragma unroll
        for (int j = 0; j < NM_VALS; ++j) {
            // Beyond the width c is 0, and h does not count.
            h[j] = (h[j] - mean) * rstd;
            if (PARAMS) {
                dg[j] = fmaf(c[j], h[j], dg[j]);
                db[j] += c[j];
            }
            c[j] *= gain[j];
            s.x += c[j];
            s.y = fmaf(c[j], h[j], s.y);
        }
        if (!a.dx) continue;
        s = group_sum2<G>(s, red[i & 1]);
        const float mc = a.rms ? 0.0f : s.x * inv_n, mch = s.y * inv_n;
        if (r < a.rows) {
#pragma unroll
            for (int j = 0; j < NM_VALS; ++j) h[j] = rstd * (c[j] - mc - h[j] * mch);
            RowPart<T, G, VEC>::store((T *)a.dx + r * a.dx_stride, lane, a.width, h);
        }
    }
    if constexpr (PARAMS) {
        float *w = a.workspace + (int64_t)blockIdx.x * 2 * a.width;
        if (GROUPS > 1) __syncthreads();
        for (int g = 0; g < GROUPS; ++g) {
            if (group == g) {
                float *to = g == GROUPS - 1 ? w : joined;
#pragma unroll
                for (int l = 0; l < P::LOADS; ++l)
#pragma unroll
                    for (int j = 0; j < P::N; ++j) {
                        const int e = P::at(lane, l) + j;
                        if (e >= a.width) continue;
                        to[e] = g ? joined[e] + dg[l * P::N + j] : dg[l * P::N + j];
                        to[a.width + e] = g ? joined[a.width + e] + db[l * P::N + j] : db[l * P::N + j];
                    }
            }
            if (g + 1 < GROUPS) __syncthreads();
        }
    }
}

template <class T>
__global__ void __launch_bounds__(NM_NT) norm_wide_dx_k(NormGradArgs a) {
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
__global__ void __launch_bounds__(NM_NT) norm_wide_param_k(NormGradArgs a) {
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

template <class Args>
cudaError_t launch(void (*kern)(Args), const Args &a, int64_t grid, int nt, int smem, cudaStream_t st) {
    if (smem > 40000) {
        cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (e != cudaSuccess) return e;
    }
    kern<<<(unsigned)grid, nt, smem, st>>>(a);
    return cudaGetLastError();
}

template <class T, int G, bool VEC>
cudaError_t forward_g(const NormArgs &a, cudaStream_t st) {
    constexpr int NT = G > NM_NT ? G : NM_NT;
    constexpr int smem = RowQueue<T, G, VEC, NT, FWD_DEPTH, 1>::BYTES;
    return launch(norm_rows_k<T, G, VEC>, a, blocks(a.rows, NT / G, NT > NM_NT ? 1 : 3), NT, smem, st);
}
template <class T, bool VEC>
cudaError_t forward_v(const NormArgs &a, cudaStream_t st) {
    if (a.width <= 32 * NM_VALS) return forward_g<T, 32, VEC>(a, st);
    if (a.width <= 64 * NM_VALS) return forward_g<T, 64, VEC>(a, st);
    if (a.width <= 128 * NM_VALS) return forward_g<T, 128, VEC>(a, st);
    if (a.width <= 256 * NM_VALS) return forward_g<T, 256, VEC>(a, st);
    return forward_g<T, 512, VEC>(a, st);
}
template <class T>
cudaError_t forward(const NormArgs &a, cudaStream_t st) {
    if (a.width > NM_WIDE) {
        norm_wide_rows_k<T><<<(unsigned)a.rows, NM_NT, 0, st>>>(a);
        return cudaGetLastError();
    }
    const bool vec = a.width % Vec<T>::N == 0 && aligned16(a.x, a.x_stride, sizeof(T)) && aligned16(a.y, a.y_stride, sizeof(T));
    return vec ? forward_v<T, true>(a, st) : forward_v<T, false>(a, st);
}

// The partial rows of dgain and dbias: what `blocks` gives at most.
int partial_rows(int64_t rows) { return (int)std::min<int64_t>(std::max<int64_t>(rows, 1), PARTIAL_ROWS); }

template <class T, int G, bool VEC>
cudaError_t backward_g(const NormGradArgs &a, bool params, int64_t &parts, cudaStream_t st) {
    constexpr int NT = G > NM_NT ? G : NM_NT, GROUPS = NT / G;
    parts = blocks(a.rows, GROUPS, NT > 256 ? 1 : 2);
    const int join = params && GROUPS > 1 ? 2 * a.width * (int)sizeof(float) : 0;
    const int smem = std::max(join, RowQueue<T, G, VEC, NT, BWD_DEPTH, 2>::BYTES);
    return params ? launch(norm_backward_k<T, G, VEC, true>, a, parts, NT, smem, st)
                  : launch(norm_backward_k<T, G, VEC, false>, a, parts, NT, smem, st);
}
template <class T, bool VEC>
cudaError_t backward_v(const NormGradArgs &a, bool params, int64_t &parts, cudaStream_t st) {
    if (a.width <= 32 * NM_VALS) return backward_g<T, 32, VEC>(a, params, parts, st);
    if (a.width <= 64 * NM_VALS) return backward_g<T, 64, VEC>(a, params, parts, st);
    if (a.width <= 128 * NM_VALS) return backward_g<T, 128, VEC>(a, params, parts, st);
    if (a.width <= 256 * NM_VALS) return backward_g<T, 256, VEC>(a, params, parts, st);
    return backward_g<T, 512, VEC>(a, params, parts, st);
}

template <class T>
cudaError_t backward(const NormGradArgs &a, cudaStream_t st) {
    const bool params = a.dgain || a.dbias;
    int64_t parts = 0;
    if (a.rows && a.width <= NM_WIDE) {
        bool vec = a.width % Vec<T>::N == 0 && aligned16(a.x, a.x_stride, sizeof(T)) &&
                   aligned16(a.dy, a.dy_stride, sizeof(T)) && (!a.dx || aligned16(a.dx, a.dx_stride, sizeof(T)));
        cudaError_t e = vec ? backward_v<T, true>(a, params, parts, st) : backward_v<T, false>(a, params, parts, st);
        if (e != cudaSuccess) return e;
    } else if (a.rows) {
        // The parameters' sums first: dx may be the array of dy.
        if (params) {
            parts = std::min<int64_t>(a.rows, 64);
            norm_wide_param_k<T><<<dim3((unsigned)((a.width + NM_NT - 1) / NM_NT), (unsigned)parts), NM_NT, 0, st>>>(a);
            if (cudaError_t e = cudaGetLastError()) return e;
        }
        if (a.dx) norm_wide_dx_k<T><<<(unsigned)a.rows, NM_NT, 0, st>>>(a);
        if (cudaError_t e = cudaGetLastError()) return e;
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
