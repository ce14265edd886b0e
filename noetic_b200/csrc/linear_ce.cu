// linear_ce.cu -- softmax cross entropy of logits z = x w^T that are not kept,
// and its gradients (the logits product and softmax_ce of Lm::loss,
// model.rs:209-234, autograd.rs:579-624).
//
//   loss = (m - z_t) + log s,  m = max_j z_j,  s = sum_j exp(z_j - m)
//   G = grad_scale row_weight (exp(z - m - log s) - [t]),  dx = G w,  dw = G^T x
//
// Forward: a tile of logits is reduced where it is computed, to the maximum and
// the sum of each of its rows; joining a row's tiles gives m and s.  Backward:
// the logits of a piece of the vocabulary are computed again and become G, from
// which the two products take their part; G of one piece is all that is kept.

#include <cuda.h>
#include <cudaTypedefs.h>

#include <algorithm>
#include <mutex>

#include "ce_gemm.cuh"
#include "nk_train.h"

namespace nk {

namespace {

using ce::Gemm;
using ce::Head;

constexpr uint64_t PIECE_BYTES = 256ull << 20;  // of G
// K-blocks that 16-bit outputs may take as one chain on the tensor cores.  Where all terms
// have one sign it is off by 4.3e-8 of the result for each 16 of K, all one way (65536 rows
// of f16: 1.8e-4): up to a quarter of the output's half step.
constexpr int longest_chain(bool bf16) { return bf16 ? 5632 : 704; }
// G is at most 1 before its scale: f16 keeps it down to 2^-38.
constexpr float G_SCALE = 16384.0f;

// nk_linear_ce_withhold: 1 + the Mode whose product's wait is to run out, or 0.
thread_local int g_withhold = 0;

constexpr size_t round_up(size_t n, size_t to) { return (n + to - 1) / to * to; }

// A block joins the tiles of 8 rows, in a fixed order: 32 threads a row.  row_of null:
// the rows are as the caller has them, and those without a token get zeros.
__global__ void __launch_bounds__(256) ce_join_k(LinearCeArgs a, const Head *head, const uint32_t *row_of, const float2 *part,
                                                 int64_t part_ld, const float *zt, int tiles) {
    pdl_trigger();
    pdl_wait();
    __shared__ float2 red[8][33];
    const int at = threadIdx.x & 7, slot = threadIdx.x >> 3, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t i = (int64_t)blockIdx.x * 8 + at, n = row_of ? (int64_t)head->live : a.rows;
    if ((int64_t)blockIdx.x * 8 >= n) return;
    float m = -INFINITY, s = 0.0f;
    if (i < n)
        for (int t0 = slot; t0 < tiles; t0 += 256) {
            float2 q[8];  // (eight loads at once: one after the other they took most of the time)
            float now = m;
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                q[u] = t0 + 32 * u < tiles ? part[(t0 + 32 * u) * part_ld + i] : make_float2(-INFINITY, 0.0f);
                now = fmaxf(now, q[u].x);
            }
            const float base = now == -INFINITY ? 0.0f : now;
            s *= ex2((m - base) * LOG2E);
#pragma unroll
            for (int u = 0; u < 8; ++u) s = fmaf(q[u].y, ex2((q[u].x - base) * LOG2E), s);
            m = now;
        }
    red[at][slot] = make_float2(m, s);
    __syncthreads();
    // Warp w finishes row w.
    const float2 q = red[warp][lane];
    float top = q.x;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    s = warp_sum(q.y * ex2((q.x - (top == -INFINITY ? 0.0f : top)) * LOG2E));
    const int64_t mine = (int64_t)blockIdx.x * 8 + warp;
    if (lane != 0 || mine >= n) return;
    const int64_t row = row_of ? row_of[mine] : mine;
    float loss = 0.0f, ls = 0.0f;
    if (row_of || a.targets[row] < (uint32_t)a.vocab) {
        ls = logf(s);
        loss = (top - zt[mine]) + ls;
        // Not a number, or a wait in the product ran out.
        if (!(isfinite(loss) && isfinite(ls)) || (head && head->err)) top = ls = loss = NAN;
    } else {
        top = 0.0f;
    }
    if (a.loss) a.loss[row] = loss;
    if (a.stats) a.stats[2 * row] = top, a.stats[2 * row + 1] = ls;
}

// ---------------------------------------------------------------- few rows
// Where the product is small the bound is reading w once (or launches): f32 fmas on
// the CUDA cores, 8 rows of x in shared memory, and a warp that multiplies them with
// COLS rows of w at a time, straight from memory.
constexpr int FEW_WARPS = 8;
constexpr int COLS = 4;

// N sums over the warp at once: lane l ends with that of value l % N (N a power of
// two up to 32), for N - 1 + log2(32 / N) shuffles.
template <int N>
__device__ __forceinline__ float warp_sums(float (&v)[N]) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int h = N / 2; h >= 1; h >>= 1) {
        const bool up = lane & h;
#pragma unroll
        for (int i = 0; i < h; ++i) {
            const float keep = up ? v[i + h] : v[i], give = up ? v[i] : v[i + h];
            v[i] = keep + __shfl_xor_sync(0xffffffffu, give, h);
        }
    }
    float s = v[0];
#pragma unroll
    for (int o = N; o < 32; o <<= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    return s;
}

template <class T, int R>
__global__ void __launch_bounds__(32 * FEW_WARPS, R <= 2 ? 4 : 2) ce_few_k(LinearCeArgs a, float2 *part, int64_t part_ld, float *zt) {
    pdl_trigger();
    pdl_wait();
    constexpr int PER = 16 / (int)sizeof(T), N = R * COLS;
    extern __shared__ __align__(16) float xs[];  // [R][width up to whole vectors]
    __shared__ float2 red[FEW_WARPS][R];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, d = a.width, whole = d / PER, ld = (d + PER - 1) / PER * PER;
    const int64_t r0 = (int64_t)blockIdx.y * R;
    for (int r = warp; r < R; r += FEW_WARPS) {
        // (A row without a token is not read.)
        const bool in = r0 + r < a.rows && a.targets[r0 + r] < (uint32_t)a.vocab;
        const T *x = (const T *)a.x + (r0 + r) * a.x_stride;
#pragma unroll 8
        for (int k = lane; k < ld; k += 32) xs[r * ld + k] = in && k < d ? to_f32(x[k]) : 0.0f;
    }
    __syncthreads();
    // The lane's own row and column of w among the N products.
    const int mine = lane % N, my_row = mine / COLS, my_col = mine % COLS;
    const uint32_t target = r0 + my_row < a.rows ? a.targets[r0 + my_row] : NO_TOKEN;
    float m = -INFINITY, s = 0.0f;
    const int step = gridDim.x * FEW_WARPS * COLS;
    for (int v0 = (blockIdx.x * FEW_WARPS + warp) * COLS; v0 < a.vocab; v0 += step) {
        float acc[N] = {};
        const T *w[COLS];
#pragma unroll
        for (int c = 0; c < COLS; ++c) w[c] = (const T *)a.w + (int64_t)min(v0 + c, a.vocab - 1) * a.w_stride;
#pragma unroll(R >= 8 ? 1 : 2)
        for (int u = lane; u < whole; u += 32) {
            uint4 q[COLS];
#pragma unroll
            for (int c = 0; c < COLS; ++c) q[c] = __ldg(reinterpret_cast<const uint4 *>(w[c] + u * PER));
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int e = 0; e < PER; e += 4) {
                    const float4 x = *reinterpret_cast<const float4 *>(&xs[r * ld + u * PER + e]);
#pragma unroll
                    for (int c = 0; c < COLS; ++c) {
                        const T *y = reinterpret_cast<const T *>(&q[c]) + e;
                        float &t = acc[r * COLS + c];
                        t = fmaf(x.x, to_f32(y[0]), t);
                        t = fmaf(x.y, to_f32(y[1]), t);
                        t = fmaf(x.z, to_f32(y[2]), t);
                        t = fmaf(x.w, to_f32(y[3]), t);
                    }
                }
        }
        if (lane < d - whole * PER) {
            const int k = whole * PER + lane;
#pragma unroll
            for (int c = 0; c < COLS; ++c) {
                const float y = to_f32(w[c][k]);
#pragma unroll
                for (int r = 0; r < R; ++r) acc[r * COLS + c] = fmaf(xs[r * ld + k], y, acc[r * COLS + c]);
            }
        }
        const float z = warp_sums<N>(acc);
        const int col = v0 + my_col;
        if (col < a.vocab && lane < N) {
            if ((uint32_t)col == target) zt[r0 + my_row] = z;
            const float now = fmaxf(m, z), base = now == -INFINITY ? 0.0f : now;
            s = fmaf(s, ex2((m - base) * LOG2E), ex2((z - base) * LOG2E));
            m = now;
        }
    }
    // The lanes of a row (COLS neighbours), then the warps.
#pragma unroll
    for (int o = COLS / 2; o >= 1; o >>= 1) {
        const float m2 = __shfl_xor_sync(0xffffffffu, m, o), s2 = __shfl_xor_sync(0xffffffffu, s, o);
        const float now = fmaxf(m, m2), base = now == -INFINITY ? 0.0f : now;
        s = s * ex2((m - base) * LOG2E) + s2 * ex2((m2 - base) * LOG2E);
        m = now;
    }
    if (lane < N && my_col == 0) red[warp][my_row] = make_float2(m, s);
    __syncthreads();
    if (threadIdx.x < R && r0 + threadIdx.x < a.rows) {
        m = -INFINITY, s = 0.0f;
        for (int w = 0; w < FEW_WARPS; ++w) {
            const float2 q = red[w][threadIdx.x];
            const float now = fmaxf(m, q.x), base = now == -INFINITY ? 0.0f : now;
            s = s * ex2((m - base) * LOG2E) + q.y * ex2((q.x - base) * LOG2E);
            m = now;
        }
        part[blockIdx.x * part_ld + r0 + threadIdx.x] = make_float2(m, s);
    }
}

// ---------------------------------------------------------------- rows that count
// What the rows that count have, in their order.
struct Index {
    Head *head;
    uint32_t *row_of, *place;  // the row of each that counts; the place of each row, or NO_TOKEN
    uint32_t *target;
    float2 *stats;   // backward
    float *weight;   // backward
};

// One block, 8192 rows at a time: a thread looks at 8, and a prefix sum of the warps'
// counts gives each its place.  (Neighbouring threads take neighbouring rows: with 8
// rows in a row to a thread this took 31 us of 8192 rows.)
__global__ void __launch_bounds__(1024) ce_index_k(LinearCeArgs a, Index ix, bool backward) {
    pdl_trigger();
    pdl_wait();
    __shared__ uint32_t counts[8 * 32];
    __shared__ uint32_t all;
    __shared__ float tops[32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    uint32_t carry = 0;
    float top = 0.0f;
    for (int64_t r0 = 0; r0 < a.rows; r0 += 8192) {
        uint32_t t[8], votes[8];
        float w[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int64_t r = r0 + i * 1024 + tid;
            t[i] = r < a.rows ? a.targets[r] : NO_TOKEN;
            w[i] = backward && a.row_weight && r < a.rows ? a.row_weight[r] : 1.0f;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const bool counts_in = t[i] < (uint32_t)a.vocab && w[i] != 0.0f;
            // (A weight that is not finite breaks its own row alone.)
            if (counts_in && isfinite(w[i])) top = fmaxf(top, fabsf(w[i]));
            votes[i] = __ballot_sync(0xffffffffu, counts_in);
            if (lane == 0) counts[i * 32 + warp] = __popc(votes[i]);
        }
        __syncthreads();
        if (warp == 0) {
            uint32_t n[8], sum = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) n[i] = counts[lane * 8 + i], sum += n[i];
            uint32_t upto = sum;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t v = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= o) upto += v;
            }
            uint32_t before = upto - sum;
#pragma unroll
            for (int i = 0; i < 8; ++i) counts[lane * 8 + i] = before, before += n[i];
            if (lane == 31) all = upto;
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int64_t r = r0 + i * 1024 + tid;
            if (r >= a.rows) continue;
            if (!(votes[i] >> lane & 1)) {
                ix.place[r] = NO_TOKEN;
                if (!backward) {
                    if (a.loss) a.loss[r] = 0.0f;
                    if (a.stats) a.stats[2 * r] = a.stats[2 * r + 1] = 0.0f;
                }
                continue;
            }
            const uint32_t at = carry + counts[i * 32 + warp] + __popc(votes[i] & ((1u << lane) - 1));
            ix.place[r] = at;
            ix.row_of[at] = (uint32_t)r;
            ix.target[at] = t[i];
            if (backward) {
                ix.stats[at] = make_float2(a.in_stats[2 * r], a.in_stats[2 * r + 1]);
                ix.weight[at] = w[i];
            }
        }
        carry += all;
        __syncthreads();
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (lane == 0) tops[warp] = top;
    __syncthreads();
    if (warp == 0) {
        top = tops[lane];
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        if (lane == 0) *ix.head = Head{0u, carry, backward ? top : 1.0f, 0u, 0u};
    }
}

// The largest finite |x| of a warp's row, on every lane.
__device__ __forceinline__ float row_absmax(const float *p, int d) {
    const int lane = threadIdx.x & 31;
    float top = 0.0f;
    int c = 0;
    if (((uintptr_t)p & 15) == 0) {
        c = d & ~3;
        for (int i0 = lane * 4; i0 < c; i0 += 1024) {
            float4 q[8];
#pragma unroll
            for (int u = 0; u < 8; ++u)
                q[u] = i0 + u * 128 < c ? *reinterpret_cast<const float4 *>(p + i0 + u * 128) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const float v[4] = {q[u].x, q[u].y, q[u].z, q[u].w};
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (isfinite(v[e])) top = fmaxf(top, fabsf(v[e]));
            }
        }
    }
    for (int i = c + lane; i < d; i += 32)
        if (isfinite(p[i])) top = fmaxf(top, fabsf(p[i]));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    return top;
}

// Rows to lay out for the products.
struct Rows {
    const void *src;
    int64_t stride, rows;
    const uint32_t *place;  // where each goes, or NO_TOKEN (nullable: its own place)
    void *dst;
    int64_t part;           // f32: from the high parts to the low ones, in elements
    int fill;               // rows of zeros behind the last that has a place, within `room`
    int64_t room;
    void *zero;             // nullable: where rows without a place become zeros (dx)
    int64_t zero_stride;
    uint32_t *top;          // f32: bits of the largest finite number, for one scale; null: a scale for each row
    float *undo;            // f32: what undoes the scale, or those of the rows
};

// f32: the largest finite number of the rows of x that count, and of w.
__global__ void __launch_bounds__(256) ce_absmax_k(Rows x, Rows w, int d) {
    pdl_trigger();
    pdl_wait();
    float top[2] = {0.0f, 0.0f};
    const int64_t step = (int64_t)gridDim.x * 8;
    for (int64_t r = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); r < x.rows + w.rows; r += step) {
        const bool of_w = r >= x.rows;
        if (!of_w && x.place[r] == NO_TOKEN) continue;
        const float t = row_absmax(of_w ? (const float *)w.src + (r - x.rows) * w.stride : (const float *)x.src + r * x.stride, d);
        top[of_w] = fmaxf(top[of_w], t);
    }
    // (Bits of numbers that are not negative are in their order; a maximum does not
    // depend on who comes first.)
    if ((threadIdx.x & 31) == 0) {
        if (top[0] > 0.0f) atomicMax(x.top, __float_as_uint(top[0]));
        if (top[1] > 0.0f) atomicMax(w.top, __float_as_uint(top[1]));
    }
}

// The power of two that brings the largest of a matrix or a row to [2^14, 2^15).
__device__ __forceinline__ float part_scale(float top) {
    if (!(top > 0.0f)) return 1.0f;
    return exp2f((float)min(max(14 - ilogbf(top), -126), 126));
}

// A warp's row: 16-bit elements as they are, f32 ones as two scaled f16 parts, high
// and low, 22 bits together; from a 128-byte line on, zeros up to ld.
template <class T>
__device__ __forceinline__ void lay_out_row(const Rows &j, const T *p, bool real, int64_t to, int d, int64_t ld) {
    const int lane = threadIdx.x & 31;
    if constexpr (sizeof(T) == 2) {
        T *o = (T *)j.dst + to * ld;
        // A row that starts within a unit of 16 bytes is read in whole units (no more of
        // them than it touches), each shifted together with the next lane's.
        const uint32_t off = (uintptr_t)p & 15, units = (off + 2 * d + 15) / 16;
        const uint4 *from = reinterpret_cast<const uint4 *>((uintptr_t)p - off);
        for (int i0 = 0; i0 < ld; i0 += 1024) {
            uint4 q4[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const uint32_t u = i0 / 8 + 32 * k + lane;
                q4[k] = real && u < units ? from[u] : make_uint4(0, 0, 0, 0);
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const uint32_t u = i0 / 8 + 32 * k + lane;
                uint4 q = q4[k];
                if (off) {  // (the warp's one row)
                    uint4 n;
                    n.x = __shfl_down_sync(0xffffffffu, q.x, 1);
                    n.y = __shfl_down_sync(0xffffffffu, q.y, 1);
                    n.z = __shfl_down_sync(0xffffffffu, q.z, 1);
                    n.w = __shfl_down_sync(0xffffffffu, q.w, 1);
                    if (lane == 31) n = real && u + 1 < units ? from[u + 1] : make_uint4(0, 0, 0, 0);
                    const uint32_t w[8] = {q.x, q.y, q.z, q.w, n.x, n.y, n.z, n.w};
                    const uint32_t words = off / 4, bits = off % 4 * 8;
                    uint32_t x[5];
#pragma unroll
                    for (int e = 0; e < 5; ++e) x[e] = words == 0 ? w[e] : words == 1 ? w[e + 1] : words == 2 ? w[e + 2] : w[min(e + 3, 7)];
                    q = make_uint4(__funnelshift_r(x[0], x[1], bits), __funnelshift_r(x[1], x[2], bits), __funnelshift_r(x[2], x[3], bits),
                                   __funnelshift_r(x[3], x[4], bits));
                }
                const int i = u * 8;
                if (i + 8 > d) {
                    T *e = reinterpret_cast<T *>(&q);
#pragma unroll
                    for (int t = 0; t < 8; ++t)
                        if (i + t >= d) e[t] = from_f32<T>(0.0f);
                }
                if (i < ld) *reinterpret_cast<uint4 *>(o + i) = q;
            }
        }
    } else {
        __half *o = (__half *)j.dst + to * ld;
        // (With a scale of its own a row is read twice, the second time from the cache.)
        const float scale = part_scale(j.top ? __uint_as_float(*j.top) : real ? row_absmax(p, d) : 0.0f);
        if (!j.top && lane == 0) j.undo[to] = 1.0f / scale;
        const bool vec = real && ((uintptr_t)p & 15) == 0;
        for (int i = lane * 8; i < ld; i += 256) {
            float v[8] = {};
            if (vec && i + 8 <= d) {
                const float4 a = *reinterpret_cast<const float4 *>(p + i), b = *reinterpret_cast<const float4 *>(p + i + 4);
                v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
            } else if (real) {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (i + e < d) v[e] = p[i + e];
            }
            uint4 hi, lo;
            __half *h = reinterpret_cast<__half *>(&hi), *l = reinterpret_cast<__half *>(&lo);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float y = v[e] * scale;
                h[e] = __float2half_rn(y);
                l[e] = __float2half_rn(isfinite(y) ? y - __half2float(h[e]) : 0.0f);
            }
            *reinterpret_cast<uint4 *>(o + i) = hi;
            *reinterpret_cast<uint4 *>(o + j.part + i) = lo;
        }
    }
}

// x (its rows that count, in their order, and rows of zeros behind them) and, where it
// has to be laid out, w (else it has no rows here).
template <class T>
__global__ void __launch_bounds__(256) ce_lay_out_k(Rows x, Rows w, int d, int64_t ld, const Head *head) {
    pdl_trigger();
    pdl_wait();
    const int lane = threadIdx.x & 31;
    if (sizeof(T) == 4 && blockIdx.x == 0 && threadIdx.x == 0 && x.top) {
        *x.undo = 1.0f / part_scale(__uint_as_float(*x.top));
        *w.undo = 1.0f / part_scale(__uint_as_float(*w.top));
    }
    const int64_t step = (int64_t)gridDim.x * 8, xs = x.rows + x.fill;
    for (int64_t r = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); r < xs + w.rows; r += step) {
        if (r >= xs) {
            lay_out_row<T>(w, (const T *)w.src + (r - xs) * w.stride, true, r - xs, d, ld);
            continue;
        }
        const bool real = r < x.rows;
        const T *p = (const T *)x.src + r * x.stride;
        int64_t to = (int64_t)head->live + (r - x.rows);
        if (real) {
            const uint32_t place = x.place[r];
            if (place == NO_TOKEN) {
                if (x.zero)
                    for (int i = lane; i < d; i += 32) ((T *)x.zero)[r * x.zero_stride + i] = from_f32<T>(0.0f);
                continue;
            }
            to = place;
        }
        if (to < x.room) lay_out_row<T>(x, p, real, to, d, ld);
    }
}

// The sums of a product whose K was split, in their order, rounded on the way out.
template <class T>
__device__ __forceinline__ void reduce(const Gemm &p, int splits) {
    const int rows = p.live_dim == 0 ? (int)p.head->live : p.M;
    const float factor = ce::out_factor(p);
    const int64_t n = (int64_t)rows * p.ld_acc / 4;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        const int64_t row = i * 4 / p.ld_acc;
        const int col = (int)(i * 4 - row * p.ld_acc);
        if (col >= p.n_valid) continue;
        const float *a = p.acc + row * p.ld_acc + col;
        float4 v = *reinterpret_cast<const float4 *>(a);
        for (int s = 1; s < splits; ++s) {
            const float4 q = *reinterpret_cast<const float4 *>(a + s * p.acc_split);
            v.x += q.x, v.y += q.y, v.z += q.z, v.w += q.w;
        }
        const float f[4] = {v.x * factor, v.y * factor, v.z * factor, v.w * factor};
        T *o = (T *)p.out + (p.out_row ? (int64_t)p.out_row[row] : row + p.out_row0) * p.out_ld + col;
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (col + j < p.n_valid) o[j] = from_f32<T>(p.out_add ? f[j] + to_f32(o[j]) : f[j]);
    }
}
template <class T, class W>
__global__ void __launch_bounds__(256) ce_reduce_k(Gemm x, int x_splits, Gemm w, int w_splits) {
    pdl_trigger();
    pdl_wait();
    if (x_splits) reduce<T>(x, x_splits);
    if (w_splits) reduce<W>(w, w_splits);
}

// ---------------------------------------------------------------- host
PFN_cuTensorMapEncodeTiled_v12000 encoder() {
    static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        void *p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            fn = (PFN_cuTensorMapEncodeTiled_v12000)p;
    });
    return fn;
}

// Boxes of 64 columns and box_rows rows of a 16-bit matrix, 128-byte swizzle.
bool make_map(CUtensorMap *map, const void *base, bool bf16, int64_t rows, int64_t cols, int64_t ld, int box_rows) {
    auto fn = encoder();
    if (!fn) return false;
    const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)ld * 2};
    const cuuint32_t box[2] = {64, (cuuint32_t)box_rows}, one[2] = {1, 1};
    return fn(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, const_cast<void *>(base),
              dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Where everything is in the workspace, and how the work is cut.
struct Plan {
    int64_t mp = 0;      // rows, up to whole tiles
    int64_t dp = 0;      // columns of laid out rows
    bool split = false;  // f32: two parts
    bool few = false;    // forward on the CUDA cores
    bool copy_w = false;
    int tiles = 0;       // partial results of a row
    int piece = 0;       // tokens of G at a time
    int64_t ldg = 0, ld_acc = 0;
    int dx_splits = 1, dw_splits = 1;
    size_t head = 0, row_of = 0, place = 0, target = 0, stats = 0, weight = 0, scales = 0, x = 0, w = 0, part = 0, zt = 0, g = 0,
           dx = 0, dw = 0, bytes = 0;
};

constexpr int PAIRS = 74;  // of 148 SMs: the workspace does not go by the device
// An item's time in K-blocks: its own, or its sums' way out, which the next item's
// K-blocks cover; and a piece's sums on their way to memory and back.
constexpr int STORE_COST = 24, SPLIT_COST = 16;
int item_cost(int64_t kblocks, bool split) { return (int)std::max<int64_t>(kblocks, STORE_COST) + 4 + (split ? SPLIT_COST : 0); }

// Pieces of K for dx and dw, of 8 K-blocks at least: those that end first where the
// two share the pairs (ce::Deal).
void pick_splits(int64_t tx, int64_t kx, int64_t tw, int64_t kw, int pairs, int &sx, int &sw) {
    static const int tries[] = {1, 2, 3, 4, 6, 8, 12, 16, 24, 32, 48, 64};
    double least = 1e300;
    sx = sw = 1;
    for (const int i : tries)
        for (const int j : tries) {
            if ((i > 1 && (kx / i < 8 || tx * i > 4 * pairs)) || (j > 1 && (kw / j < 8 || tw * j > 4 * pairs))) continue;
            const int cx = item_cost((kx + i - 1) / i, i > 1), cw = item_cost((kw + j - 1) / j, j > 1);
            const ce::Deal d((int)(tx * i), cx, (int)(tw * j), cw, pairs);
            const double q = (double)(tx * i / pairs);
            const double a = d.more ? (q + 1) * cx + (double)d.n[0] * cw : 0.0, b = q * cx + (double)d.n[1] * cw;
            const double cost = std::max(a, b);
            if (cost < least * 0.97) least = cost, sx = i, sw = j;
        }
}

// Whether the forward call takes the few rows' kernel: w's rows in whole 16-byte units,
// 8 of x within shared memory, and a product below what the other way's launches and
// (f32) its passes over w cost, about 12 us and 2.4 us a million elements of w where
// the few rows' kernel makes 12.5 million products a us.  Measured (us, this and the
// other way): f32 1 x 1024 x 32768 31 and 100, 16 rows 54 and 100, 32 rows 95 and 101,
// 64 rows 168 and 101; 96 x 768 x 16384 99 and 45; 256 x 192 x 1024 13 and 26; 512 x
// 512 x 1024 26 and 25; bf16 4 x 1024 x 32768 26 and 28, 8 rows 35 and 28; 256 x 192 x
// 1024 13 and 18, 512 x 512 x 1024 29 and 18, 32 x 512 x 8192 17 and 18.
bool few_rows(int dtype, int64_t rows, int width, int vocab, const void *w, int64_t w_stride) {
    const int es = dtype == NK_F32 ? 4 : 2;
    if (((uintptr_t)w & 15) != 0 || w_stride * es % 16 != 0 || width > 4096 || rows > 4096) return false;
    const double products = (double)rows * width * vocab;
    return dtype == NK_F32 ? products <= 1.5e8 + 30.0 * width * vocab : rows <= 4 || products <= 1e8;
}
int few_blocks(int64_t rows, int vocab) {
    const int r = rows >= 8 ? 8 : rows > 2 ? 4 : (int)std::max<int64_t>(rows, 1);
    const int64_t groups = (rows + r - 1) / r, cols = (int64_t)FEW_WARPS * COLS;
    // (148 SMs, four blocks on each, or two of 8 rows: the workspace does not go by the device.)
    const int64_t whole = (vocab + cols - 1) / cols, most = std::max<int64_t>(1, (groups > 1 ? 296 : 592) / groups);
    const int64_t rounds = (whole + most - 1) / most;
    return (int)((whole + rounds - 1) / rounds);
}

// lines_pay: w is copied where its rows start on 16-byte but not on 128-byte boundaries and
// that pays.
Plan make_plan(int dtype, int64_t rows, int width, int vocab, const void *w, int64_t w_stride, bool backward, bool lines_pay) {
    Plan p;
    auto room = [&](size_t n) {
        const size_t at = p.bytes;
        p.bytes += round_up(n, 256);
        return at;
    };
    p.mp = (int64_t)round_up((size_t)std::max<int64_t>(rows, 1), ce::TM);
    // Rows of whole 128-byte lines: boxes that straddle them make a product 30% slower
    // (1000 columns: 275 us of 9472 x 16384 rows, and 210 with 1024).  A copy of w costs
    // about as much as a third of the product with 1024 rows, or with 2048 where the
    // product is the only one; below that, rows from 16 bytes on are taken as they are.
    p.dp = (int64_t)round_up((size_t)width, 64);
    p.split = dtype == NK_F32;
    const bool lines = ((uintptr_t)w & 127) == 0 && w_stride % 64 == 0, units = ((uintptr_t)w & 15) == 0 && w_stride % 8 == 0;
    p.copy_w = p.split || !units || (lines_pay && !lines && rows >= (backward ? 1024 : 2048));
    const size_t parts = p.split ? 2 : 1;
    p.head = room(sizeof(Head));
    if (p.split) p.scales = room(((size_t)p.mp + round_up((size_t)vocab, ce::TN)) * 4);
    p.row_of = room((size_t)rows * 4);
    p.place = room((size_t)rows * 4);
    p.target = room((size_t)rows * 4);
    p.x = room((size_t)p.mp * p.dp * 2 * parts);
    if (p.copy_w) p.w = room((size_t)vocab * p.dp * 2 * parts);
    if (!backward) {
        p.few = few_rows(dtype, rows, width, vocab, w, w_stride);
        if (p.few) {
            p.bytes = 0;
            p.tiles = few_blocks(rows, vocab);
            p.mp = rows;
            p.part = room((size_t)rows * p.tiles * 8);
            p.zt = room((size_t)rows * 4);
            return p;
        }
        p.tiles = 2 * ((vocab + ce::TN - 1) / ce::TN);
        p.part = room((size_t)p.mp * p.tiles * 8);
        p.zt = room((size_t)rows * 4);
        return p;
    }
    p.stats = room((size_t)rows * 8);
    p.weight = room((size_t)rows * 4);
    const uint64_t fit = PIECE_BYTES / 2 / parts / std::max<uint64_t>(1, (uint64_t)p.mp) / ce::TN * ce::TN;
    p.piece = (int)std::min<uint64_t>(std::max<uint64_t>(fit, 4 * ce::TN), (uint64_t)vocab);
    p.ldg = (int64_t)round_up((size_t)p.piece, ce::TN);
    p.g = room((size_t)p.mp * p.ldg * 2 * parts);
    p.ld_acc = (int64_t)round_up((size_t)width, ce::TN);
    const int pairs = PAIRS;
    const int64_t nt = p.ld_acc / ce::TN, segs = p.split ? 3 : 1;
    pick_splits(p.mp / ce::TM * nt, p.ldg / ce::BK * segs, p.ldg / ce::TN * nt, p.mp / ce::BK * segs, pairs, p.dx_splits, p.dw_splits);
    if (p.dx_splits > 1 || p.piece < vocab) p.dx = room((size_t)p.dx_splits * p.mp * p.ld_acc * 4);
    if (p.dw_splits > 1) p.dw = room((size_t)p.dw_splits * p.ldg * p.ld_acc * 4);
    return p;
}

// What any call of up to `rows` rows takes at most.  Everything in a plan grows with the rows
// but three things, which have bounds that do: G (PIECE_BYTES, or 1024 tokens of all rows), the
// sums of a split dx or dw (256 x 256 sums of 4 items a pair at most, and no more splits than K
// has 8 K-blocks for), and the few rows' partial results.
size_t most_bytes(int dtype, int64_t rows, int width, int vocab, const void *w, int64_t w_stride, bool backward) {
    Plan p = make_plan(dtype, rows, width, vocab, w, w_stride, backward, true);
    const auto whole = [](uint64_t n) { return round_up(n, 256); };
    if (!backward) {
        if (((uintptr_t)w & 15) != 0) return p.bytes;
        const uint64_t cols = (uint64_t)(vocab + FEW_WARPS * COLS - 1) / (FEW_WARPS * COLS), some = std::min<int64_t>(rows, 4096);
        const size_t few = whole(8 * std::min(some * cols, std::max(592 * std::min<uint64_t>(some, 8), some))) + whole(some * 4);
        return std::max(p.bytes, few);
    }
    const uint64_t parts = p.split ? 2 : 1, segs = p.split ? 3 : 1, mp = (uint64_t)p.mp, tokens = round_up((size_t)vocab, ce::TN);
    const uint64_t row = (uint64_t)p.ld_acc * 4, split = 4 * PAIRS * (uint64_t)ce::TM * ce::TN * 4;
    const uint64_t kx = std::min<uint64_t>(tokens * segs / (8 * ce::BK), 64), kw = std::min<uint64_t>(mp * segs / (8 * ce::BK), 64);
    const uint64_t g = std::min(mp * tokens * 2 * parts, std::max(PIECE_BYTES, mp * std::min<uint64_t>(tokens, 4 * ce::TN) * 2 * parts));
    uint64_t dx = kx > 1 ? std::min(split, kx * mp * row) : 0;
    if (p.piece < vocab) dx = std::max(dx, mp * row);
    const uint64_t dw = kw > 1 ? std::min(split, kw * tokens * row) : 0;
    return p.g + whole(g) + whole(dx) + whole(dw);
}

// Instruction descriptor: f32 sums, f16 or bf16 factors, 256 x 256, majors.
uint32_t instruction(bool bf16, bool a_mn, bool b_mn) {
    return (1u << 4) | (bf16 ? (1u << 7) | (1u << 10) : 0u) | (a_mn ? 1u << 15 : 0u) | (b_mn ? 1u << 16 : 0u) |
           ((uint32_t)(ce::TN >> 3) << 17) | ((uint32_t)(ce::TM >> 4) << 24);
}

// T: the type of x and w; P: that of the parts the products take.
template <class T, class P>
struct Call {
    static constexpr bool SPLIT = sizeof(T) == 4;
    static constexpr bool BF16 = std::is_same_v<P, __nv_bfloat16>;
    const LinearCeArgs &a;
    Plan p;
    int sms;
    cudaStream_t st;
    char *ws;
    Index ix;
    float *scales;
    const P *w;      // as the products take it
    int64_t w_ld, w_cols;

    Call(const LinearCeArgs &args, bool backward, int n_sms, cudaStream_t stream)
        : a(args), p(make_plan(args.dtype, args.rows, args.width, args.vocab, args.w, args.w_stride, backward, args.copy_lines)), sms(n_sms), st(stream),
          ws((char *)args.workspace) {
        ix = {at<Head>(p.head), at<uint32_t>(p.row_of), at<uint32_t>(p.place), at<uint32_t>(p.target), at<float2>(p.stats), at<float>(p.weight)};
        scales = at<float>(p.scales);
        w = p.copy_w ? at<P>(p.w) : (const P *)a.w;
        w_ld = p.copy_w ? p.dp : a.w_stride;
        w_cols = p.copy_w ? p.dp : a.width;
    }
    cudaError_t err = cudaSuccess;  // the first launch's that failed: none follows it

    template <class... K, class... A>
    void go(void (*k)(K...), dim3 grid, int threads, int shared, A &&...args) {
        if (err == cudaSuccess) err = pdl_launch(k, grid, dim3((unsigned)threads), (size_t)shared, st, args...);
    }
    template <int MODE, bool LONG>
    void product(ce::Products &ps) {
        ps.wait_ns = g_withhold ? ce::TEST_WAIT_NS : ce::WAIT_NS;
        ps.withhold = g_withhold == MODE + 1;
        auto *k = ce::gemm_k<MODE, P, SPLIT, LONG>;
        constexpr int shared = ce::smem_bytes(MODE != ce::ROWS);
        if (err == cudaSuccess) err = allow_shared(k, shared);
        int64_t items = 0;
        for (const Gemm &g : ps.g) items += (int64_t)((g.M + ce::TM - 1) / ce::TM) * ((g.N + ce::TN - 1) / ce::TN) * g.splits;
        const int pairs = (int)std::max<int64_t>(1, std::min<int64_t>(sms / 2, items));
        go(k, 2 * pairs, ce::THREADS, shared, ps);
    }
    template <class U>
    U *at(size_t o) const {
        return (U *)(ws + o);
    }
    unsigned blocks(int64_t rows) const { return (unsigned)std::min<int64_t>((rows + 7) / 8, (int64_t)sms * 8); }

    // The index, x and, where it has to be, w laid out.
    // (Zero rows follow the rows that count: up to a whole K-block of dw.)
    void begin(bool backward) {
        go(ce_index_k, 1, 1024, 0, a, ix, backward);
        Rows x{a.x, a.x_stride, a.rows, ix.place, at<void>(p.x), p.mp * p.dp, ce::BK - 1, p.mp, a.dx, a.dx_stride, nullptr, scales};
        Rows w{a.w, a.w_stride, a.vocab, nullptr, at<void>(p.w), (int64_t)a.vocab * p.dp, 0, a.vocab, nullptr, 0, nullptr, scales + p.mp};
        if (SPLIT && backward) {
            // (dx and dw sum over tokens and rows: a scale for each matrix.)
            x.top = &ix.head->x_max;
            w.top = &ix.head->w_max;
            go(ce_absmax_k, blocks(a.rows + a.vocab), 256, 0, x, w, a.width);
        }
        if (!p.copy_w) w.rows = 0;
        go(ce_lay_out_k<T>, blocks(a.rows + w.rows + ce::BK), 256, 0, x, w, a.width, p.dp, ix.head);
    }

    bool map_x(CUtensorMap (&m)[2], int box) const {
        for (int i = 0; i < (SPLIT ? 2 : 1); ++i)
            if (!make_map(&m[i], at<P>(p.x) + i * p.mp * p.dp, BF16, p.mp, p.dp, p.dp, box)) return false;
        if (!SPLIT) m[1] = m[0];
        return true;
    }
    bool map_w(CUtensorMap (&m)[2], int box) const {
        for (int i = 0; i < (SPLIT ? 2 : 1); ++i)
            if (!make_map(&m[i], w + i * (int64_t)a.vocab * p.dp, BF16, a.vocab, w_cols, w_ld, box)) return false;
        if (!SPLIT) m[1] = m[0];
        return true;
    }
    bool map_g(CUtensorMap (&m)[2], int box) const {
        for (int i = 0; i < (SPLIT ? 2 : 1); ++i)
            if (!make_map(&m[i], at<P>(p.g) + i * p.mp * p.ldg, BF16, p.mp, p.ldg, p.ldg, box)) return false;
        if (!SPLIT) m[1] = m[0];
        return true;
    }
    Gemm gemm(int M, int N, int K, int live_dim, bool a_mn, bool b_mn, int splits) const {
        Gemm g{};
        g.M = M;
        g.N = g.n_valid = N;
        g.K = K;
        g.live_dim = live_dim;
        // high * low, low * high, high * high: the small products first.
        g.segs = SPLIT ? 3 : 1;
        g.sa = SPLIT ? 2u : 0u;
        g.sb = SPLIT ? 1u : 0u;
        g.idesc = instruction(BF16, a_mn, b_mn);
        g.m_fast = 0;
        g.group_m = 32;
        g.splits = splits;
        const int total = (K + ce::BK - 1) / ce::BK * g.segs;
        g.kps = std::max(1, (total + splits - 1) / splits);
        g.head = ix.head;
        return g;
    }

    template <int R>
    cudaError_t few() {
        auto *k = ce_few_k<T, R>;
        const int shared = R * (int)round_up((size_t)a.width, 16 / sizeof(T)) * 4;
        err = allow_shared(k, R * 4096 * 4);
        go(k, dim3((unsigned)p.tiles, (unsigned)((a.rows + R - 1) / R)), 32 * FEW_WARPS, shared, a, at<float2>(p.part), p.mp,
                                                                                                      at<float>(p.zt));
        go(ce_join_k, (unsigned)((a.rows + 7) / 8), 256, 0, a, nullptr, nullptr, at<float2>(p.part), p.mp, at<float>(p.zt), p.tiles);
        return err;
    }

    cudaError_t forward() {
        if (p.few) return a.rows >= 8 ? few<8>() : a.rows > 2 ? few<4>() : a.rows == 2 ? few<2>() : few<1>();
        begin(false);
        ce::Products ps{};
        if (!map_x(ps.a[0], 128) || !map_w(ps.b[0], 128)) return cudaErrorInvalidValue;
        Gemm &g = ps.g[0];
        g = gemm((int)a.rows, a.vocab, a.width, 0, false, false, 1);
        ps.cost[0] = ps.cost[1] = 1;
        g.m_fast = 1;
        if (SPLIT) g.x_scale = scales, g.w_scale = scales + p.mp;
        g.part = at<float2>(p.part);
        g.part_ld = p.mp;
        g.zt = at<float>(p.zt);
        g.target = ix.target;
        product<ce::ROWS, true>(ps);
        go(ce_join_k, (unsigned)((a.rows + 7) / 8), 256, 0, a, ix.head, ix.row_of, g.part, p.mp, g.zt, p.tiles);
        return err;
    }

    cudaError_t backward() {
        begin(true);
        ce::Products pg{}, ps{};
        if (!map_x(pg.a[0], 128) || !map_w(pg.b[0], 128) || !map_g(pg.c, 32) || !map_g(ps.a[0], 128) || !map_w(ps.b[0], 64) ||
            !map_g(ps.a[1], 64) || !map_x(ps.b[1], 64))
            return cudaErrorInvalidValue;
        const float g_scale = BF16 ? 1.0f : G_SCALE;
        for (int v0 = 0; v0 < a.vocab; v0 += p.piece) {
            const int n = std::min(p.piece, a.vocab - v0);
            const bool last = v0 + n == a.vocab;
            Gemm &g = pg.g[0];
            g = gemm((int)a.rows, n, a.width, 0, false, false, 1);
            g.m_fast = 1;
            g.b_row0 = v0;
            if (SPLIT) g.x_scale = scales, g.w_scale = scales + p.mp;
            g.target = ix.target;
            g.stats = ix.stats;
            g.weight = ix.weight;
            g.col0 = v0;
            g.g_scale = g_scale;
            pg.cost[0] = pg.cost[1] = 1;
            if (a.rows) product<ce::GRAD, true>(pg);
            Gemm &x = ps.g[0], &w = ps.g[1];
            x = gemm(a.dx ? (int)a.rows : 0, a.width, n, a.dx ? 0 : 2, false, true, p.dx_splits);
            x.b_row0 = v0;
            if (SPLIT) x.w_scale = scales + p.mp;
            x.acc = p.dx ? at<float>(p.dx) : nullptr;
            x.ld_acc = p.ld_acc;
            x.acc_split = p.mp * p.ld_acc;
            x.add = v0 != 0;
            x.keep = !last || p.dx_splits > 1;
            x.out = a.dx;
            x.out_ld = a.dx_stride;
            x.out_dtype = a.dtype;
            x.out_row = ix.row_of;
            x.out_scale = a.grad_scale / g_scale;
            w = gemm(a.dw ? n : 0, a.width, (int)a.rows, 1, true, true, p.dw_splits);
            if (SPLIT) w.x_scale = scales;
            w.acc = p.dw ? at<float>(p.dw) : nullptr;
            w.ld_acc = p.ld_acc;
            w.acc_split = p.ldg * p.ld_acc;
            w.keep = p.dw_splits > 1;
            w.out = a.dw;
            w.out_ld = a.dw_stride;
            w.out_row0 = v0;
            w.out_dtype = a.dw_dtype;
            w.out_add = a.accumulate;
            w.out_scale = a.grad_scale / g_scale;
            ps.cost[0] = item_cost(x.kps, p.dx_splits > 1);
            ps.cost[1] = item_cost(w.kps, p.dw_splits > 1);
            if (SPLIT || (a.dw && a.dw_dtype == NK_F32) || std::max(a.dx ? x.kps : 0, a.dw ? w.kps : 0) > longest_chain(BF16))
                product<ce::STORE, true>(ps);
            else
                product<ce::STORE, false>(ps);
            const int sx = a.dx && last && p.dx_splits > 1 ? p.dx_splits : 0, sw = a.dw && p.dw_splits > 1 ? p.dw_splits : 0;
            if (sx || sw) {
                const int64_t most = std::max<int64_t>(sx ? a.rows : 0, sw ? n : 0) * p.ld_acc / 4;
                const unsigned grid = (unsigned)std::max<int64_t>(1, std::min<int64_t>((most + 255) / 256, (int64_t)sms * 8));
                if (a.dw_dtype == NK_F32)
                    go(ce_reduce_k<T, float>, grid, 256, 0, x, sx, w, sw);
                else
                    go(ce_reduce_k<T, T>, grid, 256, 0, x, sx, w, sw);
            }
        }
        return err;
    }
};

}  // namespace

void linear_ce_withhold(int product) { g_withhold = product; }

size_t linear_ce_workspace_bytes(int dtype, int64_t rows, int width, int vocab, const void *w, int64_t w_stride,
                                 bool backward, bool copy_lines) {
    return make_plan(dtype, rows, width, vocab, w, w_stride, backward, copy_lines).bytes;
}

size_t linear_ce_most_workspace_bytes(int dtype, int64_t rows, int width, int vocab, const void *w, int64_t w_stride, bool backward) {
    return most_bytes(dtype, rows, width, vocab, w, w_stride, backward);
}

cudaError_t linear_ce(const LinearCeArgs &a, int sms, cudaStream_t st) {
    if (a.dtype == NK_F32) return Call<float, __half>(a, false, sms, st).forward();
    if (a.dtype == NK_F16) return Call<__half, __half>(a, false, sms, st).forward();
    return Call<__nv_bfloat16, __nv_bfloat16>(a, false, sms, st).forward();
}

cudaError_t linear_ce_backward(const LinearCeArgs &a, int sms, cudaStream_t st) {
    if (a.dtype == NK_F32) return Call<float, __half>(a, true, sms, st).backward();
    if (a.dtype == NK_F16) return Call<__half, __half>(a, true, sms, st).backward();
    return Call<__nv_bfloat16, __nv_bfloat16>(a, true, sms, st).backward();
}

}  // namespace nk
