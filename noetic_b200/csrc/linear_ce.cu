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

#include <algorithm>

#include "nk_head.cuh"
#include "nk_train.h"

namespace nk {

namespace {

constexpr int TILE = 64, TILE_K = 16;
constexpr uint64_t PIECE_BYTES = 256ull << 20;  // of G

size_t round256(size_t n) { return (n + 255) / 256 * 256; }

// ---------------------------------------------------------------- logits in f32
// A 64 x 64 tile of z per block of 256 threads, 4 x 4 to a thread, 16 columns of
// x and w staged in shared memory at a time.
template <class T>
__device__ __forceinline__ void z_tile(const T *x, int64_t xs, const T *w, int64_t ws, const uint32_t *targets,
                                       int64_t rows, int d, int vocab, int64_t r0, int c0, int c_end, float (&acc)[4][4]) {
    __shared__ __align__(16) float As[TILE_K][TILE + 4];
    __shared__ __align__(16) float Bs[TILE_K][TILE + 4];
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = 0.0f;
    for (int k0 = 0; k0 < d; k0 += TILE_K) {
#pragma unroll
        for (int l = 0; l < TILE * TILE_K / 256; ++l) {
            const int i = threadIdx.x + l * 256, k = i % TILE_K, r = i / TILE_K;
            const bool kin = k0 + k < d;
            // (A row without a target is not read.)
            As[k][r] = kin && r0 + r < rows && targets[r0 + r] < (uint32_t)vocab ? to_f32(x[(r0 + r) * xs + k0 + k]) : 0.0f;
            Bs[k][r] = kin && c0 + r < c_end ? to_f32(w[(int64_t)(c0 + r) * ws + k0 + k]) : 0.0f;
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < TILE_K; ++k) {
            const float4 a4 = *reinterpret_cast<const float4 *>(&As[k][ty * 4]), b4 = *reinterpret_cast<const float4 *>(&Bs[k][tx * 4]);
            const float a[4] = {a4.x, a4.y, a4.z, a4.w}, b[4] = {b4.x, b4.y, b4.z, b4.w};
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(a[i], b[j], acc[i][j]);
        }
        __syncthreads();
    }
}

// part[row][tile] = the tile's maximum and its sum relative to it; zt[row] = the
// target's logit.
template <class T>
__global__ void __launch_bounds__(256) ce_tile_k(LinearCeArgs a, float2 *part, float *zt, int tiles) {
    float z[4][4];
    const int64_t r0 = (int64_t)blockIdx.y * TILE;
    const int c0 = blockIdx.x * TILE;
    z_tile((const T *)a.x, a.x_stride, (const T *)a.w, a.w_stride, a.targets, a.rows, a.width, a.vocab, r0, c0, a.vocab, z);
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int64_t row = r0 + ty * 4 + i;
        const uint32_t t = row < a.rows ? a.targets[row] : NO_TOKEN;
        float m = -INFINITY;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int col = c0 + tx * 4 + j;
            if (col >= a.vocab) z[i][j] = -INFINITY;
            if ((uint32_t)col == t && t < (uint32_t)a.vocab) zt[row] = z[i][j];
            m = fmaxf(m, z[i][j]);
        }
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        float s = 0.0f;
        const float base = m == -INFINITY ? 0.0f : m;
#pragma unroll
        for (int j = 0; j < 4; ++j) s += ex2((z[i][j] - base) * LOG2E);
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        if (tx == 0 && row < a.rows) part[row * tiles + blockIdx.x] = make_float2(m, s);
    }
}

// A warp joins a row's tiles, in a fixed order.
__global__ void __launch_bounds__(256) ce_join_k(LinearCeArgs a, const float2 *part, const float *zt, int tiles) {
    const int64_t row = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    if (row >= a.rows) return;
    float loss = 0.0f, m = 0.0f, ls = 0.0f;
    if (a.targets[row] < (uint32_t)a.vocab) {
        const float2 *p = part + row * tiles;
        m = -INFINITY;
        for (int i = lane; i < tiles; i += 32) m = fmaxf(m, p[i].x);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        float s = 0.0f;
        for (int i = lane; i < tiles; i += 32) s = fmaf(p[i].y, ex2((p[i].x - m) * LOG2E), s);
        s = warp_sum(s);
        ls = logf(s);
        loss = (m - zt[row]) + ls;
        if (!isfinite(s)) m = ls = loss = NAN;
    }
    if (lane == 0) {
        if (a.loss) a.loss[row] = loss;
        if (a.stats) a.stats[2 * row] = m, a.stats[2 * row + 1] = ls;
    }
}

// G of columns [v0, v0 + n) of the vocabulary, f32 [rows][n].
template <class T>
__global__ void __launch_bounds__(256) ce_grad_tile_k(LinearCeArgs a, float *g, int v0, int n) {
    float z[4][4];
    const int64_t r0 = (int64_t)blockIdx.y * TILE;
    const int c0 = v0 + blockIdx.x * TILE;
    z_tile((const T *)a.x, a.x_stride, (const T *)a.w, a.w_stride, a.targets, a.rows, a.width, a.vocab, r0, c0, v0 + n, z);
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int64_t row = r0 + ty * 4 + i;
        if (row >= a.rows) continue;
        const uint32_t t = a.targets[row];
        float h = a.grad_scale * (a.row_weight ? a.row_weight[row] : 1.0f);
        const bool live = t < (uint32_t)a.vocab && h != 0.0f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int col = c0 + tx * 4 + j;
            if (col >= v0 + n) continue;
            float v = 0.0f;
            if (live) {
                v = ex2(((z[i][j] - a.in_stats[2 * row]) - a.in_stats[2 * row + 1]) * LOG2E);
                if ((uint32_t)col == t) v -= 1.0f;
                v *= h;
            }
            g[row * n + col - v0] = v;
        }
    }
}

// C[i][j] = sum_k A(i, k) B[k][j], A(i, k) = a[i as + k ak].  A zero of A skips
// its product: what stands in a row that does not count can be anything.
// sum: added to (nullable: 0); out: f32, or rounded to T with out_t.
template <class T>
__global__ void __launch_bounds__(256) ce_product_k(const float *A, int64_t as, int64_t ak, const T *B, int64_t bs, int64_t M,
                                                    int N, int64_t K, float *acc, bool add, T *out_t, float *out_f,
                                                    int64_t os, bool out_add) {
    __shared__ __align__(16) float As[TILE_K][TILE + 4];
    __shared__ __align__(16) float Bs[TILE_K][TILE];
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    const int64_t m0 = (int64_t)blockIdx.y * TILE;
    const int n0 = blockIdx.x * TILE;
    float c[4][4] = {};
    for (int64_t k0 = 0; k0 < K; k0 += TILE_K) {
#pragma unroll
        for (int l = 0; l < TILE * TILE_K / 256; ++l) {
            const int i = threadIdx.x + l * 256;
            const int kk = ak == 1 ? i % TILE_K : i / TILE, r = ak == 1 ? i / TILE_K : i % TILE;
            As[kk][r] = k0 + kk < K && m0 + r < M ? A[(m0 + r) * as + (k0 + kk) * ak] : 0.0f;
            const int kb = i / TILE, n = i % TILE;
            Bs[kb][n] = k0 + kb < K && n0 + n < N ? to_f32(B[(k0 + kb) * bs + n0 + n]) : 0.0f;
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < TILE_K; ++k)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float x = As[k][ty * 4 + i];
                if (x != 0.0f)
#pragma unroll
                    for (int j = 0; j < 4; ++j) c[i][j] = fmaf(x, Bs[k][tx * 4 + j], c[i][j]);
            }
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int64_t row = m0 + ty * 4 + i;
        if (row >= M) continue;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int col = n0 + tx * 4 + j;
            if (col >= N) continue;
            float v = c[i][j];
            if (acc) {
                if (add) v += acc[row * N + col];
                acc[row * N + col] = v;
            }
            if (out_t) out_t[row * os + col] = from_f32<T>(out_add ? v + to_f32(out_t[row * os + col]) : v);
            if (out_f) out_f[row * os + col] = out_add ? v + out_f[row * os + col] : v;
        }
    }
}

struct Plan {
    int tiles = 0;
    int piece = 0;  // columns of G at a time
    size_t part = 0, zt = 0, g = 0, dx = 0, bytes = 0;
};

Plan make_plan(int64_t rows, int width, int vocab, bool backward) {
    Plan p;
    auto room = [&](size_t n) {
        const size_t at = p.bytes;
        p.bytes += round256(n);
        return at;
    };
    p.tiles = (vocab + TILE - 1) / TILE;
    if (!backward) {
        p.part = room((size_t)rows * p.tiles * 8);
        p.zt = room((size_t)rows * 4);
    } else {
        const uint64_t fit = PIECE_BYTES / 4 / std::max<uint64_t>(1, (uint64_t)rows) / TILE * TILE;
        p.piece = (int)std::min<uint64_t>(std::max<uint64_t>(fit, 1024), (uint64_t)vocab);
        p.g = room((size_t)rows * p.piece * 4);
        p.dx = room((size_t)rows * width * 4);
    }
    return p;
}

template <class T>
cudaError_t forward(const LinearCeArgs &a, cudaStream_t st) {
    const Plan p = make_plan(a.rows, a.width, a.vocab, false);
    float2 *part = (float2 *)((char *)a.workspace + p.part);
    float *zt = (float *)((char *)a.workspace + p.zt);
    ce_tile_k<T><<<dim3((unsigned)p.tiles, (unsigned)((a.rows + TILE - 1) / TILE)), 256, 0, st>>>(a, part, zt, p.tiles);
    ce_join_k<<<(unsigned)((a.rows + 7) / 8), 256, 0, st>>>(a, part, zt, p.tiles);
    return cudaGetLastError();
}

template <class T>
cudaError_t backward(const LinearCeArgs &a, cudaStream_t st) {
    const Plan p = make_plan(a.rows, a.width, a.vocab, true);
    float *g = (float *)((char *)a.workspace + p.g), *acc = (float *)((char *)a.workspace + p.dx);
    const unsigned by = (unsigned)((a.rows + TILE - 1) / TILE), bd = (unsigned)((a.width + TILE - 1) / TILE);
    for (int v0 = 0; v0 < a.vocab; v0 += p.piece) {
        const int n = std::min(p.piece, a.vocab - v0);
        const unsigned bv = (unsigned)((n + TILE - 1) / TILE);
        if (a.rows) ce_grad_tile_k<T><<<dim3(bv, by), 256, 0, st>>>(a, g, v0, n);
        if (a.dx && a.rows)
            ce_product_k<T><<<dim3(bd, by), 256, 0, st>>>(g, n, 1, (const T *)a.w + v0 * a.w_stride, a.w_stride, a.rows,
                                                          a.width, n, acc, v0 != 0,
                                                          v0 + n == a.vocab ? (T *)a.dx : nullptr, nullptr, a.dx_stride, false);
        if (a.dw) {
            const bool f32 = a.dw_dtype == NK_F32;
            ce_product_k<T><<<dim3(bd, bv), 256, 0, st>>>(g, 1, n, (const T *)a.x, a.x_stride, n, a.width, a.rows, nullptr,
                                                          false, f32 ? nullptr : (T *)a.dw + v0 * a.dw_stride,
                                                          f32 ? (float *)a.dw + v0 * a.dw_stride : nullptr, a.dw_stride,
                                                          a.accumulate != 0);
        }
    }
    return cudaGetLastError();
}

}  // namespace

size_t linear_ce_workspace_bytes(int dtype, int64_t rows, int width, int vocab, const void *w, int64_t w_stride,
                                 bool backward) {
    return make_plan(rows, width, vocab, backward).bytes;
}

cudaError_t linear_ce(const LinearCeArgs &a, int sms, cudaStream_t st) {
    return a.dtype == NK_F32 ? forward<float>(a, st) : a.dtype == NK_F16 ? forward<__half>(a, st) : forward<__nv_bfloat16>(a, st);
}

cudaError_t linear_ce_backward(const LinearCeArgs &a, int sms, cudaStream_t st) {
    return a.dtype == NK_F32 ? backward<float>(a, st) : a.dtype == NK_F16 ? backward<__half>(a, st) : backward<__nv_bfloat16>(a, st);
}

}  // namespace nk
