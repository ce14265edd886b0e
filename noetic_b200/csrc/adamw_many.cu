// adamw_many.cu -- one AdamW step (optim.rs:33-72) over all of a model's
// tensors, with moments in 32 bits or in 8 bits and a scale for each block of
// 256, and the gradients' norm that the step can clip them by.
//
//   g = grad c,  m' = b1 m + (1 - b1) g,  v' = b2 v + (1 - b2) g g,
//   val' = val - lr (m' / (1 - b1^t) / (sqrt(v' / (1 - b2^t)) + eps) + wd val)
//
// Bound: HBM.  An element moves 8 bytes of val, 2 or 4 of gradient, 16 (32-bit)
// or 4 (8-bit) of moments and 2 of the optional copy, and the norm reads the
// gradients once more before.

#include <algorithm>
#include <cuda_fp8.h>

#include "nk_head.cuh"
#include "nk_train.h"

namespace nk {

namespace {

constexpr float E4M3_MAX = 448.0f;
constexpr float E4M3_TINY = 0.001953125f;  // 2^-9, the smallest number above 0
// Blocks whose largest value is below this are stored as zeros: 448 / value
// would leave f32's range (values like that come of gradients below 1e-30).
constexpr float SCALE_MIN = 7.8886090522101181e-31f;  // 2^-100
constexpr float V_MAX = 3e38f;
constexpr float MOMENT_MAX = 1.2676506002282294e30f;  // 2^100: m / (1 - b1^t) stays in range

// Four gradients from element 4 i on.
template <class G>
__device__ __forceinline__ void load4(const G *p, float (&g)[4]) {
    if constexpr (sizeof(G) == 4) {
        const float4 q = __ldcs(reinterpret_cast<const float4 *>(p));
        g[0] = q.x, g[1] = q.y, g[2] = q.z, g[3] = q.w;
    } else {
        const uint2 q = __ldcs(reinterpret_cast<const uint2 *>(p));
        const G *h = reinterpret_cast<const G *>(&q);
#pragma unroll
        for (int i = 0; i < 4; ++i) g[i] = to_f32(h[i]);
    }
}

// ---------------------------------------------------------------- norm
// (Four vectors of 16 bytes to a thread at once: with 8 bytes the pass was at 2.4 TB/s.)
template <class G>
__device__ __forceinline__ double chunk_squares(const G *grad, uint32_t n, bool vec) {
    constexpr uint32_t PER = 16 / sizeof(G);
    double s = 0.0;
    const uint32_t vectors = vec ? n / PER : 0;
    const uint4 *p = reinterpret_cast<const uint4 *>(grad);
    for (uint32_t i = threadIdx.x; i < vectors; i += 4 * blockDim.x) {
        uint4 q[4];
#pragma unroll
        for (uint32_t u = 0; u < 4; ++u) q[u] = i + u * blockDim.x < vectors ? __ldcs(p + i + u * blockDim.x) : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            // (A vector in f32, the vectors in 64 bits.)
            const G *g = reinterpret_cast<const G *>(&q[u]);
            float a = 0.0f, b = 0.0f;
#pragma unroll
            for (uint32_t e = 0; e < PER; e += 2) {
                const float x = to_f32(g[e]), y = to_f32(g[e + 1]);
                a = fmaf(x, x, a);
                b = fmaf(y, y, b);
            }
            // (Squares that leave f32's range: gradients above 4e18, or below 1e-16.)
            if (a + b > 1e-30f && a + b < 1e37f) {
                s += (double)(a + b);
            } else {
#pragma unroll
                for (uint32_t e = 0; e < PER; ++e) s += (double)to_f32(g[e]) * (double)to_f32(g[e]);
            }
        }
    }
    for (uint32_t i = vectors * PER + threadIdx.x; i < n; i += blockDim.x) {
        const double g = (double)to_f32(grad[i]);
        s += g * g;
    }
    return s;
}

__device__ __forceinline__ double block_sum_d(double v, double *red) {
    v = warp_sum_d(v);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    __syncthreads();
    if (lane == 0) red[warp] = v;
    __syncthreads();
    return warp_sum_d(lane < (int)(blockDim.x >> 5) ? red[lane] : 0.0);
}

__device__ __forceinline__ bool aligned(const void *p, uint32_t to) { return ((uintptr_t)p & (to - 1)) == 0; }

// Each block's sum of squares, of the chunks that its number gives it, to its own
// place; the block that finishes last adds them in a fixed order, so the norm does
// not depend on scheduling.
__global__ void __launch_bounds__(256) adamw_norm_k(AdamwMany p, float grad_scale, float max_norm, float *norm,
                                                    uint32_t *bad) {
    pdl_trigger();
    pdl_wait();
    __shared__ double red[32];
    __shared__ bool last;
    double sum = 0.0;
    for (uint32_t c = blockIdx.x; c < p.n_chunks; c += gridDim.x) {
        const AdamwChunk ch = p.chunks[c];
        const nk_adamw_tensor &t = p.tensors[ch.tensor];
        double s;
        if (t.grad_dtype == NK_F32) {
            const float *g = (const float *)t.grad + ch.first;
            s = chunk_squares(g, ch.n, aligned(g, 16));
        } else if (t.grad_dtype == NK_F16) {
            const __half *g = (const __half *)t.grad + ch.first;
            s = chunk_squares(g, ch.n, aligned(g, 16));
        } else {
            const __nv_bfloat16 *g = (const __nv_bfloat16 *)t.grad + ch.first;
            s = chunk_squares(g, ch.n, aligned(g, 16));
        }
        sum += s;
    }
    sum = block_sum_d(sum, red);
    if (threadIdx.x == 0) {
        p.partial[blockIdx.x] = sum;
        __threadfence();
        last = atomicAdd(p.ticket, 1u) == gridDim.x - 1;
    }
    __syncthreads();
    if (!last) return;
    __threadfence();
    double s = 0.0;
    for (uint32_t c = threadIdx.x; c < gridDim.x; c += blockDim.x) s += __ldcg(p.partial + c);
    s = block_sum_d(s, red);
    if (threadIdx.x == 0) {
        const float all = (float)(sqrt(s) * fabs((double)grad_scale));
        if (norm) *norm = all;
        if (max_norm > 0.0f) {
            const bool fine = isfinite(all);
            p.clip[0] = all > max_norm ? __fmul_rn(grad_scale, __fmul_rn(max_norm, __frcp_rn(all))) : grad_scale;
            p.clip[1] = fine ? 1.0f : 0.0f;
            if (!fine && bad) *bad = 1u;
        }
        *p.ticket = 0u;
    }
}

// ---------------------------------------------------------------- the step
// The reference's operations, each correctly rounded, in its order.  False: the
// element stays as it is.
__device__ __forceinline__ bool adamw_element(float &val, float grad, float c, float &m, float &v, const AdamwParams &a,
                                              bool decay) {
    const float g = __fmul_rn(grad, c);
    if (!isfinite(g) || !isfinite(val)) return false;
    m = __fadd_rn(__fmul_rn(a.b1, m), __fmul_rn(__fsub_rn(1.0f, a.b1), g));
    v = __fadd_rn(__fmul_rn(a.b2, v), __fmul_rn(__fmul_rn(__fsub_rn(1.0f, a.b2), g), g));
    const float mh = __fmul_rn(m, a.inv_bc1), vh = __fmul_rn(v, a.inv_bc2);
    float upd = __fdiv_rn(mh, __fadd_rn(__fsqrt_rn(vh), a.eps));
    if (decay) upd = __fadd_rn(upd, __fmul_rn(a.wd, val));
    val = __fsub_rn(val, __fmul_rn(a.lr, upd));
    return true;
}

__device__ __forceinline__ void store_copy(void *copy, int dtype, uint64_t i, float v) {
    if (dtype == NK_F16)
        ((__half *)copy)[i] = from_f32<__half>(v);
    else
        ((__nv_bfloat16 *)copy)[i] = from_f32<__nv_bfloat16>(v);
}
// Four values from element i on, a multiple of 4 of an 8-byte aligned copy.
__device__ __forceinline__ void store_copy4(void *copy, int dtype, uint64_t i, const float (&v)[4]) {
    uint2 q;
    if (dtype == NK_F16) {
        __half *h = reinterpret_cast<__half *>(&q);
#pragma unroll
        for (int e = 0; e < 4; ++e) h[e] = from_f32<__half>(v[e]);
    } else {
        __nv_bfloat16 *h = reinterpret_cast<__nv_bfloat16 *>(&q);
#pragma unroll
        for (int e = 0; e < 4; ++e) h[e] = from_f32<__nv_bfloat16>(v[e]);
    }
    __stcs(reinterpret_cast<uint2 *>((char *)copy + 2 * i), q);
}

template <class G>
__device__ __forceinline__ bool chunk_step32(const nk_adamw_tensor &t, const AdamwChunk &ch, const AdamwParams &a,
                                             float c, bool decay) {
    float *val = t.val + ch.first, *m = (float *)t.m + ch.first, *v = (float *)t.v + ch.first;
    const G *grad = (const G *)t.grad + ch.first;
    bool ok = true;
    uint32_t done = 0;
    if (aligned(val, 16) && aligned(m, 16) && aligned(v, 16) && aligned(grad, 4 * sizeof(G)) &&
        (!t.copy || aligned((char *)t.copy + 2 * ch.first, 8))) {
        done = ch.n & ~3u;
        for (uint32_t i = threadIdx.x * 4; i < done; i += blockDim.x * 4) {
            float g[4];
            load4(grad + i, g);
            const float4 pq = __ldcs(reinterpret_cast<float4 *>(val + i)), mq = __ldcs(reinterpret_cast<float4 *>(m + i)),
                         vq = __ldcs(reinterpret_cast<float4 *>(v + i));
            float pv[4] = {pq.x, pq.y, pq.z, pq.w}, mv[4] = {mq.x, mq.y, mq.z, mq.w}, vv[4] = {vq.x, vq.y, vq.z, vq.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) ok &= adamw_element(pv[e], g[e], c, mv[e], vv[e], a, decay);
            __stcs(reinterpret_cast<float4 *>(val + i), make_float4(pv[0], pv[1], pv[2], pv[3]));
            __stcs(reinterpret_cast<float4 *>(m + i), make_float4(mv[0], mv[1], mv[2], mv[3]));
            __stcs(reinterpret_cast<float4 *>(v + i), make_float4(vv[0], vv[1], vv[2], vv[3]));
            if (t.copy) store_copy4(t.copy, t.copy_dtype, ch.first + i, pv);
        }
    }
    for (uint32_t i = done + threadIdx.x; i < ch.n; i += blockDim.x) {
        float pv = val[i], mv = m[i], vv = v[i];
        ok &= adamw_element(pv, to_f32(grad[i]), c, mv, vv, a, decay);
        val[i] = pv;
        m[i] = mv;
        v[i] = vv;
        if (t.copy) store_copy(t.copy, t.copy_dtype, ch.first + i, pv);
    }
    return ok;
}

// Two e4m3 numbers, exactly.
__device__ __forceinline__ float2 from_e4m3(uint32_t two) {
    return __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)two, __NV_E4M3)));
}
// To nearest, ties to even.
__device__ __forceinline__ uint32_t to_e4m3(float lo, float hi) {
    return __nv_cvt_float2_to_fp8x2(make_float2(lo, hi), __NV_SATFINITE, __NV_E4M3);
}

// What the moments' rounding by chance takes from the call.
struct Chance {
    bool m, v;
    uint32_t t;
};
// Above this factor a step forgets less than half a step of the grid (1/32 to 1/16 of a
// value), so that to nearest a byte returns to where it was: roots whose gradients fell to
// a tenth stood at 6.6 times the formula's after 600 steps at b2 = 0.99, and means of
// gradients that turned round had not turned after 750 steps at b1 = 0.98.  Rounded up or
// down in proportion they are at 1.00 and 0.04 off.  Below, noisy gradients move the block's
// scale by enough (1.00 at b2 = 0.95), and to nearest is the more exact: 0.075 off where
// chance is 0.107, and takes less time (361M elements, bf16 gradients and copy: 1245 us, by
// chance 1570).
constexpr float MOST_TO_NEAREST = 0.95f;

// 24 bits of an element and a step, in [0, 1): odd multiples of it (2^32 by the golden
// ratio, by sqrt 2 and by sqrt 3), folded.  `m`: another 24.
__device__ __forceinline__ float chance_of(uint64_t element, uint32_t t, float val, float grad, bool m) {
    uint32_t x = (uint32_t)element * 0x9E3779B9u + (uint32_t)(element >> 32) + t * 0x6A09E667u;
    x ^= x >> 16;
    x = (x ^ __float_as_uint(val)) * 0xBB67AE85u;
    x ^= x >> 15;
    x = (x + __float_as_uint(grad)) * 0x9E3779B9u;
    x ^= x >> 16;
    x *= 0x6A09E667u;
    if (m) x = (x ^ x >> 13) * 0xBB67AE85u;
    return (float)((x ^ x >> 15) & 0xFFFFFFu) * 5.9604645e-8f;
}

// One of the two numbers of the grid beside y >= 0, whose mean (SQUARE: whose square's mean)
// is y's.
template <bool SQUARE>
__device__ __forceinline__ float by_chance(float y, float u) {
    const uint32_t e = max(__float_as_uint(y) & 0x7F800000u, 121u << 23);  // (2^-6: below, one step)
    const float step = __uint_as_float(e - (3u << 23)), q = y * __uint_as_float((257u << 23) - e), n = floorf(q), f = q - n;
    const bool up = SQUARE ? u * (2.0f * n + 1.0f) < f * (q + n) : u < f;
    return (up ? n + 1.0f : n) * step;
}

// 448 times the reciprocal of top (correctly rounded but for one in a million).
__device__ __forceinline__ float grid_scale(float top) {
    const float r = __fdividef(1.0f, top);
    return E4M3_MAX * fmaf(fmaf(-top, r, 1.0f), r, r);
}

__device__ __forceinline__ float rcp(float x) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float rsqrt_fast(float x) {
    float r;
    asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

__device__ __forceinline__ float2 both(float x) { return make_float2(x, x); }

// Two sums, each rounded, of products that are rounded: apart, since the assembler makes
// one fma of a packed product and a packed sum.
__device__ __forceinline__ float2 plus(float2 a, float2 b) { return make_float2(__fadd_rn(a.x, b.x), __fadd_rn(a.y, b.y)); }

// What a block's steps need of the call, worked out once a thread.
struct Step8 {
    float c, b1, g1, b2, g2, inv_bc1, root_bc2, eps, lr, wd;
    __device__ __forceinline__ Step8(const AdamwParams &a, float factor)
        : c(factor), b1(a.b1), g1(1.0f - a.b1), b2(a.b2), g2(1.0f - a.b2), inv_bc1(a.inv_bc1),
          root_bc2(sqrtf(a.inv_bc2)), eps(fmaxf(a.eps, 1.1754944e-38f)), lr(a.lr), wd(a.wd) {}
};

// A block of 256 elements on its way to a warp: copies into shared memory that
// need no registers, so that each warp has STAGES8 - 1 blocks (2.5 KB each) in flight
// while it works on one.  16 warps on an SM with four stages: 24 warps with three, 32
// with two and 16 with six measured 1272, 1348 and 1419 us where this takes 1259 (361M
// elements, bf16 gradients and copy, the norm's 112 us with it); chunks of 128 blocks
// rather than 32, and plain stores rather than streaming ones, took 55 us off that.
constexpr int STAGES8 = 4, WARPS8 = 8;
struct __align__(16) Stage8 {
    float val[NK_ADAMW_BLOCK];
    uint32_t grad[NK_ADAMW_BLOCK];  // up to 4 bytes an element
    uint32_t m[NK_ADAMW_BLOCK / 4], v[NK_ADAMW_BLOCK / 4];
    float scale[4];  // of m and of v
};

__device__ __forceinline__ float grad_of(const void *grad, int dtype, uint64_t i) {
    return dtype == NK_F32 ? ((const float *)grad)[i] : dtype == NK_F16 ? to_f32(((const __half *)grad)[i]) : to_f32(((const __nv_bfloat16 *)grad)[i]);
}

// A warp steps one block of up to 256 elements: lane l holds elements 4 l .. + 3
// and 128 + 4 l .. + 3, so the block's largest |m| and sqrt(v) are two shuffles'
// reductions and nothing is read twice.  Correctly rounded roots and quotients, as
// the 32-bit step has them, took 116 instructions an element and 2.4 TB/s; here one
// root (a reciprocal root and Newton's step, which rounds correctly but for one in a
// million) serves the update and the moment, and the quotient is a product with a
// reciprocal: 2^-22 of an update, which is below the rounding of val.  What the
// moments are made of is rounded operation by operation, as in the 32-bit step: a
// byte at the middle between two others then goes the same way wherever the formula
// is computed, where an fma here sent one in a million the other way, and the next
// step of such an element is an eighth longer or shorter.
//
// The careful form: short blocks, tensors that start off 16 bytes, elements that are
// not finite or beyond the range of what is stored.  Its operations are those of the other
// form, so that an element's result does not depend on where it lies.
__device__ __noinline__ bool careful_step8(const nk_adamw_tensor *tp, uint64_t first, uint32_t n, AdamwParams params, float factor, Chance chance) {
    const int lane = threadIdx.x & 31;
    const nk_adamw_tensor &t = *tp;
    const Step8 a(params, factor);
    const float wd = t.decay ? a.wd : 0.0f;
    float *val = t.val + first;
    uint8_t *m = (uint8_t *)t.m + first, *v = (uint8_t *)t.v + first;
    float ms, vs, pv[2][4], g[2][4], rv[2][4], um[2][4], uv[2][4];
    uint32_t mb[2], vb[2];
    ms = t.m_scale[first / NK_ADAMW_BLOCK], vs = t.v_scale[first / NK_ADAMW_BLOCK];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const uint32_t at = h * 128 + lane * 4;
        mb[h] = vb[h] = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const bool in = at + e < n;
            pv[h][e] = in ? val[at + e] : 0.0f;
            g[h][e] = in ? grad_of(t.grad, t.grad_dtype, first + at + e) : 0.0f;
            mb[h] |= in ? (uint32_t)m[at + e] << (8 * e) : 0u;
            vb[h] |= in ? (uint32_t)v[at + e] << (8 * e) : 0u;
        }
    }
    bool ok = true;
    float top_m = 0.0f, top_r = 0.0f;
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float2 mc = from_e4m3(e < 2 ? mb[h] & 0xFFFFu : mb[h] >> 16), vc = from_e4m3(e < 2 ? vb[h] & 0xFFFFu : vb[h] >> 16);
            const float mq = e & 1 ? mc.y : mc.x, r = (e & 1 ? vc.y : vc.x) * vs;
            // (A moment that is not finite stays so, and is no part of the block's scale.)
            const float gc = g[h][e] * a.c, m0 = fabsf(mq * ms) < INFINITY ? mq * ms : NAN, r0 = fabsf(r) < INFINITY ? r : NAN;
            um[h][e] = chance.m ? chance_of(first + h * 128 + lane * 4 + e, chance.t, pv[h][e], gc, true) : 0.0f;
            uv[h][e] = chance.v ? chance_of(first + h * 128 + lane * 4 + e, chance.t, pv[h][e], gc, false) : 0.0f;
            const bool fine = fabsf(gc) < INFINITY && fabsf(pv[h][e]) < INFINITY && !isnan(m0) && !isnan(r0);
            ok &= fine;
            float mm = __fadd_rn(__fmul_rn(__fmul_rn(mq, ms), a.b1), __fmul_rn(gc, a.g1));
            const float v1 = __fadd_rn(__fmul_rn(__fmul_rn(r, r), a.b2), __fmul_rn(__fmul_rn(gc, a.g2), gc)), vv = fminf(v1, V_MAX);
            // sqrt(vv); below 2^-126 (a gradient below 1e-18) it counts as 0.
            const float q = rsqrt_fast(vv);
            float u = vv * q;
            u = fmaf(fmaf(-u, u, vv) * 0.5f, q, u);
            u = vv < 1.1754944e-38f ? 0.0f : u;
            // (A v beyond f32's range divides to 0.)
            const float inv = v1 > V_MAX ? 0.0f : rcp(fmaf(u, a.root_bc2, a.eps));
            pv[h][e] = fine ? pv[h][e] + fmaf(mm * inv, -a.lr * a.inv_bc1, -a.lr * wd * pv[h][e]) : pv[h][e];
            mm = fminf(fmaxf(mm, -MOMENT_MAX), MOMENT_MAX);
            g[h][e] = fine ? mm : m0;  // the new m
            rv[h][e] = fine ? u : r0;
            top_m = fmaxf(top_m, fabsf(g[h][e]));
            top_r = fmaxf(top_r, rv[h][e]);
        }
    top_m = warp_max1(top_m);
    top_r = warp_max1(top_r);
    const float km = top_m >= SCALE_MIN ? grid_scale(top_m) : 0.0f;
    const float kr = top_r >= SCALE_MIN ? grid_scale(top_r) : 0.0f;
    // A root above 0 stays above 0: a later step divides by it.
    const float least = kr > 0.0f ? E4M3_TINY : 0.0f;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const uint32_t at = h * 128 + lane * 4;
        float y[4], z[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            y[e] = g[h][e] * km;
            z[e] = rv[h][e] > 0.0f ? fmaxf(rv[h][e] * kr, least) : rv[h][e];
            if (chance.m) y[e] = copysignf(by_chance<false>(fabsf(y[e]), um[h][e]), y[e]);
            if (chance.v) z[e] = by_chance<true>(z[e], uv[h][e]);
        }
        const uint32_t mo = to_e4m3(y[0], y[1]) | to_e4m3(y[2], y[3]) << 16, vo = to_e4m3(z[0], z[1]) | to_e4m3(z[2], z[3]) << 16;
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (at + e < n) {
                val[at + e] = pv[h][e];
                m[at + e] = (uint8_t)(mo >> (8 * e));
                v[at + e] = (uint8_t)(vo >> (8 * e));
                if (t.copy) store_copy(t.copy, t.copy_dtype, first + at + e, pv[h][e]);
            }
    }
    if (lane == 0) {
        // (The scale of what was stored, 0 for zeros.)
        t.m_scale[first / NK_ADAMW_BLOCK] = km > 0.0f ? top_m * (1.0f / E4M3_MAX) : 0.0f;
        t.v_scale[first / NK_ADAMW_BLOCK] = kr > 0.0f ? top_r * (1.0f / E4M3_MAX) : 0.0f;
    }
    return ok;
}

// The same for a whole block in shared memory, two elements to an instruction.  What
// is not finite, or out of range, shows in a sum of products with 0 and in the largest
// moment; such a block, of which nothing is stored yet, goes to the careful form.
template <class G, bool CHANCE>
__device__ __forceinline__ bool block_step8(const nk_adamw_tensor &t, uint64_t first, const Stage8 &st, const Step8 &a, const AdamwParams &params,
                                            float wd, const Chance &chance) {
    const int lane = threadIdx.x & 31;
    const float ms = st.scale[0], vs = st.scale[1];
    const float2 b1 = both(a.b1), c = both(a.c), g1 = both(a.g1), b2 = both(-a.b2), g2 = both(-a.g2), zero = both(0.0f);
    float2 pv[4], mv[4], root[4], um[4], uv[4], strange = zero;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const uint32_t at = h * 128 + lane * 4;
        const float4 q = *reinterpret_cast<const float4 *>(&st.val[at]);
        pv[2 * h] = make_float2(q.x, q.y);
        pv[2 * h + 1] = make_float2(q.z, q.w);
        float2 g[2];
        if constexpr (sizeof(G) == 4) {
            const float4 k = *reinterpret_cast<const float4 *>(&st.grad[at]);
            g[0] = make_float2(k.x, k.y);
            g[1] = make_float2(k.z, k.w);
        } else {
            const uint2 k = *reinterpret_cast<const uint2 *>(&st.grad[at / 2]);
            const G *e = reinterpret_cast<const G *>(&k);
            g[0] = make_float2(to_f32(e[0]), to_f32(e[1]));
            g[1] = make_float2(to_f32(e[2]), to_f32(e[3]));
        }
        const uint32_t mb = st.m[at / 4], vb = st.v[at / 4];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int o = 2 * h + i;
            const float2 r = mul2(from_e4m3(i ? vb >> 16 : vb & 0xFFFFu), both(vs)), gc = mul2(g[i], c);
            if (CHANCE) {
                const uint64_t e = first + at + 2 * i;
                uv[o] = make_float2(chance_of(e, chance.t, pv[o].x, gc.x, false), chance_of(e + 1, chance.t, pv[o].y, gc.y, false));
                if (chance.m) um[o] = make_float2(chance_of(e, chance.t, pv[o].x, gc.x, true), chance_of(e + 1, chance.t, pv[o].y, gc.y, true));
            }
            mv[o] = plus(mul2(mul2(from_e4m3(i ? mb >> 16 : mb & 0xFFFFu), both(ms)), b1), mul2(gc, g1));
            const float2 nv = plus(mul2(mul2(r, r), b2), mul2(mul2(gc, g2), gc));  // -v'
            strange = fma2(mv[o], zero, strange);
            strange = fma2(nv, zero, strange);
            strange = fma2(pv[o], zero, strange);
            const float2 s = make_float2(rsqrt_fast(-nv.x), rsqrt_fast(-nv.y));
            float2 u = mul2(nv, s);  // -sqrt(v')
            u = fma2(fma2(u, u, nv), mul2(s, both(0.5f)), u);
            // (0 gave 0 times infinity.)
            root[o] = make_float2(fmaxf(-u.x, 0.0f), fmaxf(-u.y, 0.0f));
        }
    }
    float top_m = 0.0f, top_r = 0.0f;
#pragma unroll
    for (int o = 0; o < 4; ++o) {
        top_m = fmaxf(top_m, fmaxf(fabsf(mv[o].x), fabsf(mv[o].y)));
        top_r = fmaxf(top_r, fmaxf(root[o].x, root[o].y));
    }
    top_m = warp_max1(top_m);
    top_r = warp_max1(top_r);
    if (__any_sync(0xffffffffu, !(strange.x + strange.y == 0.0f)) || top_m > MOMENT_MAX)
        return careful_step8(&t, first, NK_ADAMW_BLOCK, params, a.c, chance);
    const float km = top_m >= SCALE_MIN ? grid_scale(top_m) : 0.0f;
    const float kr = top_r >= SCALE_MIN ? grid_scale(top_r) : 0.0f;
    const float least = kr > 0.0f ? E4M3_TINY : 0.0f;
    const float2 root_bc2 = both(a.root_bc2), eps = both(a.eps), rate = both(-a.lr * a.inv_bc1), fade = both(-a.lr * wd);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const uint32_t at = h * 128 + lane * 4;
        uint32_t mo[2], vo[2];
        float p[4];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int o = 2 * h + i;
            const float2 den = fma2(root[o], root_bc2, eps);
            const float2 q = mul2(mv[o], make_float2(rcp(den.x), rcp(den.y)));
            const float2 now = add2(pv[o], fma2(q, rate, mul2(fade, pv[o])));
            p[2 * i] = now.x, p[2 * i + 1] = now.y;
            float2 y = mul2(mv[o], both(km)), z = mul2(root[o], both(kr));
            const float2 big = mul2(root[o], both(1e25f));
            // A root above 0 (then above 1e-19) stays above 0: a later step divides by it.
            z = make_float2(fminf(fmaxf(z.x, least), big.x), fminf(fmaxf(z.y, least), big.y));
            if (CHANCE) {
                if (chance.v) z = make_float2(by_chance<true>(z.x, uv[o].x), by_chance<true>(z.y, uv[o].y));
                if (chance.m)
                    y = make_float2(copysignf(by_chance<false>(fabsf(y.x), um[o].x), y.x), copysignf(by_chance<false>(fabsf(y.y), um[o].y), y.y));
            }
            mo[i] = to_e4m3(y.x, y.y);
            vo[i] = to_e4m3(z.x, z.y);
        }
        *reinterpret_cast<float4 *>(t.val + first + at) = make_float4(p[0], p[1], p[2], p[3]);
        *reinterpret_cast<uint32_t *>((uint8_t *)t.m + first + at) = mo[0] | mo[1] << 16;
        *reinterpret_cast<uint32_t *>((uint8_t *)t.v + first + at) = vo[0] | vo[1] << 16;
        if (t.copy) store_copy4(t.copy, t.copy_dtype, first + at, p);
    }
    if (lane == 0) {
        // (The scale of what was stored, 0 for zeros.)
        t.m_scale[first / NK_ADAMW_BLOCK] = km > 0.0f ? top_m * (1.0f / E4M3_MAX) : 0.0f;
        t.v_scale[first / NK_ADAMW_BLOCK] = kr > 0.0f ? top_r * (1.0f / E4M3_MAX) : 0.0f;
    }
    return true;
}

// The copies of a whole block into a warp's stage.
template <class G>
__device__ __forceinline__ void issue8(const nk_adamw_tensor &t, uint64_t e, Stage8 &st) {
    const int lane = threadIdx.x & 31;
    copy_async16(&st.val[lane * 4], t.val + e + lane * 4);
    copy_async16(&st.val[128 + lane * 4], t.val + e + 128 + lane * 4);
    if constexpr (sizeof(G) == 4) {
        copy_async16(&st.grad[lane * 4], (const G *)t.grad + e + lane * 4);
        copy_async16(&st.grad[128 + lane * 4], (const G *)t.grad + e + 128 + lane * 4);
    } else {
        copy_async16(&st.grad[lane * 4], (const G *)t.grad + e + lane * 8);
    }
    if (lane < 16)
        copy_async16(&st.m[lane * 4], (const uint8_t *)t.m + e + lane * 16);
    else
        copy_async16(&st.v[lane * 4 - 64], (const uint8_t *)t.v + e + lane * 16 - 256);
    if (lane < 2) copy_async4(&st.scale[lane], (lane ? t.v_scale : t.m_scale) + e / NK_ADAMW_BLOCK);
}

// A warp's chunk, STAGES8 - 1 blocks ahead.
template <class G, bool CHANCE>
__device__ __forceinline__ bool chunk_step8(const nk_adamw_tensor &t, const AdamwChunk &ch, const Step8 &a, const AdamwParams &params,
                                            Stage8 *ring, const Chance &chance) {
    const float wd = t.decay ? a.wd : 0.0f;
    const bool vec = aligned(t.val, 16) && aligned(t.m, 16) && aligned(t.v, 16) && aligned(t.grad, 16) && (!t.copy || aligned(t.copy, 8));
    const uint32_t whole = vec ? ch.n / NK_ADAMW_BLOCK : 0;
    bool ok = true;
#pragma unroll
    for (uint32_t s = 0; s < STAGES8 - 1; ++s) {
        if (s < whole) issue8<G>(t, ch.first + s * NK_ADAMW_BLOCK, ring[s]);
        copy_commit();
    }
    int from = 0, to = STAGES8 - 1;
    for (uint32_t b = 0; b < whole; ++b) {
        if (b + STAGES8 - 1 < whole) issue8<G>(t, ch.first + (b + STAGES8 - 1) * NK_ADAMW_BLOCK, ring[to]);
        copy_commit();
        copy_wait<STAGES8 - 1>();
        __syncwarp();  // the other lanes' copies, too
        ok &= block_step8<G, CHANCE>(t, ch.first + b * NK_ADAMW_BLOCK, ring[from], a, params, wd, chance);
        __syncwarp();  // (before the next copies into it)
        from = from + 1 == STAGES8 ? 0 : from + 1;
        to = to + 1 == STAGES8 ? 0 : to + 1;
    }
    for (uint32_t at = whole * NK_ADAMW_BLOCK; at < ch.n; at += NK_ADAMW_BLOCK)
        ok &= careful_step8(&t, ch.first + at, min(ch.n - at, (uint32_t)NK_ADAMW_BLOCK), params, a.c, chance);
    return ok;
}

// 32-bit moments: a block of threads takes chunks block, block + blocks, ...
__global__ void __launch_bounds__(256, 6) adamw32_k(AdamwMany p, AdamwParams a, float grad_scale, bool with_clip, uint32_t *bad) {
    pdl_trigger();
    pdl_wait();
    float c = grad_scale;
    if (with_clip) {
        if (p.clip[1] == 0.0f) return;
        c = p.clip[0];
    }
    bool ok = true;
    for (uint32_t i = blockIdx.x; i < p.n_chunks32; i += gridDim.x) {
        const AdamwChunk ch = p.chunks[i];
        const nk_adamw_tensor t = p.tensors[ch.tensor];
        const bool decay = t.decay && a.wd != 0.0f;
        ok &= t.grad_dtype == NK_F32   ? chunk_step32<float>(t, ch, a, c, decay)
              : t.grad_dtype == NK_F16 ? chunk_step32<__half>(t, ch, a, c, decay)
                                       : chunk_step32<__nv_bfloat16>(t, ch, a, c, decay);
    }
    if (!ok && bad) *bad = 1u;
}

// 8-bit moments: each warp takes chunks of its own, a ring of blocks ahead.  CHANCE: m's
// or v's bytes are rounded by chance.
template <bool CHANCE>
__global__ void __launch_bounds__(32 * WARPS8, 2) adamw8_k(AdamwMany p, AdamwParams a, float grad_scale, bool with_clip, uint32_t *bad,
                                                           Chance chance) {
    pdl_trigger();
    pdl_wait();
    extern __shared__ Stage8 rings[];
    float c = grad_scale;
    if (with_clip) {
        if (p.clip[1] == 0.0f) return;
        c = p.clip[0];
    }
    const Step8 a8(a, c);
    Stage8 *ring = rings + (threadIdx.x >> 5) * STAGES8;
    bool ok = true;
    uint32_t i = p.n_chunks32 + blockIdx.x * WARPS8 + (threadIdx.x >> 5);
    AdamwChunk next = i < p.n_chunks ? p.chunks[i] : AdamwChunk{};
    while (i < p.n_chunks) {
        const AdamwChunk ch = next;
        i += gridDim.x * WARPS8;
        if (i < p.n_chunks) next = p.chunks[i];
        const nk_adamw_tensor &t = p.tensors[ch.tensor];
        ok &= t.grad_dtype == NK_F32   ? chunk_step8<float, CHANCE>(t, ch, a8, a, ring, chance)
              : t.grad_dtype == NK_F16 ? chunk_step8<__half, CHANCE>(t, ch, a8, a, ring, chance)
                                       : chunk_step8<__nv_bfloat16, CHANCE>(t, ch, a8, a, ring, chance);
    }
    if (!ok && bad) *bad = 1u;
}

}  // namespace

uint32_t adamw_chunk_elements(uint64_t total, int sms, int bits) {
    if (bits == 32) {
        // Enough chunks for eight blocks of threads on every SM, of 1024 to 16384 elements.
        const uint64_t want = total / ((uint64_t)sms * 8) / 1024 * 1024;
        return (uint32_t)std::min<uint64_t>(std::max<uint64_t>(want, 1024), 16384);
    }
    // The same number for each warp, of 128 blocks at most.
    const uint64_t blocks = total / NK_ADAMW_BLOCK + 1, warps = (uint64_t)sms * 2 * WARPS8;
    const uint64_t rounds = (blocks + warps * 128 - 1) / (warps * 128);
    return NK_ADAMW_BLOCK * (uint32_t)((blocks + warps * rounds - 1) / (warps * rounds));
}

uint32_t adamw_partials(int sms) { return (uint32_t)sms * 8; }

cudaError_t adamw_many_norm(const AdamwMany &p, float grad_scale, float max_norm, float *norm, uint32_t *bad, int sms,
                            cudaStream_t st) {
    const unsigned blocks = std::max(1u, std::min<unsigned>(p.n_chunks, adamw_partials(sms)));
    return pdl_launch(adamw_norm_k, dim3(blocks), dim3(256), 0, st, p, grad_scale, max_norm, norm, bad);
}

cudaError_t adamw_many_step(const AdamwMany &p, const AdamwParams &a, uint32_t t, float grad_scale, bool with_clip, uint32_t *bad,
                            int sms, cudaStream_t st) {
    const uint32_t n8 = p.n_chunks - p.n_chunks32;
    if (p.n_chunks32) {
        const cudaError_t e = pdl_launch(adamw32_k, dim3(std::min<unsigned>(p.n_chunks32, (unsigned)sms * 8)), dim3(256), 0, st, p, a,
                                         grad_scale, with_clip, bad);
        if (e != cudaSuccess) return e;
    }
    if (n8) {
        constexpr int shared = WARPS8 * STAGES8 * (int)sizeof(Stage8);
        const Chance chance{a.b1 > MOST_TO_NEAREST, a.b2 > MOST_TO_NEAREST, t};
        auto *k = chance.m || chance.v ? adamw8_k<true> : adamw8_k<false>;
        cudaError_t e = allow_shared(k, shared);
        if (e != cudaSuccess) return e;
        return pdl_launch(k, dim3(std::min<unsigned>((n8 + WARPS8 - 1) / WARPS8, (unsigned)sms * 2)), dim3(32 * WARPS8), shared, st,
                          p, a, grad_scale, with_clip, bad, chance);
    }
    return cudaSuccess;
}

}  // namespace nk
