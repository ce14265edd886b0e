// nk_head.cuh -- device helpers of the operators at the model's end.
#pragma once

#include <cmath>
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <type_traits>

#include "nk_common.cuh"

namespace nk {

constexpr uint32_t NO_TOKEN = 0xFFFFFFFFu;
constexpr float LN2 = 0.693147180559945309f;
constexpr float LOG2E = 1.44269504088896341f;

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }

// Rounded to nearest, ties to even.
template <class T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) {
    return x;
}
template <>
__device__ __forceinline__ __half from_f32<__half>(float x) {
    return __float2half_rn(x);
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) {
    return __float2bfloat16_rn(x);
}

// 2^x by the special-function unit (error about 2 ulp, subnormal results 0).
__device__ __forceinline__ float ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// Sum over the block in a fixed order; `red` holds 32 values.
__device__ __forceinline__ float block_sum(float v, float *red) {
    v = warp_sum(v);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    __syncthreads();
    if (lane == 0) red[warp] = v;
    __syncthreads();
    return warp_sum(lane < (int)(blockDim.x >> 5) ? red[lane] : 0.0f);
}

// Order-preserving u32 of a float; -0 counts as +0.
__device__ __forceinline__ uint32_t order_key(float x) {
    const uint32_t b = __float_as_uint(x + 0.0f);
    return b ^ ((b >> 31) ? 0xFFFFFFFFu : 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) {
    return __uint_as_float(k ^ ((k >> 31) ? 0x80000000u : 0xFFFFFFFFu));
}

// Lets a kernel be launched with `most` bytes of dynamic shared memory.  The limit
// belongs to the function on its device, not to a call, so `most` is the most that
// any call of this function asks for: set to the call's own need, a call of another
// host thread could lower it between this and the launch.
template <class K>
inline cudaError_t allow_shared(K *kern, int most) {
    return cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
}

// ---------------------------------------------------------------- 16-byte vectors
// A row of n elements is `head` elements up to a 16-byte boundary, n_vec
// vectors, and `tail` elements, so that any row start gets wide loads.
template <class T>
struct Vec {
    static constexpr int N = 16 / (int)sizeof(T);
};

struct RowSpan {
    int head, n_vec, tail;
};
template <class T>
__device__ __forceinline__ RowSpan row_span(const T *row, int n) {
    const int off = (int)((uintptr_t)row & 15);
    RowSpan s;
    s.head = off ? (16 - off) / (int)sizeof(T) : 0;
    if (s.head > n) s.head = n;
    s.n_vec = (n - s.head) / Vec<T>::N;
    s.tail = n - s.head - s.n_vec * Vec<T>::N;
    return s;
}

__device__ __forceinline__ uint4 load16(const void *p) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "l"(p));
    return v;
}
// For arrays that the same kernel writes (in place).
__device__ __forceinline__ uint4 load16_rw(const void *p) {
    uint4 v;
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "l"(p));
    return v;
}
// (Not a barrier to the compiler: loads of what it does not overwrite may pass.)
__device__ __forceinline__ void store16(void *p, uint4 v) {
    asm volatile("st.global.v4.u32 [%0], {%1, %2, %3, %4};" ::"l"(p), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w));
}

template <class T>
__device__ __forceinline__ void unpack(uint4 v, float (&x)[Vec<T>::N]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (sizeof(T) == 4) {
            x[i] = __uint_as_float(w[i]);
        } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
            x[2 * i] = __uint_as_float(w[i] << 16);
            x[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
        } else {
            const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
            x[2 * i] = f.x;
            x[2 * i + 1] = f.y;
        }
    }
}
template <class T>
__device__ __forceinline__ uint4 pack(const float (&x)[Vec<T>::N]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (sizeof(T) == 4) {
            w[i] = __float_as_uint(x[i]);
        } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
            const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
            w[i] = *reinterpret_cast<const uint32_t *>(&h);
        } else {
            const __half2 h = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
            w[i] = *reinterpret_cast<const uint32_t *>(&h);
        }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}
// A vector of -infinity.
template <class T>
__device__ __forceinline__ uint4 masked16() {
    const uint32_t w = sizeof(T) == 4 ? 0xFF800000u : std::is_same<T, __half>::value ? 0xFC00FC00u : 0xFF80FF80u;
    return make_uint4(w, w, w, w);
}

// Two f32 operations in one instruction.
__device__ __forceinline__ float2 add2(float2 a, float2 b) { return __fadd2_rn(a, b); }
__device__ __forceinline__ float2 mul2(float2 a, float2 b) { return __fmul2_rn(a, b); }
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) { return __ffma2_rn(a, b, c); }

// Maximum that keeps a NaN.
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// ---------------------------------------------------------------- softmax sums
// Running softmax sums of one thread: the maximum m of what it has seen (a
// NaN is passed over), and relative to it s = sum 2^y and t = sum 2^y y with y
// = (z - m) scale, scale = log2(e) / temperature.  The difference z - m is
// taken before the product, so a common offset of the logits costs no
// accuracy.  y is held at -256, where 2^y is 0: masked logits (-infinity, or a
// type's lowest value) then add 0 to t and not 0 * infinity.  A NaN or
// +infinity makes s NaN.
//
// FINE sums count the logits that equal the maximum in n and leave their ones
// out of s: beside a sure token (log s near 0) the small rest then keeps its
// own 24 bits instead of those that 1 + rest leaves it.  It costs two
// instructions per logit; n is 0 otherwise.
struct SoftSums {
    float m = -INFINITY, s = 0.0f, t = 0.0f, n = 0.0f;

    // Makes v the maximum if it is above the present one.
    __device__ __forceinline__ void raise(float v, float scale) {
        if (v > m) {
            const float dy = fmaxf((m - v) * scale, -256.0f), f = ex2(dy), all = s + n;
            t = f * fmaf(dy, all, t);
            s = all * f;
            n = 0.0f;
            m = v;
        }
    }
    // What z is measured from: the maximum, or 0 while there is none.
    __device__ __forceinline__ float base() const { return m == -INFINITY ? 0.0f : m; }
    // One logit (the maximum counts it already).
    template <bool FINE = false>
    __device__ __forceinline__ void add(float z, float scale) {
        const float y = max_nan((z - base()) * scale, -256.0f), e = ex2(y);
        if (FINE && y == 0.0f)
            n += 1.0f;
        else
            s += e;
        t = fmaf(e, y, t);
    }
    // log(s + n).
    template <bool FINE = false>
    __device__ __forceinline__ float log_sum() const {
        return FINE ? (float)log((double)n + (double)s) : logf(s);
    }
};

// The largest of U vectors' elements; a NaN is passed over.  16-bit types are
// compared in pairs.
template <class T, int U>
__device__ __forceinline__ float batch_max(const uint4 (&raw)[U]) {
    if constexpr (sizeof(T) == 4) {
        float m = -INFINITY;
#pragma unroll
        for (int u = 0; u < U; ++u)
            m = fmaxf(m, fmaxf(fmaxf(__uint_as_float(raw[u].x), __uint_as_float(raw[u].y)),
                               fmaxf(__uint_as_float(raw[u].z), __uint_as_float(raw[u].w))));
        return m;
    } else {
        using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
        auto as = [](uint32_t w) { return *reinterpret_cast<T2 *>(&w); };
        T2 m = as(masked16<T>().x);
#pragma unroll
        for (int u = 0; u < U; ++u)
            m = __hmax2(m, __hmax2(__hmax2(as(raw[u].x), as(raw[u].y)), __hmax2(as(raw[u].z), as(raw[u].w))));
        return fmaxf(to_f32(m.x), to_f32(m.y));
    }
}

// Adds U vectors to a thread's sums (t only with ENT); returns their maximum.
// (Masked logits are not counted in n: y is not 0 there, as base is 0 while
// there is no maximum.)  Two partial sums each, one of a vector's even elements and one of its odd
// ones, in pairs of f32 operations.
template <class T, int U, bool ENT, bool FINE = false>
__device__ __forceinline__ float add_batch(const uint4 (&raw)[U], SoftSums &a, float scale) {
    const float bm = batch_max<T, U>(raw);
    a.raise(bm, scale);
    const float base = a.base();
    const float2 nb = make_float2(-base, -base), sc = make_float2(scale, scale);
    float2 s = make_float2(0.0f, 0.0f), t = s;
#pragma unroll
    for (int u = 0; u < U; ++u) {
        float x[Vec<T>::N];
        unpack<T>(raw[u], x);
#pragma unroll
        for (int i = 0; i < Vec<T>::N; i += 2) {
            float2 y = mul2(add2(make_float2(x[i], x[i + 1]), nb), sc);
            if (ENT) y = make_float2(max_nan(y.x, -256.0f), max_nan(y.y, -256.0f));
            float2 e = make_float2(ex2(y.x), ex2(y.y));
            if (ENT) t = fma2(e, y, t);
            if (FINE) {
                a.n += (y.x == 0.0f ? 1.0f : 0.0f) + (y.y == 0.0f ? 1.0f : 0.0f);
                e = make_float2(y.x == 0.0f ? 0.0f : e.x, y.y == 0.0f ? 0.0f : e.y);
            }
            s = add2(s, e);
        }
    }
    a.s += s.x + s.y;
    if (ENT) a.t += t.x + t.y;
    return bm;
}
// The same for those of U vectors that lie at v, v + NT, ... below v1.
template <class T, int NT, int U, bool ENT, bool FINE = false>
__device__ __forceinline__ float add_some(const uint4 (&raw)[U], int v, int v1, SoftSums &a, float scale) {
    float bm = -INFINITY;
#pragma unroll
    for (int u = 0; u < U; ++u)
        if (v + u * NT < v1) {
            const uint4 one[1] = {raw[u]};
            bm = fmaxf(bm, add_batch<T, 1, ENT, FINE>(one, a, scale));
        }
    return bm;
}

// Adds the vectors v0 <= v < v1 of `body` to the sums of a team of NT threads,
// of which this is thread `tid`, U to a thread at a time.  each(batch, maximum)
// is called for every U; returns the number of these.  With MASK a last batch
// that is not full counts its missing vectors as masked ones.  (Other warps'
// work covers the loads: fetching the next batch ahead measured 213 us a pass
// over 4096 rows of 131072 bf16, eight vectors at a time without it 207 in the same run.)
template <class T, int NT, int U, bool ENT, bool MASK = false, bool FINE = false, class F>
__device__ __forceinline__ int stream_sums(const T *body, int v0, int v1, int tid, float scale, SoftSums &sums, F &&each) {
    int batch = 0, v = v0 + tid;
    const uint4 *at = (const uint4 *)body + v;
    for (; v < v1; ++batch) {
        uint4 raw[U];
        if (v + (U - 1) * NT < v1) {
#pragma unroll
            for (int u = 0; u < U; ++u) raw[u] = load16_rw(at + u * NT);
            each(batch, add_batch<T, U, ENT, FINE>(raw, sums, scale));
        } else {
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (v + u * NT < v1)
                    raw[u] = load16_rw(at + u * NT);
                else if (MASK)
                    raw[u] = masked16<T>();
            each(batch, MASK ? add_batch<T, U, ENT, FINE>(raw, sums, scale) : add_some<T, NT, U, ENT, FINE>(raw, v, v1, sums, scale));
        }
        at += U * NT;
        v += U * NT;
    }
    return batch;
}

// Asynchronous copies to shared memory: 16 bytes, a group of them, and the
// wait until at most N groups of this thread are still on their way.
__device__ __forceinline__ void copy_async16(void *to, const void *from) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(to)), "l"(from) : "memory");
}
// The first `bytes` of 16, the rest zeros (none of it is read); 4 bytes.
__device__ __forceinline__ void copy_async16_part(void *to, const void *from, int bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"((uint32_t)__cvta_generic_to_shared(to)), "l"(from), "r"(bytes)
                 : "memory");
}
__device__ __forceinline__ void copy_async4(void *to, const void *from) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"((uint32_t)__cvta_generic_to_shared(to)), "l"(from) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// The cluster's barrier; what a thread wrote before cluster_arrive is seen after the
// wait, the relaxed one promises nothing.  Every thread of the cluster takes part.
__device__ __forceinline__ void cluster_arrive_relaxed() { asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

// The largest of a warp's values; a NaN is passed over.
__device__ __forceinline__ float warp_max1(float v) {
    float r;
    asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
    return r;
}

// A warp's sums joined, in all its lanes (t only with ENT, n only with FINE).
template <bool ENT, bool FINE = false>
__device__ __forceinline__ SoftSums warp_join(SoftSums a, float scale) {
    SoftSums r;
    r.m = warp_max1(a.m);
    // A thread without a logit above -infinity holds s = 0, or NaN.
    if (a.m != -INFINITY) a.raise(r.m, scale);
    r.s = warp_sum(a.s);
    if (ENT) r.t = warp_sum(a.t);
    if (FINE) r.n = warp_sum(a.n);
    return r;
}

// The parts that n <= 32 places hold, joined in a fixed order in every lane of a warp.
template <bool ENT, bool FINE = false>
__device__ __forceinline__ SoftSums join_places(const float4 *places, int n, float scale) {
    SoftSums a;
    const int lane = threadIdx.x & 31;
    if (lane < n) {
        const float4 p = places[lane];
        a.m = p.x;
        a.s = p.y;
        a.t = p.z;
        a.n = p.w;
    }
    return warp_join<ENT, FINE>(a, scale);
}

// Every thread's sums joined over a block of NT with one barrier; all threads
// get the result.  `places` holds a float4 per warp and must not be in use.
template <int NT, bool FINE>
__device__ __forceinline__ SoftSums block_join(const SoftSums &a, float scale, float4 *places) {
    const SoftSums w = warp_join<true, FINE>(a, scale);
    if ((threadIdx.x & 31) == 0) places[threadIdx.x >> 5] = make_float4(w.m, w.s, w.t, w.n);
    __syncthreads();
    return join_places<true, FINE>(places, NT / 32, scale);
}

}  // namespace nk
