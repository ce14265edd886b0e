// nk_head.cuh -- device helpers of the operators at the model's end.
#pragma once

#include <cmath>
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

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

__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

__device__ __forceinline__ float block_max(float v, float *red) {
    v = warp_max(v);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    __syncthreads();
    if (lane == 0) red[warp] = v;
    __syncthreads();
    return warp_max(lane < (int)(blockDim.x >> 5) ? red[lane] : -INFINITY);
}

// Order-preserving u32 of a float; -0 counts as +0.
__device__ __forceinline__ uint32_t order_key(float x) {
    const uint32_t b = __float_as_uint(x + 0.0f);
    return b ^ ((b >> 31) ? 0xFFFFFFFFu : 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) {
    return __uint_as_float(k ^ ((k >> 31) ? 0x80000000u : 0xFFFFFFFFu));
}

// Running softmax sums of one thread: the maximum m of what it has seen, and
// relative to it s = sum 2^y and t = sum 2^y y with y = (z - m) scale, scale =
// log2(e) / temperature.  The difference z - m is taken before the product, so
// a common offset of the logits costs no accuracy.  y is held at -256 in t, where 2^y is 0: masked
// logits (-infinity, or a type's lowest value) add 0 and not 0 * infinity.
struct SoftSums {
    float m = -INFINITY, s = 0.0f, t = 0.0f;

    // Makes v the maximum if it is above the present one.
    __device__ __forceinline__ void raise(float v, float scale) {
        if (v > m) {
            const float dy = fmaxf((m - v) * scale, -256.0f), f = ex2(dy);
            t = f * fmaf(dy, s, t);
            s *= f;
            m = v;
        }
    }
    // What z is measured from: the maximum, or 0 while there is none.
    __device__ __forceinline__ float base() const { return m == -INFINITY ? 0.0f : m; }
    __device__ __forceinline__ void add(float z, float base, float scale) {
        const float y = (z - base) * scale, e = ex2(y);
        s += e;
        t = fmaf(e, fmaxf(y, -256.0f), t);
    }
};

// Every thread's sums joined over the block in a fixed order; all threads get
// the result.
__device__ __forceinline__ SoftSums block_join(SoftSums a, float scale, float *red) {
    SoftSums r;
    r.m = block_max(a.m, red);
    // A thread without a logit above -infinity holds s = 0, or NaN.
    const float keep_s = a.s, keep_t = a.t;
    if (a.m != -INFINITY) a.raise(r.m, scale);
    r.s = block_sum(a.m == -INFINITY ? keep_s : a.s, red);
    r.t = block_sum(a.m == -INFINITY ? keep_t : a.t, red);
    return r;
}

}  // namespace nk
