// The sums that log probabilities and entropies are made of, and joining them.
#pragma once
#include <cuda_runtime.h>

#define LOGPROBS_FAR (-1e30f)  // a distance below the maximum at which nothing is left, and a finite one
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// Two float32 operations at once.
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(*(unsigned long long *)&r) : "l"(*(unsigned long long *)&a), "l"(*(unsigned long long *)&b));
    return r;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    float2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(*(unsigned long long *)&r) : "l"(*(unsigned long long *)&a), "l"(*(unsigned long long *)&b));
    return r;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(*(unsigned long long *)&r) : "l"(*(unsigned long long *)&a), "l"(*(unsigned long long *)&b), "l"(*(unsigned long long *)&c));
    return r;
}
// Maximum m; l = sum e^(x - m) and t = sum (x - m) e^(x - m). Without elements m is the lowest number and l is zero.
struct __align__(16) RowSums {
    float m, l, t, pad;
};
__device__ __forceinline__ RowSums joined(RowSums a, RowSums b) {
    RowSums r;
    r.m = fmaxf(a.m, b.m), r.pad = 0.0f;
    const float da = fmaxf(a.m - r.m, LOGPROBS_FAR), db = fmaxf(b.m - r.m, LOGPROBS_FAR);
    const float ea = ex2(da * 1.4426950408889634f), eb = ex2(db * 1.4426950408889634f);
    r.l = fmaf(a.l, ea, b.l * eb);
    r.t = fmaf(fmaf(a.l, da, a.t), ea, fmaf(b.l, db, b.t) * eb);
    return r;
}
// Of the 2 * `half` neighbouring lanes together, in every one of them.
__device__ __forceinline__ RowSums joined_lanes(RowSums a, int half) {
    for (int o = half; o > 0; o >>= 1) {
        RowSums b;
        b.m = __shfl_xor_sync(0xffffffffu, a.m, o), b.l = __shfl_xor_sync(0xffffffffu, a.l, o), b.t = __shfl_xor_sync(0xffffffffu, a.t, o);
        a = joined(a, b);
    }
    return a;
}
