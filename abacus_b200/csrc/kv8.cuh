// The 8-bit cache's numbers: blocks of 16 tokens with a scale, in two forms (csrc/kv8.cu says how they are made).
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <stdint.h>
#include <type_traits>

#include "common.cuh"

#define KV8_PAGE 64
#define KV8_BLOCK 16
#define KV8_PAGE_BLOCKS (KV8_PAGE / KV8_BLOCK)
enum { KV8_INT8 = 0, KV8_E4M3 = 1 };

template <int FORM> __host__ __device__ constexpr float kv8_top() { return FORM == KV8_INT8 ? 127.0f : 448.0f; }

// Eight bfloat16 values in 8 bits each, `most` the largest magnitude of their block (0: all come out as zero).
template <int FORM> __device__ __forceinline__ uint2 kv8_pack(uint4 x, float most) {
    const __nv_bfloat162 *h = (const __nv_bfloat162 *)&x;
    uint32_t out[2] = {0, 0};
    // x * (top / 128) and most / 128 are exact, and stay below infinity
    const float top = kv8_top<FORM>() / 512.0f, whole = most / 512.0f;
#pragma unroll
    for (int e = 0; e < 4; e++) {
        float2 f = __bfloat1622float2(h[e]);
        f.x = whole > 0.0f ? f.x * top / whole : 0.0f, f.y = whole > 0.0f ? f.y * top / whole : 0.0f;
        uint32_t pair;
        if constexpr (FORM == KV8_INT8) {
            const int lo = __float2int_rn(fminf(fmaxf(f.x, -127.0f), 127.0f)) + 128, hi = __float2int_rn(fminf(fmaxf(f.y, -127.0f), 127.0f)) + 128;
            pair = (uint32_t)lo | (uint32_t)hi << 8;
        } else {
            pair = __nv_cvt_float2_to_fp8x2(f, __NV_SATFINITE, __NV_E4M3);
        }
        out[e >> 1] |= pair << (16 * (e & 1));
    }
    return make_uint2(out[0], out[1]);
}
// Four numbers of a word as float32 (without the scale).
template <int FORM> __device__ __forceinline__ void kv8_unpack(uint32_t w, float *v) {
    if constexpr (FORM == KV8_INT8) {
#pragma unroll
        for (int e = 0; e < 4; e++) v[e] = (float)((int)(w >> (8 * e) & 0xff) - 128);
    } else {
#pragma unroll
        for (int e = 0; e < 2; e++) {
            const __half2_raw r = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w >> (16 * e) & 0xffff), __NV_E4M3);
            const float2 f = __half22float2(*(const __half2 *)&r);
            v[2 * e] = f.x, v[2 * e + 1] = f.y;
        }
    }
}

// The page of a position, 0 where the table names one that is not among the pool's n_pages (and a status bit says so: nothing
// outside the pool is touched).
#define KV8_BAD_PAGE 2
__device__ __forceinline__ int kv8_page(const PagedCache &c, int n_pages, int slot, int pos, int *status) {
    const int page = cache_page(c, slot, pos);
    if ((unsigned)page < (unsigned)n_pages) return page;
    atomicOr(status + 2, KV8_BAD_PAGE);
    return 0;
}

// The largest i in [0, n) with below(values[i], i), -1 if there is none; below is true up to some place and false from there on.
// A whole warp looks together, 32 places a step.
template <typename Below>
__device__ __forceinline__ int last_not_above(const int *values, int n, int lane, Below below) {
    int lo = 0, hi = n;  // the answer + 1 is in [lo, hi]
    while (lo < hi) {
        const int step = (hi - lo + 31) / 32;
        const int at = lo + step * (lane + 1) - 1;  // the last place of this lane's run
        const unsigned yes = __ballot_sync(0xffffffffu, at < hi && below(values[at], at));
        const int runs = __popc(yes);  // runs that are below to their last place
        lo += runs * step;
        hi = min(hi, lo + step - 1);
    }
    return lo - 1;
}
