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

// An 8-bit cache of one schedule entry, as the launchers get it (kernels/ops.py: Kv8Cache has the same fields in the same order).
struct Kv8Cache {
    void *k, *v;        // [pages, kv heads, 64, head_dim]
    float *scales;      // [pages, kv heads, 2 (keys, values), 4]
    void *open;         // bfloat16 [slots, 2, kv heads, 16, head_dim]
    const int *page_table;
    int *status;
    int table_width, ring_pages, n_pages, n_slots, n_kv_heads, head_dim, form, pad;
};

template <int FORM> __host__ __device__ constexpr float kv8_top() { return FORM == KV8_INT8 ? 127.0f : 448.0f; }

// Eight bfloat16 values in 8 bits each; `by` and `inverse` as kv8_steps makes them of the block's largest magnitude.
// 127 x / most comes as x times a reciprocal, up to 2^-22 off, and is then rounded to 18 bits: where it is halfway between two steps it
// is exactly that again (8 bits), and where it is not it is 2^-16 or more away, relative to itself (2 * 127 x and an odd number times most are
// whole numbers of 16 bits, at least 1 apart; 254 and 255 come closest, 126.50196; 448 x with fewer bits), which is more than the 2^-18
// that the rounding moves it. So the rounding to a step is that of the exact quotient, ties to even. A
// division takes three times as long.
struct Kv8Steps {
    float by, inverse;
};
template <int FORM> __device__ __forceinline__ Kv8Steps kv8_steps(float most) {
    const float by = most < 5e-20f ? 1.8446744073709552e19f : 1.0f;  // 2^64: no reciprocal overflows
    return {by, most > 0.0f ? kv8_top<FORM>() / (most * by) : 0.0f};
}
template <int FORM> __device__ __forceinline__ uint2 kv8_pack(uint4 x, Kv8Steps s) {
    const uint32_t h[4] = {x.x, x.y, x.z, x.w};
    uint32_t out[2];
#pragma unroll
    for (int e = 0; e < 2; e++) {
        float q[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float f = __uint_as_float(i & 1 ? h[2 * e + i / 2] & 0xffff0000u : h[2 * e + i / 2] << 16);
            const float y = __fmul_rn(__fmul_rn(f, s.by), s.inverse), t = __fmul_rn(y, 65.0f);
            q[i] = __fsub_rn(t, __fsub_rn(t, y));
        }
        if constexpr (FORM == KV8_INT8) {  // + 1.5 * 2^23: the whole number in the low bits; + 128
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; i++) w[i] = __float_as_uint(__fadd_rn(q[i], 12582912.0f)) + 128u;
            out[e] = __byte_perm(__byte_perm(w[0], w[1], 0x0040), __byte_perm(w[2], w[3], 0x0040), 0x5410);
        } else {
            const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(q[0], q[1]), __NV_SATFINITE, __NV_E4M3);
            const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(q[2], q[3]), __NV_SATFINITE, __NV_E4M3);
            out[e] = lo | hi << 16;
        }
    }
    return make_uint2(out[0], out[1]);
}
// Four numbers of a word as float32 (without the scale).
template <int FORM> __device__ __forceinline__ void kv8_unpack(uint32_t w, float *v) {
    if constexpr (FORM == KV8_INT8) {  // 2^23 + b, less 2^23 + 128
        v[0] = __uint_as_float(__byte_perm(w, 0x4b000000u, 0x7440)) - 8388736.0f, v[1] = __uint_as_float(__byte_perm(w, 0x4b000000u, 0x7441)) - 8388736.0f;
        v[2] = __uint_as_float(__byte_perm(w, 0x4b000000u, 0x7442)) - 8388736.0f, v[3] = __uint_as_float(__byte_perm(w, 0x4b000000u, 0x7443)) - 8388736.0f;
    } else {
#pragma unroll
        for (int e = 0; e < 2; e++) {
            const __half2_raw r = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w >> (16 * e) & 0xffff), __NV_E4M3);
            const float2 f = __half22float2(*(const __half2 *)&r);
            v[2 * e] = f.x, v[2 * e + 1] = f.y;
        }
    }
}

// The page of a position, 0 where the table names one that is not among the pool's n_pages (and a bit of `bad`, or of the status, says
// so: nothing outside the pool is touched).
#define KV8_BAD_PAGE 2
#define KV8_BAD_SLOT 4
__device__ __forceinline__ int kv8_page(const PagedCache &c, int n_pages, int slot, int pos, int &bad) {
    const int page = cache_page(c, slot, pos);
    if ((unsigned)page < (unsigned)n_pages) return page;
    bad |= KV8_BAD_PAGE;
    return 0;
}
__device__ __forceinline__ int kv8_page(const PagedCache &c, int n_pages, int slot, int pos, int *status) {
    int bad = 0;
    const int page = kv8_page(c, n_pages, slot, pos, bad);
    if (bad) atomicOr(status + 2, bad);
    return page;
}

// The slot, 0 where it is not one of the cache's n_slots (a bit says so).
__device__ __forceinline__ int kv8_slot(int slot, int n_slots, int &bad) {
    if ((unsigned)slot < (unsigned)n_slots) return slot;
    bad |= KV8_BAD_SLOT;
    return 0;
}
__device__ __forceinline__ int kv8_slot(int slot, int n_slots, int *status) {
    int bad = 0;
    slot = kv8_slot(slot, n_slots, bad);
    if (bad) atomicOr(status + 2, bad);
    return slot;
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
