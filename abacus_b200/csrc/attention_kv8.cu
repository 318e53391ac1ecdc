// Attention of a step's rows over a cache held in 8 bits (csrc/kv8.cu): a few new tokens a sequence against everything the
// cache holds of it, each row to its own position.
//
// out = sum_j softmax_j(scale q . k_j) v_j over the keys j <= position (and within the window): keys of whole blocks are
// q_j s_b with the block's scale s_b, so a score is s_b (q . q_j) and a value's weight p_j s_b; keys of the sequence's open
// block are bfloat16.
//
// A cluster of up to 8 CTAs takes a row, a kv head and up to 16 of its query heads, the pages dealt out among its CTAs. One warp
// of a CTA keeps a ring of pages (keys, values, scales) coming by TMA; four warps take a block of 16 tokens of every page
// each, with the block's two scales. Both products run on warp-level tensor-core instructions of 16-bit floats, the query heads
// as the 16 rows: an 8-bit number is a float16 number exactly, and q is one too once each head's row is brought
// below 1 by a power of two (what of a head lies 2^-14 below its largest element keeps an absolute error of 2^-25 of that).
// The softmax weights are p_j s_b 2^-u in float16, 2^-12 off at most, u chosen per row so that the largest ever seen is about
// 1: a block of small values with large weights counts as precisely as one of large values. Scores, maximum, sum and output are float32.
// The open block's keys and values go through the same products in bfloat16, its weights as two bfloat16 parts.
//
// An 8-bit number's way into a register pair: bytes 0 and 1 of a word with 0x64 above each are the float16 numbers 1024 + b, and
// 1152 less is q (one permute and one subtraction for two numbers); e4m3 has a conversion for two. The instructions' own order of the
// inner dimension is free as long as both operands follow it: a thread's four neighbouring bytes of a key row are the pairs
// that the instruction calls (2c, 2c + 1) and (2c + 8, 2c + 9), and q is read in that order. Values come transposed, two
// tokens and two columns to a word, so that even columns are one tile of eight and odd columns another.
#define ABK_DEFINE_ERROR
#include "common.cuh"
#include "tc_common.cuh"
#include "tensor_map.cuh"
#include "mma_tiles.cuh"
#include "kv8.cuh"

#define KV8_HEADS 16  // query heads a cluster takes at once: the rows of the tensor-core tile
#define KV8_MAX_STAGES 24
#define KV8_RING_BYTES (96 * 1024)  // keys and values in flight a CTA when an SM holds two
#define KV8_THREADS 160
#define KV8_MAX_SPLITS 8

struct AttnKv8 {
    const __nv_bfloat16 *q;
    long long q_row;
    __nv_bfloat16 *out;
    int n_heads, n_kv_heads, runs;
    float scale_log2;
    int window;
    const int *token_seq, *token_pos, *seq_slot, *seq_len_after;
    PagedCache cache;
    const float *scales;
    const __nv_bfloat16 *open;
    int n_pages, *status, stages;
};

__device__ __forceinline__ void mma_f16(float *c, const uint32_t *a, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
    __half2 t = __floats2half2_rn(lo, hi);
    return *(uint32_t *)&t;
}
// Numbers of the bytes of `w` that `select` names, as two float16.
template <int FORM, int LO, int HI> __device__ __forceinline__ uint32_t f16_of_bytes(uint32_t w) {
    if constexpr (FORM == KV8_INT8) {
        const uint32_t biased = __byte_perm(w, 0x64646464u, 0x4040 | LO | HI << 8);
        const __half2 t = __hsub2(*(const __half2 *)&biased, __half2half2(__ushort_as_half(0x6480)));  // 1152
        return *(const uint32_t *)&t;
    } else {
        const __half2_raw t = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(__byte_perm(w, 0, LO | HI << 4) & 0xffff), __NV_E4M3);
        return (uint32_t)t.x | (uint32_t)t.y << 16;
    }
}
// Shared address of 16-byte piece `piece` of token `t` in a page of HD-byte rows, written by TMA as rows of 128 bytes with the
// 128-byte swizzle (two tokens to a row where HD is 64).
template <int HD> __device__ __forceinline__ uint32_t token_piece(uint32_t base, int t, int piece) {
    if constexpr (HD == 128) return sw128(base, t, piece);
    return sw128(base, t >> 1, (t & 1) * 4 + piece);
}
// 2^u > |x| for the u returned, tight to a factor of two (x a float32 number; -126 for zero)
__device__ __forceinline__ float power_above(float x) { return (float)((__float_as_int(x) >> 23 & 0xff) - 126); }

template <int HD, int FORM>
__global__ void __launch_bounds__(KV8_THREADS, 2) attention_kv8_kernel(const __grid_constant__ CUtensorMap k_map,
                                                                    const __grid_constant__ CUtensorMap v_map, AttnKv8 p) {
    constexpr int TILE_BYTES = KV8_PAGE * HD, KS = HD / 16;
    extern __shared__ uint8_t kv8_raw[];
    uint8_t *smem = (uint8_t *)(((uintptr_t)kv8_raw + 1023) & ~(uintptr_t)1023);
    const int stages = p.stages, group = p.n_heads / p.n_kv_heads;
    const int kvh = blockIdx.y / p.runs, g0 = (blockIdx.y - kvh * p.runs) * KV8_HEADS, heads = min(KV8_HEADS, group - g0);
    uint8_t *k_s = smem, *v_s = k_s + stages * TILE_BYTES;
    float *scale_s = (float *)(v_s + stages * TILE_BYTES);  // [stages][2][4]
    float *cta_o = scale_s + stages * 2 * KV8_PAGE_BLOCKS;  // [heads][HD]: what the other CTAs read
    float *cta_mlu = cta_o + heads * HD;                    // [heads][4]: maximum, sum, the output's exponent
    float *warp_o = cta_mlu + heads * 4;                    // [4 warps][heads][HD]
    float *warp_mlu = warp_o + 4 * heads * HD;              // [4 warps][heads][4]
    __shared__ uint64_t full[KV8_MAX_STAGES], empty[KV8_MAX_STAGES];
    __shared__ int failed;

    const int split = (int)tc::cluster_rank(), splits = (int)tc::cluster_size(), r = blockIdx.z;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        failed = 0;
        for (int s = 0; s < stages; s++) tc::mbar_init(&full[s], 1), tc::mbar_init(&empty[s], 4);
        tc::mbar_init_fence();
        tc::tma_prefetch_map(&k_map), tc::tma_prefetch_map(&v_map);
    }
    pdl_wait();
    __syncthreads();
    __nv_bfloat16 *out = p.out + ((long long)r * p.n_heads + kvh * group + g0) * HD;
    const int seq = p.token_seq[r];
    if (seq < 0) {  // padding: zeros, written by the first CTA; the whole cluster leaves here
        if (split == 0)
            for (int i = threadIdx.x; i < heads * HD; i += KV8_THREADS) out[i] = __float2bfloat16_rn(0.0f);
        return;
    }
    const int pos = p.token_pos[r], slot = p.seq_slot[seq], closed = p.seq_len_after[seq] / KV8_BLOCK;
    const int lo = p.window > 0 && pos - p.window + 1 > 0 ? pos - p.window + 1 : 0;
    const int first_page = lo / KV8_PAGE, last_page = pos / KV8_PAGE, n_pages = last_page - first_page + 1;
    const int active = min(splits, n_pages);  // CTAs with fewer pages than ranks have nothing to add
    const int mine = split < n_pages ? (n_pages - 1 - split) / splits + 1 : 0;  // this CTA's pages

    if (warp == 4) {
        int issued = 0;
        bool go = true;
        for (int base = 0; base < mine && go; base += 32) {
            int page_lane = 0;  // every lane looks up one of the next 32 pages
            if (base + lane < mine)
                page_lane = kv8_page(p.cache, p.n_pages, slot, (first_page + split + (base + lane) * splits) * KV8_PAGE, p.status);
            const int n = min(32, mine - base);
            for (int i = 0; i < n && go; i++, issued++) {
                const long long tile = (long long)__shfl_sync(0xffffffffu, page_lane, i) * p.n_kv_heads + kvh;
                int bad = 0;
                if (lane == 0) {
                    const int s = issued % stages;
                    if (!tc::mbar_wait(&empty[s], ((issued / stages) & 1) ^ 1)) {
                        bad = 1;
                    } else {
                        tc::mbar_expect_tx(&full[s], 2 * TILE_BYTES + 2 * KV8_PAGE_BLOCKS * 4);
                        tc::tma_load_2d(k_s + s * TILE_BYTES, &k_map, 0, (int)(tile * (TILE_BYTES / 128)), &full[s]);
                        tc::tma_load_2d(v_s + s * TILE_BYTES, &v_map, 0, (int)(tile * (TILE_BYTES / 128)), &full[s]);
                        tc::bulk_load(scale_s + s * 2 * KV8_PAGE_BLOCKS, p.scales + tile * 2 * KV8_PAGE_BLOCKS, 2 * KV8_PAGE_BLOCKS * 4, &full[s]);
                    }
                }
                if (__shfl_sync(0xffffffffu, bad, 0)) go = false;
            }
        }
        if (!go && lane == 0) {  // let the copies in flight land before the CTA's memory goes away
            failed = 1;
            issued--;  // the copy that was not issued
            for (int i = max(0, issued - stages); i < issued; i++) tc::mbar_wait(&full[i % stages], (i / stages) & 1);
        }
    } else if (mine > 0) {
        const int row_lo = lane >> 2, row_hi = row_lo + 8, c4 = 4 * (lane & 3);  // this thread's two rows: query heads
        const __nv_bfloat16 *q_lo = p.q + (long long)r * p.q_row + (long long)(kvh * group + g0 + row_lo) * HD + c4, *q_hi = q_lo + 8 * HD;
        uint32_t qf[KS][4];
        float unit_lo, unit_hi;  // what a row's scores are multiplied by
        {
            uint2 raw_lo[KS], raw_hi[KS];
            float most_lo = 0.0f, most_hi = 0.0f;
#pragma unroll
            for (int ks = 0; ks < KS; ks++) {
                raw_lo[ks] = row_lo < heads ? *(const uint2 *)(q_lo + 16 * ks) : make_uint2(0, 0);
                raw_hi[ks] = row_hi < heads ? *(const uint2 *)(q_hi + 16 * ks) : make_uint2(0, 0);
            }
            auto largest = [](float most, uint32_t w) {
                const float2 f = __bfloat1622float2(*(const __nv_bfloat162 *)&w);
                return fmaxf(most, fmaxf(fabsf(f.x), fabsf(f.y)));
            };
#pragma unroll
            for (int ks = 0; ks < KS; ks++) {
                most_lo = largest(largest(most_lo, raw_lo[ks].x), raw_lo[ks].y);
                most_hi = largest(largest(most_hi, raw_hi[ks].x), raw_hi[ks].y);
            }
            const float down_lo = exp2f(-power_above(quad_max(most_lo))), down_hi = exp2f(-power_above(quad_max(most_hi)));
            unit_lo = p.scale_log2 / down_lo, unit_hi = p.scale_log2 / down_hi;
            auto scaled = [](uint32_t w, float by) {
                const float2 f = __bfloat1622float2(*(const __nv_bfloat162 *)&w);
                return pack_f16(f.x * by, f.y * by);
            };
#pragma unroll
            for (int ks = 0; ks < KS; ks++) {
                qf[ks][0] = scaled(raw_lo[ks].x, down_lo), qf[ks][1] = scaled(raw_hi[ks].x, down_hi);
                qf[ks][2] = scaled(raw_lo[ks].y, down_lo), qf[ks][3] = scaled(raw_hi[ks].y, down_hi);
            }
        }
        float o[2 * KS][4];  // tile 2c: the even columns of 16 c .., tile 2c + 1: the odd ones
#pragma unroll
        for (int nt = 0; nt < 2 * KS; nt++) o[nt][0] = o[nt][1] = o[nt][2] = o[nt][3] = 0.0f;
        float m_lo = -INFINITY, m_hi = -INFINITY, l_lo = 0.0f, l_hi = 0.0f, u_lo = -INFINITY, u_hi = -INFINITY;
        bool ok = true;
        int s = 0, phase = 0;
        const int j8 = lane >> 3, r8 = lane & 7;
        // scores (in units of log2) to weights: sc becomes p_j 2^-n, l and m follow, o is brought to its new exponent; v_scale is
        // the block's. What is left to multiply a row's weights with is returned in f_lo, f_hi.
        auto softmax = [&](float (*sc)[4], int key0, float by_lo, float by_hi, float v_scale, float &f_lo, float &f_hi) {
            float mx_lo = -INFINITY, mx_hi = -INFINITY;
#pragma unroll
            for (int nt = 0; nt < 2; nt++) {
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const int key = key0 + 8 * nt + 2 * (lane & 3) + (e & 1);
                    sc[nt][e] = key >= lo && key <= pos ? sc[nt][e] * (e < 2 ? by_lo : by_hi) : -INFINITY;
                }
                mx_lo = fmaxf(mx_lo, fmaxf(sc[nt][0], sc[nt][1]));
                mx_hi = fmaxf(mx_hi, fmaxf(sc[nt][2], sc[nt][3]));
            }
            // at least one of the 16 keys is visible, so the maxima are finite; references are whole powers of two
            const float a_lo = ceilf(quad_max(mx_lo)), a_hi = ceilf(quad_max(mx_hi)), above = power_above(v_scale);
            const float n_lo = fmaxf(m_lo, a_lo), n_hi = fmaxf(m_hi, a_hi);
            const float w_lo = fmaxf(u_lo, a_lo + above), w_hi = fmaxf(u_hi, a_hi + above);
            if (__any_sync(0xffffffffu, w_lo != u_lo || w_hi != u_hi)) {
                const float d_lo = exp2f(u_lo - w_lo), d_hi = exp2f(u_hi - w_hi);
#pragma unroll
                for (int nt = 0; nt < 2 * KS; nt++) o[nt][0] *= d_lo, o[nt][1] *= d_lo, o[nt][2] *= d_hi, o[nt][3] *= d_hi;
                u_lo = w_lo, u_hi = w_hi;
            }
            l_lo *= exp2f(m_lo - n_lo), l_hi *= exp2f(m_hi - n_hi);
            m_lo = n_lo, m_hi = n_hi;
#pragma unroll
            for (int nt = 0; nt < 2; nt++) {
                sc[nt][0] = exp2f(sc[nt][0] - n_lo), sc[nt][1] = exp2f(sc[nt][1] - n_lo);
                sc[nt][2] = exp2f(sc[nt][2] - n_hi), sc[nt][3] = exp2f(sc[nt][3] - n_hi);
                l_lo += sc[nt][0] + sc[nt][1], l_hi += sc[nt][2] + sc[nt][3];
            }
            f_lo = v_scale * exp2f(n_lo - u_lo), f_hi = v_scale * exp2f(n_hi - u_hi);
        };
        for (int pg = first_page + split; pg <= last_page; pg += splits) {
            if (!tc::mbar_wait(&full[s], phase)) {
                ok = false;
                break;
            }
            const int key0 = pg * KV8_PAGE + KV8_BLOCK * warp;  // this warp's block of the page
            if (key0 <= pos && key0 + KV8_BLOCK > lo) {
                float sc[2][4] = {}, f_lo, f_hi;
                if (key0 / KV8_BLOCK < closed) {
                    const uint32_t k_base = tc::smem_addr(k_s + s * TILE_BYTES), v_base = tc::smem_addr(v_s + s * TILE_BYTES);
                    const float k_scale = scale_s[s * 2 * KV8_PAGE_BLOCKS + warp], v_scale = scale_s[(s * 2 + 1) * KV8_PAGE_BLOCKS + warp];
#pragma unroll
                    for (int ks = 0; ks < KS; ks += 2) {
                        uint32_t w[4];
                        ldsm_x4(token_piece<HD>(k_base, KV8_BLOCK * warp + 8 * (j8 & 1) + r8, ks + (j8 >> 1)), w[0], w[1], w[2], w[3]);
#pragma unroll
                        for (int i = 0; i < 4; i++)
                            mma_f16(sc[i & 1], qf[ks + (i >> 1)], f16_of_bytes<FORM, 0, 1>(w[i]), f16_of_bytes<FORM, 2, 3>(w[i]));
                    }
                    softmax(sc, key0, unit_lo * k_scale, unit_hi * k_scale, v_scale, f_lo, f_hi);
                    uint32_t pf[4];
#pragma unroll
                    for (int nt = 0; nt < 2; nt++) {
                        pf[2 * nt] = pack_f16(sc[nt][0] * f_lo, sc[nt][1] * f_lo);
                        pf[2 * nt + 1] = pack_f16(sc[nt][2] * f_hi, sc[nt][3] * f_hi);
                    }
#pragma unroll
                    for (int c = 0; c < KS; c += 2) {
                        uint32_t w[4];
                        ldsm_x4_t(token_piece<HD>(v_base, KV8_BLOCK * warp + 8 * (j8 & 1) + r8, c + (j8 >> 1)), w[0], w[1], w[2], w[3]);
#pragma unroll
                        for (int i = 0; i < 2; i++) {
                            mma_f16(o[2 * (c + i)], pf, f16_of_bytes<FORM, 0, 2>(w[2 * i]), f16_of_bytes<FORM, 0, 2>(w[2 * i + 1]));
                            mma_f16(o[2 * (c + i) + 1], pf, f16_of_bytes<FORM, 1, 3>(w[2 * i]), f16_of_bytes<FORM, 1, 3>(w[2 * i + 1]));
                        }
                    }
                } else {  // the open block, as it came: once a row, by one warp of the cluster
                    const __nv_bfloat16 *open_k = p.open + ((long long)slot * 2 * p.n_kv_heads + kvh) * (KV8_BLOCK * HD),
                                        *open_v = open_k + (long long)p.n_kv_heads * (KV8_BLOCK * HD);
#pragma unroll
                    for (int ks = 0; ks < KS; ks++) {
                        const uint2 a = row_lo < heads ? *(const uint2 *)(q_lo + 16 * ks) : make_uint2(0, 0);
                        const uint2 b = row_hi < heads ? *(const uint2 *)(q_hi + 16 * ks) : make_uint2(0, 0);
                        const uint32_t qb[4] = {a.x, b.x, a.y, b.y};
#pragma unroll
                        for (int nt = 0; nt < 2; nt++) {
                            const uint2 k = *(const uint2 *)(open_k + (8 * nt + (lane >> 2)) * HD + 16 * ks + c4);
                            mma_bf16(sc[nt], qb, k.x, k.y);
                        }
                    }
                    softmax(sc, key0, p.scale_log2, p.scale_log2, 1.0f, f_lo, f_hi);
                    uint32_t high[4], low[4];
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const float f = i & 1 ? f_hi : f_lo, x = sc[i >> 1][2 * (i & 1)] * f, y = sc[i >> 1][2 * (i & 1) + 1] * f;
                        high[i] = pack_bf16(x, y);
                        const float2 back = __bfloat1622float2(*(const __nv_bfloat162 *)&high[i]);
                        low[i] = pack_bf16(x - back.x, y - back.y);
                    }
#pragma unroll
                    for (int c = 0; c < KS; c++) {
                        uint32_t v[4];  // tokens 2 c', 2 c' + 1, 2 c' + 8, 2 c' + 9; a token behind the position may hold anything
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            const int t = 2 * (lane & 3) + (i & 1) + 8 * (i >> 1);
                            v[i] = key0 + t <= pos ? *(const uint32_t *)(open_v + t * HD + 16 * c + 2 * (lane >> 2)) : 0u;
                        }
                        const uint32_t e0 = __byte_perm(v[0], v[1], 0x5410), e1 = __byte_perm(v[2], v[3], 0x5410);
                        const uint32_t d0 = __byte_perm(v[0], v[1], 0x7632), d1 = __byte_perm(v[2], v[3], 0x7632);
                        mma_bf16(o[2 * c], high, e0, e1), mma_bf16(o[2 * c], low, e0, e1);
                        mma_bf16(o[2 * c + 1], high, d0, d1), mma_bf16(o[2 * c + 1], low, d0, d1);
                    }
                }
            }
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(&empty[s]);
            if (++s == stages) s = 0, phase ^= 1;
        }
        if (!ok) failed = 1;
        l_lo = quad_sum(l_lo), l_hi = quad_sum(l_hi);
#pragma unroll
        for (int c = 0; c < KS; c++) {
            const int d = 16 * c + c4;
            if (row_lo < heads) *(float4 *)(warp_o + (warp * heads + row_lo) * HD + d) = make_float4(o[2 * c][0], o[2 * c + 1][0], o[2 * c][1], o[2 * c + 1][1]);
            if (row_hi < heads) *(float4 *)(warp_o + (warp * heads + row_hi) * HD + d) = make_float4(o[2 * c][2], o[2 * c + 1][2], o[2 * c][3], o[2 * c + 1][3]);
        }
        if ((lane & 3) == 0) {
            if (row_lo < heads) *(float4 *)(warp_mlu + (warp * heads + row_lo) * 4) = make_float4(m_lo, l_lo, u_lo, 0.0f);
            if (row_hi < heads) *(float4 *)(warp_mlu + (warp * heads + row_hi) * 4) = make_float4(m_hi, l_hi, u_hi, 0.0f);
        }
    }
    __syncthreads();
    if (failed && threadIdx.x == 0) atomicOr(p.status + 2, 1);
    auto share = [](float from, float to) { return from == -INFINITY ? 0.0f : exp2f(from - to); };
    // fold the four warps, in warp order, into this CTA's partial result
    if (mine > 0) {
        for (int i = threadIdx.x; i < heads * HD; i += KV8_THREADS) {
            const int g = i / HD, d = i - g * HD;
            float4 part[4];
            float m = -INFINITY, u = -INFINITY, l = 0.0f, acc = 0.0f;
            for (int w = 0; w < 4; w++) part[w] = *(const float4 *)(warp_mlu + (w * heads + g) * 4), m = fmaxf(m, part[w].x), u = fmaxf(u, part[w].z);
            for (int w = 0; w < 4; w++) {
                acc = fmaf(share(part[w].z, u), warp_o[(w * heads + g) * HD + d], acc);
                l = fmaf(share(part[w].x, m), part[w].y, l);
            }
            cta_o[i] = acc;
            if (d == 0) *(float4 *)(cta_mlu + g * 4) = make_float4(m, l, u, 0.0f);
        }
    }
    tc::cluster_sync();
    // every CTA folds its share of the output (four columns a thread) over the partial results, in CTA order
    const uint32_t o_addr = tc::smem_addr(cta_o), mlu_addr = tc::smem_addr(cta_mlu);
    for (int i = split + splits * threadIdx.x; i < heads * (HD / 4); i += splits * KV8_THREADS) {
        const int g = i / (HD / 4), d = 4 * (i - g * (HD / 4));
        float4 part[KV8_MAX_SPLITS], ov[KV8_MAX_SPLITS];
#pragma unroll
        for (int c = 0; c < KV8_MAX_SPLITS; c++) {
            if (c < active) {
                part[c] = tc::ld_cluster_f4(tc::peer_smem(mlu_addr + g * 16, c));
                ov[c] = tc::ld_cluster_f4(tc::peer_smem(o_addr + (g * HD + d) * 4, c));
            }
        }
        float m = -INFINITY, u = -INFINITY;
#pragma unroll
        for (int c = 0; c < KV8_MAX_SPLITS; c++)
            if (c < active) m = fmaxf(m, part[c].x), u = fmaxf(u, part[c].z);
        float l = 0.0f, a0 = 0.0f, a1 = 0.0f, a2 = 0.0f, a3 = 0.0f;
#pragma unroll
        for (int c = 0; c < KV8_MAX_SPLITS; c++) {
            if (c < active) {
                const float w = share(part[c].z, u);
                l = fmaf(share(part[c].x, m), part[c].y, l);
                a0 = fmaf(w, ov[c].x, a0), a1 = fmaf(w, ov[c].y, a1), a2 = fmaf(w, ov[c].z, a2), a3 = fmaf(w, ov[c].w, a3);
            }
        }
        const float by = exp2f(u - m) / l;
        *(uint2 *)(out + (long long)g * HD + d) = make_uint2(pack_bf16(a0 * by, a1 * by), pack_bf16(a2 * by, a3 * by));
    }
    tc::cluster_sync();  // nobody leaves while its partial result may still be read
}

// How many clusters of `splits` CTAs with `smem` bytes each the device holds at once (looked up once per shape).
static int kv8_resident_clusters(const void *kernel, int splits, int smem) {
    static std::mutex lock;
    static std::map<std::pair<const void *, std::pair<int, int>>, std::map<int, int>> known;  // .. -> device -> clusters
    int device = 0;
    cudaGetDevice(&device);
    std::lock_guard<std::mutex> guard(lock);
    auto &of_device = known[{kernel, {splits, smem}}];
    auto it = of_device.find(device);
    if (it != of_device.end()) return it->second;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(splits, 1, 1), cfg.blockDim = dim3(KV8_THREADS), cfg.dynamicSmemBytes = smem;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = splits, attr[0].val.clusterDim.y = 1, attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr, cfg.numAttrs = 1;
    int clusters = 0;
    if (cudaOccupancyMaxActiveClusters(&clusters, kernel, &cfg) != cudaSuccess) {
        cudaGetLastError();
        clusters = 0;
    }
    return of_device[device] = clusters;
}

// max_positions: no row's position reaches it (with the number of rows it fixes the grid; a captured graph passes its bound).
extern "C" int abk_attention_kv8(const void *q, long long q_row, void *out, int n_rows, int n_heads, int n_kv_heads, int head_dim,
                                 int form, float scale, int window, const int *token_seq, const int *token_pos, const int *seq_slot,
                                 const int *seq_len_after, const void *k, const void *v, const float *scales, const void *open,
                                 const int *page_table, int table_width, int ring_pages, int pool_pages, int max_positions, int *status,
                                 void *stream) {
    if (n_rows <= 0) return 0;
    if (head_dim != 64 && head_dim != 128) ABK_REFUSE("attention_kv8: head_dim %d is not 64 or 128", head_dim);
    if (form != KV8_INT8 && form != KV8_E4M3) ABK_REFUSE("attention_kv8: no 8-bit form %d", form);
    if (n_kv_heads < 1 || n_heads < 1 || n_heads % n_kv_heads) ABK_REFUSE("attention_kv8: %d heads do not divide into %d kv heads", n_heads, n_kv_heads);
    const int group = n_heads / n_kv_heads, runs = (group + KV8_HEADS - 1) / KV8_HEADS, heads = group < KV8_HEADS ? group : KV8_HEADS;
    if ((long long)n_kv_heads * runs > 65535 || n_rows > 65535) ABK_REFUSE("attention_kv8: %d rows or %d heads exceed a grid", n_rows, n_heads);
    if ((((uintptr_t)q | (uintptr_t)out) & 7) || (q_row & 3) || (((uintptr_t)scales | (uintptr_t)open) & 15))
        ABK_REFUSE("attention_kv8: q and out must be 8-byte aligned, scales and open blocks 16-byte aligned");
    CUtensorMap km, vm;
    const long long pool_rows = (long long)pool_pages * n_kv_heads * KV8_PAGE * head_dim / 128;
    int rc = tmap::bytes_in_rows_of_128(k, pool_rows, KV8_PAGE * head_dim / 128, &km);
    if (!rc) rc = tmap::bytes_in_rows_of_128(v, pool_rows, KV8_PAGE * head_dim / 128, &vm);
    if (rc) return rc;
    AttnKv8 p;
    p.q = (const __nv_bfloat16 *)q, p.q_row = q_row, p.out = (__nv_bfloat16 *)out, p.n_heads = n_heads, p.n_kv_heads = n_kv_heads;
    p.scale_log2 = scale * 1.4426950408889634f, p.window = window, p.token_seq = token_seq, p.token_pos = token_pos;
    p.seq_slot = seq_slot, p.seq_len_after = seq_len_after, p.cache.page_table = page_table, p.cache.table_width = table_width;
    p.cache.ring_pages = ring_pages, p.cache.tokens_per_page = KV8_PAGE, p.scales = scales, p.open = (const __nv_bfloat16 *)open;
    p.n_pages = pool_pages, p.status = status, p.runs = runs;
    void (*kernel)(CUtensorMap, CUtensorMap, AttnKv8) = nullptr;
    if (head_dim == 64) kernel = form == KV8_INT8 ? attention_kv8_kernel<64, KV8_INT8> : attention_kv8_kernel<64, KV8_E4M3>;
    else kernel = form == KV8_INT8 ? attention_kv8_kernel<128, KV8_INT8> : attention_kv8_kernel<128, KV8_E4M3>;
    const cudaError_t e = abk_allow_shared_memory((const void *)kernel, 224 * 1024);
    if (e != cudaSuccess) return (int)e;
    // CTAs to a row and kv head: as many as a cluster holds (8) and the pages allow, as long as all of the grid's clusters are on
    // the device at once; a grid so small that they still are with one CTA to an SM gets a ring twice as deep.
    const long long pairs = (long long)n_rows * n_kv_heads * runs;
    int seen = max_positions;
    if (window > 0 && window + KV8_PAGE < seen) seen = window + KV8_PAGE;
    const int pages = (seen + KV8_PAGE - 1) / KV8_PAGE, stage = 2 * KV8_PAGE * head_dim + 2 * KV8_PAGE_BLOCKS * 4;
    const int fold_bytes = 5 * heads * (head_dim + 4) * 4 + 1024 + 64;
    const int stages = KV8_RING_BYTES / (2 * KV8_PAGE * head_dim);
    int deep = (224 * 1024 - fold_bytes) / stage;
    if (deep > 2 * stages) deep = 2 * stages;
    auto resident = [&](int s, int st) { return kv8_resident_clusters((const void *)kernel, s, st * stage + fold_bytes); };
    int splits = pages < 1 ? 1 : pages < KV8_MAX_SPLITS ? pages : KV8_MAX_SPLITS;
    while (splits > 1 && resident(splits, stages) < pairs) splits--;
    p.stages = resident(splits, deep) >= pairs ? deep : stages;
    abk_launch_clusters(kernel, dim3(splits, n_kv_heads * runs, n_rows), dim3(KV8_THREADS), p.stages * stage + fold_bytes,
                        (cudaStream_t)stream, splits, km, vm, p);
    return ABK_LAUNCH_RESULT();
}
