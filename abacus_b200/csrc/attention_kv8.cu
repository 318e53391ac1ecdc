// Attention of a step's rows over a cache held in 8 bits (csrc/kv8.cu): a few new tokens a sequence against everything the
// cache holds of it, each row to its own position.
//
// out = sum_j softmax_j(scale q . k_j) v_j over the keys j <= position (and within the window): keys of whole blocks are
// q_j s_b with the block's scale s_b, so a score is s_b (q . q_j) and a value's weight p_j s_b; keys of the sequence's open
// block are bfloat16.
//
// The work is cut along the keys: the pages that a (row, kv head, up to 16 of its query heads) sees, one such pair after the
// other, are one long line, and every CTA takes an equal piece of it, whatever the rows' lengths. A pair that lies in one CTA's piece is
// finished there; of the others each CTA leaves its part (weighted values, maximum, sum) and a second kernel folds the parts
// in the order of the keys. A CTA takes at most two parts of pairs that are not its own, so the memory for them goes by the grid.
//
// One warp of a CTA keeps a ring of pages (keys, values, scales) coming by TMA, across the borders of pairs; four warps take a block
// of 16 tokens of every page each, with the block's two scales. Both products run on warp-level tensor-core instructions of 16-bit
// floats with the query heads as the 8 columns (two tiles of them from 9 heads on): scores are keys x heads, the
// output columns x heads, so nothing is spent on heads that are not there beyond the eighth. An 8-bit number is a float16 number exactly,
// and q is one too once each head's row is brought below 1 by a power of two (what of a head lies 2^-14 below its largest
// element keeps an absolute error of 2^-25 of that). The softmax weights are p_j s_b 2^-u in float16: 2^-11 off at most down
// to 2^-14 of the largest contribution, below that to within 2^-25 of it (N keys that are all below 2^-25 of it are lost, N 2^-25 of the
// output at most; the sums that it is divided by are float32 and have them), u
// chosen per head so that the largest ever seen is about 1: a block of small values with large weights counts as precisely
// as one of large values. Scores, maximum, sum and output are float32. The open block's keys and values go through the same products
// in bfloat16, its weights as two bfloat16 parts.
//
// An 8-bit number's way into a register pair: bytes 0 and 1 of a word with 0x64 above each are the float16 numbers 1024 + b, and
// 1152 less is q (one permute and one subtraction for two numbers); e4m3 has a conversion for two. The instructions' own order of the
// inner dimension is free as long as both operands follow it: a thread's four neighbouring bytes of a key row are the pairs
// that the instruction calls (2c, 2c + 1) and (2c + 8, 2c + 9), and q is read in that order. Values come transposed, two
// tokens and two columns to a word: even columns are the upper eight rows of a tile and odd columns the lower eight.
//
// Measured (attention and fold, without the write): 32 rows over 128 to 4,096 tokens, 32 query and 8 kv heads of 128, int8, in 32 us
// (139 MB); 8 rows over 32,768 in 87 (6.2 TB/s); two rows over 131,071 and 100,000 e4m3 tokens in 87; one row over 2,176 in 7.5. A page's block
// takes a warp some 260 instructions (int8), half of them the way from bytes to float16: at the copy rate 0.4 of what an SM issues.
#define ABK_DEFINE_ERROR
#include "common.cuh"
#include "tc_common.cuh"
#include "tensor_map.cuh"
#include "mma_tiles.cuh"
#include "kv8.cuh"

#define KV8_HEADS 16  // query heads of a pair at most: two tiles of eight columns
#define KV8_MAX_STAGES 16
#define KV8_THREADS 160
#define KV8_ROWS 512  // rows of a launch
// CTAs an SM holds. Three with heads of 64 (int8, 8 kv heads, 32 rows over 128 to 4,096 tokens: 4 heads to each 22.4 us, not 25.6, 16 to
// each 37.7, not 38.2; 8 rows over 32,768: 55.9, not 69.1, and 83.6, not 89.4; e4m3, 8 rows over 8,448: 20.1, not 22.3, and 29.3, not
// 30.0; one row over 2,176 0.2 to 0.4 longer), though 16 to 40 bytes a thread spill. Two with heads of 128, where three take longer (two
// documents of 131,071 and 100,000 tokens 95 us, not 89).
#define KV8_CTAS(dim) ((dim) == 64 ? 3 : 2)
#define KV8_START 4   // pages that starting a pair costs as much as

struct AttnKv8 {
    const __nv_bfloat16 *q;
    long long q_row;
    __nv_bfloat16 *out;
    int n_heads, n_kv_heads, runs;
    float scale_log2;
    int window;
    const int *token_seq, *token_pos, *seq_slot, *seq_pos0, *seq_len_after;
    PagedCache cache;
    const float *scales;
    const __nv_bfloat16 *open;
    int n_pages, n_slots, *status, stages;
    int early;               // this step's kv8_write has been launched: what came before it is there
    int n_rows, pairs;       // rows of the launch; pairs of a row: n_kv_heads * runs
    int first_row;           // of the step, of this launch
    float *parts;            // [2 * grid][heads of a pair][HD + 4]
};
// A pair's piece of the line: KV8_START units for what a pair costs beside its pages (its query heads, the open block, the fold of the
// warps), then one unit a page of keys. Nothing for padding.
__device__ __forceinline__ int units_of(int pos, int lo) { return KV8_START + pos / KV8_PAGE - lo / KV8_PAGE + 1; }
__device__ __forceinline__ int row_units(const AttnKv8 &p, int r) {
    if (p.token_seq[p.first_row + r] < 0) return 0;
    const int pos = p.token_pos[p.first_row + r];
    return units_of(pos, p.window > 0 && pos - p.window + 1 > 0 ? pos - p.window + 1 : 0);
}

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
// The numbers of a word's four bytes as float16 in two pairs: of bytes 0, 1 and 2, 3, or (STRIDED) of bytes 0, 2 and 1, 3.
template <int FORM, bool STRIDED> __device__ __forceinline__ void f16_of_word(uint32_t w, uint32_t &first, uint32_t &second) {
    if constexpr (FORM == KV8_INT8) {
        const __half2 less = __half2half2(__ushort_as_half(0x6480));  // 1152
        const uint32_t x = __byte_perm(w, 0x64646464u, STRIDED ? 0x4240 : 0x4140), y = __byte_perm(w, 0x64646464u, STRIDED ? 0x4341 : 0x4342);
        const __half2 p = __hsub2(*(const __half2 *)&x, less), q = __hsub2(*(const __half2 *)&y, less);
        first = *(const uint32_t *)&p, second = *(const uint32_t *)&q;
    } else {
        if (STRIDED) w = __byte_perm(w, 0, 0x3120);
        asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\tcvt.rn.f16x2.e4m3x2 %1, hi;\n\t}" : "=r"(first), "=r"(second) : "r"(w));
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

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// 8 x 8 numbers of 16 bits, a row to four lanes, transposed.
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
// Maximum over the lanes that hold the same heads (lanes of the same number modulo 4), and their sum.
__device__ __forceinline__ float heads_max(float v) {
    v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 4));
    v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 8));
    return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 16));
}
__device__ __forceinline__ float heads_sum(float v) {
    v += __shfl_xor_sync(0xffffffffu, v, 4);
    v += __shfl_xor_sync(0xffffffffu, v, 8);
    return v + __shfl_xor_sync(0xffffffffu, v, 16);
}
// What a part with exponent `from` is multiplied by where the common exponent is `to` (a part without keys: nothing).
__device__ __forceinline__ float share(float from, float to) { return from == -INFINITY ? 0.0f : exp2f(from - to); }

// A barrier over the four warps that compute, which tells all of them whether any brings true.
__device__ __forceinline__ bool any_of_the_four_warps(bool x) {
    uint32_t any;
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbar.red.or.pred q, 1, 128, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
                 : "=r"(any) : "r"((uint32_t)x) : "memory");
    return any;
}

// A run of pages of one pair, in one CTA.
struct Kv8Segment {
    int row, pair, page, pages, units;  // row of the launch; the run's first page among the row's, how many (maybe none), its units
};

template <int HD, int FORM, int NT>
__global__ void __launch_bounds__(KV8_THREADS, KV8_CTAS(HD)) attention_kv8_kernel(const __grid_constant__ CUtensorMap k_map,
                                                                              const __grid_constant__ CUtensorMap v_map, AttnKv8 p) {
    constexpr int TILE_BYTES = KV8_PAGE * HD, KS = HD / 16;
    extern __shared__ uint8_t kv8_raw[];
    uint8_t *smem = (uint8_t *)(((uintptr_t)kv8_raw + 1023) & ~(uintptr_t)1023);
    const int stages = p.stages, group = p.n_heads / p.n_kv_heads, most_heads = min(KV8_HEADS, group);
    uint8_t *k_s = smem, *v_s = k_s + stages * TILE_BYTES;
    float *scale_s = (float *)(v_s + stages * TILE_BYTES);  // [stages][2][4]
    float *warp_o = scale_s + stages * 2 * KV8_PAGE_BLOCKS;  // [4 warps][heads][HD]
    float *warp_mlu = warp_o + 4 * most_heads * HD;          // [4 warps][heads][4]: maximum, sum, the output's exponent
    __shared__ uint64_t full[KV8_MAX_STAGES], empty[KV8_MAX_STAGES];
    __shared__ int first_unit[KV8_ROWS + 1];  // of a pair of the rows before a row
    __shared__ int4 row_info[KV8_ROWS];       // position, slot, blocks in 8 bits, first visible key
    __shared__ int fresh_page[KV8_ROWS];      // the first page that the step itself writes to
    __shared__ int failed, bad_s;  // a wait ran out; pages and slots that are not there (said to the host at the end: not before pdl_wait())

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        failed = 0, bad_s = 0;
        for (int s = 0; s < stages; s++) tc::mbar_init(&full[s], 1), tc::mbar_init(&empty[s], 4);
        tc::mbar_init_fence();
        tc::tma_prefetch_map(&k_map), tc::tma_prefetch_map(&v_map);
    }
    // Where kv8_write of this very step has been launched, the launch just before this one is that or a later one: what came before kv8_write
    // is there, and is read before pdl_wait(): the step's index arrays and the page table, and (by the copy warp) the pages before
    // those that the step's own tokens are in. Under a ring such a page may be one that kv8_write is putting blocks into at that moment; it
    // puts one only where no row sees any token of the block that was there (the step's rows and the window fit the ring, as
    // the launcher's caller checks), so what is torn belongs to blocks that are behind no row's first key and are never looked at. Otherwise
    // all of it waits for the launch before, whatever that is.
    if (!p.early) pdl_wait();
    int bad = 0;
    for (int r = threadIdx.x; r < p.n_rows; r += KV8_THREADS) {
        const int seq = p.token_seq[p.first_row + r], pos = p.token_pos[p.first_row + r];
        const int lo = p.window > 0 && pos - p.window + 1 > 0 ? pos - p.window + 1 : 0;
        first_unit[r + 1] = seq < 0 ? 0 : units_of(pos, lo);
        fresh_page[r] = seq < 0 ? 0 : p.seq_pos0[seq] / KV8_PAGE;
        row_info[r] = seq < 0 ? make_int4(0, 0, 0, 0) : make_int4(pos, kv8_slot(p.seq_slot[seq], p.n_slots, bad), p.seq_len_after[seq] / KV8_BLOCK, lo);
    }
    __syncthreads();
    if (bad) atomicOr(&bad_s, bad), bad = 0;
    if (warp == 0) {
        int before = 0;
        if (lane == 0) first_unit[0] = 0;
        for (int r0 = 0; r0 < p.n_rows; r0 += 32) {
            int x = r0 + lane < p.n_rows ? first_unit[r0 + lane + 1] : 0;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int y = __shfl_up_sync(0xffffffffu, x, o);
                if (lane >= o) x += y;
            }
            if (r0 + lane < p.n_rows) first_unit[r0 + lane + 1] = before + x;
            before += __shfl_sync(0xffffffffu, x, 31);
        }
    }
    __syncthreads();
    const long long units = (long long)p.pairs * first_unit[p.n_rows], per = (units + gridDim.x - 1) / gridDim.x;
    const long long begin = per * blockIdx.x, end = min(units, begin + per);
    if (begin >= end) {
        pdl_wait();
        return;
    }
    // the run of pages that starts at `unit`
    auto segment_at = [&](long long unit) {
        int lo = 0, hi = p.n_rows;  // the last row that starts at or before the unit (rows without pages start where the next one does)
        while (hi - lo > 1) {
            const int mid = (lo + hi) / 2;
            if ((long long)p.pairs * first_unit[mid] <= unit) lo = mid;
            else hi = mid;
        }
        const int all = first_unit[lo + 1] - first_unit[lo], in_row = (int)(unit - (long long)p.pairs * first_unit[lo]);
        Kv8Segment s;
        s.row = lo, s.pair = in_row / all;
        const int from = in_row - s.pair * all, to = (int)min((long long)all, from + end - unit);
        s.units = to - from, s.page = max(from - KV8_START, 0), s.pages = max(to - KV8_START, 0) - s.page;
        return s;
    };

    if (warp == 4) {
        int issued = 0;
        bool go = true, waited = !p.early;
        for (long long unit = begin; unit < end && go;) {
            const Kv8Segment seg = segment_at(unit);
            const int4 info = row_info[seg.row];
            const int kvh = seg.pair / p.runs, first = info.w / KV8_PAGE + seg.page;
            for (int base = 0; base < seg.pages && go; base += 32) {
                int page_lane = 0;  // every lane looks up one of the next 32 pages
                if (base + lane < seg.pages) page_lane = kv8_page(p.cache, p.n_pages, info.y, (first + base + lane) * KV8_PAGE, bad);
                const int n = min(32, seg.pages - base);
                for (int i = 0; i < n && go; i++, issued++) {
                    const long long tile = (long long)__shfl_sync(0xffffffffu, page_lane, i) * p.n_kv_heads + kvh;
                    int bad = 0;
                    if (!waited && first + base + i >= fresh_page[seg.row]) pdl_wait(), waited = true;
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
            unit += seg.units;
        }
        if (bad) atomicOr(&bad_s, bad);
        pdl_wait();
        if (!go && lane == 0) {  // let the copies in flight land before the CTA's memory goes away
            failed = 1;
            issued--;  // the copy that was not issued
            for (int i = max(0, issued - stages); i < issued; i++) tc::mbar_wait(&full[i % stages], (i / stages) & 1);
        }
    } else {
        const int i8 = lane >> 2, c4 = 4 * (lane & 3), j8 = lane >> 3, r8 = lane & 7;
        bool ok = true;
        int s = 0, phase = 0, done = 0;
        pdl_wait();
        for (long long unit = begin; unit < end && ok;) {
            const Kv8Segment seg = segment_at(unit);
            unit += seg.units;
            if (seg.pages == 0) continue;
            const int4 info = row_info[seg.row];
            const int pos = info.x, slot = info.y, closed = info.z, lo = info.w;
            const int kvh = seg.pair / p.runs, g0 = (seg.pair - kvh * p.runs) * KV8_HEADS, heads = min(KV8_HEADS, group - g0);
            const int first = lo / KV8_PAGE + seg.page;
            const long long row = p.first_row + seg.row;
            const __nv_bfloat16 *q = p.q + row * p.q_row + (long long)(kvh * group + g0) * HD + c4;
            // q of head i8 (and i8 + 8): the products' right operand, and what the scores of heads 2 c, 2 c + 1 are multiplied by
            uint32_t qf[NT][KS][2];
            float unit_of[NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
                uint2 raw[KS];
                float most = 0.0f;
#pragma unroll
                for (int ks = 0; ks < KS; ks++) raw[ks] = 8 * nt + i8 < heads ? *(const uint2 *)(q + (8 * nt + i8) * HD + 16 * ks) : make_uint2(0, 0);
                auto largest = [](float most, uint32_t w) {
                    const float2 f = __bfloat1622float2(*(const __nv_bfloat162 *)&w);
                    return fmaxf(most, fmaxf(fabsf(f.x), fabsf(f.y)));
                };
#pragma unroll
                for (int ks = 0; ks < KS; ks++) most = largest(largest(most, raw[ks].x), raw[ks].y);
                const float down = exp2f(-power_above(quad_max(most))), up = p.scale_log2 / down;
                auto scaled = [](uint32_t w, float by) {
                    const float2 f = __bfloat1622float2(*(const __nv_bfloat162 *)&w);
                    return pack_f16(f.x * by, f.y * by);
                };
#pragma unroll
                for (int ks = 0; ks < KS; ks++) qf[nt][ks][0] = scaled(raw[ks].x, down), qf[nt][ks][1] = scaled(raw[ks].y, down);
                unit_of[nt][0] = __shfl_sync(0xffffffffu, up, 8 * (lane & 3)), unit_of[nt][1] = __shfl_sync(0xffffffffu, up, 8 * (lane & 3) + 4);
            }
            float o[NT][KS][4];  // tile c: columns 16 c + 2 i8 (0, 1: heads 2 c, 2 c + 1) and 16 c + 2 i8 + 1 (2, 3)
            float m[NT][2], l[NT][2], u[NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
#pragma unroll
                for (int c = 0; c < KS; c++) o[nt][c][0] = o[nt][c][1] = o[nt][c][2] = o[nt][c][3] = 0.0f;
#pragma unroll
                for (int e = 0; e < 2; e++) m[nt][e] = -INFINITY, l[nt][e] = 0.0f, u[nt][e] = -INFINITY;
            }
            // Scores of keys i8 and i8 + 8 (in units of log2) to weights: sc becomes p_j 2^-m, l and m follow, o is brought to its
            // new exponent; what is left to multiply a head's weights with is returned in f. v_scale is the block's, and at
            // least one of its keys is visible, so the maxima are finite; references are whole powers of two.
            auto softmax = [&](float (*sc)[4], float (*f)[2], float v_scale) {
                const float above = power_above(v_scale);
                bool moved = false;
                float was[NT][2];
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        const float a = ceilf(heads_max(fmaxf(sc[nt][e], sc[nt][e + 2]))), n = fmaxf(m[nt][e], a);
                        l[nt][e] *= ex2(m[nt][e] - n), m[nt][e] = n;
                        was[nt][e] = u[nt][e], u[nt][e] = fmaxf(u[nt][e], a + above);
                        moved |= was[nt][e] != u[nt][e];
                        sc[nt][e] = ex2(sc[nt][e] - n), sc[nt][e + 2] = ex2(sc[nt][e + 2] - n);
                        l[nt][e] += sc[nt][e] + sc[nt][e + 2];
                        f[nt][e] = v_scale * ex2(n - u[nt][e]);
                    }
                }
                if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
                    for (int nt = 0; nt < NT; nt++) {
                        const float d0 = ex2(was[nt][0] - u[nt][0]), d1 = ex2(was[nt][1] - u[nt][1]);
#pragma unroll
                        for (int c = 0; c < KS; c++) o[nt][c][0] *= d0, o[nt][c][1] *= d1, o[nt][c][2] *= d0, o[nt][c][3] *= d1;
                    }
                }
            };
            auto mask = [&](float (*sc)[4], int key0) {  // keys behind the position or before the window
                const int key = key0 + i8;
                const bool sees0 = key >= lo && key <= pos, sees8 = key + 8 >= lo && key + 8 <= pos;
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
                    if (!sees0) sc[nt][0] = sc[nt][1] = -INFINITY;
                    if (!sees8) sc[nt][2] = sc[nt][3] = -INFINITY;
                }
            };
            // The open block, as it came: once a pair, by one warp, ahead of the pages, which may still be on their way.
            if (pos / KV8_BLOCK >= closed && pos / KV8_PAGE >= first && pos / KV8_PAGE < first + seg.pages && pos % KV8_PAGE / KV8_BLOCK == warp) {
                const int key0 = pos / KV8_BLOCK * KV8_BLOCK;
                float sc[NT][4] = {}, f[NT][2];
                const __nv_bfloat16 *open_k = p.open + ((long long)slot * 2 * p.n_kv_heads + kvh) * (KV8_BLOCK * HD),
                                    *open_v = open_k + (long long)p.n_kv_heads * (KV8_BLOCK * HD);
#pragma unroll
                for (int ks = 0; ks < KS; ks++) {
                    const uint2 k0 = *(const uint2 *)(open_k + i8 * HD + 16 * ks + c4), k8 = *(const uint2 *)(open_k + (i8 + 8) * HD + 16 * ks + c4);
                    const uint32_t a[4] = {k0.x, k8.x, k0.y, k8.y};
#pragma unroll
                    for (int nt = 0; nt < NT; nt++) {
                        const uint2 b = 8 * nt + i8 < heads ? *(const uint2 *)(q + (8 * nt + i8) * HD + 16 * ks) : make_uint2(0, 0);
                        mma_bf16(sc[nt], a, b.x, b.y);
                    }
                }
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
#pragma unroll
                    for (int e = 0; e < 4; e++) sc[nt][e] *= p.scale_log2;
                mask(sc, key0);
                softmax(sc, f, 1.0f);
                uint32_t high[NT][2], low[NT][2];
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
#pragma unroll
                    for (int i = 0; i < 2; i++) {
                        const float x = sc[nt][2 * i] * f[nt][0], y = sc[nt][2 * i + 1] * f[nt][1];
                        const uint32_t h = pack_bf16(x, y);
                        const float2 back = __bfloat1622float2(*(const __nv_bfloat162 *)&h);
                        high[nt][i] = transposed(h), low[nt][i] = transposed(pack_bf16(x - back.x, y - back.y));
                    }
#pragma unroll
                for (int c = 0; c < KS; c++) {
                    uint32_t v[4];  // tokens 2 c', 2 c' + 1, 2 c' + 8, 2 c' + 9; one that the row does not see may hold anything
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const int t = 2 * (lane & 3) + (i & 1) + 8 * (i >> 1);
                        v[i] = key0 + t <= pos && key0 + t >= lo ? *(const uint32_t *)(open_v + t * HD + 16 * c + 2 * i8) : 0u;
                    }
                    const uint32_t a[4] = {__byte_perm(v[0], v[1], 0x5410), __byte_perm(v[0], v[1], 0x7632),
                                           __byte_perm(v[2], v[3], 0x5410), __byte_perm(v[2], v[3], 0x7632)};
#pragma unroll
                    for (int nt = 0; nt < NT; nt++) mma_bf16(o[nt][c], a, high[nt][0], high[nt][1]), mma_bf16(o[nt][c], a, low[nt][0], low[nt][1]);
                }
            }
            for (int pg = first; pg < first + seg.pages; pg++) {
                ok = __all_sync(0xffffffffu, tc::mbar_wait(&full[s], phase));
                if (!ok) break;
                const int key0 = pg * KV8_PAGE + KV8_BLOCK * warp;  // this warp's block of the page
                if (key0 / KV8_BLOCK < closed && key0 <= pos && key0 + KV8_BLOCK > lo) {
                    float sc[NT][4] = {}, f[NT][2];
                    const uint32_t k_base = tc::smem_addr(k_s + s * TILE_BYTES), v_base = tc::smem_addr(v_s + s * TILE_BYTES);
                    const float k_scale = scale_s[s * 2 * KV8_PAGE_BLOCKS + warp], v_scale = scale_s[(s * 2 + 1) * KV8_PAGE_BLOCKS + warp];
#pragma unroll
                    for (int ks = 0; ks < KS; ks += 2) {
                        uint32_t w[4];
                        ldsm_x4(token_piece<HD>(k_base, KV8_BLOCK * warp + 8 * (j8 & 1) + r8, ks + (j8 >> 1)), w[0], w[1], w[2], w[3]);
#pragma unroll
                        for (int i = 0; i < 2; i++) {
                            uint32_t a[4];
                            f16_of_word<FORM, false>(w[2 * i], a[0], a[2]), f16_of_word<FORM, false>(w[2 * i + 1], a[1], a[3]);
#pragma unroll
                            for (int nt = 0; nt < NT; nt++) mma_f16(sc[nt], a, qf[nt][ks + i][0], qf[nt][ks + i][1]);
                        }
                    }
#pragma unroll
                    for (int nt = 0; nt < NT; nt++)
#pragma unroll
                        for (int e = 0; e < 4; e++) sc[nt][e] *= unit_of[nt][e & 1] * k_scale;
                    if (key0 < lo || key0 + KV8_BLOCK - 1 > pos) mask(sc, key0);
                    softmax(sc, f, v_scale);
                    uint32_t pf[NT][2];
#pragma unroll
                    for (int nt = 0; nt < NT; nt++) {
                        pf[nt][0] = transposed(pack_f16(sc[nt][0] * f[nt][0], sc[nt][1] * f[nt][1]));
                        pf[nt][1] = transposed(pack_f16(sc[nt][2] * f[nt][0], sc[nt][3] * f[nt][1]));
                    }
#pragma unroll
                    for (int c = 0; c < KS; c += 2) {
                        uint32_t w[4];
                        ldsm_x4_t(token_piece<HD>(v_base, KV8_BLOCK * warp + 8 * (j8 & 1) + r8, c + (j8 >> 1)), w[0], w[1], w[2], w[3]);
#pragma unroll
                        for (int i = 0; i < 2; i++) {
                            uint32_t a[4];
                            f16_of_word<FORM, true>(w[2 * i], a[0], a[1]), f16_of_word<FORM, true>(w[2 * i + 1], a[2], a[3]);
#pragma unroll
                            for (int nt = 0; nt < NT; nt++) mma_f16(o[nt][c + i], a, pf[nt][0], pf[nt][1]);
                        }
                    }
                }
                __syncwarp();
                if (lane == 0) tc::mbar_arrive(&empty[s]);
                if (++s == stages) s = 0, phase ^= 1;
            }
            // fold the four warps, in warp order
            if (done) asm volatile("bar.sync 1, 128;" ::: "memory");  // the last run's fold has been read
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    const int g = 8 * nt + 2 * (lane & 3) + e;
                    const float sum = heads_sum(l[nt][e]);
                    if (g < heads) {
                        float *dst = warp_o + (warp * most_heads + g) * HD + 2 * i8;
#pragma unroll
                        for (int c = 0; c < KS; c++) *(float2 *)(dst + 16 * c) = make_float2(o[nt][c][e], o[nt][c][e + 2]);
                        if (i8 == 0) *(float4 *)(warp_mlu + (warp * most_heads + g) * 4) = make_float4(m[nt][e], sum, u[nt][e], 0.0f);
                    }
                }
            }
            ok = !any_of_the_four_warps(!ok);  // all stop behind this run or none: every barrier is passed by all of them
            const bool whole = seg.pages == first_unit[seg.row + 1] - first_unit[seg.row] - KV8_START;
            float *part = p.parts + (2 * (long long)blockIdx.x + (done > 0)) * most_heads * (HD + 4);
            done++;
            __nv_bfloat16 *out = p.out + (row * p.n_heads + kvh * group + g0) * HD;
            for (int i = threadIdx.x; i < heads * (HD / 4); i += 128) {
                const int g = i / (HD / 4), d = 4 * (i - g * (HD / 4));
                float4 mlu[4], acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                float mm = -INFINITY, uu = -INFINITY, ll = 0.0f;
#pragma unroll
                for (int w = 0; w < 4; w++) mlu[w] = *(const float4 *)(warp_mlu + (w * most_heads + g) * 4), mm = fmaxf(mm, mlu[w].x), uu = fmaxf(uu, mlu[w].z);
#pragma unroll
                for (int w = 0; w < 4; w++) {
                    const float by = share(mlu[w].z, uu);
                    const float4 x = *(const float4 *)(warp_o + (w * most_heads + g) * HD + d);
                    acc.x = fmaf(by, x.x, acc.x), acc.y = fmaf(by, x.y, acc.y), acc.z = fmaf(by, x.z, acc.z), acc.w = fmaf(by, x.w, acc.w);
                    ll = fmaf(share(mlu[w].x, mm), mlu[w].y, ll);
                }
                if (whole) {
                    const float by = exp2f(uu - mm) / ll;
                    *(uint2 *)(out + (long long)g * HD + d) = make_uint2(pack_bf16(acc.x * by, acc.y * by), pack_bf16(acc.z * by, acc.w * by));
                } else {
                    *(float4 *)(part + g * HD + d) = acc;
                    if (d == 0) *(float4 *)(part + most_heads * HD + g * 4) = make_float4(mm, ll, uu, 0.0f);
                }
            }
        }
        if (!ok) failed = 1;
    }
    __syncthreads();
    if ((failed | bad_s) && threadIdx.x == 0) atomicOr(p.status + 2, (failed ? 1 : 0) | bad_s);
}

// The pairs that several CTAs have parts of, folded in the order of the keys, a CTA a head; zeros for rows that are padding. `grid`:
// the CTAs of the kernel above. The parts' shares come first, a thread a part; then every thread adds up four columns over a
// KV8_FOLD_THREADS * 4 / HD th of the parts, all loads under way together.
#define KV8_FOLD_THREADS 128
#define KV8_MAX_GRID 512
template <int HD> __global__ void __launch_bounds__(KV8_FOLD_THREADS, 10) attention_kv8_fold_kernel(AttnKv8 p, int grid) {
    constexpr int COLS = HD / 4, GROUPS = KV8_FOLD_THREADS / COLS;
    __shared__ float weight[KV8_MAX_GRID], scratch[33];
    __shared__ float4 sums[GROUPS][COLS];
    __shared__ int before_s, all_s;
    const int group = p.n_heads / p.n_kv_heads, most_heads = min(KV8_HEADS, group);
    const int r = blockIdx.y, pair = blockIdx.x / most_heads, g = blockIdx.x - pair * most_heads, lane = threadIdx.x & 31;
    const int kvh = pair / p.runs, g0 = (pair - kvh * p.runs) * KV8_HEADS;
    if (threadIdx.x == 0) before_s = 0, all_s = 0;
    // (the step's rows are not the kernel above's to write: they are counted while it runs)
    if (g0 + g >= group) {
        pdl_wait();
        return;
    }
    __syncthreads();
    int before = 0, all = 0;
    for (int i = threadIdx.x; i < p.n_rows; i += KV8_FOLD_THREADS) {
        const int n = row_units(p, i);
        all += n, before += i < r ? n : 0;
    }
    before = __reduce_add_sync(0xffffffffu, before), all = __reduce_add_sync(0xffffffffu, all);
    if (lane == 0) atomicAdd(&before_s, before), atomicAdd(&all_s, all);
    __syncthreads();
    const int mine = row_units(p, r);
    pdl_wait();
    __nv_bfloat16 *out = p.out + ((long long)(p.first_row + r) * p.n_heads + kvh * group + g0 + g) * HD;
    if (mine == 0) {
        if (threadIdx.x < COLS) *(uint2 *)(out + 4 * threadIdx.x) = make_uint2(0, 0);
        return;
    }
    const long long units = (long long)p.pairs * all_s, per = (units + grid - 1) / grid;
    const long long begin = (long long)p.pairs * before_s + (long long)pair * mine, first_page = begin + KV8_START, last = begin + mine - 1;
    const int c0 = (int)(first_page / per), n = (int)(last / per) - c0 + 1;  // the CTAs that have pages of the pair
    if (n == 1) return;
    const long long size = (long long)most_heads * (HD + 4);
    // of the first CTA it is the second part where the CTA's piece starts with another pair's pages
    auto part = [&](int c) { return p.parts + (2ll * (c0 + c) + (c == 0 && per * c0 < begin)) * size; };
    // everything that most pairs need is asked for at once: a thread's first part's numbers and its first four parts' columns
    const int col = threadIdx.x % COLS, of = threadIdx.x / COLS;
    float4 x[4];
    auto columns = [&](int c) {
#pragma unroll
        for (int i = 0; i < 4; i++) x[i] = c + i * GROUPS < n ? *(const float4 *)(part(c + i * GROUPS) + g * HD + 4 * col) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    };
    auto numbers = [&](int c) { return c < n ? *(const float4 *)(part(c) + most_heads * HD + 4 * g) : make_float4(-INFINITY, 0.0f, -INFINITY, 0.0f); };
    const float4 mine_mlu = numbers(threadIdx.x);
    columns(of);
    float m = mine_mlu.x, u = mine_mlu.z, l = 0.0f;
    for (int c = threadIdx.x + KV8_FOLD_THREADS; c < n; c += KV8_FOLD_THREADS) {
        const float4 mlu = numbers(c);
        m = fmaxf(m, mlu.x), u = fmaxf(u, mlu.z);
    }
    m = block_max(m, scratch), u = block_max(u, scratch);
    for (int c = threadIdx.x; c < n; c += KV8_FOLD_THREADS) {
        const float4 mlu = c == threadIdx.x ? mine_mlu : numbers(c);
        l = fmaf(share(mlu.x, m), mlu.y, l), weight[c] = share(mlu.z, u);
    }
    l = block_sum(l, scratch);  // (a barrier: the weights are there)
    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int c = of; c < n; c += 4 * GROUPS) {
        if (c != of) columns(c);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float w = c + i * GROUPS < n ? weight[c + i * GROUPS] : 0.0f;
            acc.x = fmaf(w, x[i].x, acc.x), acc.y = fmaf(w, x[i].y, acc.y), acc.z = fmaf(w, x[i].z, acc.z), acc.w = fmaf(w, x[i].w, acc.w);
        }
    }
    sums[of][col] = acc;
    __syncthreads();
    if (threadIdx.x < COLS) {
        for (int i = 1; i < GROUPS; i++) acc.x += sums[i][col].x, acc.y += sums[i][col].y, acc.z += sums[i][col].z, acc.w += sums[i][col].w;
        const float by = exp2f(u - m) / l;
        *(uint2 *)(out + 4 * col) = make_uint2(pack_bf16(acc.x * by, acc.y * by), pack_bf16(acc.z * by, acc.w * by));
    }
}

// Floats of memory for the parts of pairs that several CTAs share.
extern "C" long long abk_attention_kv8_part_floats(int n_heads, int n_kv_heads, int head_dim) {
    const int group = n_kv_heads > 0 ? n_heads / n_kv_heads : 1;
    return 2ll * KV8_CTAS(head_dim) * abk_sm_count() * (group < KV8_HEADS ? group : KV8_HEADS) * (head_dim + 4);
}
extern "C" int abk_attention_kv8(const void *q, long long q_row, void *out, int n_rows, int n_heads, float scale, int window,
                                 const int *token_seq, const int *token_pos, const int *seq_slot, const int *seq_pos0,
                                 const int *seq_len_after, const Kv8Cache *cache, float *parts, long long part_floats, int early,
                                 void *stream) {
    const Kv8Cache &c = *cache;
    const int head_dim = c.head_dim, n_kv_heads = c.n_kv_heads, form = c.form;
    if (n_rows <= 0) return 0;
    if (head_dim != 64 && head_dim != 128) ABK_REFUSE("attention_kv8: head_dim %d is not 64 or 128", head_dim);
    if (form != KV8_INT8 && form != KV8_E4M3) ABK_REFUSE("attention_kv8: no 8-bit form %d", form);
    if (n_kv_heads < 1 || n_heads < 1 || n_heads % n_kv_heads) ABK_REFUSE("attention_kv8: %d heads do not divide into %d kv heads", n_heads, n_kv_heads);
    const int group = n_heads / n_kv_heads, runs = (group + KV8_HEADS - 1) / KV8_HEADS, heads = group < KV8_HEADS ? group : KV8_HEADS;
    if ((((uintptr_t)q | (uintptr_t)out) & 7) || (q_row & 3) || (((uintptr_t)c.scales | (uintptr_t)c.open | (uintptr_t)parts) & 15))
        ABK_REFUSE("attention_kv8: q and out must be 8-byte aligned, scales, open blocks and parts 16-byte aligned");
    const int ctas = KV8_CTAS(head_dim), grid = ctas * abk_sm_count();
    if (grid > KV8_MAX_GRID) ABK_REFUSE("attention_kv8: %d CTAs are more than the fold has room for", grid);
    if (part_floats < abk_attention_kv8_part_floats(n_heads, n_kv_heads, head_dim))
        ABK_REFUSE("attention_kv8: room for %lld floats of parts is too little", part_floats);
    CUtensorMap km, vm;
    const long long pool_rows = (long long)c.n_pages * n_kv_heads * KV8_PAGE * head_dim / 128;
    int rc = tmap::bytes_in_rows_of_128(c.k, pool_rows, KV8_PAGE * head_dim / 128, &km);
    if (!rc) rc = tmap::bytes_in_rows_of_128(c.v, pool_rows, KV8_PAGE * head_dim / 128, &vm);
    if (rc) return rc;
    AttnKv8 p;
    p.q = (const __nv_bfloat16 *)q, p.q_row = q_row, p.out = (__nv_bfloat16 *)out, p.n_heads = n_heads, p.n_kv_heads = n_kv_heads;
    p.scale_log2 = scale * 1.4426950408889634f, p.window = window, p.token_seq = token_seq, p.token_pos = token_pos;
    p.seq_slot = seq_slot, p.seq_pos0 = seq_pos0, p.seq_len_after = seq_len_after, p.cache.page_table = c.page_table, p.cache.table_width = c.table_width;
    p.cache.ring_pages = c.ring_pages, p.cache.tokens_per_page = KV8_PAGE, p.scales = c.scales, p.open = (const __nv_bfloat16 *)c.open;
    p.n_pages = c.n_pages, p.n_slots = c.n_slots, p.status = c.status, p.runs = runs, p.pairs = n_kv_heads * runs, p.parts = parts, p.early = early;
    void (*kernel)(CUtensorMap, CUtensorMap, AttnKv8) = nullptr;
    auto of_dim = [&](auto hd, auto tiles) {
        constexpr int HD = decltype(hd)::value, NT = decltype(tiles)::value;
        return form == KV8_INT8 ? attention_kv8_kernel<HD, KV8_INT8, NT> : attention_kv8_kernel<HD, KV8_E4M3, NT>;
    };
    using std::integral_constant;
    if (head_dim == 64) kernel = heads <= 8 ? of_dim(integral_constant<int, 64>(), integral_constant<int, 1>()) : of_dim(integral_constant<int, 64>(), integral_constant<int, 2>());
    else kernel = heads <= 8 ? of_dim(integral_constant<int, 128>(), integral_constant<int, 1>()) : of_dim(integral_constant<int, 128>(), integral_constant<int, 2>());
    const int stage = 2 * KV8_PAGE * head_dim + 2 * KV8_PAGE_BLOCKS * 4, fold_bytes = 4 * heads * (head_dim + 4) * 4 + 1024;
    p.stages = ((226 - 14 * ctas) * 1024 / ctas - fold_bytes) / stage;  // (14 KB: a CTA's table of rows, and what every CTA takes)
    if (p.stages > KV8_MAX_STAGES) p.stages = KV8_MAX_STAGES;
    const int smem = p.stages * stage + fold_bytes;
    const cudaError_t e = abk_allow_shared_memory((const void *)kernel, smem);
    if (e != cudaSuccess) return (int)e;
    for (int first = 0; first < n_rows; first += KV8_ROWS) {
        p.first_row = first, p.n_rows = n_rows - first < KV8_ROWS ? n_rows - first : KV8_ROWS;
        abk_launch(kernel, dim3(grid), dim3(KV8_THREADS), smem, (cudaStream_t)stream, km, vm, p);
        rc = ABK_LAUNCH_RESULT();
        if (rc) return rc;
        const dim3 pairs(p.pairs * heads, p.n_rows);
        if (head_dim == 64) abk_launch(attention_kv8_fold_kernel<64>, pairs, dim3(KV8_FOLD_THREADS), 0, (cudaStream_t)stream, p, grid);
        else abk_launch(attention_kv8_fold_kernel<128>, pairs, dim3(KV8_FOLD_THREADS), 0, (cudaStream_t)stream, p, grid);
        rc = ABK_LAUNCH_RESULT();
        if (rc) return rc;
    }
    return 0;
}
