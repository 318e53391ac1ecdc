// The log probability of a given token and the entropy under the logits x . w^T (src/model.c:324), which never reach memory: the
// product on the tensor cores (tcgen05, pairs of CTAs on tiles of 256 rows of x and 256 of w, as csrc/gemm_tc.cu has it), and
// where that kernel stores a tile this one adds it to running sums, m = max, l = sum e^(x - m), t = sum (x - m) e^(x - m).
//
// The tiles go through the rows of x first, so that the pairs work on the same few tiles of w at a time and w comes from
// the L2 for all but the first; up to LP_GROUP tiles of rows (2,048 rows) are a group, and w is read once a group. A pair takes
// every pairs-th tile of the line. A thread that reads the accumulator has one row and 128 of a tile's columns; the sums of the
// group's rows wait in shared memory for the row's next tile, and at the group's end every pair leaves its own for every row.
// The tensor cores' own sums are cut off, not rounded, at every step of 16 products: over K = 4,096 that leaves log probabilities
// 1.6e-6 off (against 4e-7 over 1,024), relative to their size, and the entropies of few rows twice as much. So a long K is multiplied in segments
// of up to 1,024, each into an accumulator of its own, and the reading threads add them up, in registers, while the tensor cores are on the
// next one. Of 3,000 drawn products of 1 to 4,500 rows 3 had an output more than 1e-6 off; with segments of up to 1,536 30, with 768
// one, but then K = 1,024 takes two: 2,048 rows 613 us, not 516.
// A second kernel joins the pairs' sums, a warp a row. Measured: 2,048 rows of 1,024 against 151,936 in 516 us, 1,235 TFLOP/s (cuBLAS
// sustains 1,377 under the power cap); 4,999 rows of 4,096 in 5,140, four segments, 1,210 TFLOP/s (5,020 in three). The eight warps that read need 6.5 instructions and one exponential a logit:
// at K = 1,024 half of the time that the tensor cores take for it.
//
// Few rows (up to LP_FEW, few_wins): w is all there is to read, and a tile of 256 rows of x of which a few are there costs the tensor cores as much
// time as w takes to come. So the operands change sides: a CTA's tile is up to 128 rows of w, the rows of x are its 16 to 64 columns, and
// a thread that reads the accumulator has one token of the vocabulary and keeps the sums of 32 rows of x in registers over all of its
// CTA's tiles. The tiles are as high as makes all CTAs take the same number of full ones (115 for 151,936 on 148 SMs). 37 rows of 1,024
// against 151,936: 61 us, with the tiles above 77 (the matrix at the copy rate: 48).
#define ABK_DEFINE_ERROR
#include "common.cuh"
#include "tc_common.cuh"
#include "tensor_map.cuh"
#include "logprobs.cuh"

#define LP_ROWS 128      // rows of x a CTA holds of a tile; a pair has two of it
#define LP_COLS 256      // rows of w a tile has; each CTA of a pair brings half
#define LP_K 64
#define LP_STAGES 6
#define LP_GROUP 8
#define LP_THREADS 320   // one warp that loads, one that multiplies, eight that read
#define LP_SEGMENT 16    // blocks of K to a segment at most
#define LP_MOST_ROWS 16384  // rows of a launch

struct GemmLogProbs {
    int rows, vocab, k_blocks, segment_blocks, segments, m_tiles, v_tiles, tiles, groups;
    const int *tokens;
    float *given;  // [rows]: the given token's logit, where there is one
    float4 *parts;  // [pairs][rows]
    int *status;
};
struct LpTile {
    int group, in_group, row0, col0;
};
__device__ __forceinline__ LpTile tile_at(const GemmLogProbs &g, int t) {
    const int per = LP_GROUP * g.v_tiles;
    LpTile r;
    r.group = t / per;
    const int rest = t - r.group * per, wide = min(LP_GROUP, g.m_tiles - r.group * LP_GROUP), v = rest / wide;
    r.in_group = rest - v * wide;
    r.row0 = (r.group * LP_GROUP + r.in_group) * 2 * LP_ROWS, r.col0 = v * LP_COLS;
    return r;
}
#define LP_A_BYTES (LP_ROWS * LP_K * 2)
#define LP_B_BYTES (LP_COLS / 2 * LP_K * 2)
#define LP_STATE_BYTES (LP_GROUP * 2 * LP_ROWS * 16)
#define LP_SMEM (LP_STAGES * (LP_A_BYTES + LP_B_BYTES) + LP_STATE_BYTES + 1024 /* alignment */ + 256 /* barriers */)

template <bool SEGMENTS>
__global__ void __launch_bounds__(LP_THREADS) gemm_logprobs_kernel(const __grid_constant__ CUtensorMap map_x,
                                                                   const __grid_constant__ CUtensorMap map_w, GemmLogProbs g) {
    extern __shared__ uint8_t lp_raw[];
    uint8_t *smem = (uint8_t *)(((uintptr_t)lp_raw + 1023) & ~(uintptr_t)1023);
    uint8_t *a_tiles = smem, *b_tiles = smem + LP_STAGES * LP_A_BYTES;
    float4 *state = (float4 *)(b_tiles + LP_STAGES * LP_B_BYTES);  // [tile of the group][half of the columns][row]
    uint64_t *full = (uint64_t *)((uint8_t *)state + LP_STATE_BYTES);
    uint64_t *empty = full + LP_STAGES, *acc_full = empty + LP_STAGES, *acc_empty = acc_full + 2;
    uint32_t *tmem_holder = (uint32_t *)(acc_empty + 2);
    volatile int *flags = (volatile int *)(tmem_holder + 1);  // [0]: a wait ran out
    constexpr uint32_t TMEM_COLS = 2 * LP_COLS;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = (int)tc::cluster_rank();  // 0: the leader, 1: its peer
    const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
    if (threadIdx.x == 0) {
        for (int s = 0; s < LP_STAGES; s++) tc::mbar_init(&full[s], 1), tc::mbar_init(&empty[s], 1);
        for (int b = 0; b < 2; b++) tc::mbar_init(&acc_full[b], 1), tc::mbar_init(&acc_empty[b], 16);  // every reading warp of both CTAs
        flags[0] = 0;
        tc::mbar_init_fence();
        tc::tma_prefetch_map(&map_x), tc::tma_prefetch_map(&map_w);
    }
    if (warp == 1) tc::tmem_alloc_pair(tmem_holder, TMEM_COLS);
    tc::fence_before_sync();
    tc::cluster_sync();  // both CTAs' barriers are there before either signals the other's
    tc::fence_after_sync();
    const uint32_t tmem = *tmem_holder;

    if (warp == 0) {
        if (lane == 0) {
            // A stage is full when both CTAs' copies have landed: all of them report to the leader's barrier.
            constexpr uint32_t STAGE_BYTES = 2 * (LP_A_BYTES + LP_B_BYTES);
            pdl_wait();
            int issued = 0;
            for (int t = pair; t < g.tiles && !flags[0]; t += pairs) {
                const LpTile at = tile_at(g, t);
                const int p0 = at.row0 + rank * LP_ROWS, q0 = at.col0 + rank * (LP_COLS / 2);
                for (int kb = 0; kb < g.k_blocks; kb++, issued++) {
                    const int s = issued % LP_STAGES;
                    const uint32_t bar = tc::peer_smem(tc::smem_addr(&full[s]), 0);
                    if (!tc::mbar_wait(&empty[s], ((issued / LP_STAGES) & 1) ^ 1)) {  // (its own: the commit reaches both)
                        flags[0] = 1;
                        break;
                    }
                    if (rank == 0) tc::mbar_expect_tx(&full[s], STAGE_BYTES);
                    tc::tma_load_2d_pair(b_tiles + s * LP_B_BYTES, &map_w, kb * LP_K, q0, bar);
                    tc::tma_load_2d_pair(a_tiles + s * LP_A_BYTES, &map_x, kb * LP_K, p0, bar);
                }
            }
        }
    } else if (warp == 1) {
        if (lane == 0 && rank == 0) {
            constexpr uint32_t idesc = tc::idesc_bf16_f32(2 * LP_ROWS, LP_COLS);
            int done = 0, it = 0;
            for (int t = pair; t < g.tiles && !flags[0]; t += pairs) {
                for (int kb = 0; kb < g.k_blocks && !flags[0]; it++) {
                    const int b = it & 1, kb_end = SEGMENTS ? min(kb + g.segment_blocks, g.k_blocks) : g.k_blocks;
                    if (!tc::mbar_wait(&acc_empty[b], ((it >> 1) & 1) ^ 1)) {  // both CTAs are done with this accumulator
                        flags[0] = 1;
                        break;
                    }
                    tc::fence_after_sync();
                    for (bool more = false; kb < kb_end; kb++, done++) {
                        const int s = done % LP_STAGES;
                        if (!tc::mbar_wait(&full[s], (done / LP_STAGES) & 1)) {
                            flags[0] = 1;
                            break;
                        }
                        tc::fence_after_sync();
                        const uint32_t a = tc::smem_addr(a_tiles + s * LP_A_BYTES), bq = tc::smem_addr(b_tiles + s * LP_B_BYTES);
#pragma unroll
                        for (int k = 0; k < LP_K / 16; k++, more = true)
                            tc::mma_ss_pair(tmem + b * LP_COLS, tc::smem_desc_k_sw128(a + k * 32), tc::smem_desc_k_sw128(bq + k * 32), idesc, more);
                        tc::mma_commit_pair(&empty[s]);
                    }
                    if (!flags[0]) tc::mma_commit_pair(&acc_full[b]);
                }
            }
        }
    } else {
        // warp w reads lanes 32 * (w % 4) .. + 31 of the accumulator: rows; and half of its columns
        const int quarter = warp & 3, half = (warp - 2) >> 2, row = quarter * 32 + lane;
        const float4 nothing = make_float4(-3.402823466e38f, 0.0f, 0.0f, 0.0f);
        auto clear = [&]() {
            for (int i = 0; i < LP_GROUP; i++) state[(i * 2 + half) * LP_ROWS + row] = nothing;
        };
        auto leave = [&](int group) {  // the group's sums of this pair, the halves joined
            asm volatile("bar.sync 1, 256;" ::: "memory");
            const int wide = min(LP_GROUP, g.m_tiles - group * LP_GROUP);
            for (int i = half; i < wide; i += 2) {
                const int p = (group * LP_GROUP + i) * 2 * LP_ROWS + rank * LP_ROWS + row;
                const float4 u = state[i * 2 * LP_ROWS + row], v = state[(i * 2 + 1) * LP_ROWS + row];
                const RowSums s = joined({u.x, u.y, u.z, 0.0f}, {v.x, v.y, v.z, 0.0f});
                if (p < g.rows) g.parts[(long long)pair * g.rows + p] = make_float4(s.m, s.l, s.t, 0.0f);
            }
            asm volatile("bar.sync 1, 256;" ::: "memory");
            clear();
        };
        clear();
        int it = 0, group = 0;
        const int segments = SEGMENTS ? g.segments : 1;
        float sum[SEGMENTS ? LP_COLS / 2 : 1];  // of the segments so far, this thread's columns
        pdl_wait();
        bool ok = true;
        for (int t = pair; t < g.tiles && ok; t += pairs) {
            const LpTile at = tile_at(g, t);
            while (group < at.group) leave(group++);
            const int p = at.row0 + rank * LP_ROWS + row, col0 = at.col0 + half * (LP_COLS / 2);
            const bool mine = p < g.rows;
            const int wanted = (mine ? g.tokens[p] : -1) - col0;  // the given token's place among this thread's columns
            float4 &kept = state[(at.in_group * 2 + half) * LP_ROWS + row];
            const float4 s = kept;
            const bool any = __any_sync(0xffffffffu, mine);
            for (int segment = 0; segment < segments; segment++, it++) {
                const int b = it & 1;
                ok = __all_sync(0xffffffffu, !flags[0] && tc::mbar_wait(&acc_full[b], (it >> 1) & 1));
                if (!ok) {
                    flags[0] = 1;
                    break;
                }
                tc::fence_after_sync();
                const uint32_t acc = tmem + ((uint32_t)(quarter * 32) << 16) + b * LP_COLS + half * (LP_COLS / 2);
                if (any && segment < segments - 1) {
                    if constexpr (SEGMENTS) {
#pragma unroll
                        for (int c0 = 0; c0 < LP_COLS / 2; c0 += 16) {
                            uint32_t w[16];
                            tc::tmem_ld16(acc + c0, w);
                            tc::tmem_ld_wait();
#pragma unroll
                            for (int j = 0; j < 16; j++) sum[c0 + j] = segment ? sum[c0 + j] + __uint_as_float(w[j]) : __uint_as_float(w[j]);
                        }
                    }
                } else if (any) {
                    float2 l = make_float2(s.y, 0.0f), tt = make_float2(s.z, 0.0f);
                    float m = s.x;
                    const bool here = __any_sync(0xffffffffu, wanted >= 0 && wanted < LP_COLS / 2 && wanted + col0 < g.vocab);
                    auto columns = [&](int c0) {
                        __align__(8) uint32_t w[32];
                        tc::tmem_ld16(acc + c0, w), tc::tmem_ld16(acc + c0 + 16, w + 16);
                        tc::tmem_ld_wait();
                        float *v = (float *)w;
                        if constexpr (SEGMENTS) {
#pragma unroll
                            for (int j = 0; j < 32; j++) v[j] += sum[c0 + j];
                        }
                        const bool edge = col0 + c0 + 32 > g.vocab;
                        if (edge) {  // columns behind the vocabulary, until they are left out below: the first one again
#pragma unroll
                            for (int j = 1; j < 32; j++)
                                if (col0 + c0 + j >= g.vocab) v[j] = v[0];
                        }
                        if (here) {
#pragma unroll
                            for (int j = 0; j < 32; j++)
                                if (wanted == c0 + j && col0 + c0 + j < g.vocab) g.given[p] = v[j];
                        }
                        float most = v[0], least = v[0];
#pragma unroll
                        for (int j = 1; j < 32; j++) most = fmaxf(most, v[j]), least = fminf(least, v[j]);
                        if (most > m) {
                            const float d = fmaxf(m - most, LOGPROBS_FAR), e = ex2(d * 1.4426950408889634f);
                            tt = mul2(make_float2(e, e), fma2(l, make_float2(d, d), tt)), l = mul2(make_float2(e, e), l), m = most;
                        }
                        // The end of the vocabulary, or a distance that float32 does not hold (0 times it would be NaN): one by one,
                        // with the same roundings (the warp's other rows come this way too).
                        if (__any_sync(0xffffffffu, edge || least - m < LOGPROBS_FAR)) {
#pragma unroll
                            for (int j = 0; j < 32; j++) {
                                const float d = v[j] - m, e = ex2(d * 1.4426950408889634f);
                                if (col0 + c0 + j >= g.vocab) continue;
                                float &l1 = j & 1 ? l.y : l.x, &t1 = j & 1 ? tt.y : tt.x;
                                l1 += v[j] == -INFINITY ? __int_as_float(0x7fffffff) : e, t1 = fmaf(e, fmaxf(d, LOGPROBS_FAR), t1);
                            }
                            return;
                        }
                        const float2 down = make_float2(-m, -m), unit = make_float2(1.4426950408889634f, 1.4426950408889634f);
#pragma unroll
                        for (int j = 0; j < 16; j++) {
                            const float2 d = add2(((const float2 *)v)[j], down), y = mul2(d, unit), e = make_float2(ex2(y.x), ex2(y.y));
                            l = add2(l, e), tt = fma2(e, d, tt);
                        }
                    };
                    if constexpr (SEGMENTS) {  // (the sums are registers: every column by its own number)
#pragma unroll
                        for (int c0 = 0; c0 < LP_COLS / 2; c0 += 32)
                            if (col0 + c0 < g.vocab) columns(c0);
                    } else {
#pragma unroll 1
                        for (int c0 = 0; c0 < LP_COLS / 2 && col0 + c0 < g.vocab; c0 += 32) columns(c0);
                    }
                    kept = make_float4(m, l.x + l.y, tt.x + tt.y, 0.0f);
                }
                tc::fence_before_sync();
                __syncwarp();
                if (lane == 0) tc::mbar_arrive_in_cluster(tc::peer_smem(tc::smem_addr(&acc_empty[b]), 0));
            }
        }
        while (group < g.groups) leave(group++);
    }
    // Nobody leaves while the other CTA may still signal its barriers or write its tensor memory. (After a wait that ran
    // out, copies may still be on their way into this CTA's shared memory: give them a tenth of a millisecond.)
    if (flags[0]) {
        const uint64_t t0 = tc::global_ns();
        while (tc::global_ns() - t0 < 100000) __nanosleep(1000);
    }
    tc::fence_before_sync();
    tc::cluster_sync();
    if (flags[0] && threadIdx.x == 0) atomicOr(g.status + 1, 1);
    if (warp == 1) {
        tc::fence_after_sync();
        tc::tmem_free_pair(tmem, TMEM_COLS);
    }
}

// ------------------------------------------------------------------ few rows
#define LP_FEW 64
#define LP_FEW_STAGES 8
#define LP_FEW_SMEM (LP_FEW_STAGES * (LP_A_BYTES + LP_FEW * LP_K * 2) + 1024 /* alignment */ + 256 /* barriers */)

struct FewLogProbs {
    int rows, columns, vocab, high, tiles, k_blocks, segment_blocks, segments;  // columns: the rows of x, up to a multiple of 16; high: rows of w a tile
    const int *tokens;
    float *given;
    float4 *parts;  // [CTAs][rows]
    int *status;
};

__global__ void __launch_bounds__(LP_THREADS) gemm_logprobs_few_kernel(const __grid_constant__ CUtensorMap map_w,
                                                                       const __grid_constant__ CUtensorMap map_x, FewLogProbs g) {
    extern __shared__ uint8_t lp_raw[];
    uint8_t *smem = (uint8_t *)(((uintptr_t)lp_raw + 1023) & ~(uintptr_t)1023);
    const int b_bytes = g.columns * LP_K * 2;
    uint8_t *a_tiles = smem, *b_tiles = smem + LP_FEW_STAGES * LP_A_BYTES;
    uint64_t *full = (uint64_t *)(b_tiles + LP_FEW_STAGES * LP_FEW * LP_K * 2);
    uint64_t *empty = full + LP_FEW_STAGES, *acc_full = empty + LP_FEW_STAGES, *acc_empty = acc_full + 2;
    uint32_t *tmem_holder = (uint32_t *)(acc_empty + 2);
    volatile int *flags = (volatile int *)(tmem_holder + 1);  // [0]: a wait ran out
    __shared__ int token_s[LP_FEW];
    __shared__ float4 sums_s[4][LP_FEW];
    constexpr uint32_t TMEM_COLS = 2 * LP_FEW;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int s = 0; s < LP_FEW_STAGES; s++) tc::mbar_init(&full[s], 1), tc::mbar_init(&empty[s], 1);
        for (int b = 0; b < 2; b++) tc::mbar_init(&acc_full[b], 1), tc::mbar_init(&acc_empty[b], 8);
        flags[0] = 0;
        tc::mbar_init_fence();
        tc::tma_prefetch_map(&map_x), tc::tma_prefetch_map(&map_w);
    }
    if (warp == 1) tc::tmem_alloc(tmem_holder, TMEM_COLS);
    pdl_wait();
    if (threadIdx.x < g.rows) token_s[threadIdx.x] = g.tokens[threadIdx.x];
    tc::fence_before_sync();
    __syncthreads();
    tc::fence_after_sync();
    const uint32_t tmem = *tmem_holder;

    if (warp == 0) {
        if (lane == 0) {
            int issued = 0;
            for (int t = blockIdx.x; t < g.tiles && !flags[0]; t += gridDim.x) {
                for (int kb = 0; kb < g.k_blocks; kb++, issued++) {
                    const int s = issued % LP_FEW_STAGES;
                    if (!tc::mbar_wait(&empty[s], ((issued / LP_FEW_STAGES) & 1) ^ 1)) {
                        flags[0] = 1;
                        break;
                    }
                    tc::mbar_expect_tx(&full[s], g.high * LP_K * 2 + b_bytes);
                    tc::tma_load_2d(a_tiles + s * LP_A_BYTES, &map_w, kb * LP_K, t * g.high, &full[s]);
                    tc::tma_load_2d(b_tiles + s * b_bytes, &map_x, kb * LP_K, 0, &full[s]);
                }
            }
            if (flags[0])  // let the copies still in flight land before the CTA's memory goes away
                for (int i = max(0, issued - LP_FEW_STAGES); i < issued; i++) tc::mbar_wait(&full[i % LP_FEW_STAGES], (i / LP_FEW_STAGES) & 1);
        }
    } else if (warp == 1) {
        if (lane == 0) {
            const uint32_t idesc = tc::idesc_bf16_f32(LP_ROWS, g.columns);
            int done = 0, it = 0;
            for (int t = blockIdx.x; t < g.tiles && !flags[0]; t += gridDim.x) {
                for (int kb = 0; kb < g.k_blocks && !flags[0]; it++) {
                    const int b = it & 1, kb_end = min(kb + g.segment_blocks, g.k_blocks);
                    if (!tc::mbar_wait(&acc_empty[b], ((it >> 1) & 1) ^ 1)) {
                        flags[0] = 1;
                        break;
                    }
                    tc::fence_after_sync();
                    for (bool more = false; kb < kb_end; kb++, done++) {
                        const int s = done % LP_FEW_STAGES;
                        if (!tc::mbar_wait(&full[s], (done / LP_FEW_STAGES) & 1)) {
                            flags[0] = 1;
                            break;
                        }
                        tc::fence_after_sync();
                        const uint32_t a = tc::smem_addr(a_tiles + s * LP_A_BYTES), bq = tc::smem_addr(b_tiles + s * b_bytes);
#pragma unroll
                        for (int k = 0; k < LP_K / 16; k++, more = true)
                            tc::mma_ss(tmem + b * LP_FEW, tc::smem_desc_k_sw128(a + k * 32), tc::smem_desc_k_sw128(bq + k * 32), idesc, more);
                        tc::mma_commit(&empty[s]);
                    }
                    if (!flags[0]) tc::mma_commit(&acc_full[b]);
                }
            }
        }
    } else {
        // warp w reads lanes 32 * (w % 4) .. + 31 of the accumulator, tokens of the vocabulary, and 32 of the rows of x
        constexpr int COLS = LP_FEW / 2;
        static_assert(COLS == 32, "a column a lane at the end");
        const int quarter = warp & 3, half = (warp - 2) >> 2, col0 = half * COLS;
        float m[COLS], l[COLS], tt[COLS];
#pragma unroll
        for (int j = 0; j < COLS; j++) m[j] = -3.402823466e38f, l[j] = 0.0f, tt[j] = 0.0f;
        bool ok = true;
        int it = 0;
        for (int t = blockIdx.x; t < g.tiles && ok; t += gridDim.x) {
            const int in_tile = quarter * 32 + lane, token = t * g.high + in_tile;
            const bool mine = in_tile < g.high && token < g.vocab;
            float sum[COLS];
            for (int segment = 0; segment < g.segments; segment++, it++) {
                const int b = it & 1;
                ok = __all_sync(0xffffffffu, !flags[0] && tc::mbar_wait(&acc_full[b], (it >> 1) & 1));
                if (!ok) {
                    flags[0] = 1;
                    break;
                }
                tc::fence_after_sync();
#pragma unroll
                for (int c0 = 0; c0 < COLS; c0 += 16) {
                    if (col0 + c0 >= g.columns) continue;
                    uint32_t w[16];
                    tc::tmem_ld16(tmem + ((uint32_t)(quarter * 32) << 16) + b * LP_FEW + col0 + c0, w);
                    tc::tmem_ld_wait();
#pragma unroll
                    for (int j = 0; j < 16; j++) sum[c0 + j] = segment ? sum[c0 + j] + __uint_as_float(w[j]) : __uint_as_float(w[j]);
                }
                tc::fence_before_sync();
                __syncwarp();
                if (lane == 0) tc::mbar_arrive(&acc_empty[b]);
            }
            if (ok && mine) {
#pragma unroll
                for (int j = 0; j < COLS; j++) {
                    if (col0 + j >= g.rows) continue;
                    const float v = sum[j], n = fmaxf(m[j], v), dm = fmaxf(m[j] - n, LOGPROBS_FAR), dv = v - n;
                    const float a = ex2(dm * 1.4426950408889634f), e = ex2(dv * 1.4426950408889634f);
                    tt[j] = fmaf(a, fmaf(l[j], dm, tt[j]), e * fmaxf(dv, LOGPROBS_FAR));
                    l[j] = v == -INFINITY ? __int_as_float(0x7fffffff) : fmaf(l[j], a, e), m[j] = n;
                    if (token_s[col0 + j] == token) g.given[col0 + j] = v;
                }
            }
            __syncwarp();
        }
        // The lanes' sums of 32 columns joined to a column a lane: at every step a lane gives away half of its columns and takes the
        // other lane's share of the half it keeps (31 joins a lane, where every column for itself would take 160).
#pragma unroll
        for (int n = COLS / 2; n > 0; n >>= 1) {
            const bool upper = lane & n;
#pragma unroll
            for (int j = 0; j < n; j++) {
                const RowSums keep = {upper ? m[j + n] : m[j], upper ? l[j + n] : l[j], upper ? tt[j + n] : tt[j], 0.0f};
                RowSums come;
                come.m = __shfl_xor_sync(0xffffffffu, upper ? m[j] : m[j + n], n);
                come.l = __shfl_xor_sync(0xffffffffu, upper ? l[j] : l[j + n], n);
                come.t = __shfl_xor_sync(0xffffffffu, upper ? tt[j] : tt[j + n], n);
                const RowSums both = joined(keep, come);
                m[j] = both.m, l[j] = both.l, tt[j] = both.t;
            }
        }
        sums_s[quarter][col0 + lane] = make_float4(m[0], l[0], tt[0], 0.0f);
    }
    tc::fence_before_sync();
    __syncthreads();
    if (threadIdx.x < g.rows) {
        RowSums s = {-3.402823466e38f, 0.0f, 0.0f, 0.0f};
        for (int q = 0; q < 4; q++) {
            const float4 x = sums_s[q][threadIdx.x];
            s = joined(s, {x.x, x.y, x.z, 0.0f});
        }
        g.parts[(long long)blockIdx.x * g.rows + threadIdx.x] = make_float4(s.m, s.l, s.t, 0.0f);
    }
    if (flags[0] && threadIdx.x == 0) atomicOr(g.status + 1, 1);
    if (warp == 1) {
        tc::fence_after_sync();
        tc::tmem_free(tmem, TMEM_COLS);
    }
}

// A warp a row: the pairs' sums joined.
__global__ void __launch_bounds__(128) logprobs_join_kernel(const float4 *__restrict__ parts, int pairs, int rows, int vocab,
                                                            const int *__restrict__ tokens, const float *__restrict__ given,
                                                            float *__restrict__ logprob, float *__restrict__ entropy) {
    pdl_wait();
    const int row = blockIdx.x * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (row >= rows) return;
    RowSums s = {-3.402823466e38f, 0.0f, 0.0f, 0.0f};
    for (int c0 = 0; c0 < pairs; c0 += 128) {
        float4 x[4];
#pragma unroll
        for (int i = 0; i < 4; i++)
            x[i] = c0 + 32 * i + lane < pairs ? parts[(long long)(c0 + 32 * i + lane) * rows + row] : make_float4(-3.402823466e38f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int i = 0; i < 4; i++) s = joined(s, {x[i].x, x[i].y, x[i].z, 0.0f});
    }
    s = joined_lanes(s, 16);
    if (lane == 0) {
        const int token = tokens[row];
        const float log_l = logf(s.l), nan = __int_as_float(0x7fffffff);
        const bool none = !(s.l > 0.0f) || !(s.t == s.t);  // (a NaN or an infinity among the logits)
        logprob[row] = none || token < 0 || token >= vocab ? nan : given[row] - s.m - log_l;
        if (entropy) entropy[row] = none ? nan : log_l - s.t / s.l;
    }
}

// Whether few rows against this matrix go to the kernel made for them: the fewer the rows and the larger the matrix, the longer its reading
// lasts beside what that kernel does at its end. us, that kernel and the one above: 151,936 x 1,024 with 1 row 55 and 84, 33 60 and 74, 64 63 and
// 65; x 4,096 with 64 203 and 254; 64,000 x 1,024 with 16 31 and 35, 48 35 and 36, 64 36 and 33; 32,000 x 1,024 with 16 18.6 and 21,
// 48 22.2 and 21.8; 16,000 x 1,024 with 1 12.5 and 15.5, 16 13.5 and 13.6, 33 15.4 and 13.7; 8,000 x 512 with 16 10.7 and 10.1.
static bool few_wins(int M, int V, int K) { return M <= LP_FEW && (long long)M * 1400000 <= (long long)V * K; }

// Floats of memory for the sums of `rows` rows: 4 a row and pair of CTAs, and the given tokens' logits.
extern "C" long long abk_gemm_logprobs_floats(int rows) {
    const long long most = rows < LP_MOST_ROWS ? rows : LP_MOST_ROWS;
    return most * (4 * (rows <= LP_FEW ? abk_sm_count() : abk_sm_count() / 2) + 1) + 4;
}
extern "C" int abk_gemm_logprobs(const void *x, const void *w, int M, int V, int K, long long ldx, long long ldw, const int *tokens,
                                 float *logprob, float *entropy, float *memory, long long floats, int *status, void *stream) {
    if (M <= 0) return 0;
    if (V < 1 || K < 1 || K % 8) ABK_REFUSE("gemm_logprobs: a vocabulary of %d and rows of %d (a multiple of 8)", V, K);
    if (((uintptr_t)x & 15) || ((uintptr_t)w & 15) || ldx % 8 || ldw % 8 || ((uintptr_t)memory & 15))
        ABK_REFUSE("gemm_logprobs: operands must be 16-byte aligned with pitches of a multiple of 8");
    if (floats < abk_gemm_logprobs_floats(M)) ABK_REFUSE("gemm_logprobs: room for %lld floats is too little", floats);
    const int k_blocks = (K + LP_K - 1) / LP_K, pieces = (k_blocks + LP_SEGMENT - 1) / LP_SEGMENT;  // segments as equal as whole blocks allow
    const int segment_blocks = (k_blocks + pieces - 1) / pieces, segments = (k_blocks + segment_blocks - 1) / segment_blocks;
    if (few_wins(M, V, K)) {
        const int ctas = abk_sm_count();
        FewLogProbs g;
        const long long waves = (V + (long long)ctas * LP_ROWS - 1) / ((long long)ctas * LP_ROWS);
        g.high = (int)((V + waves * ctas - 1) / (waves * ctas));
        if (g.high < 16) g.high = 16;
        g.rows = M, g.columns = (M + 15) / 16 * 16, g.vocab = V, g.tiles = (V + g.high - 1) / g.high;
        g.k_blocks = k_blocks, g.segment_blocks = segment_blocks, g.segments = segments, g.tokens = tokens, g.status = status;
        const int grid = g.tiles < ctas ? g.tiles : ctas;
        g.parts = (float4 *)memory, g.given = memory + 4ll * grid * M;
        CUtensorMap mx, mw;
        int rc = tmap::bf16_rows_of_128_bytes(x, M, K, ldx, g.columns, &mx);
        if (!rc) rc = tmap::bf16_rows_of_128_bytes(w, V, K, ldw, g.high, &mw);
        if (rc) return rc;
        if (cudaError_t e = abk_allow_shared_memory((const void *)gemm_logprobs_few_kernel, LP_FEW_SMEM)) return (int)e;
        abk_launch(gemm_logprobs_few_kernel, dim3(grid), dim3(LP_THREADS), LP_FEW_SMEM, (cudaStream_t)stream, mw, mx, g);
        rc = ABK_LAUNCH_RESULT();
        if (rc) return rc;
        abk_launch(logprobs_join_kernel, dim3((M + 3) / 4), dim3(128), 0, (cudaStream_t)stream, (const float4 *)g.parts, grid, M, V, tokens,
                   (const float *)g.given, logprob, entropy);
        return ABK_LAUNCH_RESULT();
    }
    auto kernel = k_blocks > LP_SEGMENT ? gemm_logprobs_kernel<true> : gemm_logprobs_kernel<false>;
    if (cudaError_t e = abk_allow_shared_memory((const void *)kernel, LP_SMEM)) return (int)e;
    for (int first = 0; first < M; first += LP_MOST_ROWS) {
        const int rows = M - first < LP_MOST_ROWS ? M - first : LP_MOST_ROWS;
        CUtensorMap mx, mw;
        int rc = tmap::bf16_rows_of_128_bytes((const char *)x + 2ll * first * ldx, rows, K, ldx, LP_ROWS, &mx);
        if (!rc) rc = tmap::bf16_rows_of_128_bytes(w, V, K, ldw, LP_COLS / 2, &mw);
        if (rc) return rc;
        GemmLogProbs g;
        g.rows = rows, g.vocab = V, g.k_blocks = k_blocks, g.segment_blocks = segment_blocks, g.segments = segments, g.m_tiles = (rows + 2 * LP_ROWS - 1) / (2 * LP_ROWS);
        g.v_tiles = (V + LP_COLS - 1) / LP_COLS, g.groups = (g.m_tiles + LP_GROUP - 1) / LP_GROUP;
        if ((long long)g.m_tiles * g.v_tiles > 0x3fffffff) ABK_REFUSE("gemm_logprobs: a vocabulary of %d is too many tiles", V);
        g.tiles = g.m_tiles * g.v_tiles, g.tokens = tokens + first, g.status = status;
        int pairs = abk_sm_count() / 2;
        if (g.tiles < pairs) pairs = g.tiles;
        g.parts = (float4 *)memory, g.given = memory + 4ll * pairs * rows;
        abk_launch_clusters(kernel, dim3(2 * pairs), dim3(LP_THREADS), LP_SMEM, (cudaStream_t)stream, 2, mx, mw, g);
        rc = ABK_LAUNCH_RESULT();
        if (rc) return rc;
        abk_launch(logprobs_join_kernel, dim3((rows + 3) / 4), dim3(128), 0, (cudaStream_t)stream, (const float4 *)g.parts, pairs, rows, V,
                   g.tokens, (const float *)g.given, logprob + first, entropy ? entropy + first : nullptr);
        rc = ABK_LAUNCH_RESULT();
        if (rc) return rc;
    }
    return 0;
}
