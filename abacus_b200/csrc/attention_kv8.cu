// Attention of a step's rows over a cache held in 8 bits (csrc/kv8.cu): a few new tokens a sequence against everything the
// cache holds of it, each row to its own position.
//
// out = sum_j softmax_j(scale q . k_j) v_j over the keys j <= position (and within the window): keys of whole blocks are
// q_j s_b with the block's scale s_b, so a score is s_b (q . q_j) and a value's weight p_j s_b; keys of the sequence's open
// block are bfloat16. Scores, the running maximum and sum, and the weighted values are float32.
#define ABK_DEFINE_ERROR
#include "common.cuh"
#include "kv8.cuh"

#define KV8_HEADS 16  // query heads a CTA takes at once

struct AttnKv8 {
    const __nv_bfloat16 *q;
    long long q_row;
    __nv_bfloat16 *out;
    int n_heads, n_kv_heads, runs;
    float scale_log2;
    int window;
    const int *token_seq, *token_pos, *seq_slot, *seq_len_after;
    PagedCache cache;
    const uint8_t *k, *v;
    const float *scales;
    const __nv_bfloat16 *open;
    int n_pages, *status;
};

template <int HD, int FORM>
__global__ void __launch_bounds__(128) attention_kv8_kernel(AttnKv8 p) {
    constexpr int E = HD / 32;
    __shared__ float q_s[KV8_HEADS][HD], part_o[KV8_HEADS][HD], part_m[4][KV8_HEADS], part_l[4][KV8_HEADS];
    pdl_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = blockIdx.z;
    const int group = p.n_heads / p.n_kv_heads, kvh = blockIdx.y, g0 = blockIdx.x * KV8_HEADS, heads = min(KV8_HEADS, group - g0);
    const int h0 = kvh * group + g0, seq = p.token_seq[r];
    __nv_bfloat16 *out = p.out + ((long long)r * p.n_heads + h0) * HD;
    if (seq < 0) {
        for (int i = threadIdx.x; i < heads * HD; i += 128) out[i] = __float2bfloat16_rn(0.0f);
        return;
    }
    const int pos = p.token_pos[r], slot = p.seq_slot[seq], closed = p.seq_len_after[seq] / KV8_BLOCK;
    const int lo = p.window > 0 ? max(0, pos - p.window + 1) : 0;
    for (int i = threadIdx.x; i < heads * HD; i += 128) q_s[i / HD][i % HD] = __bfloat162float(p.q[r * p.q_row + (long long)h0 * HD + i]);
    __syncthreads();
    float o[KV8_HEADS][E], m[KV8_HEADS], l[KV8_HEADS];
#pragma unroll
    for (int g = 0; g < KV8_HEADS; g++) {
        m[g] = -INFINITY, l[g] = 0.0f;
#pragma unroll
        for (int e = 0; e < E; e++) o[g][e] = 0.0f;
    }
    for (int b = lo / KV8_BLOCK + warp; b <= pos / KV8_BLOCK; b += 4) {
        const bool whole = b < closed;
        const int page = whole ? kv8_page(p.cache, p.n_pages, slot, b * KV8_BLOCK, p.status) : 0;
        const long long at = cache_offset(p.cache, page, kvh, p.n_kv_heads, b * KV8_BLOCK, HD);
        const float *sc = p.scales + ((long long)page * p.n_kv_heads + kvh) * 2 * KV8_PAGE_BLOCKS + b % KV8_PAGE_BLOCKS;
        const float ks = whole ? sc[0] : 1.0f, vs = whole ? sc[KV8_PAGE_BLOCKS] : 1.0f;
        const __nv_bfloat16 *ok = p.open + ((long long)slot * 2 * p.n_kv_heads + kvh) * (KV8_BLOCK * HD),
                            *ov = ok + (long long)p.n_kv_heads * (KV8_BLOCK * HD);
        for (int t = max(0, lo - b * KV8_BLOCK); t < KV8_BLOCK && b * KV8_BLOCK + t <= pos; t++) {
            float k[E], v[E];
#pragma unroll
            for (int e = 0; e < E; e++) {
                const int d = lane * E + e;
                if (whole) {
                    float four[4];
                    kv8_unpack<FORM>(p.k[at + t * HD + d], four), k[e] = four[0];
                    kv8_unpack<FORM>(p.v[at + t * HD + d], four), v[e] = four[0];
                } else {
                    k[e] = __bfloat162float(ok[t * HD + d]), v[e] = __bfloat162float(ov[t * HD + d]);
                }
            }
#pragma unroll
            for (int g = 0; g < KV8_HEADS; g++) {
                if (g >= heads) break;
                float s = 0.0f;
#pragma unroll
                for (int e = 0; e < E; e++) s = fmaf(q_s[g][lane * E + e], k[e], s);
                s = warp_sum(s) * (p.scale_log2 * ks);
                const float n = fmaxf(m[g], s), c = m[g] == n ? 1.0f : exp2f(m[g] - n), w = exp2f(s - n);
                m[g] = n, l[g] = l[g] * c + w;
#pragma unroll
                for (int e = 0; e < E; e++) o[g][e] = o[g][e] * c + w * vs * v[e];
            }
        }
    }
    for (int w = 0; w < 4; w++) {  // the warps' results one after another
        if (warp == w) {
#pragma unroll
            for (int g = 0; g < KV8_HEADS; g++) {
                if (g >= heads) break;
                const float before = w ? part_m[0][g] : -INFINITY, n = fmaxf(before, m[g]);
                const float a = before == -INFINITY ? 0.0f : exp2f(before - n), c = m[g] == -INFINITY ? 0.0f : exp2f(m[g] - n);
                __syncwarp();
#pragma unroll
                for (int e = 0; e < E; e++) part_o[g][lane * E + e] = (w ? part_o[g][lane * E + e] * a : 0.0f) + o[g][e] * c;
                if (lane == 0) part_m[0][g] = n, part_l[0][g] = (w ? part_l[0][g] * a : 0.0f) + l[g] * c;
                __syncwarp();
            }
        }
        __syncthreads();
    }
    for (int i = threadIdx.x; i < heads * HD; i += 128) out[i] = __float2bfloat16_rn(part_o[i / HD][i % HD] / part_l[0][i / HD]);
}

// max_positions: no row's position reaches it.
extern "C" int abk_attention_kv8(const void *q, long long q_row, void *out, int n_rows, int n_heads, int n_kv_heads, int head_dim,
                                 int form, float scale, int window, const int *token_seq, const int *token_pos, const int *seq_slot,
                                 const int *seq_len_after, const void *k, const void *v, const float *scales, const void *open,
                                 const int *page_table, int table_width, int ring_pages, int pool_pages, int *status,
                                 void *stream) {
    if (n_rows <= 0) return 0;
    if (head_dim != 64 && head_dim != 128) ABK_REFUSE("attention_kv8: head_dim %d is not 64 or 128", head_dim);
    if (form != KV8_INT8 && form != KV8_E4M3) ABK_REFUSE("attention_kv8: no 8-bit form %d", form);
    if (n_kv_heads < 1 || n_heads % n_kv_heads) ABK_REFUSE("attention_kv8: %d heads do not divide into %d kv heads", n_heads, n_kv_heads);
    if (n_kv_heads > 65535 || n_rows > 65535) ABK_REFUSE("attention_kv8: %d rows or %d kv heads exceed a grid", n_rows, n_kv_heads);
    AttnKv8 p;
    p.q = (const __nv_bfloat16 *)q, p.q_row = q_row, p.out = (__nv_bfloat16 *)out, p.n_heads = n_heads, p.n_kv_heads = n_kv_heads;
    p.scale_log2 = scale * 1.4426950408889634f, p.window = window, p.token_seq = token_seq, p.token_pos = token_pos;
    p.seq_slot = seq_slot, p.seq_len_after = seq_len_after, p.cache.page_table = page_table, p.cache.table_width = table_width;
    p.cache.ring_pages = ring_pages, p.cache.tokens_per_page = KV8_PAGE, p.k = (const uint8_t *)k, p.v = (const uint8_t *)v;
    p.scales = scales, p.open = (const __nv_bfloat16 *)open, p.n_pages = pool_pages, p.status = status;
    p.runs = (n_heads / n_kv_heads + KV8_HEADS - 1) / KV8_HEADS;
    const dim3 grid(p.runs, n_kv_heads, n_rows), block(128);
    auto go = [&](auto kernel) { abk_launch(kernel, grid, block, 0, (cudaStream_t)stream, p); };
    if (head_dim == 64) form == KV8_INT8 ? go(attention_kv8_kernel<64, KV8_INT8>) : go(attention_kv8_kernel<64, KV8_E4M3>);
    else form == KV8_INT8 ? go(attention_kv8_kernel<128, KV8_INT8>) : go(attention_kv8_kernel<128, KV8_E4M3>);
    return ABK_LAUNCH_RESULT();
}
