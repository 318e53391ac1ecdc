// Keys and values held in 8 bits: a step's new ones into the cache, and a sequence's read back as pages.
//
// Blocks of KV8_BLOCK = 16 tokens of a sequence and kv head have one scale each for keys and for values:
// x ~ q * s with s = max|x| / 127 and q = rint(127 x / max|x|) a whole number (stored as q + 128), or
// s = max|x| / 448 and q the nearest e4m3 number. The quotient is taken of 127 x (448 x), which is a float32 number whatever the
// bfloat16 x, so a value halfway between two steps is seen as that and goes to the even one. A block of zeros has the scale
// zero; a block with a value that is not finite reads back as NaN.
// A block is put into 8 bits when its last token comes; until then its tokens lie as they came in the slot's open block,
// so that no value is ever rounded twice and a token's place in the 8-bit pages is written once.
// A warp takes one block of one head's keys or values, 16 rows of the step in 16-byte pieces, in registers from load to store. Measured:
// prompts of 5,745 tokens, 8 heads of 128, 35 MB in and out, in 10 us, read back as float32 in 13 (59 MB); single tokens of 32 sequences in 3.
#define ABK_DEFINE_ERROR
#include "common.cuh"
#include "kv8.cuh"
#include "qkv_prep.cuh"

#define KV8_WARPS 4

struct Kv8Write {
    const __nv_bfloat16 *qkv;  // k head h of row r at qkv + r * row + (n_heads + h) * head_dim, v n_kv_heads heads further
    long long row;
    int n_heads, n_kv_heads, n_seqs, one_each;
    const int *seq_start, *seq_pos0, *seq_len_after, *seq_slot;
    PagedCache cache;
    uint8_t *k, *v;
    float *scales;
    __nv_bfloat16 *open;
    int n_pages, n_slots, *status;
};

// A warp holds a block in pieces of 8 elements: token t, elements 8 c .., in piece i of a lane with 32 i + lane = t * HD / 8 + c.
// A whole block into 8 bits, by a warp.
template <int HD, int FORM>
__device__ __forceinline__ void close_block(const Kv8Write &p, const uint4 *x, int slot, int head, int j, int pos0, int lane) {
    constexpr int PIECES = KV8_BLOCK * HD / 256;
    __nv_bfloat162 top2 = __floats2bfloat162_rn(0.0f, 0.0f);
#pragma unroll
    for (int i = 0; i < PIECES; i++) {
        const __nv_bfloat162 *h = (const __nv_bfloat162 *)&x[i];
#pragma unroll
        for (int e = 0; e < 4; e++) top2 = __hmax2_nan(top2, __habs2(h[e]));
    }
    const float2 two = __bfloat1622float2(top2);
    const bool odd = __any_sync(0xffffffffu, !(two.x < INFINITY) || !(two.y < INFINITY));  // a value that is not finite
    const float most = warp_max(fmaxf(two.x, two.y));
    const Kv8Steps steps = kv8_steps<FORM>(odd ? 0.0f : most);
    const int page = kv8_page(p.cache, p.n_pages, slot, pos0, p.status);
    uint8_t *dst = (j == 0 ? p.k : p.v) + cache_offset(p.cache, page, head, p.n_kv_heads, pos0, HD);
#pragma unroll
    for (int i = 0; i < PIECES; i++) *(uint2 *)(dst + 8 * (32 * i + lane)) = kv8_pack<FORM>(x[i], steps);
    if (lane == 0)
        p.scales[(((long long)page * p.n_kv_heads + head) * 2 + j) * KV8_PAGE_BLOCKS + (pos0 % KV8_PAGE) / KV8_BLOCK] =
            odd ? __int_as_float(0x7fffffff) : most / kv8_top<FORM>();
}

template <int HD, int FORM>
__global__ void __launch_bounds__(32 * KV8_WARPS) kv8_write_kernel(Kv8Write p) {
    constexpr int LPR = HD / 8, PIECES = KV8_BLOCK * HD / 256;  // lanes to a row of 16-byte pieces
    pdl_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int which = blockIdx.y * KV8_WARPS + warp;  // keys of the heads, then values of the heads
    if (which >= 2 * p.n_kv_heads) return;
    const int j = which / p.n_kv_heads, head = which - j * p.n_kv_heads;
    // the sequence and its block: block k of a sequence that brings n tokens from row a on has its first row at f_k; unit
    // a / 16 + 2 s is block 0 and unit f_k / 16 + 2 s + 1 block k > 0 of sequence s, so units of different blocks differ
    int s = blockIdx.x, first = 0, unit = blockIdx.x;
    if (!p.one_each) {
        s = last_not_above(p.seq_start, p.n_seqs, lane, [&](int start, int i) { return start / KV8_BLOCK + 2 * i <= unit; });
        if (s < 0) return;
    }
    const int a = p.seq_start[s], n = p.seq_start[s + 1] - a;
    if (n <= 0) return;
    const int start = p.seq_pos0[s], after = p.seq_len_after[s], o = start % KV8_BLOCK;
    if (!p.one_each && unit != a / KV8_BLOCK + 2 * s) {
        const int q = unit - 2 * s - 1;
        if (q * KV8_BLOCK + KV8_BLOCK <= a) return;
        first = max(1, (q * KV8_BLOCK - a + o + KV8_BLOCK - 1) / KV8_BLOCK);
        const int row = a + first * KV8_BLOCK - o;
        if (row / KV8_BLOCK != q || row >= a + n) return;
    }
    if ((unsigned)p.seq_slot[s] >= (unsigned)p.n_slots) {  // nothing is written
        kv8_slot(p.seq_slot[s], p.n_slots, p.status);
        return;
    }
    const int slot = p.seq_slot[s];
    const int b0 = start / KV8_BLOCK, last = (after - 1) / KV8_BLOCK;
    // The open block's place holds the first block's earlier tokens until they have been read: where the step also leaves an
    // open block behind, one warp does both, in that order.
    const bool both = o != 0 && last > b0 && after % KV8_BLOCK != 0;
    int b = b0 + first;
    if (both && b == last) return;
    __nv_bfloat16 *open = p.open + (((long long)slot * 2 + j) * p.n_kv_heads + head) * (KV8_BLOCK * HD);
    const __nv_bfloat16 *src = p.qkv + (p.n_heads + j * p.n_kv_heads + head) * (long long)HD;
    for (;;) {
        const int pos0 = b * KV8_BLOCK;
        const bool whole = pos0 + KV8_BLOCK <= after;
        uint4 x[PIECES];
#pragma unroll
        for (int i = 0; i < PIECES; i++) {
            const int t = (32 * i + lane) / LPR, c = (32 * i + lane) % LPR, pos = pos0 + t;
            if (pos >= start && pos < after) x[i] = *(const uint4 *)(src + (long long)(a + pos - start) * p.row + 8 * c);
            else if (pos < start && whole) x[i] = *(const uint4 *)(open + t * HD + 8 * c);
        }
        if (!whole) {
#pragma unroll
            for (int i = 0; i < PIECES; i++) {
                const int t = (32 * i + lane) / LPR, c = (32 * i + lane) % LPR, pos = pos0 + t;
                if (pos >= start && pos < after) *(uint4 *)(open + t * HD + 8 * c) = x[i];
            }
        } else if (cache_keeps(p.cache, pos0 + KV8_BLOCK - 1, after)) {  // (a place goes to the later block with its last token)
            close_block<HD, FORM>(p, x, slot, head, j, pos0, lane);
        }
        if (!both || b != b0) return;
        __syncwarp();  // every lane has read its pieces of the old open block
        b = last;
    }
}

// A step of one token a sequence with its preparation (qkv_prep.cuh) taken in: q normed and rotated in place, the new token's key and value
// into the open block, or, the sixteenth of its block, with the fifteen before it into 8 bits. A warp takes 256 / HD query heads of a
// row, or one key or value head.
struct Kv8Prepare {
    __nv_bfloat16 *qkv;
    const int *token_seq, *token_pos;
    const float *q_norm, *k_norm;  // [HD]; null: no norm
    const float *cos, *sin;        // [positions, HD / 2]; null: no rotation
    float eps;
};
template <int HD, int FORM>
__global__ void __launch_bounds__(32 * KV8_WARPS) kv8_prepare_write_kernel(Kv8Write p, Kv8Prepare e) {
    constexpr int LPH = HD / 8, HPW = 32 / LPH, PIECES = KV8_BLOCK * HD / 256;
    pdl_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = blockIdx.x, sub = lane / LPH, l = lane % LPH;
    const int q_warps = (p.n_heads + HPW - 1) / HPW, unit = blockIdx.y * KV8_WARPS + warp;
    if (unit >= q_warps + 2 * p.n_kv_heads) return;
    const int seq = e.token_seq[r];
    if (seq < 0) return;
    const int pos = e.token_pos[r];
    const bool upper = l >= LPH / 2;
    float cs[8], sn[8];
    if (e.cos) {
        const int at = (upper ? l - LPH / 2 : l) * 8;
        const float4 *c4 = (const float4 *)(e.cos + (long long)pos * (HD / 2) + at), *s4 = (const float4 *)(e.sin + (long long)pos * (HD / 2) + at);
        const float4 c0 = c4[0], c1 = c4[1], s0 = s4[0], s1 = s4[1];
        cs[0] = c0.x, cs[1] = c0.y, cs[2] = c0.z, cs[3] = c0.w, cs[4] = c1.x, cs[5] = c1.y, cs[6] = c1.z, cs[7] = c1.w;
        sn[0] = s0.x, sn[1] = s0.y, sn[2] = s0.z, sn[3] = s0.w, sn[4] = s1.x, sn[5] = s1.y, sn[6] = s1.z, sn[7] = s1.w;
    }
    __nv_bfloat16 *row = e.qkv + (long long)r * p.row + 8 * l;
    if (unit < q_warps) {
        const int h = unit * HPW + sub;
        const uint4 raw = h < p.n_heads ? *(const uint4 *)(row + (long long)h * HD) : make_uint4(0, 0, 0, 0);
        const uint4 done = prep_head_values<HD>(raw, true, e.q_norm, e.eps, e.cos != nullptr, l, upper, cs, sn);
        if (h < p.n_heads) *(uint4 *)(row + (long long)h * HD) = done;
        return;
    }
    const int which = unit - q_warps, j = which / p.n_kv_heads, head = which - j * p.n_kv_heads;
    const uint4 raw = *(const uint4 *)(row + (long long)(p.n_heads + which) * HD);
    const uint4 mine = prep_head_values<HD>(raw, j == 0, e.k_norm, e.eps, e.cos != nullptr, l, upper, cs, sn);  // (the same in every run of LPH lanes)
    if ((unsigned)p.seq_slot[seq] >= (unsigned)p.n_slots) {  // nothing is written
        kv8_slot(p.seq_slot[seq], p.n_slots, p.status);
        return;
    }
    const int slot = p.seq_slot[seq], t = pos % KV8_BLOCK;
    __nv_bfloat16 *open = p.open + (((long long)slot * 2 + j) * p.n_kv_heads + head) * (KV8_BLOCK * HD);
    if (t < KV8_BLOCK - 1) {
        if (sub == 0) *(uint4 *)(open + t * HD + 8 * l) = mine;
        return;
    }
    uint4 x[PIECES];
#pragma unroll
    for (int i = 0; i < PIECES; i++) x[i] = (32 * i + lane) / LPH < KV8_BLOCK - 1 ? *(const uint4 *)(open + 8 * (32 * i + lane)) : mine;
    close_block<HD, FORM>(p, x, slot, head, j, pos - t, lane);
}

struct Kv8Read {
    const int *first_page;  // [n_seqs + 1]: sequence s goes to pages first_page[s] .. first_page[s + 1] - 1 of the copies
    const int *seq_len_after, *seq_slot;
    int n_seqs, n_kv_heads;
    PagedCache cache;
    const uint8_t *k, *v;
    const float *scales;
    const __nv_bfloat16 *open;
    void *out_k, *out_v;
    int n_pages, n_slots, *status;
};

__device__ __forceinline__ void store_piece(float *dst, const float *v) { *(float4 *)dst = make_float4(v[0], v[1], v[2], v[3]); }
__device__ __forceinline__ void store_piece(__nv_bfloat16 *dst, const float *v) {
    __nv_bfloat162 h[4];
#pragma unroll
    for (int e = 0; e < 4; e++) h[e] = __floats2bfloat162_rn(v[2 * e], v[2 * e + 1]);
    *(uint4 *)dst = *(const uint4 *)h;
}

// A warp a block of 16 tokens of one head's keys or values: 8 of them to a page and head.
template <int HD, int FORM, typename T>
__global__ void __launch_bounds__(256) kv8_read_kernel(Kv8Read p) {
    constexpr int N = 16 / sizeof(T), PIECES = KV8_BLOCK * HD / (32 * N);  // a lane stores 16 bytes at a time, N elements
    pdl_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int page_out = blockIdx.x, head = blockIdx.y, j = warp >> 2, block = warp & 3;
    const int s = last_not_above(p.first_page, p.n_seqs, lane, [&](int first, int) { return first <= page_out; });
    if (s < 0 || page_out < p.first_page[s] || page_out >= p.first_page[s + 1]) return;
    const int after = p.seq_len_after[s], slot = kv8_slot(p.seq_slot[s], p.n_slots, p.status);
    const int pos0 = (page_out - p.first_page[s]) * KV8_PAGE + block * KV8_BLOCK;
    T *dst = (T *)(j == 0 ? p.out_k : p.out_v) +
             (((long long)page_out * p.n_kv_heads + head) * KV8_PAGE + block * KV8_BLOCK) * HD;
    if (pos0 + KV8_BLOCK <= after) {
        const int page = kv8_page(p.cache, p.n_pages, slot, pos0, p.status);
        const uint8_t *src = (j == 0 ? p.k : p.v) + cache_offset(p.cache, page, head, p.n_kv_heads, pos0, HD);
        const float scale = p.scales[(((long long)page * p.n_kv_heads + head) * 2 + j) * KV8_PAGE_BLOCKS + block];
        uint32_t x[PIECES][N / 4];
#pragma unroll
        for (int i = 0; i < PIECES; i++) {
            if constexpr (N == 4) {
                x[i][0] = *(const uint32_t *)(src + N * (32 * i + lane));
            } else {
                const uint2 two = *(const uint2 *)(src + N * (32 * i + lane));
                x[i][0] = two.x, x[i][N / 4 - 1] = two.y;
            }
        }
#pragma unroll
        for (int i = 0; i < PIECES; i++) {
            float v[N];
#pragma unroll
            for (int e = 0; e < N / 4; e++) kv8_unpack<FORM>(x[i][e], v + 4 * e);
#pragma unroll
            for (int e = 0; e < N; e++) v[e] *= scale;
            store_piece(dst + N * (32 * i + lane), v);
        }
    } else {
        const __nv_bfloat16 *open = p.open + (((long long)slot * 2 + j) * p.n_kv_heads + head) * (KV8_BLOCK * HD);
#pragma unroll
        for (int i = 0; i < PIECES; i++) {
            const int at = N * (32 * i + lane);
            float v[N];
#pragma unroll
            for (int e = 0; e < N; e++) v[e] = pos0 + at / HD < after ? __bfloat162float(open[at + e]) : 0.0f;  // behind the last token: zeros
            store_piece(dst + at, v);
        }
    }
}

extern "C" int abk_kv8_cache_bytes() { return (int)sizeof(Kv8Cache); }
static Kv8Write kv8_write_args(const void *qkv, long long row, int n_heads, const int *seq_slot, const Kv8Cache &c) {
    Kv8Write p = {};
    p.qkv = (const __nv_bfloat16 *)qkv, p.row = row, p.n_heads = n_heads, p.n_kv_heads = c.n_kv_heads, p.seq_slot = seq_slot;
    p.cache.page_table = c.page_table, p.cache.table_width = c.table_width, p.cache.ring_pages = c.ring_pages;
    p.cache.tokens_per_page = KV8_PAGE, p.k = (uint8_t *)c.k, p.v = (uint8_t *)c.v, p.scales = c.scales, p.open = (__nv_bfloat16 *)c.open;
    p.n_pages = c.n_pages, p.n_slots = c.n_slots, p.status = c.status;
    return p;
}
// Rows of one token each. q_norm, k_norm, cos and sin may be null (no norm, no rotation).
extern "C" int abk_kv8_prepare_write(void *qkv, long long row, int n_rows, int n_heads, const int *token_seq, const int *token_pos,
                                     const int *seq_slot, const float *q_norm, const float *k_norm, float eps, const float *cos,
                                     const float *sin, const Kv8Cache *cache, void *stream) {
    const Kv8Cache &c = *cache;
    if (n_rows <= 0) return 0;
    if (c.head_dim != 64 && c.head_dim != 128) ABK_REFUSE("kv8_write: head_dim %d is not 64 or 128", c.head_dim);
    if (c.form != KV8_INT8 && c.form != KV8_E4M3) ABK_REFUSE("kv8_write: no 8-bit form %d", c.form);
    if ((((uintptr_t)qkv | (uintptr_t)c.k | (uintptr_t)c.v | (uintptr_t)c.open | (uintptr_t)q_norm | (uintptr_t)k_norm | (uintptr_t)cos |
          (uintptr_t)sin) & 15) || (row & 7) || ((uintptr_t)c.scales & 3) || !cos != !sin)
        ABK_REFUSE("kv8_write: rows, norms, angles, pools and open blocks must be 16-byte aligned");
    const int warps = (n_heads + 256 / c.head_dim - 1) / (256 / c.head_dim) + 2 * c.n_kv_heads, groups = (warps + KV8_WARPS - 1) / KV8_WARPS;
    if (c.n_kv_heads < 1 || n_heads < 1 || groups > 65535) ABK_REFUSE("kv8_write: %d heads, %d kv heads", n_heads, c.n_kv_heads);
    const Kv8Write p = kv8_write_args(qkv, row, n_heads, seq_slot, c);
    const Kv8Prepare e = {(__nv_bfloat16 *)qkv, token_seq, token_pos, q_norm, k_norm, cos, sin, eps};
    auto go = [&](auto kernel) { abk_launch(kernel, dim3(n_rows, groups), dim3(32 * KV8_WARPS), 0, (cudaStream_t)stream, p, e); };
    if (c.head_dim == 64) c.form == KV8_INT8 ? go(kv8_prepare_write_kernel<64, KV8_INT8>) : go(kv8_prepare_write_kernel<64, KV8_E4M3>);
    else c.form == KV8_INT8 ? go(kv8_prepare_write_kernel<128, KV8_INT8>) : go(kv8_prepare_write_kernel<128, KV8_E4M3>);
    return ABK_LAUNCH_RESULT();
}
extern "C" int abk_kv8_write(const void *qkv, long long row, int n_rows, int n_heads, int n_seqs, int one_each, const int *seq_start,
                             const int *seq_pos0, const int *seq_len_after, const int *seq_slot, const Kv8Cache *cache, void *stream) {
    const Kv8Cache &c = *cache;
    if (n_rows <= 0 || n_seqs <= 0) return 0;
    if (c.head_dim != 64 && c.head_dim != 128) ABK_REFUSE("kv8_write: head_dim %d is not 64 or 128", c.head_dim);
    if (c.form != KV8_INT8 && c.form != KV8_E4M3) ABK_REFUSE("kv8_write: no 8-bit form %d", c.form);
    if ((((uintptr_t)qkv | (uintptr_t)c.k | (uintptr_t)c.v | (uintptr_t)c.open) & 15) || (row & 7) || ((uintptr_t)c.scales & 3))
        ABK_REFUSE("kv8_write: rows, pools and open blocks must be 16-byte aligned");
    const int units = one_each ? n_seqs : n_rows / KV8_BLOCK + 2 * n_seqs + 1;
    const int groups = (2 * c.n_kv_heads + KV8_WARPS - 1) / KV8_WARPS;
    if (c.n_kv_heads < 1 || groups > 65535) ABK_REFUSE("kv8_write: %d kv heads", c.n_kv_heads);
    Kv8Write p = kv8_write_args(qkv, row, n_heads, seq_slot, c);
    p.n_seqs = n_seqs, p.one_each = one_each, p.seq_start = seq_start, p.seq_pos0 = seq_pos0, p.seq_len_after = seq_len_after;
    const dim3 grid(units, groups), block(32 * KV8_WARPS);
    auto go = [&](auto kernel) { abk_launch(kernel, grid, block, 0, (cudaStream_t)stream, p); };
    if (c.head_dim == 64) c.form == KV8_INT8 ? go(kv8_write_kernel<64, KV8_INT8>) : go(kv8_write_kernel<64, KV8_E4M3>);
    else c.form == KV8_INT8 ? go(kv8_write_kernel<128, KV8_INT8>) : go(kv8_write_kernel<128, KV8_E4M3>);
    return ABK_LAUNCH_RESULT();
}

extern "C" int abk_kv8_read(const Kv8Cache *cache, int n_seqs, const int *seq_len_after, const int *seq_slot, const int *first_page,
                            int n_pages, void *out_k, void *out_v, int out_dtype, void *stream) {
    const Kv8Cache &c = *cache;
    if (n_pages <= 0 || n_seqs <= 0) return 0;
    if (c.head_dim != 64 && c.head_dim != 128) ABK_REFUSE("kv8_read: head_dim %d is not 64 or 128", c.head_dim);
    if (c.form != KV8_INT8 && c.form != KV8_E4M3) ABK_REFUSE("kv8_read: no 8-bit form %d", c.form);
    if (((uintptr_t)c.k | (uintptr_t)c.v | (uintptr_t)c.open | (uintptr_t)out_k | (uintptr_t)out_v) & 15)
        ABK_REFUSE("kv8_read: pools, open blocks and copies must be 16-byte aligned");
    if (c.n_kv_heads < 1 || c.n_kv_heads > 65535) ABK_REFUSE("kv8_read: %d kv heads", c.n_kv_heads);
    Kv8Read p;
    p.first_page = first_page, p.seq_len_after = seq_len_after, p.seq_slot = seq_slot, p.n_seqs = n_seqs, p.n_kv_heads = c.n_kv_heads;
    p.cache.page_table = c.page_table, p.cache.table_width = c.table_width, p.cache.ring_pages = 0, p.cache.tokens_per_page = KV8_PAGE;
    p.k = (const uint8_t *)c.k, p.v = (const uint8_t *)c.v, p.scales = c.scales, p.open = (const __nv_bfloat16 *)c.open;
    p.out_k = out_k, p.out_v = out_v, p.n_pages = c.n_pages, p.n_slots = c.n_slots, p.status = c.status;
    const dim3 grid(n_pages, c.n_kv_heads), block(256);
    auto go = [&](auto kernel) { abk_launch(kernel, grid, block, 0, (cudaStream_t)stream, p); };
    auto by_form = [&](auto hd) {
        constexpr int HD = decltype(hd)::value;
        if (out_dtype == ABK_F32) c.form == KV8_INT8 ? go(kv8_read_kernel<HD, KV8_INT8, float>) : go(kv8_read_kernel<HD, KV8_E4M3, float>);
        else c.form == KV8_INT8 ? go(kv8_read_kernel<HD, KV8_INT8, __nv_bfloat16>) : go(kv8_read_kernel<HD, KV8_E4M3, __nv_bfloat16>);
    };
    if (c.head_dim == 64) by_form(std::integral_constant<int, 64>());
    else by_form(std::integral_constant<int, 128>());
    return ABK_LAUNCH_RESULT();
}
