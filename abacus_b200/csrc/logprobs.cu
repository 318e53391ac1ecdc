// How likely given tokens are under rows of logits: with m = max x and l = sum e^(x - m), the log probability of token t is
// x_t - m - log l, the entropy log l - sum e^(x - m) (x - m) / l; and the most likely tokens with their log probabilities, the
// larger logit first, the lower index first among equals (the order of src/main.c:43-48).
//
// A logit of -inf is a token that cannot come: it adds nothing, and its log probability is -inf. A row with a NaN or +inf, or
// with nothing but -inf, is no distribution: its numbers are NaN and its tokens -1. A token outside the vocabulary has the log
// probability NaN.
//
// A row is read once, by a CTA or, where there are few rows, by a cluster of up to 8 CTAs, a slice each. Every thread keeps a
// running maximum and the two sums over its elements, 16 at a time; nothing in the walk waits for another warp. The most
// likely tokens: every warp keeps its best 32 (or 64) so far sorted across its lanes. An element is looked at only where it reaches a
// bound that at least k elements of the slice reach, the smallest of the warps' ceil(k / 8)-th best, which the warps leave in
// shared memory as they go (a bound that is out of date is only lower). A warp meets its elements by rising index, so among
// equals the one it has comes before the one it meets. Sorted lists are merged by counting: an element's place is its place in
// its own list and, by halving, the elements of the other lists before it; the warps' first, then the cluster's.
#define ABK_DEFINE_ERROR
#include "common.cuh"
#include "tc_common.cuh"

#define LOGPROBS_MAX_TOP 64
#define LOGPROBS_WARPS 8
#define LOGPROBS_THREADS (32 * LOGPROBS_WARPS)
#define LOGPROBS_MAX_SPLITS 8
#define LOGPROBS_FAR (-1e30f)  // a distance below the maximum at which nothing is left, and a finite one

struct LogProbs {
    const void *logits;
    long long stride;
    int vocab, top, slice;  // elements of a CTA's slice (whole pieces of 16 bytes)
    const int *tokens;
    float *logprob, *entropy;
    int *top_ids;
    float *top_logprobs;
};
struct __align__(8) Ranked {
    float v;
    int i;
};
__device__ __forceinline__ bool ranks_before(Ranked a, Ranked b) { return a.v > b.v || (a.v == b.v && a.i < b.i); }
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
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
// The next float32 number above x (which is not NaN).
__device__ __forceinline__ float next_up(float x) {
    if (x == 0.0f) return __int_as_float(1);
    return __int_as_float(__float_as_int(x) + (x > 0.0f ? 1 : -1));
}

// Elements of a 16-byte piece.
template <typename T> struct Piece;
template <> struct Piece<float> {
    static constexpr int N = 4;
    __device__ __forceinline__ static void floats(uint4 w, float *v) {
        v[0] = __uint_as_float(w.x), v[1] = __uint_as_float(w.y), v[2] = __uint_as_float(w.z), v[3] = __uint_as_float(w.w);
    }
    __device__ __forceinline__ static uint4 nothing() { return make_uint4(0xff800000u, 0xff800000u, 0xff800000u, 0xff800000u); }
};
template <> struct Piece<__nv_bfloat16> {
    static constexpr int N = 8;
    __device__ __forceinline__ static void floats(uint4 w, float *v) {
        const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int e = 0; e < 4; e++) v[2 * e] = __uint_as_float(u[e] << 16), v[2 * e + 1] = __uint_as_float(u[e] & 0xffff0000u);
    }
    __device__ __forceinline__ static uint4 nothing() { return make_uint4(0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u); }
};

// A warp's best so far, the best first: element 32 r + lane in v[r], i[r]; NaN where there is none yet.
template <int R> struct Best {
    float v[R > 0 ? R : 1];
    int i[R > 0 ? R : 1];
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int r = 0; r < R; r++) v[r] = __int_as_float(0x7fffffff), i[r] = 0x7fffffff;
    }
    __device__ __forceinline__ float at(int n) const {
        float x = __shfl_sync(0xffffffffu, v[0], n & 31);
        if (R > 1) {
            const float y = __shfl_sync(0xffffffffu, v[R - 1], n & 31);
            x = n < 32 ? x : y;
        }
        return x;
    }
    // x at index xi, which is larger than that of every equal element that is here
    __device__ __forceinline__ void insert(float x, int xi, int lane) {
        int pos = 0;
#pragma unroll
        for (int r = 0; r < R; r++) pos += __popc(__ballot_sync(0xffffffffu, v[r] >= x));
#pragma unroll
        for (int r = R - 1; r >= 0; r--) {
            float up = __shfl_up_sync(0xffffffffu, v[r], 1);
            int up_i = __shfl_up_sync(0xffffffffu, i[r], 1);
            if (r > 0) {
                const float over = __shfl_sync(0xffffffffu, v[0], 31);
                const int over_i = __shfl_sync(0xffffffffu, i[0], 31);
                if (lane == 0) up = over, up_i = over_i;
            }
            const int n = 32 * r + lane;
            if (n > pos) v[r] = up, i[r] = up_i;
            else if (n == pos) v[r] = x, i[r] = xi;
        }
    }
};

// Merges sorted lists in shared memory: list c at lists + c * LOGPROBS_MAX_TOP has counts(c) elements; f(rank, element) for the first k.
template <typename Counts, typename F>
__device__ __forceinline__ void merge_lists(const Ranked *lists, int n_lists, int k, Counts counts, F f) {
    for (int j = threadIdx.x; j < n_lists * k; j += LOGPROBS_THREADS) {
        const int mine = j / k, at = j - mine * k;
        if (at >= counts(mine)) continue;
        const Ranked c = lists[mine * LOGPROBS_MAX_TOP + at];
        int rank = at;
        for (int o = 0; o < n_lists && rank < k; o++) {
            if (o == mine) continue;
            int lo = 0, hi = counts(o);
            while (lo < hi) {
                const int mid = (lo + hi) / 2;
                if (ranks_before(lists[o * LOGPROBS_MAX_TOP + mid], c)) lo = mid + 1;
                else hi = mid;
            }
            rank += lo;
        }
        if (rank < k) f(rank, c);
    }
}

template <typename T, int R>
__global__ void __launch_bounds__(LOGPROBS_THREADS) logprobs_kernel(LogProbs p) {
    constexpr int N = Piece<T>::N, U = 16 / N;  // elements of a piece, pieces a thread takes at a time
    __shared__ Ranked lists[(R ? LOGPROBS_WARPS : 1) * LOGPROBS_MAX_TOP], best[R ? LOGPROBS_MAX_TOP : 1];
    __shared__ volatile float bounds[LOGPROBS_WARPS];
    __shared__ RowSums warp_sums[LOGPROBS_WARPS], cta_sums;
    __shared__ int have[LOGPROBS_WARPS], cta_have;
    const int split = (int)tc::cluster_rank(), splits = (int)tc::cluster_size(), lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int row = blockIdx.y;
    if (threadIdx.x < LOGPROBS_WARPS) bounds[threadIdx.x] = -INFINITY;
    pdl_wait();
    __syncthreads();
    const T *x = (const T *)p.logits + row * p.stride;
    // slices start on a 16-byte boundary of memory; slice 0 also takes the elements before the first one
    const int ahead = min((int)(((16 - ((uintptr_t)x & 15)) & 15) / sizeof(T)), p.vocab);
    const int lo = split == 0 ? 0 : min(p.vocab, ahead + split * p.slice), hi = split == splits - 1 ? p.vocab : min(p.vocab, ahead + (split + 1) * p.slice);
    const int body = max(lo, ahead), pieces = (hi - body) / N, tail = body + pieces * N;  // [lo, body) and [tail, hi): less than a piece each
    const uint4 *src = (const uint4 *)(x + body);
    float m = -3.402823466e38f, l = 0.0f, t = 0.0f;
    Best<R> top;
    top.clear();
    float cut = -INFINITY;  // what an element has to reach to be looked at
    const int jth = (p.top + LOGPROBS_WARPS - 1) / LOGPROBS_WARPS - 1;
    auto sum = [&](const float *v, int n, float most) {
        if (most > m) {
            const float d = fmaxf(m - most, LOGPROBS_FAR), e = ex2(d * 1.4426950408889634f);
            t = e * fmaf(l, d, t), l *= e, m = most;
        }
#pragma unroll
        for (int e = 0; e < n; e++) {
            const float d = v[e] - m, w = ex2(d * 1.4426950408889634f);
            l += w, t = fmaf(w, fmaxf(d, LOGPROBS_FAR), t);
        }
    };
    auto meet = [&](float v, int at) {  // (the whole warp with the same element)
        if (!(v >= cut)) return;
        top.insert(v, at, lane);
        const float last = top.at(p.top - 1), mine = top.at(jth);
        cut = fmaxf(cut, last == last ? next_up(last) : -INFINITY);
        if (lane == 0 && mine > bounds[warp]) bounds[warp] = mine;
    };
    auto loose = [&](int from, int to) {  // elements outside the pieces, a lane each
        const int at = from + lane;
        const float v = at < to ? to_float(x[at]) : -INFINITY;
        if (at < to) sum(&v, 1, v);
        if (R)
            for (int i = 0; i < to - from; i++) meet(__shfl_sync(0xffffffffu, v, i), from + i);
    };
    auto load = [&](int j0, float *v) {
        uint4 w[U];
#pragma unroll
        for (int u = 0; u < U; u++) w[u] = j0 + 32 * u + lane < pieces ? __ldcs(src + j0 + 32 * u + lane) : Piece<T>::nothing();
#pragma unroll
        for (int u = 0; u < U; u++) Piece<T>::floats(w[u], v + u * N);
        float most = v[0];
#pragma unroll
        for (int e = 1; e < 16; e++) most = fmaxf(most, v[e]);
        return most;
    };
    float v[16], most = load(warp * U * 32, v);
    if (R) {  // the first bounds: ceil(k / 8) lanes of every warp have an element that reaches their warp's
        float rest = most, b = -INFINITY;
        for (int r = 0; r <= jth; r++) {
            b = warp_max(rest);
            const unsigned holders = __ballot_sync(0xffffffffu, rest == b);
            if (lane == __ffs(holders) - 1) rest = -INFINITY;  // one of them is taken out
        }
        if (lane == 0) bounds[warp] = b;
        __syncthreads();
    }
    if (warp == 0) loose(lo, body);
    for (int j0 = warp * U * 32; j0 < pieces; j0 += LOGPROBS_THREADS * U) {
        if (R) {
            float b = bounds[lane & (LOGPROBS_WARPS - 1)];
#pragma unroll
            for (int o = LOGPROBS_WARPS / 2; o > 0; o >>= 1) b = fminf(b, __shfl_xor_sync(0xffffffffu, b, o));
            cut = fmaxf(cut, b);
            if (__any_sync(0xffffffffu, most >= cut)) {
#pragma unroll
                for (int u = 0; u < U; u++) {
                    const int at = j0 + 32 * u + lane;
                    float of_piece = v[u * N];
#pragma unroll
                    for (int e = 1; e < N; e++) of_piece = fmaxf(of_piece, v[u * N + e]);
                    for (unsigned hits = __ballot_sync(0xffffffffu, of_piece >= cut && at < pieces); hits; hits &= hits - 1) {
                        const int from = __ffs(hits) - 1;
#pragma unroll
                        for (int e = 0; e < N; e++) meet(__shfl_sync(0xffffffffu, v[u * N + e], from), body + (j0 + 32 * u + from) * N + e);
                    }
                }
            }
        }
        sum(v, 16, most);
        most = load(j0 + LOGPROBS_THREADS * U, v);
    }
    if (warp == LOGPROBS_WARPS - 1) loose(tail, hi);
    RowSums mine = {m, l, t, 0.0f};
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        RowSums other;
        other.m = __shfl_xor_sync(0xffffffffu, mine.m, o), other.l = __shfl_xor_sync(0xffffffffu, mine.l, o), other.t = __shfl_xor_sync(0xffffffffu, mine.t, o);
        mine = joined(mine, other);
    }
    if (lane == 0) warp_sums[warp] = mine;
    if (R) {
        int n = 0;
#pragma unroll
        for (int r = 0; r < R; r++) {
            lists[warp * LOGPROBS_MAX_TOP + 32 * r + lane] = {top.v[r], top.i[r]};
            n += __popc(__ballot_sync(0xffffffffu, top.v[r] == top.v[r]));
        }
        if (lane == 0) have[warp] = min(n, p.top);
    }
    __syncthreads();
    if (R) {
        merge_lists(lists, LOGPROBS_WARPS, p.top, [&](int c) { return have[c]; }, [&](int rank, Ranked c) { best[rank] = c; });
        if (threadIdx.x == 0) {
            int n = 0;
            for (int w = 0; w < LOGPROBS_WARPS; w++) n += have[w];
            cta_have = min(n, p.top);
        }
    }
    if (warp == 0) {
        RowSums s = warp_sums[0];
        for (int w = 1; w < LOGPROBS_WARPS; w++) s = joined(s, warp_sums[w]);
        if (lane == 0) cta_sums = s;
    }
    if (splits > 1) tc::cluster_sync();
    else __syncthreads();
    if (split == 0) {
        RowSums s = cta_sums;
        for (int c = 1; c < splits; c++) {
            const float4 o = tc::ld_cluster_f4(tc::peer_smem(tc::smem_addr(&cta_sums), c));
            s = joined(s, {o.x, o.y, o.z, 0.0f});
        }
        const float log_l = logf(s.l), nan = __int_as_float(0x7fffffff);
        const bool none = !(s.l > 0.0f);  // nothing can come, or a NaN, or +inf (which is one less itself)
        if (threadIdx.x == 0) {
            const int token = p.tokens[row];
            p.logprob[row] = none || token < 0 || token >= p.vocab ? nan : to_float(x[token]) - s.m - log_l;
            if (p.entropy) p.entropy[row] = none ? nan : log_l - s.t / s.l;
        }
        if (R) {
            const long long at = (long long)row * p.top;
            auto put = [&](int rank, Ranked c) {
                p.top_ids[at + rank] = none ? -1 : c.i, p.top_logprobs[at + rank] = none ? nan : c.v - s.m - log_l;
            };
            if (none) {
                for (int j = threadIdx.x; j < p.top; j += LOGPROBS_THREADS) put(j, {0.0f, 0});
            } else if (splits == 1) {
                if (threadIdx.x < p.top) put(threadIdx.x, best[threadIdx.x]);
            } else {
                __shared__ int of_cta[LOGPROBS_MAX_SPLITS];
                for (int j = threadIdx.x; j < splits * p.top; j += LOGPROBS_THREADS) {
                    const int c = j / p.top, i = j - c * p.top;
                    const float2 b = tc::ld_cluster_f2(tc::peer_smem(tc::smem_addr(best + i), c));
                    lists[c * LOGPROBS_MAX_TOP + i] = {b.x, __float_as_int(b.y)};
                }
                if (threadIdx.x < splits) of_cta[threadIdx.x] = __float_as_int(tc::ld_cluster_f1(tc::peer_smem(tc::smem_addr(&cta_have), threadIdx.x)));
                __syncthreads();
                merge_lists(lists, splits, p.top, [&](int c) { return of_cta[c]; }, put);
            }
        }
    }
    if (splits > 1) tc::cluster_sync();  // nobody leaves while its numbers may still be read
}

extern "C" int abk_token_logprobs(const void *logits, int dtype, long long stride, int n_rows, int vocab, const int *tokens,
                                  float *logprob, float *entropy, int top, int *top_ids, float *top_logprobs, void *stream) {
    if (n_rows <= 0) return 0;
    if (vocab < 1) ABK_REFUSE("token_logprobs: vocabulary of %d", vocab);
    if (top < 0 || top > LOGPROBS_MAX_TOP || top > vocab)
        ABK_REFUSE("token_logprobs: %d most likely tokens of a vocabulary of %d (at most %d)", top, vocab, LOGPROBS_MAX_TOP);
    const int size = dtype == ABK_F32 ? 4 : 2, piece = 16 / size;
    if ((uintptr_t)logits % size) ABK_REFUSE("token_logprobs: logits that are not aligned to their own size");
    // CTAs to a row: until the GPU is full (8 to an SM), in slices of at least 4,096 elements, as many as a cluster holds
    const int full = 8 * abk_sm_count();
    int splits = 1;
    while (splits < LOGPROBS_MAX_SPLITS && (long long)n_rows * splits * 2 <= full && vocab / (splits * 2) >= 4096) splits *= 2;
    LogProbs p;
    p.logits = logits, p.stride = stride, p.vocab = vocab, p.top = top, p.tokens = tokens, p.logprob = logprob, p.entropy = entropy;
    p.top_ids = top_ids, p.top_logprobs = top_logprobs;
    p.slice = (vocab + splits * piece - 1) / (splits * piece) * piece;
    void (*kernel)(LogProbs) = nullptr;
    if (dtype == ABK_F32) kernel = top == 0 ? logprobs_kernel<float, 0> : top <= 32 ? logprobs_kernel<float, 1> : logprobs_kernel<float, 2>;
    else kernel = top == 0 ? logprobs_kernel<__nv_bfloat16, 0> : top <= 32 ? logprobs_kernel<__nv_bfloat16, 1> : logprobs_kernel<__nv_bfloat16, 2>;
    for (int first = 0; first < n_rows; first += 32768) {  // (rows of a grid)
        LogProbs q = p;
        const int rows = n_rows - first < 32768 ? n_rows - first : 32768;
        q.logits = (const char *)logits + first * stride * size, q.tokens = tokens + first, q.logprob = logprob + first;
        q.entropy = entropy ? entropy + first : nullptr;
        q.top_ids = top ? top_ids + (long long)first * top : nullptr, q.top_logprobs = top ? top_logprobs + (long long)first * top : nullptr;
        abk_launch_clusters(kernel, dim3(splits, rows), dim3(LOGPROBS_THREADS), 0, (cudaStream_t)stream, splits, q);
        const int rc = ABK_LAUNCH_RESULT();
        if (rc) return rc;
    }
    return 0;
}
