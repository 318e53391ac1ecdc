// How likely given tokens are under rows of logits: with m = max x and l = sum e^(x - m), the log probability of token t is
// x_t - m - log l, the entropy log l - sum e^(x - m) (x - m) / l; and the most likely tokens with their log probabilities, the
// larger logit first, the lower index first among equals (the order of src/main.c:43-48).
//
// A logit of -inf is a token that cannot come: it adds nothing, and its log probability is -inf. A row with a NaN or +inf, or
// with nothing but -inf, is no distribution: its numbers are NaN and its tokens -1. A token outside the vocabulary has the log
// probability NaN.
//
// A row is read once: a cluster of up to 8 CTAs takes it, a slice each, which stays in the CTA's shared memory as it came
// (what does not fit there is read a second time). Every CTA finds its slice's maximum, then in one walk over shared memory the
// two sums and the candidates for the most likely tokens, and the cluster folds the CTAs' numbers through distributed shared memory.
// l is kept without its maxima's ones, l = n + l', n the number of maxima: log l = log(n + l') is log1p(l' + n - 1) to all its
// digits where one token has nearly all of the weight.
//
// The most likely k of a slice: at least k elements reach the smallest of the warps' ceil(k / warps)-th largest thread maxima, so
// what reaches it is collected (some tens of elements) and each is ranked by counting those before it. Where more reach it
// than there is room for (ties; a slice that is nearly all -inf), the k-th largest is found digit by digit of the ordered bits, and of
// its equals the first are taken. CTA 0 ranks the slices' k the same way.
#define ABK_DEFINE_ERROR
#include "common.cuh"
#include "tc_common.cuh"

#define LOGPROBS_MAX_TOP 64
#define LOGPROBS_THREADS 512
#define LOGPROBS_WARPS (LOGPROBS_THREADS / 32)
#define LOGPROBS_CANDIDATES 512
#define LOGPROBS_MAX_SPLITS 8
#define LOGPROBS_KEPT_BYTES (96 * 1024)  // of a slice in shared memory, so that an SM holds two CTAs

struct LogProbs {
    const void *logits;
    long long stride;
    int vocab, top, slice, kept;  // elements of a CTA's slice (a multiple of 16 bytes), and how many of them are kept
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
// The bits of x in the order of the numbers (-0 as 0; no NaN).
__device__ __forceinline__ uint32_t ordered(float x) {
    const uint32_t b = __float_as_uint(x + 0.0f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
struct __align__(16) SliceSums {
    float m, l, t;  // maximum; sum of e^(x - m) without the maxima; sum of e^(x - m) (x - m)
    int ties;       // how many maxima
};

// Elements of a 16-byte piece.
template <typename T> struct Piece;
template <> struct Piece<float> {
    static constexpr int N = 4;
    __device__ static void floats(uint4 w, float *v) {
        v[0] = __uint_as_float(w.x), v[1] = __uint_as_float(w.y), v[2] = __uint_as_float(w.z), v[3] = __uint_as_float(w.w);
    }
};
template <> struct Piece<__nv_bfloat16> {
    static constexpr int N = 8;
    __device__ static void floats(uint4 w, float *v) {
        const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int e = 0; e < 4; e++) v[2 * e] = __uint_as_float(u[e] << 16), v[2 * e + 1] = __uint_as_float(u[e] & 0xffff0000u);
    }
};

// The k best of cand[0..n), n <= LOGPROBS_CANDIDATES, in order, into best[0..k): each is counted past by all that come before it.
__device__ __forceinline__ void rank_candidates(const Ranked *cand, int n, int k, Ranked *best) {
    for (int j = threadIdx.x; j < n; j += LOGPROBS_THREADS) {
        const Ranked c = cand[j];
        int rank = 0;
        for (int i = 0; i < n; i++) rank += ranks_before(cand[i], c);
        if (rank < k) best[rank] = c;
    }
}

template <typename T>
__global__ void __launch_bounds__(LOGPROBS_THREADS) logprobs_kernel(LogProbs p) {
    constexpr int N = Piece<T>::N;
    extern __shared__ __align__(16) uint8_t kept_raw[];
    T *kept = (T *)kept_raw;
    __shared__ float scratch[33], bound_s[LOGPROBS_WARPS];
    __shared__ Ranked cand[LOGPROBS_CANDIDATES], best[LOGPROBS_MAX_TOP];
    __shared__ SliceSums sums;
    __shared__ int count, digits[256], wanted, prefix;
    const int split = (int)tc::cluster_rank(), splits = (int)tc::cluster_size(), lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int row = blockIdx.y;
    pdl_wait();
    const T *x = (const T *)p.logits + row * p.stride;
    // slices start on a 16-byte boundary of memory: slice 0 also takes the elements before the first one
    const int skew = (int)(((16 - ((uintptr_t)x & 15)) & 15) / sizeof(T)), ahead = min(skew, p.vocab);
    const int lo = split == 0 ? 0 : min(p.vocab, ahead + split * p.slice), hi = split == splits - 1 ? p.vocab : min(p.vocab, ahead + (split + 1) * p.slice);
    const int pieces = (hi - max(lo, ahead)) / N, body = max(lo, ahead), tail = body + pieces * N;  // [lo, body) and [tail, hi) are less than a piece
    const uint4 *src = (const uint4 *)(x + body);
    const int kept_pieces = min(pieces, p.kept / N);
    float most = -INFINITY;
    bool odd = false;  // a NaN or +inf
    // every element once: into shared memory, the maximum on the way
    {
        constexpr int U = 4;
        for (int j = threadIdx.x; j < pieces; j += U * LOGPROBS_THREADS) {
            uint4 w[U];
#pragma unroll
            for (int i = 0; i < U; i++)
                if (j + i * LOGPROBS_THREADS < pieces) w[i] = __ldg(src + j + i * LOGPROBS_THREADS);
#pragma unroll
            for (int i = 0; i < U; i++) {
                const int at = j + i * LOGPROBS_THREADS;
                if (at < pieces) {
                    if (at < kept_pieces) ((uint4 *)kept)[at] = w[i];
                    float v[N];
                    Piece<T>::floats(w[i], v);
#pragma unroll
                    for (int e = 0; e < N; e++) most = fmaxf(most, v[e]), odd |= !(v[e] < INFINITY);
                }
            }
        }
    }
    const int loose = (body - lo) + (hi - tail);  // elements outside the pieces: at most 14
    float mine_loose = -INFINITY;
    int loose_at = 0;
    if (threadIdx.x < loose) {
        loose_at = threadIdx.x < body - lo ? lo + threadIdx.x : tail + threadIdx.x - (body - lo);
        mine_loose = to_float(x[loose_at]);
        most = fmaxf(most, mine_loose), odd |= !(mine_loose < INFINITY);
    }
    // f(value, index) for every element of the slice, the thread's own as above
    auto each = [&](auto f) {
        for (int j = threadIdx.x; j < pieces; j += LOGPROBS_THREADS) {
            const uint4 w = j < kept_pieces ? ((const uint4 *)kept)[j] : __ldg(src + j);
            float v[N];
            Piece<T>::floats(w, v);
#pragma unroll
            for (int e = 0; e < N; e++) f(v[e], body + j * N + e);
        }
        if (threadIdx.x < loose) f(mine_loose, loose_at);
    };
    if (threadIdx.x == 0) count = 0;
    const int k = min(p.top, hi - lo);  // of this slice
    if (k > 0) {  // this warp's ceil(k / warps)-th largest thread maximum
        float v = most, m = -INFINITY;
        for (int r = 0; r < (k + LOGPROBS_WARPS - 1) / LOGPROBS_WARPS; r++) {
            m = warp_max(v);
            const unsigned holders = __ballot_sync(0xffffffffu, v == m);
            if (lane == __ffs(holders) - 1) v = -INFINITY;  // one of them is taken out
        }
        if (lane == 0) bound_s[warp] = m;
    }
    const float m = block_max(most, scratch);
    odd = __syncthreads_or(odd);
    float bound = INFINITY;
    if (k > 0)
        for (int w = 0; w < LOGPROBS_WARPS; w++) bound = fminf(bound, bound_s[w]);
    float l = 0.0f, t = 0.0f;
    int ties = 0;
    const float m2 = m == -INFINITY ? 0.0f : m;
    each([&](float v, int at) {
        const float d = v - m2, e = ex2(d * 1.4426950408889634f);
        ties += v == m, l += v == m ? 0.0f : e, t = fmaf(e, fmaxf(d, -1e30f), t);
        if (v >= bound) {
            const int c = atomicAdd(&count, 1);
            if (c < LOGPROBS_CANDIDATES) cand[c] = {v, at};
        }
    });
    l = block_sum(l, scratch), t = block_sum(t, scratch);
    const float n_ties = block_sum((float)ties, scratch);
    if (threadIdx.x == 0) sums = {odd ? NAN : m, l, t, (int)n_ties};
    if (k > 0) {
        if (count > LOGPROBS_CANDIDATES) {  // (the same for the whole CTA) the k-th largest, eight bits of the ordered numbers at a time
            if (threadIdx.x == 0) wanted = k, prefix = 0;
            for (int shift = 24; shift >= 0; shift -= 8) {
                for (int i = threadIdx.x; i < 256; i += LOGPROBS_THREADS) digits[i] = 0;
                __syncthreads();
                const uint32_t above = shift == 24 ? 0 : 0xffffffffu << (shift + 8), have = (uint32_t)prefix;
                each([&](float v, int) {
                    const uint32_t b = ordered(v);
                    if ((b & above) == have) atomicAdd(&digits[b >> shift & 255], 1);
                });
                __syncthreads();
                if (threadIdx.x == 0) {
                    int left = wanted, d = 255;
                    while (d > 0 && digits[d] < left) left -= digits[d], d--;
                    wanted = left, prefix = (int)(have | (uint32_t)d << shift);
                }
                __syncthreads();
            }
            // all above it, and of its equals the `wanted` first ones
            const uint32_t kth = (uint32_t)prefix;
            if (threadIdx.x == 0) count = 0;
            __syncthreads();
            each([&](float v, int at) {
                if (ordered(v) > kth) cand[atomicAdd(&count, 1)] = {v, at};
            });
            __syncthreads();
            int found = 0;
            for (int j0 = lo; j0 < hi && found < wanted; j0 += LOGPROBS_THREADS) {
                const int j = j0 + threadIdx.x;
                const float v = j < hi ? to_float(x[j]) : 0.0f;
                const bool same = j < hi && ordered(v) == kth;
                const unsigned votes = __ballot_sync(0xffffffffu, same);
                if (lane == 0) digits[warp] = __popc(votes);
                __syncthreads();
                int before = found, all = 0;
                for (int w = 0; w < LOGPROBS_WARPS; w++) before += w < warp ? digits[w] : 0, all += digits[w];
                before += __popc(votes & ((1u << lane) - 1));
                if (same && before < wanted) cand[k - wanted + before] = {v, j};
                found += all;
                __syncthreads();
            }
            if (threadIdx.x == 0) count = k;
        }
        __syncthreads();
        rank_candidates(cand, min(count, LOGPROBS_CANDIDATES), k, best);
    }
    if (splits > 1) tc::cluster_sync();
    else __syncthreads();
    // the row's numbers, in every CTA that needs them
    auto of_cta = [&](const void *at, int c) { return tc::peer_smem(tc::smem_addr(at), c); };
    if (split == 0) {
        float mm = -INFINITY;
        bool none = false;
        for (int c = 0; c < splits; c++) {
            const float4 s = tc::ld_cluster_f4(of_cta(&sums, c));
            none |= !(s.x == s.x), mm = fmaxf(mm, s.x);
        }
        none |= mm == -INFINITY;
        float ll = 0.0f, tt = 0.0f;
        int n = 0;
        for (int c = 0; c < splits; c++) {
            const float4 s = tc::ld_cluster_f4(of_cta(&sums, c));
            const int n_c = __float_as_int(s.w);
            if (s.x == -INFINITY) continue;  // nothing in this slice can come
            if (s.x == mm) {
                ll += s.y, tt += s.z, n += n_c;
            } else {
                const float d = s.x - mm, e = exp2f(d * 1.4426950408889634f);
                ll = fmaf((float)n_c + s.y, e, ll), tt = fmaf(fmaf((float)n_c + s.y, d, s.z), e, tt);
            }
        }
        const float log_l = log1pf(ll + (float)(n - 1)), nan = __int_as_float(0x7fffffff);
        if (threadIdx.x == 0) {
            const int token = p.tokens[row];
            p.logprob[row] = none || token < 0 || token >= p.vocab ? nan : to_float(x[token]) - mm - log_l;
            if (p.entropy) p.entropy[row] = none ? nan : log_l - tt / (ll + (float)n);
        }
        if (p.top > 0) {
            // the slices' best, at most 8 x 64, into cand: they are at most LOGPROBS_CANDIDATES
            const int per = p.top;
            int n_cand = 0;
            __syncthreads();
            for (int c = 0; c < splits; c++) {
                const int c_lo = c == 0 ? 0 : min(p.vocab, ahead + c * p.slice), c_hi = c == splits - 1 ? p.vocab : min(p.vocab, ahead + (c + 1) * p.slice);
                const int have = min(per, c_hi - c_lo);
                for (int i = threadIdx.x; i < have; i += LOGPROBS_THREADS) {
                    const float2 b = tc::ld_cluster_f2(of_cta(best + i, c));
                    cand[n_cand + i] = {b.x, __float_as_int(b.y)};
                }
                n_cand += have;
            }
            __syncthreads();
            for (int j = threadIdx.x; j < n_cand; j += LOGPROBS_THREADS) {
                const Ranked c = cand[j];
                int rank = 0;
                for (int i = 0; i < n_cand; i++) rank += ranks_before(cand[i], c);
                if (rank < p.top && !none) {
                    p.top_ids[(long long)row * p.top + rank] = c.i;
                    p.top_logprobs[(long long)row * p.top + rank] = c.v - mm - log_l;
                }
            }
            if (none)
                for (int j = threadIdx.x; j < p.top; j += LOGPROBS_THREADS)
                    p.top_ids[(long long)row * p.top + j] = -1, p.top_logprobs[(long long)row * p.top + j] = nan;
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
    // slices of at least 4,096 elements, as many as a cluster holds
    int splits = (vocab + 4095) / 4096;
    if (splits > LOGPROBS_MAX_SPLITS) splits = LOGPROBS_MAX_SPLITS;
    LogProbs p;
    p.logits = logits, p.stride = stride, p.vocab = vocab, p.top = top, p.tokens = tokens, p.logprob = logprob, p.entropy = entropy;
    p.top_ids = top_ids, p.top_logprobs = top_logprobs;
    p.slice = (vocab + splits * piece - 1) / (splits * piece) * piece;
    p.kept = p.slice + piece;  // (the last slice may have an element or two more than the others)
    if (p.kept > LOGPROBS_KEPT_BYTES / size) p.kept = LOGPROBS_KEPT_BYTES / size;
    const int smem = p.kept * size;
    void (*kernel)(LogProbs) = dtype == ABK_F32 ? logprobs_kernel<float> : logprobs_kernel<__nv_bfloat16>;
    const cudaError_t e = abk_allow_shared_memory((const void *)kernel, smem);
    if (e != cudaSuccess) return (int)e;
    for (int first = 0; first < n_rows; first += 32768) {  // (rows of a grid)
        LogProbs q = p;
        const int rows = n_rows - first < 32768 ? n_rows - first : 32768;
        q.logits = (const char *)logits + first * stride * size, q.tokens = tokens + first, q.logprob = logprob + first;
        q.entropy = entropy ? entropy + first : nullptr;
        q.top_ids = top ? top_ids + (long long)first * top : nullptr, q.top_logprobs = top ? top_logprobs + (long long)first * top : nullptr;
        abk_launch_clusters(kernel, dim3(splits, rows), dim3(LOGPROBS_THREADS), smem, (cudaStream_t)stream, splits, q);
        const int rc = ABK_LAUNCH_RESULT();
        if (rc) return rc;
    }
    return 0;
}
