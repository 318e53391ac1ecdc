// How likely given tokens are under rows of logits: with m = max x and l = sum e^(x - m), the log probability of token t is
// x_t - m - log l, the entropy log l - sum e^(x - m) (x - m) / l; and the most likely tokens with their log probabilities, the
// larger logit first, the lower index first among equals (the order of src/main.c:43-48).
//
// A logit of -inf is a token that cannot come: it adds nothing, and its log probability is -inf. A row with a NaN or +inf, or
// with nothing but -inf, is no distribution: its numbers are NaN and its tokens -1. A token outside the vocabulary has the log
// probability NaN.
//
// A row is read once, by a CTA or, where there are few rows, by a cluster of up to 16 CTAs, a slice each. Every thread keeps a
// running maximum and the two sums over its elements, four 16-byte pieces at a time, the next four on their way; nothing in the walk waits for
// another warp. The most likely tokens: an element is noted, in the warp's own list in shared memory, only where it reaches a bound
// that at least k elements of the slice reach: every warp leaves its ceil(k / 8)-th largest thread maximum in shared memory as it goes,
// and of these the one that enough warps reach is the bound (one that is out of date is only lower). Where fewer warps have elements (a short
// slice, a mask that leaves one range of tokens) each leaves more. A list that fills up is cut to its best k; a
// warp meets its elements by rising index, so from then on an equal of the k-th need not be noted. At the end the elements that
// reach the last bound, some tens, are ranked by counting those before each, and once more those of a cluster's CTAs. Elements of -inf are
// never noted: where a row has fewer than k others, the first of them fill its places.
//
// Measured: 512 rows of 151,936 float32 logits with 5 alternatives in 61 us, 5.1 TB/s (50 without); 8 rows with 20 in 12.5 to 13.9 (9.4 without), a
// chain of three turns of loads, bounds, ranks and the cluster's fold; 200 rows of 50,261 bfloat16 logits, a twentieth not -inf, with 64
// in 24: there every turn of 1,024 elements has some to note. Short slices and ranges, with 1, 20 and 64 alternatives: 32 rows of 65,536 bfloat16 logits
// 14, 18.5 and 26, 600 rows of 6,000 9, 12 and 16, 500 rows of 1,500 float32 ones 6, 8 and 13.5, 64 rows of 151,936 with 1,000 neighbours
// left 13, 16 and 20 (float32) and 18, 21 and 33 (bfloat16). Most of a row's elements as alternatives are ranked the long way: 600 rows of 500 with 64 98.
#define ABK_DEFINE_ERROR
#include "common.cuh"
#include "tc_common.cuh"
#include "logprobs.cuh"

#define LOGPROBS_MAX_TOP 64
#define LOGPROBS_WARPS 8
#define LOGPROBS_THREADS (32 * LOGPROBS_WARPS)
#define LOGPROBS_MAX_SPLITS 16
static_assert(LOGPROBS_MAX_SPLITS >= 2 * LOGPROBS_WARPS, "room for all lists");
// 16-byte pieces a thread takes at a time: 16 elements of float32, 32 of 16-bit types. With two of these for 16-bit types 200 rows of
// 50,261 with 64 alternatives take 27.7 us, not 24.2; four spill some registers (64 bytes of stores), three (12 bytes)
// take the same 24.2, and rows without many to note show no difference.
#define LOGPROBS_PIECES 4
#define LOGPROBS_LOWEST (-3.402823466e38f)
#define LOGPROBS_NOTED 128  // elements a warp's list has room for beside those of one piece of every lane

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
// The largest number of a warp's lanes.
__device__ __forceinline__ float largest_of_lanes(float v) {
    float r;
    asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
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

// The best k of the n elements noted at `list`, in order, in its first places (by way of `spare`, room for k); returns how many those
// are. By one warp.
__device__ __noinline__ int cut_to_best(Ranked *list, Ranked *spare, int n, int k, int lane) {
    for (int j = lane; j < n; j += 32) {
        const Ranked c = list[j];
        int rank = 0;
        for (int i = 0; i < n; i++) rank += ranks_before(list[i], c);
        if (rank < k) spare[rank] = c;
    }
    __syncwarp();
    n = min(n, k);
    for (int j = lane; j < n; j += 32) list[j] = spare[j];
    __syncwarp();
    return n;
}

// What the warps of a CTA know of the most likely elements, in shared memory. At level L k elements of the slice are looked for in
// LOGPROBS_WARPS >> L warps, ceil(k / that many) in each: level 0 where all warps have elements, the others where a slice is short
// or a mask leaves one range of tokens.
#define LOGPROBS_LEVELS 4
static_assert(LOGPROBS_WARPS >> (LOGPROBS_LEVELS - 1) == 1 && LOGPROBS_LEVELS * LOGPROBS_WARPS == 32, "a lane a level and warp");
struct Bounds {
    volatile float of_warp[LOGPROBS_LEVELS][LOGPROBS_WARPS];  // what that many of a warp's elements reach
    volatile float common;                                    // what k elements of the slice reach, as of some moment
};
// Elements a warp at a level: ceil(top / warps)
__device__ __forceinline__ int in_warp_at(int top, int level) {
    const int shift = LOGPROBS_LEVELS - 1 - level;
    return (top + (1 << shift) - 1) >> shift;
}
// A warp's bounds at the first levels: the in_warp_at()-th largest of its lanes' numbers (none where it has fewer lanes).
__device__ __forceinline__ void leave_bounds(Bounds *b, float of_lane, int top, int levels, int warp, int lane) {
    float x = -INFINITY;
    for (int level = 0, r = 0; level < levels; level++) {
        const int in_warp = in_warp_at(top, level);
        if (in_warp > 32) return;
        for (; r < in_warp; r++) {
            x = largest_of_lanes(of_lane);
            const unsigned holders = __ballot_sync(0xffffffffu, of_lane == x);
            if (lane == __ffs(holders) - 1) of_lane = -INFINITY;  // one of them is taken out
        }
        if (lane == 0) b->of_warp[level][warp] = x;
    }
}
// What k elements of the slice reach: at its level a lane's warp is the `need`-th that has in_warp_at() of them that reach it. The bounds
// of this moment or earlier ones, either will do.
__device__ __forceinline__ float common_bound(const Bounds *bounds, int need, int lane) {
    const float b = (&bounds->of_warp[0][0])[lane];
    int above = 0;  // (equals in the order of the warps)
#pragma unroll
    for (int w = 0; w < LOGPROBS_WARPS; w++) {
        const float o = __shfl_sync(0xffffffffu, b, w, LOGPROBS_WARPS);
        above += o > b || (o == b && w < (lane & (LOGPROBS_WARPS - 1)));
    }
    return largest_of_lanes(above == need - 1 ? b : -INFINITY);
}
// A warp's list: n elements, and what an element has to reach to be noted.
struct Noted {
    int n;
    float cut;
};
// An element of every lane.
__device__ __forceinline__ void note(Noted &noted, Ranked *list, float v, int at, bool real, int lane) {
    const bool hit = real && v >= noted.cut;
    const unsigned hits = __ballot_sync(0xffffffffu, hit);
    if (hits) {
        if (hit) list[noted.n + __popc(hits & ((1u << lane) - 1))] = {v, at};
        noted.n += __popc(hits);
    }
}
// Room for an element of every lane's next piece.
__device__ __forceinline__ void make_room(Noted &noted, Ranked *list, Ranked *spare, int top, int lane) {
    if (noted.n <= LOGPROBS_NOTED) return;
    __syncwarp();
    noted.n = cut_to_best(list, spare, noted.n, top, lane);
    if (noted.n == top) noted.cut = fmaxf(noted.cut, next_up(list[noted.n - 1].v));
}
// The elements of a warp's 32 * U pieces (32 of every LOGPROBS_THREADS, from j0 on) that reach the cut, read again behind their sums (the walk's own copies would have
// to stay in registers for this: 512 rows of 151,936 with the 5 most likely take 71 us so, not 66).
template <typename T> __device__ __forceinline__ Noted note_pieces(const uint4 *src, int j0, int pieces, int body, Noted noted, Ranked *list,
                                                                Ranked *spare, int top, int lane) {
    constexpr int N = Piece<T>::N, U = LOGPROBS_PIECES;
    uint4 w[U];
#pragma unroll
    for (int u = 0; u < U; u++) w[u] = j0 + LOGPROBS_THREADS * u + lane < pieces ? __ldg(src + j0 + LOGPROBS_THREADS * u + lane) : Piece<T>::nothing();
#pragma unroll
    for (int u = 0; u < U; u++) {
        float v[N];
        Piece<T>::floats(w[u], v);
        float of_piece = v[0];
#pragma unroll
        for (int e = 1; e < N; e++) of_piece = fmaxf(of_piece, v[e]);
        if (!__any_sync(0xffffffffu, of_piece >= noted.cut)) continue;
        make_room(noted, list, spare, top, lane);
#pragma unroll
        for (int e = 0; e < N; e++) note(noted, list, v[e], body + (j0 + LOGPROBS_THREADS * u + lane) * N + e, j0 + LOGPROBS_THREADS * u + lane < pieces, lane);
    }
    return noted;
}
// The bound moves with a thread's maximum that counts; returns it.
__device__ __forceinline__ float move_bound(Bounds *b, float of_lane, int top, int levels, int need, int warp, int lane) {
    leave_bounds(b, of_lane, top, levels, warp, lane);
    __syncwarp();
    const float x = common_bound(b, need, lane);
    if (lane == 0) b->common = x;
    return x;
}

template <typename T, bool TOP>
__global__ void __launch_bounds__(LOGPROBS_THREADS, sizeof(T) == 4 ? 4 : 3) logprobs_kernel(LogProbs p) {
    constexpr int N = Piece<T>::N, U = LOGPROBS_PIECES, ROOM = LOGPROBS_NOTED + 32 * N;  // elements of a piece, pieces a thread takes at a time
    __shared__ Ranked lists[TOP ? LOGPROBS_WARPS : 1][TOP ? ROOM : 1], best[TOP ? LOGPROBS_MAX_TOP : 1];
    __shared__ Ranked cand[TOP ? LOGPROBS_MAX_SPLITS * LOGPROBS_MAX_TOP : 1];  // in turn: room to sort a list, all lists, the cluster's
    __shared__ Bounds bounds;
    __shared__ RowSums warp_sums[LOGPROBS_WARPS], cta_sums;
    __shared__ int count, in_cta, in_row, have[LOGPROBS_MAX_SPLITS];
    const int split = (int)tc::cluster_rank(), splits = (int)tc::cluster_size(), lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int row = blockIdx.y;
    if (threadIdx.x == 0) count = 0, bounds.common = -INFINITY;
    if (TOP && lane < LOGPROBS_LEVELS) bounds.of_warp[lane][warp] = -INFINITY;
    pdl_wait();
    const T *x = (const T *)p.logits + row * p.stride;
    // slices start on a 16-byte boundary of memory; slice 0 also takes the elements before the first one
    const int ahead = min((int)(((16 - ((uintptr_t)x & 15)) & 15) / sizeof(T)), p.vocab);
    const int lo = split == 0 ? 0 : min(p.vocab, ahead + split * p.slice), hi = split == splits - 1 ? p.vocab : min(p.vocab, ahead + (split + 1) * p.slice);
    const int body = max(lo, ahead), pieces = (hi - body) / N, tail = body + pieces * N;  // [lo, body) and [tail, hi): less than a piece each
    const uint4 *src = (const uint4 *)(x + body);
    float given = __int_as_float(0x7fffffff);  // the given token's logit
    if (split == 0 && threadIdx.x == 0) {
        const int token = p.tokens[row];
        if (token >= 0 && token < p.vocab) given = to_float(x[token]);
    }
    float m = LOGPROBS_LOWEST;
    float2 l = make_float2(0.0f, 0.0f), t = l;  // of the elements at even places and at odd ones
    auto sum = [&](const float2 *v, int pairs, float most) {
        if (most > m) {
            const float d = fmaxf(m - most, LOGPROBS_FAR), e = ex2(d * 1.4426950408889634f);
            t = mul2(make_float2(e, e), fma2(l, make_float2(d, d), t)), l = mul2(make_float2(e, e), l), m = most;
        }
        const float2 down = make_float2(-m, -m), unit = make_float2(1.4426950408889634f, 1.4426950408889634f);
#pragma unroll
        for (int i = 0; i < pairs; i++) {
            const float2 d = add2(v[i], down), y = mul2(d, unit), w = make_float2(ex2(y.x), ex2(y.y));
            l = add2(l, w), t = fma2(w, make_float2(fmaxf(d.x, LOGPROBS_FAR), fmaxf(d.y, LOGPROBS_FAR)), t);
        }
    };
    Ranked *list = lists[TOP ? warp : 0], *spare = cand + (TOP ? warp * LOGPROBS_MAX_TOP : 0);
    Noted noted = {0, LOGPROBS_LOWEST};
    // levels that a bound of the first turn needs: as many warps as it has have a piece a lane
    const int filled = min(pieces, LOGPROBS_THREADS) / 32, levels = filled >= 8 ? 1 : filled >= 4 ? 2 : filled >= 2 ? 3 : 4;
    const int in_warp = TOP ? in_warp_at(p.top, lane >> 3) : 1, need = (p.top + in_warp - 1) / in_warp;  // of the lane's level
    auto loose = [&](int from, int to) {  // elements outside the pieces, a lane each
        const int at = from + lane;
        const float v = at < to ? to_float(x[at]) : -INFINITY;
        const float2 alone = make_float2(v, -INFINITY);
        if (at < to) sum(&alone, 1, v);
        if (TOP) make_room(noted, list, spare, p.top, lane), note(noted, list, v, at, at < to, lane);
    };
    // With most likely tokens a thread's pieces lie LOGPROBS_THREADS apart: all warps have some of a short slice, and of a range of tokens that a
    // mask leaves. Without, a warp's lie side by side.
    constexpr int APART = TOP ? LOGPROBS_THREADS : 32;
    auto load = [&](int j0, uint4 *w) {
        if (j0 + APART * (U - 1) + 32 <= pieces) {
#pragma unroll
            for (int u = 0; u < U; u++) w[u] = __ldcs(src + j0 + APART * u + lane);
        } else {
#pragma unroll
            for (int u = 0; u < U; u++) w[u] = j0 + APART * u + lane < pieces ? __ldcs(src + j0 + APART * u + lane) : Piece<T>::nothing();
        }
    };
    uint4 w[U];
    const int from = warp * (TOP ? 32 : U * 32);  // of a turn's pieces
    load(from, w);
    bool first = true;
    for (int j0 = from; first || j0 < pieces; j0 += LOGPROBS_THREADS * U) {
        __align__(8) float v[U * N];
#pragma unroll
        for (int u = 0; u < U; u++) Piece<T>::floats(w[u], v + u * N);
        load(j0 + LOGPROBS_THREADS * U, w);
        float most = v[0];
#pragma unroll
        for (int e = 1; e < U * N; e++) most = fmaxf(most, v[e]);
        if (TOP) {
            if (first) {  // the first bounds
                leave_bounds(&bounds, most, p.top, levels, warp, lane);
                __syncthreads();
                noted.cut = fmaxf(noted.cut, common_bound(&bounds, need, lane));
            } else {
                noted.cut = fmaxf(noted.cut, bounds.common);
            }
        }
        if (first && warp == 0) loose(lo, body);
        const bool risen = most > m;
        sum((const float2 *)v, U * N / 2, most);
        if (TOP && __any_sync(0xffffffffu, most >= noted.cut)) {
            const bool moves = __any_sync(0xffffffffu, most >= noted.cut && risen);  // (else no thread's maximum that counts does)
            const bool none = noted.cut == LOGPROBS_LOWEST;  // no bound yet: what few warps have may give one
            if (none || (!first && moves)) noted.cut = fmaxf(noted.cut, move_bound(&bounds, m, p.top, none ? LOGPROBS_LEVELS : levels, need, warp, lane));
            noted = note_pieces<T>(src, j0, pieces, body, noted, list, spare, p.top, lane);
        }
        first = false;
    }
    if (warp == LOGPROBS_WARPS - 1) loose(tail, hi);
    const RowSums mine = joined_lanes({m, l.x + l.y, t.x + t.y, 0.0f}, 16);
    if (lane == 0) warp_sums[warp] = mine;
    if (TOP) make_room(noted, list, spare, p.top, lane);
    __syncthreads();
    if (TOP) {
        const float b = common_bound(&bounds, need, lane);
        for (int i = lane; i < noted.n; i += 32)
            if (list[i].v >= b) cand[atomicAdd(&count, 1)] = list[i];
    }
    if (warp == 0) {
        const RowSums s = joined_lanes(warp_sums[lane & (LOGPROBS_WARPS - 1)], LOGPROBS_WARPS / 2);
        if (lane == 0) cta_sums = s;
    }
    __syncthreads();
    if (TOP) {
        const int all = count;
        if (threadIdx.x == 0) in_cta = all;
        for (int j = threadIdx.x; j < all; j += LOGPROBS_THREADS) {
            const Ranked c = cand[j];
            int rank = 0;
#pragma unroll 8
            for (int i = 0; i < all; i++) rank += ranks_before(cand[i], c);
            if (rank < p.top) best[rank] = c;
        }
    }
    if (splits > 1) tc::cluster_sync();
    else __syncthreads();
    if (split == 0) {
        RowSums s = cta_sums;
        if (splits > 1) {  // a CTA's a lane
            const float4 o = tc::ld_cluster_f4(tc::peer_smem(tc::smem_addr(&cta_sums), lane & (splits - 1)));
            s = joined_lanes({o.x, o.y, o.z, 0.0f}, splits / 2);
        }
        const float log_l = logf(s.l), nan = __int_as_float(0x7fffffff);
        const bool none = !(s.l > 0.0f);  // nothing can come, or a NaN, or +inf (which is one less itself)
        if (threadIdx.x == 0) {
            p.logprob[row] = none ? nan : given - s.m - log_l;
            if (p.entropy) p.entropy[row] = none ? nan : log_l - s.t / s.l;
        }
        if (TOP) {
            const long long at = (long long)row * p.top;
            auto put = [&](int rank, Ranked c) {
                p.top_ids[at + rank] = none ? -1 : c.i, p.top_logprobs[at + rank] = none ? nan : c.v - s.m - log_l;
            };
            int found = min(in_cta, p.top);
            if (none) {
                for (int j = threadIdx.x; j < p.top; j += LOGPROBS_THREADS) put(j, {0.0f, 0});
                found = p.top;
            } else if (splits == 1) {
                if (threadIdx.x < found) put(threadIdx.x, best[threadIdx.x]);
            } else {
                // of the CTAs' best those that reach what k of them reach: the largest of their k-th, the smallest of their ceil(k / CTAs)-th
                if (threadIdx.x == 0) count = 0;
                if (warp == 0) {
                    int n_c = 0;
                    const int few = (p.top + splits - 1) / splits;
                    float kth = -INFINITY, all_have = INFINITY;
                    if (lane < splits) {
                        n_c = min(__float_as_int(tc::ld_cluster_f1(tc::peer_smem(tc::smem_addr(&in_cta), lane))), p.top);
                        const float v = tc::ld_cluster_f1(tc::peer_smem(tc::smem_addr(&best[p.top - 1].v), lane));
                        const float w = tc::ld_cluster_f1(tc::peer_smem(tc::smem_addr(&best[few - 1].v), lane));
                        have[lane] = n_c, kth = n_c == p.top ? v : -INFINITY, all_have = n_c >= few ? w : -INFINITY;
                    }
                    found = __reduce_add_sync(0xffffffffu, n_c), kth = fmaxf(warp_max(kth), -warp_max(-all_have));
                    if (lane == 0) bounds.common = kth, in_row = found;
                }
                __syncthreads();
                const float kth = bounds.common;
                for (int j = threadIdx.x; j < splits * p.top; j += LOGPROBS_THREADS) {
                    const int c = j / p.top, i = j - c * p.top;
                    if (i >= have[c]) continue;
                    const float2 b = tc::ld_cluster_f2(tc::peer_smem(tc::smem_addr(best + i), c));
                    if (b.x >= kth) cand[atomicAdd(&count, 1)] = {b.x, __float_as_int(b.y)};
                }
                __syncthreads();
                const int all = count;
                for (int j = threadIdx.x; j < all; j += LOGPROBS_THREADS) {
                    const Ranked c = cand[j];
                    int rank = 0;
#pragma unroll 8
                    for (int i = 0; i < all; i++) rank += ranks_before(cand[i], c);
                    if (rank < p.top) put(rank, c);
                }
                found = in_row;
            }
            // fewer than k tokens can come: the first of the others fill the places
            for (int j0 = 0; j0 < p.vocab && found < p.top && warp == 0; j0 += 32) {
                const bool hit = j0 + lane < p.vocab && to_float(x[j0 + lane]) == -INFINITY;
                const unsigned hits = __ballot_sync(0xffffffffu, hit);
                const int rank = found + __popc(hits & ((1u << lane) - 1));
                if (hit && rank < p.top) put(rank, {-INFINITY, j0 + lane});
                found += __popc(hits);
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
    // CTAs to a row: until the GPU is full (4 to an SM; 8: 512 rows of 151,936 with 5 alternatives 79 us, not 71), in slices of at least 4,096
    // elements, as many as a cluster holds (8 rows with 20 alternatives: one CTA a row 33 us, 16 of them 13)
    const int full = 4 * abk_sm_count();
    int splits = 1;
    while (splits < LOGPROBS_MAX_SPLITS && (long long)n_rows * splits * 2 <= full && vocab / (splits * 2) >= 4096) splits *= 2;
    LogProbs p;
    p.logits = logits, p.stride = stride, p.vocab = vocab, p.top = top, p.tokens = tokens, p.logprob = logprob, p.entropy = entropy;
    p.top_ids = top_ids, p.top_logprobs = top_logprobs;
    p.slice = (vocab + splits * piece - 1) / (splits * piece) * piece;
    void (*kernel)(LogProbs) = nullptr;
    if (dtype == ABK_F32) kernel = top == 0 ? logprobs_kernel<float, false> : logprobs_kernel<float, true>;
    else kernel = top == 0 ? logprobs_kernel<__nv_bfloat16, false> : logprobs_kernel<__nv_bfloat16, true>;
    if (splits > 8) {
        const cudaError_t e = cudaFuncSetAttribute((const void *)kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        if (e != cudaSuccess) return (int)e;
    }
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
