// How likely given tokens are under rows of logits: with m = max x and l = sum e^(x - m), the log probability of token t is
// x_t - m - log l, the entropy log l - sum e^(x - m) (x - m) / l; and the most likely tokens with their log probabilities, the
// larger logit first, the lower index first among equals (the order of src/main.c:43-48).
//
// A logit of -inf is a token that cannot come: it adds nothing, and its log probability is -inf. A row with a NaN or +inf, or
// with nothing but -inf, is no distribution: its numbers are NaN and its tokens -1. A token outside the vocabulary has the log
// probability NaN.
#define ABK_DEFINE_ERROR
#include "common.cuh"

#define LOGPROBS_MAX_TOP 64
#define LOGPROBS_THREADS 512

struct LogProbs {
    const void *logits;
    long long stride;
    int vocab, top;
    const int *tokens;
    float *logprob, *entropy;
    int *top_ids;
    float *top_logprobs;
};
struct Ranked {
    float v;
    int i;
};
__device__ __forceinline__ bool ranks_before(Ranked a, Ranked b) { return a.v > b.v || (a.v == b.v && a.i < b.i); }

template <typename T>
__global__ void __launch_bounds__(LOGPROBS_THREADS) logprobs_kernel(LogProbs p) {
    __shared__ float scratch[33];
    __shared__ Ranked best[LOGPROBS_THREADS / 32];
    pdl_wait();
    const int row = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const T *x = (const T *)p.logits + row * p.stride;
    float m = -INFINITY, l = 0.0f, t = 0.0f;
    for (int j = threadIdx.x; j < p.vocab; j += LOGPROBS_THREADS) m = fmaxf(m, to_float(x[j]));
    m = block_max(m, scratch);
    for (int j = threadIdx.x; j < p.vocab; j += LOGPROBS_THREADS) {
        const float d = to_float(x[j]) - m, e = expf(d);
        l += e, t += e * fmaxf(d, -1e30f);
    }
    l = block_sum(l, scratch), t = block_sum(t, scratch);
    const bool none = !(m < INFINITY) || m == -INFINITY || !(l >= 0.0f);
    const float nan = __int_as_float(0x7fffffff), log_l = logf(l);
    if (threadIdx.x == 0) {
        const int token = p.tokens[row];
        p.logprob[row] = none || token < 0 || token >= p.vocab ? nan : to_float(x[token]) - m - log_l;
        if (p.entropy) p.entropy[row] = none ? nan : log_l - t / l;
    }
    Ranked last = {INFINITY, -1};
    for (int k = 0; k < p.top; k++) {
        Ranked b = {-INFINITY, 0x7fffffff};
        if (!none)
            for (int j = threadIdx.x; j < p.vocab; j += LOGPROBS_THREADS) {
                const Ranked c = {to_float(x[j]), j};
                if (ranks_before(last, c) && ranks_before(c, b)) b = c;
            }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const Ranked c = {__shfl_xor_sync(0xffffffffu, b.v, o), __shfl_xor_sync(0xffffffffu, b.i, o)};
            if (ranks_before(c, b)) b = c;
        }
        __syncthreads();
        if (lane == 0) best[warp] = b;
        __syncthreads();
        for (int w = 0; w < LOGPROBS_THREADS / 32; w++)
            if (ranks_before(best[w], b)) b = best[w];
        last = b;
        if (threadIdx.x == 0) {
            p.top_ids[(long long)row * p.top + k] = none ? -1 : b.i;
            p.top_logprobs[(long long)row * p.top + k] = none ? nan : b.v - m - log_l;
        }
    }
}

extern "C" int abk_token_logprobs(const void *logits, int dtype, long long stride, int n_rows, int vocab, const int *tokens,
                                  float *logprob, float *entropy, int top, int *top_ids, float *top_logprobs, void *stream) {
    if (n_rows <= 0) return 0;
    if (vocab < 1) ABK_REFUSE("token_logprobs: vocabulary of %d", vocab);
    if (top < 0 || top > LOGPROBS_MAX_TOP || top > vocab)
        ABK_REFUSE("token_logprobs: %d most likely tokens of a vocabulary of %d (at most %d)", top, vocab, LOGPROBS_MAX_TOP);
    LogProbs p = {logits, stride, vocab, top, tokens, logprob, entropy, top_ids, top_logprobs};
    if (dtype == ABK_F32) abk_launch(logprobs_kernel<float>, dim3(n_rows), dim3(LOGPROBS_THREADS), 0, (cudaStream_t)stream, p);
    else abk_launch(logprobs_kernel<__nv_bfloat16>, dim3(n_rows), dim3(LOGPROBS_THREADS), 0, (cudaStream_t)stream, p);
    return ABK_LAUNCH_RESULT();
}
