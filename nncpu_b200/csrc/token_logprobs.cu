// Log probabilities of given tokens, the distribution's entropy and its best alternatives, row by row of logits:
//   M = max x, S = sum e^(x - M):  log p(t) = x_t - M - ln S,  entropy = ln S - sum e^(x - M) (x - M) / S,
//   the k best by (x descending, index ascending).
// A NaN counts as -inf, as everywhere in the choice of a token (crates/nncpu/src/model/forward.rs:1003-1011); a lane of -inf has
// probability 0 and adds nothing to the entropy.

#include <math.h>

#define NN_LIB token_logprobs
#include "common.cuh"

namespace {

struct Rows {
    const void* logits;      // [n, vocab]
    int dt;
    const int* targets;      // [n]
    float* logprobs;         // [n]
    float* entropy;          // [n]
    float* top;              // [n, k] or null
    int* ids;                // [n, k]
    int n, vocab, k;
};

__device__ __forceinline__ float logit(const Rows& p, size_t row, int i) {
    const float x = ld_f(p.logits, row * p.vocab + i, p.dt);
    return x != x ? -INFINITY : x;
}

constexpr int kThreads = 512;

__global__ void __launch_bounds__(kThreads) rows_kernel(const Rows p) {
    __shared__ float scratch[33];
    __shared__ unsigned long long best;
    const size_t row = blockIdx.x;
    float m = -INFINITY;
    for (int i = threadIdx.x; i < p.vocab; i += kThreads) m = fmaxf(m, logit(p, row, i));
    m = block_max(m, scratch);
    float s = 0.0f, e = 0.0f;
    for (int i = threadIdx.x; i < p.vocab; i += kThreads) {
        const float x = logit(p, row, i);
        if (x > -INFINITY) {
            const float y = x - m, w = expf(y);
            s += w;
            e = fmaf(w, y, e);
        }
    }
    s = block_sum(s, scratch);
    e = block_sum(e, scratch);
    const float logs = logf(s);
    if (threadIdx.x == 0) {
        const int t = p.targets[row];
        p.logprobs[row] = t < 0 || t >= p.vocab ? __int_as_float(0x7FC00000) : m == -INFINITY ? -INFINITY : logit(p, row, t) - m - logs;
        p.entropy[row] = m == -INFINITY ? 0.0f : logs - e / s;
    }
    // the k best, one after the other: the greatest (x, -index) below the one before
    unsigned long long before = ~0ull;
    for (int k = 0; k < p.k; ++k) {
        if (threadIdx.x == 0) best = 0;
        __syncthreads();
        unsigned long long mine = 0;
        for (int i = threadIdx.x; i < p.vocab; i += kThreads) {
            const uint32_t b = __float_as_uint(logit(p, row, i) + 0.0f);
            const unsigned long long key = (unsigned long long)(b & 0x80000000u ? ~b : b | 0x80000000u) << 32 | (uint32_t)~i;
            if (key < before && key > mine) mine = key;
        }
        atomicMax(&best, mine);
        __syncthreads();
        before = best;
        if (threadIdx.x == 0) {
            const int i = (int)~(uint32_t)before;
            p.ids[row * p.k + k] = i;
            const float x = logit(p, row, i);
            p.top[row * p.k + k] = x == -INFINITY ? -INFINITY : x - m - logs;
        }
        __syncthreads();
    }
}

}  // namespace

extern "C" int nncpu_token_logprobs(const void* logits, int dt, const int* targets, float* logprobs, float* entropy, float* top, int* ids,
                                    int n, int vocab, int k, cudaStream_t stream) {
    NN_CHECK(n >= 0 && vocab > 0 && vocab < (1 << 30), "token_logprobs: %d rows of %d logits", n, vocab);
    NN_CHECK(k >= 0 && k <= vocab && k <= 64, "token_logprobs: the best %d of %d (at most 64)", k, vocab);
    if (n == 0) return 0;
    Rows p{logits, dt, targets, logprobs, entropy, top, ids, n, vocab, k};
    rows_kernel<<<(unsigned)n, kThreads, 0, stream>>>(p);
    NN_LAUNCH_OK("token_logprobs");
    return 0;
}
