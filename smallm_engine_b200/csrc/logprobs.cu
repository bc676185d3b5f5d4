// Log probabilities from rows of logits x[0..V):
//
//   lse = m + log S0,  S0 = sum e^(x - m),  S1 = sum e^(x - m) (x - m),  m = max x
//   log p(token) = (x[token] - m) - log S0
//   entropy      = log S0 - S1 / S0
//
// and the n_top most likely tokens, largest logit first, equal logits in
// order of their ids (NaN last).  A logit of -inf has probability 0 and adds
// nothing to the entropy; a row that holds NaN or +inf, or nothing above
// -inf, has no distribution, and its log probabilities and entropy are NaN.
#include "common.cuh"
#include "engine.h"
#include "smallm_cuda.h"

namespace smallm {
namespace {

constexpr int kLpThreads = 1024;
constexpr int kLpWarps = kLpThreads / 32;

// Larger key = earlier alternative; keys are unique within a row.
__device__ __forceinline__ unsigned long long alt_key(float x, uint32_t i) {
    const uint32_t o = x == x ? float_order_key(x + 0.f) : 0u;
    return ((unsigned long long)o << 32) | (0xFFFFFFFFu - i);
}

__device__ unsigned long long block_max_key(unsigned long long k, unsigned long long* red) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const unsigned long long y = __shfl_xor_sync(0xffffffffu, k, o);
        k = y > k ? y : k;
    }
    __syncthreads();
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = k;
    __syncthreads();
    for (int w = 0; w < kLpWarps; ++w) k = red[w] > k ? red[w] : k;
    return k;
}

__global__ void __launch_bounds__(kLpThreads) smallm_logprobs_kernel(const LogprobArgs a) {
    __shared__ float red[32];
    __shared__ unsigned long long kred[kLpWarps];
    const float* x = a.logits + (size_t)blockIdx.x * a.stride;
    unsigned long long best = 0;
    bool bad = false;
    for (uint32_t i = threadIdx.x; i < a.vocab; i += kLpThreads) {
        const float v = x[i];
        bad |= !(v < INFINITY);
        const unsigned long long k = alt_key(v, i);
        best = k > best ? k : best;
    }
    best = block_max_key(best, kred);
    const float m = x[0xFFFFFFFFu - (uint32_t)best];
    bad = __syncthreads_or(bad) || m == -INFINITY;
    float s0 = 0.f, s1 = 0.f;
    for (uint32_t i = threadIdx.x; i < a.vocab; i += kLpThreads) {
        const float d = x[i] - m, e = expf(d);
        s0 += e;
        s1 += e > 0.f ? e * d : 0.f;
    }
    s0 = block_sum(s0, red);
    s1 = block_sum(s1, red);
    const float nan = __int_as_float(0x7FC00000);
    const float ls = bad ? nan : logf(s0);
    if (threadIdx.x == 0) {
        if (a.entropy) a.entropy[blockIdx.x] = ls - s1 / s0;
        if (a.tokens) {
            const uint32_t t = a.tokens[blockIdx.x];
            a.logprob[blockIdx.x] = t < a.vocab ? (x[t] - m) - ls : nan;
        }
    }
    for (uint32_t r = 0; r < a.n_top; ++r) {
        if (threadIdx.x == 0) {
            const uint32_t id = 0xFFFFFFFFu - (uint32_t)best;
            a.top_ids[(size_t)blockIdx.x * a.n_top + r] = id;
            a.top_logprobs[(size_t)blockIdx.x * a.n_top + r] = (x[id] - m) - ls;
        }
        unsigned long long next = 0;
        for (uint32_t i = threadIdx.x; i < a.vocab; i += kLpThreads) {
            const unsigned long long k = alt_key(x[i], i);
            if (k < best && k > next) next = k;
        }
        best = block_max_key(next, kred);
    }
}

}  // namespace

void launch_logprobs(const LogprobArgs& a, cudaStream_t stream) {
    if (!a.vocab) throw Error(SMALLM_ERR_INVALID, "logprobs: an empty vocabulary");
    if (a.stride < a.vocab) throw Error(SMALLM_ERR_INVALID, "logprobs: stride must be at least vocab");
    if (a.n_top > kLogprobMaxTop || a.n_top > a.vocab)
        throw Error(SMALLM_ERR_RANGE, "logprobs: at most 64 alternatives, and no more than vocab");
    if (!a.n_rows) return;
    smallm_logprobs_kernel<<<a.n_rows, kLpThreads, 0, stream>>>(a);
    SM_CUDA(cudaGetLastError());
}

}  // namespace smallm
