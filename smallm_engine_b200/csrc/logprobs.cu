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
//
// Bound by the one read of the logits.  A cluster of 1 to 16 CTAs owns a row
// (more CTAs when there are few rows), each a contiguous range of it in chunks
// of 16 KB that arrive in two shared-memory stages by bulk copies:
//   - (m, S0, S1) run per thread; a larger maximum m' rescales them,
//     S1' = e^(m - m') (S1 + (m - m') S0);
//   - alternatives are 64-bit keys (value, then lower id), unique in a row.  A
//     threshold below which nothing can be among the n_top best lets nearly
//     every chunk pass with one comparison per thread; what is above it is
//     collected in shared memory, and when much is, the list is ranked and cut
//     to n_top, its last key the new threshold.  Where half the threads or
//     more hold something above it (the first chunk; ascending rows), the
//     n_top-th largest of 128 group maxima (2 threads, 32 elements) raises it
//     first: n_top groups reach it, so at most 32 n_top elements do.
// Rank 0 joins the ranges through distributed shared memory.  509 x 151936, five
// alternatives: 58 us, 5.3 TB/s; 1 x 128256, twenty: 10 us, which is the cluster's
// start and barriers and the ranking.
#include <cooperative_groups.h>

#include <algorithm>

#include "common.cuh"
#include "engine.h"
#include "smallm_cuda.h"

namespace smallm {
namespace {

namespace cg = cooperative_groups;

constexpr int kLpThreads = 256;
constexpr int kLpVec = 4;                          // float4s of a thread per chunk
constexpr uint32_t kLpChunk = kLpThreads * kLpVec;  // float4s of a CTA per chunk
constexpr uint32_t kLpStages = 2;
constexpr uint32_t kLpMaxCluster = 16;
constexpr uint32_t kLpGroups = kLpThreads / 2;
constexpr uint32_t kLpCut = 128;  // collected keys that make a cut worth its barriers
constexpr uint32_t kLpLists = (kLpMaxCluster - 1) * kLogprobMaxTop / kLpThreads + 1;  // joined keys of a thread
constexpr uint32_t kLpKeys = kLogprobMaxTop * 2 * kLpVec * 4 + kLpCut + kLogprobMaxTop;
static_assert(kLpGroups >= kLogprobMaxTop && kLpKeys >= kLpMaxCluster * kLogprobMaxTop, "key buffer");

typedef unsigned long long u64;

struct LpShared {
    alignas(128) float4 stage[kLpStages][kLpChunk];
    uint64_t full[kLpStages];
    u64 keys[kLpKeys];          // collected
    u64 best[kLogprobMaxTop];   // ranked
    u64 group[kLpGroups];
    u64 floor;                  // only larger keys matter
    uint32_t count;
    float m, s0, s1;
    uint32_t bad;
    float wm[kLpThreads / 32], w0[kLpThreads / 32], w1[kLpThreads / 32];
};

// Larger key = earlier alternative; never 0.
__device__ __forceinline__ u64 alt_key(float x, uint32_t i) {
    const uint32_t o = x == x ? float_order_key(x + 0.f) : 0u;
    return ((u64)o << 32) | (0xFFFFFFFFu - i);
}
__device__ __forceinline__ float alt_value(u64 k) {
    const uint32_t o = (uint32_t)(k >> 32);
    return __uint_as_float(o & 0x80000000u ? o & 0x7FFFFFFFu : ~o);
}
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
constexpr float kLog2e = 1.4426950408889634f;
__device__ __forceinline__ float ex2(float t) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(t));
    return r;
}
// e^d of d <= 0; 0 below -200.  Off by 2 |d| 2^-24 + 2^-22 of itself, of which
// the sum sees e^d times that: 5e-8 to 1e-7 in a log probability of 128256, where
// f32's expf leaves 2e-8; chosen for its two instructions.
__device__ __forceinline__ float exp_neg(float d) { return ex2(d * kLog2e); }
// (m, s0, s1) joined with another range's.
__device__ __forceinline__ void join(float& m, float& s0, float& s1, float om, float o0, float o1) {
    const float M = fmaxf(m, om);
    if (M == -INFINITY) return;
    const float da = fmaxf(m - M, -200.f), db = fmaxf(om - M, -200.f);
    const float fa = exp_neg(da), fb = exp_neg(db);
    s1 = fa * fmaf(da, s0, s1) + fb * fmaf(db, o0, o1);
    s0 = fa * s0 + fb * o0;
    m = M;
}

// Rank the collected keys (unique) and keep the `want` largest: best[0..),
// largest first, and again at the front of keys.  All threads call it.
__device__ void lp_cut(LpShared& sh, uint32_t want) {
    const uint32_t c = sh.count;
    for (uint32_t i = threadIdx.x; i < c; i += kLpThreads) {
        const u64 k = sh.keys[i];
        uint32_t rank = 0;
#pragma unroll 8
        for (uint32_t j = 0; j < c; ++j) rank += sh.keys[j] > k;
        if (rank < want) sh.best[rank] = k;
    }
    __syncthreads();
    const uint32_t n = min(c, want);
    if (threadIdx.x < n) sh.keys[threadIdx.x] = sh.best[threadIdx.x];
    if (threadIdx.x == 0) {
        sh.count = n;
        if (n == want && sh.best[n - 1] > sh.floor) sh.floor = sh.best[n - 1];
    }
    __syncthreads();
}

__global__ void __launch_bounds__(kLpThreads, 4)
    smallm_logprobs_kernel(const LogprobArgs a, uint32_t per_cta, unsigned int* err) {
    extern __shared__ __align__(128) uint8_t lp_smem[];
    LpShared& sh = *reinterpret_cast<LpShared*>(lp_smem);
    cg::cluster_group cluster = cg::this_cluster();
    const uint32_t C = cluster.num_blocks(), rank = cluster.block_rank(), row = blockIdx.x / C;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const float* x = a.logits + (size_t)row * a.stride;
    // float4s of the row from the 16-byte boundary at or before its start
    const uint32_t mis = (uint32_t)(reinterpret_cast<uintptr_t>(x) >> 2) & 3u;
    const uint32_t nq = (uint32_t)(((uint64_t)a.vocab + mis + 3) / 4);
    const uint32_t qb = min(nq, rank * per_cta), qe = min(nq, qb + per_cta);
    // whole float4s of the row arrive by bulk copies; its ragged ends are read directly
    const uint32_t whole_b = mis ? 1 : 0, whole_e = (uint32_t)(((uint64_t)a.vocab + mis) / 4);
    auto whole = [&](uint32_t q0, uint32_t& b, uint32_t& e) {  // ... of the chunk from q0
        b = max(q0, whole_b);
        e = max(b, min(min(q0 + kLpChunk, qe), whole_e));
    };
    auto fetch = [&](uint32_t q0) {  // one thread
        uint32_t b, e;
        whole(q0, b, e);
        const uint32_t s = (q0 - qb) / kLpChunk % kLpStages;
        if (e > b) {
            mbar_arrive_expect_tx(&sh.full[s], (e - b) * 16);
            bulk_g2s(&sh.stage[s][b - q0], x - mis + 4ull * b, (e - b) * 16, &sh.full[s]);
        } else {
            mbar_arrive(&sh.full[s]);
        }
    };
    if (tid < (int)kLogprobMaxTop) sh.best[tid] = 0;
    pdl_wait();
    if (tid == 0) {
        for (uint32_t s = 0; s < kLpStages; ++s) mbar_init(&sh.full[s], 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        for (uint32_t s = 0; s < kLpStages; ++s)
            if (qb + s * kLpChunk < qe) fetch(qb + s * kLpChunk);
        sh.floor = 0;
        sh.count = 0;
    }
    // (on its way before it is needed)
    const uint32_t token = a.tokens && rank == 0 && tid == 0 ? a.tokens[row] : a.vocab;
    const float given = token < a.vocab ? x[token] : 0.f;
    float m = -INFINITY, s0 = 0.f, s1 = 0.f;
    bool bad = false, ok = true;
    __syncthreads();
    for (uint32_t q0 = qb, n = 0; q0 < qe; q0 += kLpChunk, ++n) {
        const uint32_t s = n % kLpStages, parity = n / kLpStages & 1;
        // (a second wait after one that gave up: no copy lands in a CTA that has left)
        ok = (mbar_wait(&sh.full[s], parity) || (mbar_wait(&sh.full[s], parity), false)) && ok;
        float v[kLpVec][4];
#pragma unroll
        for (int u = 0; u < kLpVec; ++u) *reinterpret_cast<float4*>(v[u]) = sh.stage[s][u * kLpThreads + tid];
        if (q0 < whole_b || q0 + kLpChunk > min(qe, whole_e)) {  // the row's ends
#pragma unroll
            for (int u = 0; u < kLpVec; ++u) {
                const uint32_t q = q0 + u * kLpThreads + tid;
                if (q >= whole_b && q < min(qe, whole_e)) continue;
                const uint32_t i = 4 * q - mis;  // wraps below the row's start
#pragma unroll
                for (int c = 0; c < 4; ++c) v[u][c] = q < qe && i + c < a.vocab ? x[i + c] : -INFINITY;
            }
        }
        float xm = v[0][0];
#pragma unroll
        for (int u = 0; u < kLpVec; ++u)
#pragma unroll
            for (int c = 0; c < 4; ++c) xm = max_nan(xm, v[u][c]);
        bad |= !(xm < INFINITY);
        if (xm > m) {
            const float d = fmaxf(m - xm, -200.f), f = exp_neg(d);
            s1 = f * fmaf(d, s0, s1);
            s0 *= f;
            m = xm;
        }
        const float ref = m == -INFINITY ? 0.f : m;
        // (S1 in units of log2 until the end)
        float2 c0 = make_float2(0.f, 0.f), c1 = c0;
        const float2 less = make_float2(-ref, -ref), scale = make_float2(kLog2e, kLog2e);
#pragma unroll
        for (int u = 0; u < kLpVec; ++u)
#pragma unroll
            for (int c = 0; c < 4; c += 2) {
                float2 t = mul2(add2(make_float2(v[u][c], v[u][c + 1]), less), scale);
                t.x = fmaxf(t.x, -300.f);
                t.y = fmaxf(t.y, -300.f);
                const float2 e = make_float2(ex2(t.x), ex2(t.y));
                c0 = add2(c0, e);
                c1 = fma2(e, t, c1);
            }
        s0 += c0.x + c0.y;
        s1 += (c1.x + c1.y) * (1.f / kLog2e);
        // the stage is free once every thread has its elements
        const bool more = tid == 0 && q0 + kLpStages * kLpChunk < qe;
        if (!a.n_top) {
            __syncthreads();
            if (more) fetch(q0 + kLpStages * kLpChunk);
            continue;
        }
        // ids of this thread's elements: first of float4 u, or past vocab
        auto id_of = [&](int u, int c) { return 4 * (q0 + u * kLpThreads + tid) - mis + c; };
        auto in_row = [&](int u, int c) {
            return q0 + u * kLpThreads + tid < qe && id_of(u, c) < a.vocab;
        };
        u64 floor = sh.floor;
        const bool over = !(xm < INFINITY) || float_order_key(xm + 0.f) >= (uint32_t)(floor >> 32);
        const int n_over = __syncthreads_count(over);
        if (more) fetch(q0 + kLpStages * kLpChunk);
        if (!n_over) continue;
        if (n_over > kLpThreads / 2) {
            u64 k = 0;
            if (xm < INFINITY && xm > -INFINITY) {  // the first place of the maximum
                uint32_t id = 0;
#pragma unroll
                for (int u = kLpVec - 1; u >= 0; --u)
#pragma unroll
                    for (int c = 3; c >= 0; --c)
                        if (v[u][c] == xm) id = id_of(u, c);
                k = alt_key(xm, id);
            } else {
#pragma unroll 1
                for (int u = 0; u < kLpVec; ++u)
#pragma unroll 1
                    for (int c = 0; c < 4; ++c)
                        if (in_row(u, c)) {
                            const u64 y = alt_key(x[id_of(u, c)], id_of(u, c));
                            k = y > k ? y : k;
                        }
            }
            const u64 other = __shfl_xor_sync(0xffffffffu, k, 1);
            k = other > k ? other : k;
            if (!(tid & 1)) sh.group[tid >> 1] = k;
            __syncthreads();
            // two threads for a group, half of the other groups each
            const u64 mine = sh.group[tid >> 1];
            uint32_t larger = 0;
            const ulonglong2* gk = reinterpret_cast<const ulonglong2*>(sh.group) + (tid & 1) * (kLpGroups / 4);
#pragma unroll 8
            for (uint32_t j = 0; j < kLpGroups / 4; ++j) {
                const ulonglong2 y = gk[j];
                larger += (y.x > mine) + (y.y > mine);
            }
            larger += __shfl_xor_sync(0xffffffffu, larger, 1);
            if (!(tid & 1) && mine && larger == a.n_top - 1 && mine - 1 > sh.floor) sh.floor = mine - 1;
            __syncthreads();
            floor = sh.floor;
        }
        if (over) {
            const float least = alt_value(floor);  // NaN (everything may count) where there is no floor yet
#pragma unroll
            for (int u = 0; u < kLpVec; ++u)
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    if (v[u][c] < least) continue;
                    const u64 k = alt_key(v[u][c], id_of(u, c));
                    if (k > floor && in_row(u, c)) sh.keys[atomicAdd(&sh.count, 1u)] = k;
                }
        }
        __syncthreads();
        // (a cut soon after the first chunks, while the floor still rises fast)
        if (sh.count > min(kLpCut, a.n_top + max(4u, a.n_top / 2))) lp_cut(sh, a.n_top);
    }
    if (a.n_top) lp_cut(sh, a.n_top);
    // this CTA's (m, s0, s1)
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const float om = __shfl_xor_sync(0xffffffffu, m, o), o0 = __shfl_xor_sync(0xffffffffu, s0, o),
                    o1 = __shfl_xor_sync(0xffffffffu, s1, o);
        join(m, s0, s1, om, o0, o1);
    }
    if (lane == 0) {
        sh.wm[warp] = m;
        sh.w0[warp] = s0;
        sh.w1[warp] = s1;
    }
    bad = __syncthreads_or(bad);
    if (tid == 0) {
        for (int w = 1; w < kLpThreads / 32; ++w) join(m, s0, s1, sh.wm[w], sh.w0[w], sh.w1[w]);
        sh.m = m;
        sh.s0 = s0;
        sh.s1 = s1;
        sh.bad = bad;
    }
    if (C > 1) {
        cluster.sync();
        if (rank == 0) {
            // Own ranked keys stay at the front of keys; the others' follow.  Where
            // m ranges have d keys each at or above a key and m d >= n_top, smaller
            // ones do not matter: the m-th largest of the ranges' d-th keys.
            const uint32_t top = a.n_top, d = min(top, max((top + C - 1) / C, 5u)), need = (top + d - 1) / max(d, 1u);
            u64 list[kLpLists];
#pragma unroll
            for (int j = 0; j < (int)kLpLists; ++j) {
                const uint32_t i = min(tid + j * kLpThreads, (C - 1) * top), r = i / max(top, 1u) + 1;
                list[j] = *cluster.map_shared_rank(&sh.best[i % max(top, 1u)], min(r, C - 1));
            }
            u64 least = (uint32_t)lane < C && top ? *cluster.map_shared_rank(&sh.best[d - 1], lane) : 0ull;
            uint32_t larger = 0;
#pragma unroll
            for (int r = 0; r < (int)kLpMaxCluster; ++r) larger += __shfl_sync(0xffffffffu, least, r) > least;
            const uint32_t at = __ballot_sync(0xffffffffu, (uint32_t)lane < C && least && larger == need - 1);
            const u64 bound = at ? __shfl_sync(0xffffffffu, least, __ffs(at) - 1) : 0ull;
#pragma unroll
            for (int j = 0; j < (int)kLpLists; ++j)
                if (tid + j * kLpThreads < (C - 1) * top && list[j] && list[j] >= bound)
                    sh.keys[atomicAdd(&sh.count, 1u)] = list[j];
            if (warp == 0) {  // lane r: CTA r
                const LpShared* o = cluster.map_shared_rank(&sh, (uint32_t)lane < C ? lane : 0);
                m = o->m;
                s0 = o->s0;
                s1 = o->s1;
                bad = (uint32_t)lane < C && o->bad;
                if ((uint32_t)lane >= C) m = -INFINITY, s0 = s1 = 0.f;
#pragma unroll
                for (int d = 8; d > 0; d >>= 1) {
                    const float om = __shfl_xor_sync(0xffffffffu, m, d), o0 = __shfl_xor_sync(0xffffffffu, s0, d),
                                o1 = __shfl_xor_sync(0xffffffffu, s1, d);
                    join(m, s0, s1, om, o0, o1);
                }
                bad = __any_sync(0xffffffffu, bad);
                if (lane == 0) {
                    sh.m = m;
                    sh.s0 = s0;
                    sh.s1 = s1;
                    sh.bad = bad;
                }
            }
            __syncthreads();
            if (top) lp_cut(sh, top);
        }
        cluster.sync();
        if (rank) {
            if (!ok) atomicOr(err, kErrLogprobs);
            return;
        }
    } else {
        __syncthreads();
    }
    if (!ok) atomicOr(err, kErrLogprobs);
    const float nan = __int_as_float(0x7FC00000);
    const float M = sh.m, ls = sh.bad || M == -INFINITY ? nan : logf(sh.s0);
    if (tid == 0) {
        if (a.entropy) a.entropy[row] = ls - sh.s1 / sh.s0;
        if (a.tokens) a.logprob[row] = token < a.vocab ? (given - M) - ls : nan;
    }
    for (uint32_t i = tid; i < a.n_top; i += kLpThreads) {
        const u64 k = sh.best[i];
        a.top_ids[(size_t)row * a.n_top + i] = 0xFFFFFFFFu - (uint32_t)k;
        a.top_logprobs[(size_t)row * a.n_top + i] = (alt_value(k) - M) - ls;
    }
}

}  // namespace

void launch_logprobs(const LogprobArgs& a, cudaStream_t stream) {
    if (!a.vocab) throw Error(SMALLM_ERR_INVALID, "logprobs: an empty vocabulary");
    if (a.vocab > 1u << 30) throw Error(SMALLM_ERR_RANGE, "logprobs: at most 2^30 logits per row");
    if (a.stride < a.vocab) throw Error(SMALLM_ERR_INVALID, "logprobs: stride must be at least vocab");
    if (a.n_top > kLogprobMaxTop || a.n_top > a.vocab)
        throw Error(SMALLM_ERR_RANGE, "logprobs: at most 64 alternatives, and no more than vocab");
    if (a.n_rows > 1u << 26) throw Error(SMALLM_ERR_RANGE, "logprobs: at most 2^26 rows");
    if ((reinterpret_cast<uintptr_t>(a.logits) | reinterpret_cast<uintptr_t>(a.tokens) |
         reinterpret_cast<uintptr_t>(a.logprob) | reinterpret_cast<uintptr_t>(a.entropy) |
         (a.n_top ? reinterpret_cast<uintptr_t>(a.top_ids) | reinterpret_cast<uintptr_t>(a.top_logprobs) : 0)) & 3u)
        throw Error(SMALLM_ERR_INVALID, "logprobs: pointers must be 4-byte aligned");
    if (!a.n_rows) return;
    // CTAs per row: one up to two chunks (63 x 8000: 3.4 us, by two CTAs 4.5 us),
    // then two per SM in all, each with a chunk to itself at least (1 x 12338: 4.2
    // us by four CTAs, 4.7 us by two; 1 x 32000, twenty alternatives: 7.4 us by
    // eight, 12 us by two)
    const uint32_t nq = (a.vocab + 6) / 4, sms = (uint32_t)device_sm_count();
    uint32_t C = 1;
    while (C < kLpMaxCluster && a.n_rows * C < 2 * sms && nq > std::max(C, 2u) * kLpChunk) C *= 2;
    const void* fn = (const void*)smallm_logprobs_kernel;
    if (C > 8) allow_large_clusters_once(fn);
    set_smem_limit_once(fn, (int)sizeof(LpShared));
    LogprobArgs aa = a;
    uint32_t per_cta = (nq + C - 1) / C;
    unsigned int* err = a.err ? a.err : device_error_flag();
    void* args[] = {&aa, &per_cta, &err};
    launch_cluster_ex(fn, dim3(a.n_rows * C), dim3(kLpThreads), sizeof(LpShared), C, stream, args);
}

}  // namespace smallm
