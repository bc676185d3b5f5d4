// Attention of T drafted tokens over the KV cache (verification of a draft).
//
//   s[t,h,k] = q[t,h] . K[g,k] / sqrt(hd),     g = h / (n_heads / n_kv)
//   p = softmax over the rows k that token t sees:  every k < n_past, and of
//       the drafted rows n_past + u those whose mask bit u is set (no mask:
//       u <= t, a chain)
//   out[t,h] = sum_k p[k] V[g,k];   weights[g,k] += sum over t, h of g of p[k]
//
// A token that sees nothing gets zeros and adds nothing.  Rows that a token
// does not see have no effect on it, whatever they hold.
//
// The G query heads of a KV head and the T tokens are one matrix of R = T * G
// rows (row r: token r / G, head r % G) over the KV head's n = n_past + T
// keys, so every K and V row is read once per block of rows.  The keys are
// split over CTAs; each leaves an unnormalised partial (reference exponent,
// sum, output) and a second kernel joins them: the online-softmax identity
//   sum_k e^{s_k} v_k = sum_i e^{m_i} (sum_{k in i} e^{s_k - m_i} v_k).
// Exponents are base 2: with c = log2(e) / sqrt(hd), p = 2^(s c - mc), one
// fma rounding, mc the running maximum times c.
#include <algorithm>

#include "common.cuh"
#include "engine.h"
#include "smallm_cuda.h"

namespace smallm {
namespace {

constexpr uint32_t kTile = 32;       // keys per warp tile: one lane per key in the softmax
constexpr int kVecRows = 8;          // rows per CTA
constexpr int kVecWarps = 8;
constexpr int kVecThreads = 32 * kVecWarps;

struct TreeParams {
    TreeArgs a;
    uint32_t G, R, n, words;
    uint32_t n_split, tiles_per_split;
    uint32_t sc_stride;  // floats between two rows of stored scores
    float c;             // log2(e) / sqrt(hd)
    float* part_o;       // [n_split][n_kv * R][hd]
    float2* part_ml;     // [n_split][n_kv * R] (mc, sum)
    float* scores;       // [n_kv * R][sc_stride], raw q . K, -inf where unseen
    float2* stats;       // [n_kv * R] (mc of the whole row, 1 / sum or 0)
};

__device__ __forceinline__ bool tree_sees(const TreeParams& p, uint32_t t, uint32_t key) {
    if (key < p.a.n_past) return true;
    const uint32_t u = key - p.a.n_past;
    if (u >= p.a.n_tokens) return false;
    if (!p.a.mask) return u <= t;
    return (p.a.mask[(size_t)t * p.words + (u >> 5)] >> (u & 31)) & 1u;
}

// Sum v[i] over the 8 lanes of a group; lane l8 of the group gets the sum of
// row l8 (a reduce-scatter: 7 shuffles instead of 24).
__device__ __forceinline__ float group_reduce8(float (&v)[8], int l8) {
#pragma unroll
    for (int w = 4; w >= 1; w >>= 1) {
        const bool up = (l8 & w) != 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (i < w) {
                const float keep = up ? v[i + w] : v[i];
                const float send = up ? v[i] : v[i + w];
                v[i] = keep + __shfl_xor_sync(0xffffffffu, send, w);
            }
        }
    }
    return v[0];
}

// Vector path: f32 FMAs, each warp runs its own online softmax over tiles of
// 32 keys for the CTA's 8 rows; the warps' states are joined at the end.
template <int HD>
__global__ void __launch_bounds__(kVecThreads, 2) smallm_tree_vec_kernel(const TreeParams p) {
    constexpr int DV = HD / 32;  // K float4s of a lane (8 lanes per key); V floats of a lane (32 lanes per key)
    __shared__ __align__(16) float qs[kVecRows][HD];
    __shared__ __align__(16) float ps[kVecWarps][kTile][kVecRows];
    __shared__ __align__(16) float os[kVecWarps][kVecRows][HD];
    __shared__ float wm[kVecWarps][kVecRows], wl[kVecWarps][kVecRows];
    const TreeArgs& a = p.a;
    const uint32_t split = blockIdx.x, g = blockIdx.y, r0 = blockIdx.z * kVecRows;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, l8 = lane & 7, kl = lane >> 3;
    for (int i = tid; i < kVecRows * HD; i += kVecThreads) {
        const uint32_t r = r0 + i / HD;
        qs[i / HD][i % HD] =
            r < p.R ? a.q[(size_t)(r / p.G) * a.q_stride + ((size_t)g * p.G + r % p.G) * HD + i % HD] : 0.f;
    }
    __syncthreads();
    float m[kVecRows], l[kVecRows], o[kVecRows][DV];
#pragma unroll
    for (int r = 0; r < kVecRows; ++r) {
        m[r] = -INFINITY;
        l[r] = 0.f;
#pragma unroll
        for (int e = 0; e < DV; ++e) o[r][e] = 0.f;
    }
    const float* kb = a.kcache + (size_t)g * a.max_ctx * HD;
    const float* vb = a.vcache + (size_t)g * a.max_ctx * HD;
    const uint32_t tiles = (p.n + kTile - 1) / kTile;
    const uint32_t t_end = min(tiles, (split + 1) * p.tiles_per_split);
    for (uint32_t tile = split * p.tiles_per_split + warp; tile < t_end; tile += kVecWarps) {
        const uint32_t base = tile * kTile;
        // scores: 4 keys at a time, 8 lanes per key
#pragma unroll 2
        for (int j = 0; j < 8; ++j) {
            const uint32_t key = base + 4 * j + kl;
            float4 kv[DV];
#pragma unroll
            for (int e = 0; e < DV; ++e)
                kv[e] = key < p.n ? __ldg(reinterpret_cast<const float4*>(kb + (size_t)key * HD) + l8 + 8 * e)
                                  : make_float4(0.f, 0.f, 0.f, 0.f);
            float s[kVecRows];
#pragma unroll
            for (int r = 0; r < kVecRows; ++r) {
                s[r] = 0.f;
#pragma unroll
                for (int e = 0; e < DV; ++e) {
                    const float4 q4 = reinterpret_cast<const float4*>(qs[r])[l8 + 8 * e];
                    s[r] = fmaf(q4.x, kv[e].x, s[r]);
                    s[r] = fmaf(q4.y, kv[e].y, s[r]);
                    s[r] = fmaf(q4.z, kv[e].z, s[r]);
                    s[r] = fmaf(q4.w, kv[e].w, s[r]);
                }
            }
            ps[warp][4 * j + kl][l8] = group_reduce8(s, l8);
        }
        __syncwarp();
        // online softmax: lane = key
        const uint32_t key = base + lane;
        const bool mixed = base + kTile > a.n_past;  // the tile holds drafted rows or the end
        float s[kVecRows];
        *reinterpret_cast<float4*>(&s[0]) = *reinterpret_cast<const float4*>(&ps[warp][lane][0]);
        *reinterpret_cast<float4*>(&s[4]) = *reinterpret_cast<const float4*>(&ps[warp][lane][4]);
#pragma unroll
        for (int r = 0; r < kVecRows; ++r) {
            if (mixed && (r0 + r >= p.R || !tree_sees(p, (r0 + r) / p.G, key))) s[r] = -INFINITY;
            if (p.scores && r0 + r < p.R && key < p.n)
                p.scores[((size_t)g * p.R + r0 + r) * p.sc_stride + key] = s[r];
            const float mt = warp_max(s[r]) * p.c;
            const float mn = fmaxf(m[r], mt);
            const float ref = mn == -INFINITY ? 0.f : mn;
            const float e = exp2f(fmaf(s[r], p.c, -ref));
            const float cf = exp2f(m[r] - ref);
            m[r] = mn;
            l[r] = fmaf(l[r], cf, e);
            s[r] = e;
#pragma unroll
            for (int d = 0; d < DV; ++d) o[r][d] *= cf;
        }
        *reinterpret_cast<float4*>(&ps[warp][lane][0]) = *reinterpret_cast<const float4*>(&s[0]);
        *reinterpret_cast<float4*>(&ps[warp][lane][4]) = *reinterpret_cast<const float4*>(&s[4]);
        __syncwarp();
        // o += p V: lane owns DV consecutive head dimensions
#pragma unroll 4
        for (int k = 0; k < (int)kTile; ++k) {
            float v[DV];
            const bool in = base + k < p.n;
            const float* vr = vb + (size_t)(base + k) * HD + lane * DV;
            if constexpr (DV == 4) {
                const float4 x = in ? __ldg(reinterpret_cast<const float4*>(vr)) : make_float4(0.f, 0.f, 0.f, 0.f);
                v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w;
            } else if constexpr (DV == 2) {
                const float2 x = in ? __ldg(reinterpret_cast<const float2*>(vr)) : make_float2(0.f, 0.f);
                v[0] = x.x, v[1] = x.y;
            } else {
                v[0] = in ? __ldg(vr) : 0.f;
            }
            float e[kVecRows];
            *reinterpret_cast<float4*>(&e[0]) = *reinterpret_cast<const float4*>(&ps[warp][k][0]);
            *reinterpret_cast<float4*>(&e[4]) = *reinterpret_cast<const float4*>(&ps[warp][k][4]);
#pragma unroll
            for (int r = 0; r < kVecRows; ++r)
#pragma unroll
                for (int d = 0; d < DV; ++d)
                    // an unseen row may hold anything: 0 * inf must not reach o
                    if (!mixed || e[r] != 0.f) o[r][d] = fmaf(e[r], v[d], o[r][d]);
        }
        __syncwarp();
    }
    // join the warps
#pragma unroll
    for (int r = 0; r < kVecRows; ++r) {
        const float lt = warp_sum(l[r]);
        if (lane == 0) {
            wm[warp][r] = m[r];
            wl[warp][r] = lt;
        }
#pragma unroll
        for (int d = 0; d < DV; ++d) os[warp][r][lane * DV + d] = o[r][d];
    }
    __syncthreads();
    for (int i = tid; i < kVecRows * HD; i += kVecThreads) {
        const int rr = i / HD, d = i % HD;
        const uint32_t r = r0 + rr;
        if (r >= p.R) continue;
        float M = -INFINITY;
#pragma unroll
        for (int w = 0; w < kVecWarps; ++w) M = fmaxf(M, wm[w][rr]);
        const float ref = M == -INFINITY ? 0.f : M;
        float L = 0.f, O = 0.f;
#pragma unroll
        for (int w = 0; w < kVecWarps; ++w) {
            const float f = exp2f(wm[w][rr] - ref);
            L = fmaf(f, wl[w][rr], L);
            O = fmaf(f, os[w][rr][d], O);
        }
        const size_t row = (size_t)g * p.R + r;
        if (p.n_split > 1) {
            const size_t slot = (size_t)split * a.n_kv * p.R + row;
            p.part_o[slot * HD + d] = O;
            if (d == 0) p.part_ml[slot] = make_float2(M, L);
        } else {
            const float inv = L > 0.f ? 1.f / L : (L == 0.f ? 0.f : L);
            a.out[(size_t)(r / p.G) * a.out_stride + ((size_t)g * p.G + r % p.G) * HD + d] = O * inv;
            if (d == 0 && p.scores) p.stats[row] = make_float2(ref, inv);
        }
    }
}

// Join the splits' partials: one warp per (KV head, row).
template <int HD>
__global__ void __launch_bounds__(128) smallm_tree_merge_kernel(const TreeParams p) {
    constexpr int DV = HD / 32;
    const TreeArgs& a = p.a;
    const int lane = threadIdx.x & 31;
    const size_t rows = (size_t)a.n_kv * p.R, row = (size_t)blockIdx.x * 4 + (threadIdx.x >> 5);
    if (row >= rows) return;
    float M = -INFINITY;
    for (uint32_t s = lane; s < p.n_split; s += 32) M = fmaxf(M, p.part_ml[s * rows + row].x);
    M = warp_max(M);
    const float ref = M == -INFINITY ? 0.f : M;
    float L = 0.f, O[DV];
#pragma unroll
    for (int d = 0; d < DV; ++d) O[d] = 0.f;
#pragma unroll 4
    for (uint32_t s = 0; s < p.n_split; ++s) {
        const float2 ml = p.part_ml[s * rows + row];
        const float f = exp2f(ml.x - ref);
        L = fmaf(f, ml.y, L);
#pragma unroll
        for (int d = 0; d < DV; ++d) O[d] = fmaf(f, p.part_o[(s * rows + row) * HD + lane + 32 * d], O[d]);
    }
    const float inv = L > 0.f ? 1.f / L : (L == 0.f ? 0.f : L);
    const uint32_t g = (uint32_t)(row / p.R), r = (uint32_t)(row % p.R);
    float* o = a.out + (size_t)(r / p.G) * a.out_stride + ((size_t)g * p.G + r % p.G) * HD;
#pragma unroll
    for (int d = 0; d < DV; ++d) o[lane + 32 * d] = O[d] * inv;
    if (lane == 0 && p.scores) p.stats[row] = make_float2(ref, inv);
}

// weights[g][k] += sum_r 2^(s c - mc_r) / sum_r, one thread per (KV head, key):
// rows in order, so the total does not depend on the launch.
__global__ void __launch_bounds__(256) smallm_tree_weights_kernel(const TreeParams p) {
    const uint32_t key = blockIdx.x * 256 + threadIdx.x, g = blockIdx.y;
    if (key >= p.n) return;
    float acc = 0.f;
    const float* s = p.scores + (size_t)g * p.R * p.sc_stride + key;
#pragma unroll 4
    for (uint32_t r = 0; r < p.R; ++r) {
        const float2 st = p.stats[(size_t)g * p.R + r];
        acc = fmaf(exp2f(fmaf(s[(size_t)r * p.sc_stride], p.c, -st.x)), st.y, acc);
    }
    p.a.weights[(size_t)g * p.a.max_ctx + key] += acc;
}

size_t align256(size_t x) { return (x + 255) & ~(size_t)255; }

// Split of the keys and the workspace's layout, from sizes alone.
struct TreePlan {
    uint32_t n_split, tiles_per_split, sc_stride;
    size_t off_ml, off_scores, off_stats, bytes;
};

TreePlan tree_plan(uint32_t n_heads, uint32_t n_kv, uint32_t hd, uint32_t n_past, uint32_t n_tokens, bool weights) {
    TreePlan t{};
    const uint32_t R = n_tokens * (n_heads / n_kv), n = n_past + n_tokens;
    const uint32_t blocks = n_kv * ((R + kVecRows - 1) / kVecRows), tiles = (n + kTile - 1) / kTile;
    // two CTAs per SM in all; no split below a tile for each warp of a CTA
    const uint32_t want = std::max(1u, 2 * (uint32_t)device_sm_count() / blocks);
    const uint32_t most = (tiles + kVecWarps - 1) / kVecWarps;
    t.n_split = std::min(want, most);
    t.tiles_per_split = (tiles + t.n_split - 1) / t.n_split;
    t.n_split = (tiles + t.tiles_per_split - 1) / t.tiles_per_split;
    const size_t rows = (size_t)n_kv * R;
    size_t at = t.n_split > 1 ? align256(4 * rows * t.n_split * hd) : 0;
    t.off_ml = at;
    if (t.n_split > 1) at += align256(8 * rows * t.n_split);
    t.off_scores = at;
    t.sc_stride = (n + 31) / 32 * 32;
    if (weights) at += align256(4 * rows * t.sc_stride);
    t.off_stats = at;
    if (weights) at += align256(8 * rows);
    t.bytes = at;
    return t;
}

void tree_check_shape(uint32_t n_heads, uint32_t n_kv, uint32_t hd, uint32_t n_past, uint32_t n_tokens) {
    if (!n_heads || !n_kv || n_heads % n_kv)
        throw Error(SMALLM_ERR_INVALID, "attention_tree: n_heads must be a positive multiple of n_kv_heads");
    if (n_heads / n_kv > kTreeMaxGroup || n_kv > kTreeMaxKv)
        throw Error(SMALLM_ERR_RANGE, "attention_tree: at most 64 query heads per KV head and 1024 KV heads");
    if (hd != 32 && hd != 64 && hd != 128)
        throw Error(SMALLM_ERR_INVALID, "attention_tree: head_dim must be 32, 64 or 128");
    if (n_tokens > kTreeMaxTokens) throw Error(SMALLM_ERR_RANGE, "attention_tree: at most 1024 drafted tokens");
    if ((uint64_t)n_past + n_tokens > kTreeMaxKeys)
        throw Error(SMALLM_ERR_RANGE, "attention_tree: at most 2^30 cache rows");
}

template <int HD>
void launch_tree(const TreeParams& p, cudaStream_t stream) {
    const dim3 grid(p.n_split, p.a.n_kv, (p.R + kVecRows - 1) / kVecRows);
    smallm_tree_vec_kernel<HD><<<grid, kVecThreads, 0, stream>>>(p);
    SM_CUDA(cudaGetLastError());
    if (p.n_split > 1) {
        smallm_tree_merge_kernel<HD><<<(uint32_t)(((size_t)p.a.n_kv * p.R + 3) / 4), 128, 0, stream>>>(p);
        SM_CUDA(cudaGetLastError());
    }
    if (p.a.weights) {
        smallm_tree_weights_kernel<<<dim3((p.n + 255) / 256, p.a.n_kv), 256, 0, stream>>>(p);
        SM_CUDA(cudaGetLastError());
    }
}

}  // namespace

size_t tree_workspace_bytes(uint32_t n_heads, uint32_t n_kv, uint32_t hd, uint32_t n_past, uint32_t n_tokens,
                            bool weights) {
    tree_check_shape(n_heads, n_kv, hd, n_past, n_tokens);
    return n_tokens ? tree_plan(n_heads, n_kv, hd, n_past, n_tokens, weights).bytes : 0;
}

void launch_attention_tree(const TreeArgs& a, void* work, size_t work_bytes, cudaStream_t stream) {
    tree_check_shape(a.n_heads, a.n_kv, a.hd, a.n_past, a.n_tokens);
    if ((uint64_t)a.n_past + a.n_tokens > a.max_ctx)
        throw Error(SMALLM_ERR_RANGE, "attention_tree: n_past + n_tokens must not pass max_ctx");
    if (!a.n_tokens) return;
    const uint32_t row = a.n_heads * a.hd;
    if (a.q_stride < row || a.out_stride < row || a.q_stride % 4 || a.out_stride % 4)
        throw Error(SMALLM_ERR_INVALID,
                    "attention_tree: q_stride and out_stride must be multiples of 4 of at least n_heads * head_dim");
    if ((reinterpret_cast<uintptr_t>(a.q) | reinterpret_cast<uintptr_t>(a.kcache) |
         reinterpret_cast<uintptr_t>(a.vcache) | reinterpret_cast<uintptr_t>(a.out)) & 15u)
        throw Error(SMALLM_ERR_INVALID, "attention_tree: q, kcache, vcache and out must be 16-byte aligned");
    if ((reinterpret_cast<uintptr_t>(a.mask) | reinterpret_cast<uintptr_t>(a.weights)) & 3u)
        throw Error(SMALLM_ERR_INVALID, "attention_tree: mask and weights must be 4-byte aligned");
    const TreePlan t = tree_plan(a.n_heads, a.n_kv, a.hd, a.n_past, a.n_tokens, a.weights != nullptr);
    if (t.bytes > work_bytes || (t.bytes && !work))
        throw Error(SMALLM_ERR_INVALID, "attention_tree: this call needs a workspace of " + std::to_string(t.bytes) +
                                            " bytes");
    if (t.bytes && (reinterpret_cast<uintptr_t>(work) & 15u))
        throw Error(SMALLM_ERR_INVALID, "attention_tree: the workspace must be 16-byte aligned");
    TreeParams p{};
    p.a = a;
    p.G = a.n_heads / a.n_kv;
    p.R = a.n_tokens * p.G;
    p.n = a.n_past + a.n_tokens;
    p.words = (a.n_tokens + 31) / 32;
    p.n_split = t.n_split;
    p.tiles_per_split = t.tiles_per_split;
    p.sc_stride = t.sc_stride;
    p.c = (float)(1.4426950408889634 / sqrt((double)a.hd));
    uint8_t* w = static_cast<uint8_t*>(work);
    p.part_o = reinterpret_cast<float*>(w);
    p.part_ml = reinterpret_cast<float2*>(w + t.off_ml);
    p.scores = a.weights ? reinterpret_cast<float*>(w + t.off_scores) : nullptr;
    p.stats = a.weights ? reinterpret_cast<float2*>(w + t.off_stats) : nullptr;
    if (a.hd == 32) launch_tree<32>(p, stream);
    else if (a.hd == 64) launch_tree<64>(p, stream);
    else launch_tree<128>(p, stream);
}

}  // namespace smallm
