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
#include "tcgen05.cuh"

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
    unsigned int* err;   // the device error word
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

// ---- tensor-core path --------------------------------------------------------
//
// From about a dozen rows the vector path is bound by its FMAs (R / 2 flop per
// byte of K and V), so blocks of 128 rows go to tcgen05, one CTA per SM, tiles
// of 64 keys.  f32 operands enter as two f16 halves, x 2^e = hi + lo with |lo|
// at most half a unit of hi: 22 bits, and three products (hi hi + hi lo +
// lo hi) leave out 2^-24 of the operands' size.  e brings the largest
// magnitude of the tile (K, V) or row (q) to [2^14, 2^15), so an element loses
// bits only below 2^-39 of that.  The small products are accumulated first.
//   - warps 12..19 convert: 256 threads hold the next K and V tile in
//     registers (64 KB in flight), find the tile's exponent and write hi and
//     lo in the MMA's swizzled layout, three slots for each of K and V;
//   - warp 20, one lane, issues S = Q K^T (Q in tensor memory) and, a tile
//     behind, O = P V (P in tensor memory, V MN-major);
//   - warps 0..3, lane = row: running maximum (a whole number in base 2, so
//     rescaling is exact), P = 2^(s - m + 14) as hi and lo, sum;
//   - warps 4..11, lane = row: O of each tile leaves tensor memory and is added
//     to f32 registers with the tile's exponent and the row's rescaling, which
//     keeps the long sum in rounded f32 adds.
// An infinity or NaN of K or V would reach every row through 0 * inf, so it is
// replaced by 0 and its key marked; rows that see the key turn to NaN.
// Every wait is bounded; one that gives up raises bit 8 of the error word.
constexpr uint32_t kTcRows = 128, kTcKeys = 64, kTcSlots = 3, kTcRing = 8, kTcCorr = 4;
// six warpgroups; registers per thread 80 at launch (480 over the six), then
// 104 softmax + 2 x 88 output + 2 x 88 converters + 24 issuer = 480
constexpr uint32_t kTcThreads = 32 * 24;
constexpr unsigned kErrTreeWait = 256u;
constexpr float kPShift = 14.f;

template <int HD>
struct TcTree {
    static constexpr uint32_t chunks = HD < 64 ? 1 : HD / 64;   // 128-byte columns of a tile
    static constexpr uint32_t half = chunks * kTcKeys * 128;    // bytes of a tile's hi or lo
    static constexpr uint32_t slot = 2 * half;
    static constexpr size_t smem = 1024 + 2ull * kTcSlots * slot + 8192;
    static constexpr uint32_t pv_n = HD < 64 ? 64 : HD;         // columns past HD are never read
    // tensor-memory columns
    static constexpr uint32_t q_hi = 0, q_lo = 64, s0 = 128, p0 = 256, o = 384;
    static constexpr uint32_t idesc_s = (1u << 4) | ((kTcKeys >> 3) << 17) | ((kTcRows >> 4) << 24);
    static constexpr uint32_t idesc_pv = (1u << 4) | (1u << 16) | ((pv_n >> 3) << 17) | ((kTcRows >> 4) << 24);
};

struct TcShared {
    uint64_t k_full[kTcSlots], k_empty[kTcSlots], v_full[kTcSlots], v_empty[kTcSlots];
    uint64_t s_full[2], s_empty[2], p_full[2], p_empty[2], o_full, o_empty, q_full, ml_full, done;
    float k_scale[kTcRing], v_scale[kTcRing];
    unsigned long long bad[kTcRing];
    uint32_t wmax[3][8];
    uint32_t tmem;
    float corr[kTcCorr][kTcRows];
    float2 ml[kTcRows];
};
static_assert(sizeof(TcShared) <= 8192, "shared-memory tail");

// 2^(14 - floor(log2 max)) of a magnitude given as f32 bits, and its inverse.
__device__ __forceinline__ void tc_scale(uint32_t max_bits, float& mult, float& inv) {
    const uint32_t e = max_bits >> 23, f = min(268u - e, 253u);
    mult = __uint_as_float(f << 23);
    inv = __uint_as_float((254u - f) << 23);
}
__device__ __forceinline__ void split_f16(float a, float b, uint32_t& hi, uint32_t& lo) {
    const __half2 h = __floats2half2_rn(a, b);
    const float2 f = __half22float2(h);
    const __half2 l = __floats2half2_rn(a - f.x, b - f.y);
    hi = *reinterpret_cast<const uint32_t*>(&h);
    lo = *reinterpret_cast<const uint32_t*>(&l);
}
// Barrier of the 256 converter threads; true where any of them says so.
__device__ __forceinline__ bool conv_any(bool v) {
    uint32_t r;
    asm volatile(
        "{\n .reg .pred p, q;\n setp.ne.u32 p, %1, 0;\n barrier.cta.red.or.pred q, 1, 256, p;\n"
        " selp.u32 %0, 1, 0, q;\n}"
        : "=r"(r)
        : "r"((uint32_t)v)
        : "memory");
    return r != 0;
}
__device__ __forceinline__ float ex2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// One tile's K or V of a converter thread: units of 8 consecutive floats.
template <int HD>
struct TcUnits {
    static constexpr int n = (int)(kTcKeys * (HD / 8) / 256);
    float x[n][8];
    __device__ __forceinline__ void load(const float* base, uint32_t key0, uint32_t n_keys, int tid) {
#pragma unroll
        for (int i = 0; i < n; ++i) {
            const uint32_t u = i * 256 + tid, key = key0 + u / (HD / 8);
            const float4* p = reinterpret_cast<const float4*>(base + (size_t)key * HD + u % (HD / 8) * 8);
            const float4 z = make_float4(0.f, 0.f, 0.f, 0.f);
            *reinterpret_cast<float4*>(&x[i][0]) = key < n_keys ? __ldg(p) : z;
            *reinterpret_cast<float4*>(&x[i][4]) = key < n_keys ? __ldg(p + 1) : z;
        }
    }
    __device__ __forceinline__ uint32_t max_bits() const {
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < n; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) m = max(m, __float_as_uint(x[i][j]) & 0x7FFFFFFFu);
        return m;
    }
    // Infinities and NaN become 0 and mark their key.
    __device__ __forceinline__ void clean(unsigned long long* bad, int tid) {
#pragma unroll
        for (int i = 0; i < n; ++i) {
            bool any = false;
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if ((__float_as_uint(x[i][j]) & 0x7FFFFFFFu) >= 0x7F800000u) {
                    x[i][j] = 0.f;
                    any = true;
                }
            if (any) atomicOr(bad, 1ull << ((i * 256 + tid) / (HD / 8)));
        }
    }
    __device__ __forceinline__ void store(uint8_t* slot, float mult, int tid) const {
#pragma unroll
        for (int i = 0; i < n; ++i) {
            const uint32_t u = i * 256 + tid, row = u / (HD / 8), c8 = u % (HD / 8);
            uint8_t* dst = slot + (c8 >> 3) * (kTcKeys * 128) + row * 128 + (((c8 & 7) ^ (row & 7)) << 4);
            uint4 hi, lo;
            split_f16(x[i][0] * mult, x[i][1] * mult, hi.x, lo.x);
            split_f16(x[i][2] * mult, x[i][3] * mult, hi.y, lo.y);
            split_f16(x[i][4] * mult, x[i][5] * mult, hi.z, lo.z);
            split_f16(x[i][6] * mult, x[i][7] * mult, hi.w, lo.w);
            *reinterpret_cast<uint4*>(dst) = hi;
            *reinterpret_cast<uint4*>(dst + TcTree<HD>::half) = lo;
        }
    }
};

// Bits of the 64 keys from key0 that row token t sees.
__device__ __forceinline__ unsigned long long tc_seen(const TreeParams& p, uint32_t t, uint32_t key0) {
    unsigned long long m = 0;
    const int64_t u0 = (int64_t)key0 - p.a.n_past;  // drafted index of the tile's first key
    if (u0 < 0) m = u0 <= -64 ? ~0ull : (1ull << -u0) - 1;
    for (int w = 0; w < 3; ++w) {  // mask words that overlap [u0, u0 + 64)
        const int64_t word = (u0 < 0 ? 0 : u0 >> 5) + w, at = word * 32 - u0;
        if (word >= p.words || at >= 64) break;
        uint32_t bits;
        if (p.a.mask) bits = p.a.mask[(size_t)t * p.words + word];
        else bits = t >= word * 32 + 31 ? ~0u : (t < word * 32 ? 0u : (2u << (t & 31)) - 1u);
        if (word == p.words - 1 && p.a.n_tokens % 32) bits &= (1u << (p.a.n_tokens % 32)) - 1u;
        m |= at >= 0 ? (unsigned long long)bits << at : (unsigned long long)(bits >> -at);
    }
    return m;
}

template <int HD>
__global__ void __launch_bounds__(kTcThreads, 1) smallm_tree_tc_kernel(const TreeParams p) {
    using C = TcTree<HD>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    uint8_t* ks = smem;
    uint8_t* vs = smem + kTcSlots * C::slot;
    TcShared& sh = *reinterpret_cast<TcShared*>(vs + kTcSlots * C::slot);
    const TreeArgs& a = p.a;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t r0 = blockIdx.x * kTcRows, split = blockIdx.y, g = blockIdx.z;
    const uint32_t tiles = (p.n + kTcKeys - 1) / kTcKeys;
    const uint32_t t0 = split * p.tiles_per_split, nt = min(tiles, t0 + p.tiles_per_split) - t0;

    if (threadIdx.x == 0) {
        for (uint32_t i = 0; i < kTcSlots; ++i) {
            mbar_init(&sh.k_full[i], 8);
            mbar_init(&sh.k_empty[i], 1);
            mbar_init(&sh.v_full[i], 8);
            mbar_init(&sh.v_empty[i], 1);
        }
        for (uint32_t b = 0; b < 2; ++b) {
            mbar_init(&sh.s_full[b], 2);   // the MMA's commit and the issuing thread
            mbar_init(&sh.s_empty[b], 4);
            mbar_init(&sh.p_full[b], 4);
            mbar_init(&sh.p_empty[b], 1);
        }
        mbar_init(&sh.o_full, 2);
        mbar_init(&sh.o_empty, 8);
        mbar_init(&sh.q_full, 4);
        mbar_init(&sh.ml_full, 4);
        mbar_init(&sh.done, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 20) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh.tmem)),
                     "r"(512u)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tm = sh.tmem;
    bool ok = true;

    if (warp < 4) {
        // ---- softmax: lane = row
        asm volatile("setmaxnreg.inc.sync.aligned.u32 104;");
        const uint32_t rl = threadIdx.x, r = r0 + rl;
        const uint32_t lanes = tm + ((warp * 32u) << 16);
        const bool valid = r < p.R;
        const uint32_t tok = valid ? r / p.G : 0;
        const float4* q = reinterpret_cast<const float4*>(a.q + (size_t)tok * a.q_stride +
                                                          ((size_t)g * p.G + (valid ? r % p.G : 0)) * HD);
        uint32_t mb = 0;
        for (int i = 0; i < HD / 4; ++i) {
            const float4 x = __ldg(q + i);
            mb = max(max(mb, __float_as_uint(x.x) & 0x7FFFFFFFu), __float_as_uint(x.y) & 0x7FFFFFFFu);
            mb = max(max(mb, __float_as_uint(x.z) & 0x7FFFFFFFu), __float_as_uint(x.w) & 0x7FFFFFFFu);
        }
        float mult, qinv;
        tc_scale(mb, mult, qinv);
        if (!valid) mult = 0.f;
#pragma unroll 1
        for (int i = 0; i < HD / 16; ++i) {
            uint32_t hi[8], lo[8];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float4 x = valid ? __ldg(q + 4 * i + j) : make_float4(0.f, 0.f, 0.f, 0.f);
                split_f16(x.x * mult, x.y * mult, hi[2 * j], lo[2 * j]);
                split_f16(x.z * mult, x.w * mult, hi[2 * j + 1], lo[2 * j + 1]);
            }
            tmem_st8(lanes + C::q_hi + 8 * i, hi);
            tmem_st8(lanes + C::q_lo + 8 * i, lo);
        }
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.q_full);
        float m = -INFINITY, l = 0.f;
        float* sc = p.scores && valid ? p.scores + ((size_t)g * p.R + r) * p.sc_stride : nullptr;
        for (uint32_t t = 0; t < nt; ++t) {
            const uint32_t b = t & 1, use = t >> 1, key0 = (t0 + t) * kTcKeys, ring = t % kTcRing;
            ok = mbar_wait(&sh.s_full[b], use & 1);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            tc_fence_after();
            float s[kTcKeys];
            {
                uint32_t x[32];
                tmem_ld32(lanes + C::s0 + b * kTcKeys, x);
#pragma unroll
                for (int i = 0; i < 32; ++i) s[i] = __uint_as_float(x[i]);
                tmem_ld32(lanes + C::s0 + b * kTcKeys + 32, x);
#pragma unroll
                for (int i = 0; i < 32; ++i) s[32 + i] = __uint_as_float(x[i]);
            }
            // (never 0: an unseen key's -inf times it stays -inf)
            const float raw = fmaxf(qinv * sh.k_scale[ring], 0x1p-120f);
            const unsigned long long bad = sh.bad[ring];
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.s_empty[b]);
            unsigned long long seen = ~0ull;
            if (key0 + kTcKeys > a.n_past) {
                seen = tc_seen(p, tok, key0);
#pragma unroll
                for (int i = 0; i < (int)kTcKeys; ++i)
                    if (!((seen >> i) & 1)) s[i] = -INFINITY;
            }
            if (bad & seen) {
#pragma unroll
                for (int i = 0; i < (int)kTcKeys; ++i)
                    if ((bad & seen) >> i & 1) s[i] = __uint_as_float(0x7FC00000u);
            }
            if (sc) {
#pragma unroll
                for (int i = 0; i < (int)kTcKeys; i += 4)
                    *reinterpret_cast<float4*>(sc + key0 + i) =
                        make_float4(s[i] * raw, s[i + 1] * raw, s[i + 2] * raw, s[i + 3] * raw);
            }
            float mx = s[0];
#pragma unroll
            for (int i = 1; i < (int)kTcKeys; ++i) mx = fmaxf(mx, s[i]);
            const float ct = raw * p.c;
            const float mn = fmaxf(m, mx == -INFINITY ? -INFINITY : ceilf(mx * ct));
            const float ref = mn == -INFINITY ? 0.f : mn;
            const float corr = ex2_approx(m - ref);
            sh.corr[t % kTcCorr][rl] = corr;
            m = mn;
            // P's buffer is free once the product two tiles back has read it
            if (t >= 2) {
                ok = mbar_wait(&sh.p_empty[b], (use - 1) & 1);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                tc_fence_after();
            }
            const float off = kPShift - ref;
            float sum = 0.f;
#pragma unroll
            for (int i = 0; i < (int)kTcKeys; i += 16) {
                uint32_t hi[8], lo[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float x = ex2_approx(fmaf(s[i + 2 * j], ct, off));
                    const float y = ex2_approx(fmaf(s[i + 2 * j + 1], ct, off));
                    sum += x + y;
                    split_f16(x, y, hi[j], lo[j]);
                }
                tmem_st8(lanes + C::p0 + b * 64 + i / 2, hi);
                tmem_st8(lanes + C::p0 + b * 64 + 32 + i / 2, lo);
            }
            l = fmaf(l, corr, sum);
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.p_full[b]);
        }
        sh.ml[rl] = make_float2(m, l * 0x1p-14f);
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.ml_full);
    } else if (warp < 12) {
        // ---- output: lane = row, warps 4..7 the first half of the columns, 8..11 the second
        asm volatile("setmaxnreg.inc.sync.aligned.u32 88;");
        constexpr int OC = HD / 2;
        float o[OC];
#pragma unroll
        for (int i = 0; i < OC; ++i) o[i] = 0.f;
        const uint32_t rl = (warp & 3) * 32 + lane, r = r0 + rl, col = warp < 8 ? 0 : OC;
        const uint32_t src = tm + (((warp & 3) * 32u) << 16) + C::o + col;
        for (uint32_t t = 0; t < nt; ++t) {
            ok = mbar_wait(&sh.o_full, t & 1);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            tc_fence_after();
            const float corr = sh.corr[t % kTcCorr][rl], scale = sh.v_scale[t % kTcRing] * 0x1p-14f;
#pragma unroll
            for (int c = 0; c < OC; c += 16) {
                uint32_t x[16];
                tmem_ld16(src + c, x);
#pragma unroll
                for (int i = 0; i < 16; ++i) o[c + i] = fmaf(__uint_as_float(x[i]), scale, o[c + i] * corr);
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.o_empty);
        }
        ok = mbar_wait(&sh.ml_full, 0) && ok;
        if (r < p.R) {
            const float2 ml = sh.ml[rl];
            const size_t row = (size_t)g * p.R + r;
            float* dst;
            float f = 1.f;
            if (p.n_split > 1) {
                const size_t slot = (size_t)split * a.n_kv * p.R + row;
                dst = p.part_o + slot * HD + col;
                if (col == 0) p.part_ml[slot] = ml;
            } else {
                f = ml.y > 0.f ? 1.f / ml.y : (ml.y == 0.f ? 0.f : ml.y);
                dst = a.out + (size_t)(r / p.G) * a.out_stride + ((size_t)g * p.G + r % p.G) * HD + col;
                if (col == 0 && p.scores) p.stats[row] = make_float2(ml.x == -INFINITY ? 0.f : ml.x, f);
            }
#pragma unroll
            for (int i = 0; i < OC; i += 4)
                *reinterpret_cast<float4*>(dst + i) =
                    make_float4(o[i] * f, o[i + 1] * f, o[i + 2] * f, o[i + 3] * f);
        }
    } else if (warp < 20) {
        // ---- converters
        asm volatile("setmaxnreg.inc.sync.aligned.u32 88;");
        const int tid = (int)threadIdx.x - 384;
        const uint32_t cw = warp - 12;
        const float* kb = a.kcache + (size_t)g * a.max_ctx * HD;
        const float* vb = a.vcache + (size_t)g * a.max_ctx * HD;
        TcUnits<HD> ku, vu;
        vu.load(vb, t0 * kTcKeys, p.n, tid);
        ku.load(kb, t0 * kTcKeys, p.n, tid);
        auto convert = [&](TcUnits<HD>& u, uint32_t t, int which, uint8_t* slots, uint64_t* full, uint64_t* empty,
                           float* scales) -> bool {
            const uint32_t slot = t % kTcSlots, use = t / kTcSlots, ring = t % kTcRing;
            const uint32_t mw = __reduce_max_sync(0xffffffffu, u.max_bits());
            if (lane == 0) sh.wmax[which][cw] = mw;
            if (which == 0 && tid == 0) sh.bad[ring] = 0;
            const bool stuck = use > 0 && !mbar_wait(&empty[slot], (use - 1) & 1);
            if (conv_any(stuck)) return false;
            uint32_t mx = 0;
#pragma unroll
            for (int w = 0; w < 8; ++w) mx = max(mx, sh.wmax[which][w]);
            if (mx >= 0x7F800000u) {  // the same for all 256 threads
                u.clean(&sh.bad[ring], tid);
                const uint32_t m2 = __reduce_max_sync(0xffffffffu, u.max_bits());
                if (lane == 0) sh.wmax[2][cw] = m2;
                conv_any(false);
                mx = 0;
#pragma unroll
                for (int w = 0; w < 8; ++w) mx = max(mx, sh.wmax[2][w]);
                conv_any(false);
            }
            float mult, inv;
            tc_scale(mx, mult, inv);
            u.store(slots + slot * C::slot, mult, tid);
            if (tid == 0) scales[ring] = inv;
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(&full[slot]);
            return true;
        };
        for (uint32_t t = 0; t < nt; ++t) {
            // V first: K's arrival then covers the marks of both
            ok = convert(vu, t, 0, vs, sh.v_full, sh.v_empty, sh.v_scale);
            if (!ok) break;
            if (t + 1 < nt) vu.load(vb, (t0 + t + 1) * kTcKeys, p.n, tid);
            ok = convert(ku, t, 1, ks, sh.k_full, sh.k_empty, sh.k_scale);
            if (!ok) break;
            if (t + 1 < nt) ku.load(kb, (t0 + t + 1) * kTcKeys, p.n, tid);
        }
    } else {
      asm volatile("setmaxnreg.dec.sync.aligned.u32 24;");
      if (warp == 20 && lane == 0) {
        // ---- MMA issuer
        ok = mbar_wait(&sh.q_full, 0);
        tc_fence_after();
        auto scores = [&](uint32_t t) -> bool {
            const uint32_t slot = t % kTcSlots, b = t & 1;
            if (!mbar_wait(&sh.k_full[slot], (t / kTcSlots) & 1)) return false;
            if (t >= 2 && !mbar_wait(&sh.s_empty[b], ((t >> 1) - 1) & 1)) return false;
            tc_fence_after();
            const uint8_t* hi = ks + slot * C::slot;
            const uint32_t d = tm + C::s0 + b * kTcKeys;
#pragma unroll
            for (int x = 0; x < 3; ++x) {  // lo hi, hi lo, hi hi
#pragma unroll
                for (int j = 0; j < HD / 16; ++j)
                    mma_f16_ta(d, tm + (x == 0 ? C::q_lo : C::q_hi) + 8 * j,
                               smem_desc_sw128(hi + (x == 1 ? C::half : 0) + (j >> 2) * (kTcKeys * 128)) + 2 * (j & 3),
                               C::idesc_s, (x | j) != 0);
            }
            mma_commit(&sh.k_empty[slot]);
            mma_commit(&sh.s_full[b]);
            mbar_arrive(&sh.s_full[b]);
            return true;
        };
        ok = ok && scores(0);
        for (uint32_t t = 0; ok && t < nt; ++t) {
            if (t + 1 < nt && !scores(t + 1)) {
                ok = false;
                break;
            }
            const uint32_t slot = t % kTcSlots, b = t & 1;
            ok = mbar_wait(&sh.v_full[slot], (t / kTcSlots) & 1) && mbar_wait(&sh.p_full[b], (t >> 1) & 1) &&
                 (t == 0 || mbar_wait(&sh.o_empty, (t - 1) & 1));
            if (!ok) break;
            tc_fence_after();
            const uint8_t* hi = vs + slot * C::slot;
            const uint32_t pa = tm + C::p0 + b * 64;
#pragma unroll
            for (int x = 0; x < 3; ++x) {
#pragma unroll
                for (int j = 0; j < (int)kTcKeys / 16; ++j)
                    mma_f16_ta(tm + C::o, pa + (x == 0 ? 32 : 0) + 8 * j,
                               smem_desc_sw128_mn(hi + (x == 1 ? C::half : 0) + j * 2048, kTcKeys * 128), C::idesc_pv,
                               (x | j) != 0);
            }
            mma_commit(&sh.v_empty[slot]);
            mma_commit(&sh.p_empty[b]);
            mma_commit(&sh.o_full);
            mbar_arrive(&sh.o_full);
        }
        // tensor memory is freed only after every MMA has completed
        mma_commit(&sh.done);
        ok = mbar_wait(&sh.done, 0) && ok;
      }
    }
    if (!ok) atomicOr(p.err, kErrTreeWait);
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (warp == 20) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tm), "r"(512u) : "memory");
    }
}

// ---- joining -------------------------------------------------------------------

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

#ifndef SMALLM_TREE_TC_ROWS
#define SMALLM_TREE_TC_ROWS 9u
#endif

size_t align256(size_t x) { return (x + 255) & ~(size_t)255; }

// Split of the keys and the workspace's layout, from sizes alone.
struct TreePlan {
    bool tc;
    uint32_t n_split, tiles_per_split, sc_stride;
    size_t off_ml, off_scores, off_stats, bytes;
};

TreePlan tree_plan(uint32_t n_heads, uint32_t n_kv, uint32_t hd, uint32_t n_past, uint32_t n_tokens, bool weights) {
    TreePlan t{};
    const uint32_t R = n_tokens * (n_heads / n_kv), n = n_past + n_tokens;
    t.tc = R >= SMALLM_TREE_TC_ROWS;
    const uint32_t keys = t.tc ? kTcKeys : kTile, rows_cta = t.tc ? kTcRows : kVecRows;
    const uint32_t blocks = n_kv * ((R + rows_cta - 1) / rows_cta), tiles = (n + keys - 1) / keys;
    // one CTA per SM in all on the tensor path, else two; no split below a
    // tile for each warp of a vector CTA
    const uint32_t want = std::max(1u, (t.tc ? 1 : 2) * (uint32_t)device_sm_count() / blocks);
    const uint32_t most = t.tc ? tiles : (tiles + kVecWarps - 1) / kVecWarps;
    t.n_split = std::min(want, most);
    t.tiles_per_split = (tiles + t.n_split - 1) / t.n_split;
    t.n_split = (tiles + t.tiles_per_split - 1) / t.tiles_per_split;
    const size_t rows = (size_t)n_kv * R;
    size_t at = t.n_split > 1 ? align256(4 * rows * t.n_split * hd) : 0;
    t.off_ml = at;
    if (t.n_split > 1) at += align256(8 * rows * t.n_split);
    t.off_scores = at;
    t.sc_stride = (n + 63) / 64 * 64;
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
void launch_tree(const TreeParams& p, bool tc, cudaStream_t stream) {
    if (tc) {
        set_smem_limit_once((const void*)smallm_tree_tc_kernel<HD>, (int)TcTree<HD>::smem);
        const dim3 grid((p.R + kTcRows - 1) / kTcRows, p.n_split, p.a.n_kv);
        smallm_tree_tc_kernel<HD><<<grid, kTcThreads, TcTree<HD>::smem, stream>>>(p);
    } else {
        const dim3 grid(p.n_split, p.a.n_kv, (p.R + kVecRows - 1) / kVecRows);
        smallm_tree_vec_kernel<HD><<<grid, kVecThreads, 0, stream>>>(p);
    }
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
    p.err = device_error_flag();
    uint8_t* w = static_cast<uint8_t*>(work);
    p.part_o = reinterpret_cast<float*>(w);
    p.part_ml = reinterpret_cast<float2*>(w + t.off_ml);
    p.scores = a.weights ? reinterpret_cast<float*>(w + t.off_scores) : nullptr;
    p.stats = a.weights ? reinterpret_cast<float2*>(w + t.off_stats) : nullptr;
    if (a.hd == 32) launch_tree<32>(p, t.tc, stream);
    else if (a.hd == 64) launch_tree<64>(p, t.tc, stream);
    else launch_tree<128>(p, t.tc, stream);
}

}  // namespace smallm
