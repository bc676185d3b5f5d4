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
// fma rounding, mc the running maximum times c.  The totals need the whole
// row's mc and sum, so with them the scores are stored (4 R bytes a key beside
// 8 hd of K and V) and a last kernel sums 2^(s c - mc) / sum over the rows.
// All launches are programmatic dependents: their set-up overlaps what ran
// before (2 to 3 us of a call), and they wait for it before any access.
#include <algorithm>
#include <cfloat>
#include <cmath>
#include <type_traits>

#include "common.cuh"
#include "engine.h"
#include "smallm_cuda.h"
#include "tcgen05.cuh"

namespace smallm {
namespace {

struct TreeParams {
    TreeArgs a;
    uint32_t G, R, n;
    uint32_t n_split, tiles_per_split;
    uint32_t sc_rows;    // stored scores of a key: R, padded; 0: they run along keys
    uint32_t sc_keys;    // ... and of a row: n, padded to tiles
    float c;             // log2(e) / sqrt(hd)
    float o_below;       // outputs are summed as 2^-head of them, so that n values fit: kPShift + head
    float head_up;       // 2^head
    float* part_o;       // [n_split][n_kv * R][hd], 2^-head of the sums
    float2* part_ml;     // [n_split][n_kv * R] (mc, sum)
    float* scores;       // [n_kv][sc_keys / 4][sc_rows][4] or [n_kv][R][sc_keys], raw q . K, -inf where unseen
    float2* stats;       // [n_kv * R] (mc of the whole row, 1 / sum or 0)
    unsigned int* err;   // the device error word
};

// ---- the kernel ----------------------------------------------------------------
//
// R rows need R / 2 flop per byte of K and V, more than the f32 units give from
// a dozen rows on, so blocks of 128 rows go to tcgen05, one CTA per SM, tiles of
// 64 keys.  (With fewer rows it is the copies that bound the kernel, and a form
// in f32 FMAs, two CTAs per SM, was slower for one token of 32 heads at 128:
// 55 us against 36 us over 16384 rows, 12 us against 10 us over 128.)  f32
// operands enter as two f16 halves, x 2^e = hi + lo with |lo| at most half a
// unit of hi: 22 bits, and three products (hi hi + hi lo + lo hi) leave out
// 2^-24 of the operands' size.  e brings the largest magnitude of the tile (K,
// V) or row (q) to [2^14, 2^15), so an element loses bits only below 2^-39 of
// that.  The small products are accumulated first.  (The result is nearer the
// definition in 64 bits than f32 products and sums are: 1.1e-6 of its norm
// against 3.6e-6 for 64 tokens over 32683 rows.)
// One scale for a tile holds while no row of it is 2^14 times smaller than
// another, which leaves every row 2^-25 of its own largest magnitude; else each
// row has a scale of its own, so that no row takes bits from another, seen or
// not: a K row's multiplies its scores, a V row's goes into P, which is then
// relative to the token's largest product p |v| of the tile instead of its
// largest p.  P therefore waits for V's scales (2% of 64 tokens over 32747 rows,
// 5% of one token with totals over 16384; looked at before the exponentials: by
// a wait after them, P in registers meanwhile, it was 13% and 14%).  With such
// rows in every tile 64 tokens take 2.2 times as long.
//   - warps 25 (K) and 26 (V) copy tiles of f32 rows with bulk copies into
//     three slots each (six for rows of 64 or fewer).  (Loads through registers
//     took the load/store unit twice as long as these copies and the reads of
//     them.)
//   - warps 16..19 (K) and 20..23 (V) convert in place: a group takes a tile
//     into registers, finds its exponent (or, by way of the slot again, those of
//     its rows) and, once all have theirs, writes hi and lo in the MMA's
//     swizzled layout over it.  (Slots of their own behind
//     one tile of raw rows, for eight warps each: 3% slower at 64 tokens.)
//   - warp 24 issues S = Q K^T (Q in tensor memory) and, a tile behind,
//     O = P V (P in tensor memory, over S's columns; V MN-major);
//   - warps 0..7, lane = row, two warps for a row: each takes half of the keys
//     for the running maximum (a whole number in base 2, so rescaling is
//     exact; the halves meet in shared memory), P = 2^(s - mt + 14) as hi and lo,
//     mt the tile's own maximum, and the sum;
//   - warps 8..15, lane = row, take half of the columns of a tile's O each and
//     add it to f32 registers with that tile's exponent and the row's
//     rescaling: the long sum is made of rounded f32 adds.  (By the same warps
//     as the softmax one token over 16384 rows took 2% longer, with totals 6%.)
// One token of 32 heads at 128 reads K and V at 5.9 TB/s from 16384 rows on
// (the slope of its time; copies reach 6.5), after 8 us for two launches, the
// first tile and the join.  Blocks with all 128 rows take about 2800 cycles a
// tile where the products take 1536: conversion works for 2600 of them, softmax
// and the issue of the products for 2000, in 5 instructions of 8 issue slots.
// Measured and not kept: smaller copies in a longer ring, a scale for each
// converter warp instead of each tile, six converter warps (fewer registers) or
// eight, f32 FMAs for few rows, splits that join through a cluster's shared
// memory, the mask read before the wait for the products (spills).
// An infinity or NaN of K or V would reach every row through 0 * inf, so it is
// replaced by 0 and its key marked; rows that see the key turn to NaN.
// Every wait is bounded; one that gives up raises bit 8 of the error word.
constexpr uint32_t kTcRows = 128, kTcKeys = 64, kTcMaxSlots = 6, kTcRing = 8;
// seven warpgroups; registers per thread 72 at launch (504 over the seven), then
// 2 x 72 rows + 2 x 88 output + 2 x 80 converters + 24 issuer = 504
constexpr uint32_t kTcThreads = 32 * 28;
constexpr uint32_t kConvThreads = 128, kConvWarps = kConvThreads / 32;
constexpr float kPShift = 14.f;
constexpr float kTinyShift = 100.f;
constexpr float kLargeScore = 0x1p22f;  // exponents from here on have less than two fractional bits
constexpr float kWideTile = 0x1p-14f;  // a tile's rows get scales of their own where one is this much smaller

template <int HD>
struct TcTree {
    static constexpr uint32_t chunks = HD < 64 ? 1 : HD / 64;   // 128-byte columns of a tile
    static constexpr uint32_t half = chunks * kTcKeys * 128;    // bytes of a tile's hi or lo
    static constexpr uint32_t slot = 2 * half;
    static constexpr uint32_t slots = HD > 64 ? 3 : 6;          // of K and of V each
    static constexpr size_t smem = 1024 + 2ull * slots * slot + 16384;
    static_assert(kTcKeys * HD * 4 <= slot, "a tile is converted in place");
    static_assert(kTcRows * HD * 4 <= 2 * slot, "q and the output pass through two slots");
    static_assert(slots <= kTcMaxSlots && slots + 2 <= kTcRing, "scales outlive their slots by two tiles");
    static constexpr uint32_t pv_n = HD < 64 ? 64 : HD;         // columns past HD are never read
    // tensor-memory columns; P (hi 32, lo 32) takes the place of its S
    static constexpr uint32_t q_hi = 0, q_lo = 64, s0 = 128, o0 = 256;
    static constexpr uint32_t idesc_s = (1u << 4) | ((kTcKeys >> 3) << 17) | ((kTcRows >> 4) << 24);
    static constexpr uint32_t idesc_pv = (1u << 4) | (1u << 16) | ((pv_n >> 3) << 17) | ((kTcRows >> 4) << 24);
};

struct TcShared {
    uint64_t k_full[kTcMaxSlots], k_empty[kTcMaxSlots], v_full[kTcMaxSlots], v_empty[kTcMaxSlots];
    uint64_t v_scaled[kTcMaxSlots], z_full[4];
    uint64_t raw_full[2][kTcMaxSlots];  // [K, V]
    uint64_t s_full[2], p_full[2], o_full[2], o_empty[2], q_full, done;
    float k_scale[kTcRing], v_exp[kTcRing];  // what a tile was divided by; V's as O's exponent
    unsigned long long k_bad[kTcRing], v_bad[kTcRing];
    uint2 wrange[2][2][kConvWarps];  // [K, V][tile % 2][warp] bits of the largest and smallest magnitude
    uint32_t tmem;
    float part_max[2][2][kTcRows];  // [tile % 2][half]
    float part_sum[2][kTcRows];
    uint32_t q_max[kTcRows];
    // [tile % 4] what a tile's maximum leaves of the output before it, and what O is
    // multiplied by; below f32's normal range -2^kTinyShift times that
    float2 corr[4][kTcRows];
    float factor[kTcRows];
    float part_z[2][kTcRows];
    // the rows' own scales, V's as exponents, for tiles with k_scale or v_exp infinite
    alignas(16) float row_scale[2][kTcRing][kTcKeys];
};
static_assert(sizeof(TcShared) <= 16384, "shared-memory tail");

// 2^(14 - floor(log2 max)) of a magnitude given as f32 bits, and its inverse.
__device__ __forceinline__ void tc_scale(uint32_t max_bits, float& mult, float& inv) {
    const uint32_t e = max_bits >> 23, f = min(268u - e, 253u);
    mult = __uint_as_float(f << 23);
    inv = __uint_as_float((254u - f) << 23);
}
// The exponent of an inverse that tc_scale gave: -126 to 114.
__device__ __forceinline__ int scale_exp(float inv) { return (int)(__float_as_uint(inv) >> 23) - 127; }
// hi = x rounded to f16, lo = (x - hi) rounded to f16, of two values (the
// difference as a mixed fma by -1: a mixed subtraction takes the f16 operand
// first, and the two negations after it cost an instruction each).
__device__ __forceinline__ void split_f16(float2 x, uint32_t& hi, uint32_t& lo) {
    asm("{\n .reg .f16 a, b, n;\n .reg .f32 c, d;\n"
        " cvt.rn.f16x2.f32 %0, %3, %2;\n mov.b32 {a, b}, %0;\n mov.b16 n, 0xBC00;\n"
        " fma.rn.f32.f16 c, a, n, %2;\n fma.rn.f32.f16 d, b, n, %3;\n"
        " cvt.rn.f16x2.f32 %1, d, c;\n}"
        : "=&r"(hi), "=r"(lo)
        : "f"(x.x), "f"(x.y));
}
// Barrier of the 128 threads of converter group `id`; true where any says so.
__device__ __forceinline__ bool conv_any(int id, bool v) {
    uint32_t r;
    asm volatile(
        "{\n .reg .pred p, q;\n setp.ne.u32 p, %1, 0;\n barrier.cta.red.or.pred q, %2, 128, p;\n"
        " selp.u32 %0, 1, 0, q;\n}"
        : "=r"(r)
        : "r"((uint32_t)v), "r"(id)
        : "memory");
    return r != 0;
}
__device__ __forceinline__ float ex2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// 2^e of a whole e <= 127; 0 below -126.
__device__ __forceinline__ float exp2_whole(float e) { return __int_as_float(max(__float2int_rn(e) + 127, 0) << 23); }
// The largest of three magnitudes, NaN if any is.
__device__ __forceinline__ float max3_abs_nan(float a, float b, float c) {
    float r;
    asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

__device__ __forceinline__ float max_abs_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(fabsf(b)));
    return r;
}
// 1 / sum of a row with maximum m; 0 where it sees nothing, NaN where its scores
// leave no sum.
__device__ __forceinline__ float row_inverse(float m, float sum) {
    return sum > 0.f ? 1.f / sum : (m == -INFINITY && sum == 0.f ? 0.f : __int_as_float(0x7FC00000));
}
// A row's weights are plain where its maximum is no large score and it has a sum.
__device__ __forceinline__ bool row_plain(float2 stats) {
    return fabsf(stats.x) < kLargeScore && fabsf(stats.y) < INFINITY;
}
// The weight 2^(s c - mc) / sum of a stored score; in other rows the product is
// rounded as the kernel's, and an unseen key has none even where the sum is NaN.
template <bool PLAIN>
__device__ __forceinline__ float add_weight(float acc, float s, float c, float2 stats) {
    const float y = PLAIN ? fmaf(s, c, -stats.x) : __fadd_rn(__fmul_rn(s, c), -stats.x);
    return !PLAIN && s == -INFINITY ? acc : fmaf(exp2f(y), stats.y, acc);
}
// x = f(column, x) over N * 8 f32 columns of this thread's lane of tensor
// memory, in a loop: for paths that are rarely taken and shall not hold
// registers or much code.
template <int N, typename F>
__device__ __forceinline__ void tmem_map8(uint32_t taddr, F f) {
#pragma unroll 1
    for (int c = 0; c < 8 * N; c += 8) {
        uint32_t x[8];
        tmem_ld8(taddr + c, x);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = __float_as_uint(f(c + i, __uint_as_float(x[i])));
        tmem_st8(taddr + c, x);
    }
    tmem_wait_st();
}

// Bits of the 64 keys from key0 that row token t sees.
__device__ __forceinline__ unsigned long long tc_seen(const uint32_t* mask, uint32_t n_past, uint32_t n_tokens,
                                                   uint32_t t, uint32_t key0) {
    const uint32_t words = (n_tokens + 31) / 32;
    unsigned long long m = 0;
    const int64_t u0 = (int64_t)key0 - n_past;  // drafted index of the tile's first key
    if (u0 < 0) m = u0 <= -64 ? ~0ull : (1ull << -u0) - 1;
    for (int w = 0; w < 3; ++w) {  // mask words that overlap [u0, u0 + 64)
        const int64_t word = (u0 < 0 ? 0 : u0 >> 5) + w, at = word * 32 - u0;
        if (word >= words || at >= 64) break;
        uint32_t bits;
        if (mask) bits = mask[(size_t)t * words + word];
        else bits = t >= word * 32 + 31 ? ~0u : (t < word * 32 ? 0u : (2u << (t & 31)) - 1u);
        if (word == words - 1 && n_tokens % 32) bits &= (1u << (n_tokens % 32)) - 1u;
        m |= at >= 0 ? (unsigned long long)bits << at : (unsigned long long)(bits >> -at);
    }
    return m;
}

// One lane: every copy of tiles before `end` has landed.
template <int HD>
__device__ __forceinline__ bool tc_landed(uint32_t end, uint64_t* full) {
    constexpr uint32_t S = TcTree<HD>::slots;
    bool ok = true;
    for (uint32_t t = end - min(end, S); t < end; ++t) ok = mbar_wait_soon(&full[t % S], (t / S) & 1) && ok;
    return ok;
}
// One lane: tiles from .. to - 1 of a CTA's tiles t0 .. (rows of `src` below n)
// into their slots.
template <int HD>
__device__ __forceinline__ bool tc_copy(const float* src, uint32_t n, uint32_t t0, uint32_t from, uint32_t to,
                                        uint8_t* slots, uint64_t* full, uint64_t* empty) {
    using C = TcTree<HD>;
    for (uint32_t t = from; t < to; ++t) {
        const uint32_t s = t % C::slots, row = (t0 + t) * kTcKeys, rows = min(n - row, kTcKeys);
        if (t >= C::slots && !mbar_wait_soon(&empty[s], (t / C::slots - 1) & 1)) {
            tc_landed<HD>(t, full);  // no copy may still be landing when the CTA exits
            return false;
        }
        mbar_arrive_expect_tx(&full[s], rows * HD * 4);
        bulk_g2s(slots + s * C::slot, src + (size_t)row * HD, rows * HD * 4, &full[s]);
    }
    return true;
}

// One converter group: tiles t0 .. t0 + nt - 1, in place.  V's exponents are
// left as O's.
template <int HD, int GROUP>
__device__ __forceinline__ bool tc_convert(const TreeParams& p, uint32_t t0, uint32_t nt, int tid, uint8_t* smem, TcShared& sh) {
    using C = TcTree<HD>;
    constexpr int N = (int)kTcKeys * HD / 4 / kConvThreads;  // float4s of a thread
    constexpr uint32_t W = HD / 4, STEP = kConvThreads / W;  // float4s of a row; rows between two units
    const uint32_t c4 = tid % W, row0 = tid / W;
    uint8_t* slots = smem + GROUP * C::slots * C::slot;
    uint64_t* full = GROUP ? sh.v_full : sh.k_full;
    unsigned long long* bads = GROUP ? sh.v_bad : sh.k_bad;
    auto& wrange = sh.wrange[GROUP];
    float4 x[N];
    // (STEP is a multiple of 4: the swizzle of odd units differs in one bit at most)
    const uint32_t dst0 =
        (c4 >> 4) * (kTcKeys * 128) + (c4 & 1) * 8 + row0 * 128 + ((((c4 & 15) >> 1) ^ (row0 & 7)) << 4);
    constexpr uint32_t FLIP = (STEP & 4) << 4;
    const int lane = tid & 31, cw = tid >> 5;
    for (uint32_t t = 0; t < nt; ++t) {
        const uint32_t slot = t % C::slots, ring = t % kTcRing;
        const uint32_t left = p.n - (t0 + t) * kTcKeys;  // rows from the tile's first to the last
        const bool stuck = !mbar_wait_soon(&sh.raw_full[GROUP][slot], (t / C::slots) & 1);
        const float4* src = reinterpret_cast<const float4*>(slots + slot * C::slot) + tid;
        // the largest magnitude, and the smallest (as bits less 1, so that zeros do not
        // count) of four elements' largest ones: no row of the tile is smaller.  (Of
        // three, ordinary rows beside a channel 1000 times larger are looked at more
        // closely again and again: 10% longer.)
        float m = 0.f;
        uint32_t low = ~0u;
        auto unit_max = [](const float4& v) { return max_abs_nan(max3_abs_nan(v.x, v.y, v.z), v.w); };
        auto below = [](uint32_t least, float v) { return __viaddmin_u32(__float_as_uint(v), ~0u, least); };
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = src[i * kConvThreads];
        if (left < kTcKeys) {
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (row0 + i * STEP >= left) x[i] = make_float4(0.f, 0.f, 0.f, 0.f);
        }
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            const float u = unit_max(x[i]), v = unit_max(x[i + 1]);
            m = max3_abs_nan(m, u, v);
            low = below(below(low, u), v);
        }
        auto put_range = [&](float most, uint32_t least) {
            const uint32_t a = __reduce_max_sync(0xffffffffu, __float_as_uint(most));
            const uint32_t b = __reduce_min_sync(0xffffffffu, least);
            if (lane == 0) wrange[t & 1][cw] = make_uint2(a, b);
        };
        uint32_t mx;
        auto get_range = [&] {  // true: rows may differ too much for one scale
            const uint2 r = wrange[t & 1][lane % kConvWarps];
            mx = __reduce_max_sync(0xffffffffu, r.x);
            return __uint_as_float(__reduce_min_sync(0xffffffffu, r.y)) < __uint_as_float(mx) * kWideTile;
        };
        put_range(m, low);
        if (tid == 0) bads[ring] = 0;
        // (past this barrier every thread has its elements)
        if (conv_any(1 + GROUP, stuck)) return false;
        bool wide = get_range();
        if (wide || mx >= 0x7F800000u) {  // the same for the whole group; by way of the slot, to spare registers
            float4* own = reinterpret_cast<float4*>(slots + slot * C::slot) + tid;
            auto row_max = [&](const float4& v) {
                float r = fmaxf(fmaxf(fabsf(v.x), fabsf(v.y)), fmaxf(fabsf(v.z), fabsf(v.w)));
                if constexpr (W == 32) {
                    return __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(r)));
                } else {
#pragma unroll
                    for (int o = W / 2; o > 0; o >>= 1) r = fmaxf(r, __shfl_xor_sync(0xffffffffu, r, o));
                    return r;
                }
            };
            // whole rows' magnitudes, infinities and NaN cleaned; rows of zeros do not count
            m = 0.f, low = ~0u;
#pragma unroll 4
            for (uint32_t i = 0, row = row0; i < (uint32_t)N; ++i, row += STEP) {
                float4 v = own[i * kConvThreads];
                if (row >= left) v = make_float4(0.f, 0.f, 0.f, 0.f);
                bool hurt = false;
                auto clean = [&](float& e) {
                    if (!(fabsf(e) < INFINITY)) e = 0.f, hurt = true;
                };
                clean(v.x), clean(v.y), clean(v.z), clean(v.w);
                if (hurt) atomicOr(&bads[ring], 1ull << row);
                own[i * kConvThreads] = v;
                const float r = row_max(v);
                m = fmaxf(m, r);
                low = below(low, r);
            }
            conv_any(1 + GROUP, false);  // the ranges have been read by all
            put_range(m, low);
            conv_any(1 + GROUP, false);
            wide = get_range();
            if (wide) {
#pragma unroll 4
                for (uint32_t i = 0, row = row0; i < (uint32_t)N; ++i, row += STEP) {
                    float4 v = own[i * kConvThreads];
                    float mult, inv;
                    tc_scale(__float_as_uint(row_max(v)), mult, inv);
                    own[i * kConvThreads] = make_float4(v.x * mult, v.y * mult, v.z * mult, v.w * mult);
                    if (c4 == 0) sh.row_scale[GROUP][ring][row] = GROUP ? (float)scale_exp(inv) : inv;
                }
            }
#pragma unroll
            for (int i = 0; i < N; ++i) x[i] = src[i * kConvThreads];
            conv_any(1 + GROUP, false);  // as above: every thread has its elements
        }
        float mult, inv;
        tc_scale(mx, mult, inv);
        if (tid == 0) (GROUP ? sh.v_exp : sh.k_scale)[ring] = wide ? INFINITY : (GROUP ? (float)scale_exp(inv) - p.o_below : inv);
        if (wide) mult = 1.f;
        if (GROUP) {  // P needs V's scales, and sooner than the products need V
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.v_scaled[slot]);
        }
        uint8_t* const dsts[2] = {slots + slot * C::slot + dst0, slots + slot * C::slot + (dst0 ^ FLIP)};
        const float2 mult2 = make_float2(mult, mult);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            uint2 hi, lo;
            split_f16(mul2(make_float2(x[i].x, x[i].y), mult2), hi.x, lo.x);
            split_f16(mul2(make_float2(x[i].z, x[i].w), mult2), hi.y, lo.y);
            uint8_t* dst = dsts[i & 1];
            *reinterpret_cast<uint2*>(dst + i * STEP * 128) = hi;
            *reinterpret_cast<uint2*>(dst + i * STEP * 128 + C::half) = lo;
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(&full[slot]);
    }
    return true;
}

// SCORES: the scores are stored, for the totals, along the keys (1: few rows) or
// along the rows (2).
template <int HD, int SCORES>
__global__ void __launch_bounds__(kTcThreads, 1) smallm_tree_kernel(const TreeParams p) {
    using C = TcTree<HD>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    uint8_t* ks = smem;
    uint8_t* vs = smem + C::slots * C::slot;
    TcShared& sh = *reinterpret_cast<TcShared*>(vs + C::slots * C::slot);
    const TreeArgs& a = p.a;
    const uint32_t warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const uint32_t r0 = blockIdx.x * kTcRows, split = blockIdx.y, g = blockIdx.z;
    const uint32_t tiles = (p.n + kTcKeys - 1) / kTcKeys;
    const uint32_t t0 = split * p.tiles_per_split, nt = min(tiles, t0 + p.tiles_per_split) - t0;

    pdl_launch_dependents();  // the joining kernel's launch overlaps this one
    const uint32_t quads = min(4u, (p.R - r0 + 31) / 32);  // warps' row quarters that hold rows
    const uint32_t v_first = C::slots - (quads * (32 * HD * 4) + C::slot - 1) / C::slot;  // V's slots before q's
    if (threadIdx.x == 0) {
        for (uint32_t i = 0; i < C::slots; ++i) {
            mbar_init(&sh.k_full[i], kConvWarps);
            mbar_init(&sh.k_empty[i], 1);
            mbar_init(&sh.v_full[i], kConvWarps);
            mbar_init(&sh.v_scaled[i], kConvWarps);
            mbar_init(&sh.v_empty[i], 1);
        }
        for (uint32_t b = 0; b < 2; ++b) {
            mbar_init(&sh.s_full[b], 2);   // the MMA's commit and the issuing thread
            mbar_init(&sh.p_full[b], 2 * quads);
            mbar_init(&sh.o_full[b], 2);
            mbar_init(&sh.o_empty[b], 2 * quads);
        }
        for (uint32_t i = 0; i < 4; ++i) mbar_init(&sh.z_full[i], 2);
        mbar_init(&sh.q_full, 2 * quads);
        mbar_init(&sh.done, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 24) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh.tmem)),
                     "r"(512u)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    pdl_wait();  // what came before on the stream has ended
    // the first tiles' rows are on their way while the CTA is set up (copying
    // warps: 25 K, 26 V; the last of V's slots hold q first)
    if (warp - 25 < 2 && lane == 0) {
        const uint32_t op = warp - 25;
        const float* rows_src = (op ? a.vcache : a.kcache) + (size_t)g * a.max_ctx * HD;
        for (uint32_t s = 0; s < C::slots; ++s) mbar_init(&sh.raw_full[op][s], 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        tc_copy<HD>(rows_src, p.n, t0, 0, min(nt, op ? v_first : C::slots), op ? vs : ks, sh.raw_full[op], nullptr);
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tm = __shfl_sync(0xffffffffu, sh.tmem, 0);
    bool ok = true;

    if (warp < 8) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 72;");
        constexpr int SC = (int)kTcKeys / 2;  // this thread's columns of S
        const uint32_t quad = warp & 3, half = warp >> 2;
        const uint32_t rl = quad * 32 + lane, r = r0 + rl;
        const uint32_t lanes = tm + ((quad * 32u) << 16);
        const bool valid = r < p.R;
        const uint32_t tok = valid ? r / p.G : 0;
        {
            // q: the eight warps read eight rows at a time, and their largest magnitudes,
            // into V's slots; then each row is scaled and split by its two threads
            // (rows past the last stay as they are: nothing of them is written)
            constexpr int QL = HD / 32;
            float* stage = reinterpret_cast<float*>(vs + v_first * C::slot);
#pragma unroll 1
            for (uint32_t b = warp * 8; b < kTcRows && r0 + b < p.R; b += 64) {
                uint32_t tt = (r0 + b) / p.G, hh = (r0 + b) % p.G;
                alignas(16) float x[8][QL];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float* qi = a.q + (size_t)tt * a.q_stride + ((size_t)g * p.G + hh) * HD + lane * QL;
#pragma unroll
                    for (int j = 0; j < QL; ++j) x[i][j] = 0.f;
                    if (r0 + b + i < p.R) {
                        if constexpr (QL == 4) *reinterpret_cast<float4*>(x[i]) = __ldg(reinterpret_cast<const float4*>(qi));
                        else if constexpr (QL == 2) *reinterpret_cast<float2*>(x[i]) = __ldg(reinterpret_cast<const float2*>(qi));
                        else x[i][0] = __ldg(qi);
                    }
                    if (++hh == p.G) hh = 0, ++tt;
                }
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    uint32_t m = 0;
#pragma unroll
                    for (int j = 0; j < QL; ++j) m = max(m, __float_as_uint(x[i][j]) & 0x7FFFFFFFu);
                    // (16-byte units of a row permuted by the row: no bank conflicts either way)
                    float* at = stage + (b + i) * HD + (((lane * QL >> 2) ^ (i & 7)) << 2) + (lane * QL & 3);
                    if constexpr (QL == 4) *reinterpret_cast<float4*>(at) = *reinterpret_cast<const float4*>(x[i]);
                    else if constexpr (QL == 2) *reinterpret_cast<float2*>(at) = *reinterpret_cast<const float2*>(x[i]);
                    else *at = x[i][0];
                    m = __reduce_max_sync(0xffffffffu, m);
                    if (lane == 0) sh.q_max[b + i] = m;
                }
            }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // V's rows follow
        asm volatile("barrier.cta.sync 3, 256;" ::: "memory");
        // a quarter without rows is done: what the products hold in its lanes is not read
        if (quad < quads) {
        float qinv;
        {
            const float4* src = reinterpret_cast<const float4*>(vs + v_first * C::slot) + rl * (HD / 4);
            float mult;
            tc_scale(sh.q_max[rl], mult, qinv);
            const float2 mult2 = make_float2(mult, mult);
#pragma unroll
            for (int i = 0; i < HD / 8; i += 4) {
                uint32_t hi[8], lo[8];
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const float4 x = src[(half * (HD / 8) + i + u) ^ (rl & 7)];
                    split_f16(mul2(make_float2(x.x, x.y), mult2), hi[2 * u], lo[2 * u]);
                    split_f16(mul2(make_float2(x.z, x.w), mult2), hi[2 * u + 1], lo[2 * u + 1]);
                }
                tmem_st8(lanes + C::q_hi + half * (HD / 4) + 2 * i, hi);
                tmem_st8(lanes + C::q_lo + half * (HD / 4) + 2 * i, lo);
            }
        }
        tmem_wait_st();
        tc_fence_before();
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.q_full);

        // the largest of the warp's rows (as bits: no sign, no NaN)
        const float qtop = __uint_as_float(__reduce_max_sync(0xffffffffu, valid ? __float_as_uint(qinv) : 0u));
        float m = -INFINITY, l = 0.f;
        uint32_t meets = 0;  // tiles so far in which the halves met once more
        float* sc = nullptr;
        if constexpr (SCORES == 1) sc = p.scores + ((size_t)g * p.R + r) * p.sc_keys + half * SC;
        if constexpr (SCORES == 2) sc = p.scores + ((size_t)g * p.sc_keys + half * SC) * p.sc_rows + 4 * r;
        // a wait that gave up leaves the loop running (without waits) to its
        // end, since the two warps of a row meet at a barrier in it
        for (uint32_t t = 0; t < nt; ++t) {
            const uint32_t b = t & 1, key0 = (t0 + t) * kTcKeys, ring = t % kTcRing;
            ok = ok && mbar_wait_soon(&sh.v_scaled[t % C::slots], (t / C::slots) & 1) &&
                 mbar_wait_soon(&sh.s_full[b], (t >> 1) & 1);
            ok = __all_sync(0xffffffffu, ok);
            tc_fence_after();
            const uint32_t sp = lanes + C::s0 + b * kTcKeys;
            const float k_scale = sh.k_scale[ring];
            const unsigned long long bad = sh.k_bad[ring];
            float s[SC];
            auto get_scores = [&] {
                tmem_ld32(sp + half * SC, reinterpret_cast<uint32_t(&)[SC]>(s));
            };
            auto put_scores = [&] {
#pragma unroll
                for (int i = 0; i < SC; i += 8)
                    tmem_st8(sp + half * SC + i, reinterpret_cast<const uint32_t(&)[8]>(s[i]));
                tmem_wait_st();
            };
            get_scores();
            // keys with scales of their own, or a factor beyond f32's range (which no score need be)
            const float factor = qtop * k_scale, v_exp = sh.v_exp[ring];
            const bool wide_v = v_exp == INFINITY;
            const bool far = !(factor < INFINITY);
            // (never 0: an unseen key's -inf times it stays -inf)
            const float raw = far ? 1.f : fmaxf(qinv * k_scale, 0x1p-120f);
            if (key0 + kTcKeys > a.n_past || bad || far) {
                if (far) {
                    // scores of their own size, by way of tensor memory (spares registers);
                    // q's scale first where it is below 1: no overflow on the way
                    const float* ks = &sh.row_scale[0][ring][half * SC];
                    const float qa = fminf(qinv, 1.f), qb = fmaxf(qinv, 1.f);
                    tmem_map8<SC / 8>(sp + half * SC, [&](int i, float x) {
                        return x * qa * (k_scale == INFINITY ? ks[i] : k_scale) * qb;
                    });
                    get_scores();
                }
                const uint32_t seen = (uint32_t)(tc_seen(a.mask, a.n_past, a.n_tokens, tok, key0) >> (half * SC));
                const uint32_t hurt = (uint32_t)(bad >> (half * SC));
#pragma unroll
                for (int i = 0; i < SC; ++i) {
                    if (!((seen >> i) & 1)) s[i] = -INFINITY;
                    else if ((hurt >> i) & 1) s[i] = __uint_as_float(0x7FC00000u);
                }
            }
            if (SCORES == 1 && valid) {
#pragma unroll
                for (int i = 0; i < SC; i += 4)
                    *reinterpret_cast<float4*>(sc + key0 + i) =
                        make_float4(s[i] * raw, s[i + 1] * raw, s[i + 2] * raw, s[i + 3] * raw);
            }
            if (SCORES == 2 && valid) {  // the lanes' rows are neighbours
                float* at = sc + (size_t)key0 * p.sc_rows;
#pragma unroll
                for (int i = 0; i < SC; i += 4)
                    *reinterpret_cast<float4*>(at + i * p.sc_rows) =
                        make_float4(s[i] * raw, s[i + 1] * raw, s[i + 2] * raw, s[i + 3] * raw);
            }
            float mx[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
            for (int i = 4; i < SC; ++i) mx[i & 3] = fmaxf(mx[i & 3], s[i]);
            float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
            sh.part_max[b][half][rl] = top;
            asm volatile("barrier.cta.sync %0, 64;" ::"r"(4 + quad) : "memory");
            top = fmaxf(top, sh.part_max[b][half ^ 1][rl]);
            float ct = raw * p.c;
            // P is relative to the tile's own maximum mt: relative to the row's, a
            // tile of small weights would lose bits that large values bring back
            // (-inf only where nothing is seen: scores that are all below f32's range end
            // with a sum of 0 at a finite maximum, one above it with a NaN)
            const float mt = top == -INFINITY ? -INFINITY : fmaxf(ceilf(top * ct), -FLT_MAX);
            const float mn = fmaxf(m, mt), ref = mn == -INFINITY ? 0.f : mn;
            const float corr_t = ex2_approx(m - ref), part = ex2_approx(mt - ref);
            m = mn;
            const float tref = mt == INFINITY ? __uint_as_float(0x7FC00000u) : (mt == -INFINITY ? 0.f : mt);
            float off = kPShift - tref;
            float o_exp = v_exp, wsum = 0.f;  // O's exponent besides mt's; sum of the weights where P holds more
            // (from a factor of 2^-13 on hd products below 2^30 can give a large score)
            const bool large = fabsf(tref) >= kLargeScore;
            if (wide_v || (!(factor < 0x1p-13f) && __any_sync(0xffffffffu, valid && large))) {
                // exponents of their own first, by way of tensor memory.  A product of a large
                // score is rounded before the maximum's is taken from it: by an fma the
                // maximum itself could end up anywhere between 2^-128 and 2^128.
                float z = wide_v ? -INFINITY : 0.f;  // P's exponent besides mt's
                const float* vx = &sh.row_scale[1][ring][half * SC];
                put_scores();
                tmem_map8<SC / 8>(sp + half * SC, [&](int i, float x) {
                    float y = large ? __fadd_rn(__fadd_rn(__fmul_rn(x, ct), -tref), kPShift) : fmaf(x, ct, off);
                    wsum += ex2_approx(y);
                    if (wide_v) {
                        y += vx[i];
                        z = fmaxf(z, y);
                    }
                    return y;
                });
                get_scores();
                // The halves meet: P goes where the other half's scores were, and takes up the
                // scales of V's rows relative to the token's largest product among the keys
                // that it sees.  (A bounded wait: after one that gave up the two warps may
                // disagree about this path.)
                sh.part_z[half][rl] = z;
                __syncwarp();
                if (lane == 0) mbar_arrive(&sh.z_full[quad]);
                ok = __all_sync(0xffffffffu, ok && mbar_wait_soon(&sh.z_full[quad], meets++ & 1));
                z = fmaxf(z, sh.part_z[half ^ 1][rl]);
                if (wide_v) {
                    z = z == -INFINITY ? 0.f : ceilf(z) - kPShift;
                    o_exp = z - p.o_below;
                }
                ct = 1.f, off = -z;
            }
            float2 sum = make_float2(0.f, 0.f);
            const float2 ct2 = make_float2(ct, ct), off2 = make_float2(off, off);
#pragma unroll
            for (int i = 0; i < SC; i += 16) {
                uint32_t hi[8], lo[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    float2 e = fma2(make_float2(s[i + 2 * j], s[i + 2 * j + 1]), ct2, off2);
                    e.x = ex2_approx(e.x);
                    e.y = ex2_approx(e.y);
                    sum = add2(sum, e);
                    split_f16(e, hi[j], lo[j]);
                }
                tmem_st8(sp + half * (SC / 2) + i / 2, hi);
                tmem_st8(sp + 32 + half * (SC / 2) + i / 2, lo);
            }
            if (!wide_v) wsum = sum.x + sum.y;
            if (half == 0) {
                const float e = mt - ref + o_exp;  // O's exponent
                const bool tiny = e < -126.f && e > -126.f - kTinyShift;
                sh.corr[t % 4][rl] = make_float2(corr_t, tiny ? -exp2_whole(e + kTinyShift) : exp2_whole(e));
            }
            l = fmaf(l, corr_t, wsum * part);
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.p_full[b]);
        }
        sh.part_sum[half][rl] = l;
        asm volatile("barrier.cta.sync %0, 64;" ::"r"(4 + quad) : "memory");
        l = (l + sh.part_sum[half ^ 1][rl]) * 0x1p-14f;
        const size_t row = (size_t)g * p.R + r;
        float f = 0.f;
        if (p.n_split > 1) {
            if (half == 0 && valid) p.part_ml[(size_t)split * a.n_kv * p.R + row] = make_float2(m, l);
        } else {
            f = row_inverse(m, l);
            if (SCORES && half == 0 && valid) p.stats[row] = make_float2(m == -INFINITY ? 0.f : m, f);
        }
        if (half == 0) sh.factor[rl] = p.n_split > 1 ? 1.f : f * p.head_up;
        asm volatile("barrier.cta.sync %0, 128;" ::"r"(8 + quad) : "memory");
        }
    } else if (warp < 16) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 88;");
        constexpr int OC = HD / 2;  // this thread's columns of O
        const uint32_t quad = warp & 3, half = warp >> 2 & 1;
        const uint32_t rl = quad * 32 + lane, r = r0 + rl;
        const uint32_t lanes = tm + ((quad * 32u) << 16);
        if (quad < quads) {
        float2 o[OC / 2];
#pragma unroll
        for (int i = 0; i < OC / 2; ++i) o[i] = make_float2(0.f, 0.f);
        for (uint32_t t = 0; t < nt; ++t) {  // o = o * corr + O of tile t
            const uint32_t b = t & 1;
            ok = ok && mbar_wait_soon(&sh.o_full[b], (t >> 1) & 1);
            ok = __all_sync(0xffffffffu, ok);
            tc_fence_after();
            const float2 tile = sh.corr[t % 4][rl];
            if (__any_sync(0xffffffffu, tile.x != 1.f || tile.y < 0.f)) {
                if (__any_sync(0xffffffffu, tile.y < 0.f)) {
                    const float down = tile.y < 0.f ? exp2_whole(-kTinyShift) : 1.f;
                    tmem_map8<OC / 8>(lanes + C::o0 + b * 128 + half * OC, [&](int, float x) { return x * down; });
                }
                const float2 corr2 = make_float2(tile.x, tile.x);
#pragma unroll
                for (int i = 0; i < OC / 2; ++i) o[i] = mul2(o[i], corr2);
            }
            const float scale = fabsf(tile.y);
            const float2 scale2 = make_float2(scale, scale);
            constexpr int OW = 16;
#pragma unroll
            for (int c = 0; c < OC; c += OW) {
                uint32_t x[OW];
                tmem_ld16(lanes + C::o0 + b * 128 + half * OC + c, x);
#pragma unroll
                for (int i = 0; i < OW / 2; ++i)
                    o[c / 2 + i] = fma2(make_float2(__uint_as_float(x[2 * i]), __uint_as_float(x[2 * i + 1])), scale2,
                                        o[c / 2 + i]);
            }
            const unsigned long long bad = sh.v_bad[t % kTcRing];
            if (bad && r < p.R && (bad & tc_seen(a.mask, a.n_past, a.n_tokens, r / p.G, (t0 + t) * kTcKeys))) {
#pragma unroll
                for (int i = 0; i < OC / 2; ++i)
                    o[i] = make_float2(__uint_as_float(0x7FC00000u), __uint_as_float(0x7FC00000u));
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.o_empty[b]);
        }
        asm volatile("barrier.cta.sync %0, 128;" ::"r"(8 + quad) : "memory");
        const float f = sh.factor[rl];
        // rows leave through K's slots (every MMA has completed), so that the
        // stores run along rows
        constexpr int OL = OC / 4, OX = OL < 8 ? OL - 1 : 7;  // float4s of half a row; their permutation
        float4* stage = reinterpret_cast<float4*>(ks) + (warp - 8) * 32 * OL;
#pragma unroll
        for (int i = 0; i < OC; i += 4)
            stage[lane * OL + ((i / 4) ^ (lane & OX))] =
                make_float4(o[i / 2].x * f, o[i / 2].y * f, o[i / 2 + 1].x * f, o[i / 2 + 1].y * f);
        __syncwarp();
        // STEP half rows at a time; where they go to the output, the lane's head and
        // token go up with its row (a division for each row took 1 us for 64 rows)
        constexpr uint32_t STEP = 32 / OL;
        const uint32_t row = lane / OL, c = half * OC + lane % OL * 4, last = min(32u, p.R - r0 - quad * 32);
        const float4* from = stage + row * OL;
        if (p.n_split > 1) {
            float* dst = p.part_o + ((size_t)split * a.n_kv * p.R + (size_t)g * p.R + r0 + quad * 32 + row) * HD + c;
#pragma unroll 4
            for (uint32_t i = 0; i < last; i += STEP)
                if (i + row < last)
                    *reinterpret_cast<float4*>(dst + i * HD) = from[i * OL + (lane % OL ^ (i + row & OX))];
        } else {
            uint32_t token = (r0 + quad * 32 + row) / p.G, head = (r0 + quad * 32 + row) % p.G;
            float* dst = a.out + (size_t)g * p.G * HD + c;
#pragma unroll 2
            for (uint32_t i = 0; i < last; i += STEP) {
                if (i + row < last)
                    *reinterpret_cast<float4*>(dst + (size_t)token * a.out_stride + head * HD) =
                        from[i * OL + (lane % OL ^ (i + row & OX))];
                for (head += STEP; head >= p.G; head -= p.G) ++token;
            }
        }
        }
    } else if (warp < 20) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 80;");
        ok = tc_convert<HD, 0>(p, t0, nt, (int)threadIdx.x - 512, smem, sh);
    } else if (warp < 24) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 80;");
        ok = tc_convert<HD, 1>(p, t0, nt, (int)threadIdx.x - 640, smem, sh);
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 24;");
        if (warp == 24) {
            // ---- MMA issuer: the whole warp walks the loop, one lane issues
            uint32_t leader;
            asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(leader));
            auto wait = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, mbar_wait_soon(bar, parity)); };
            ok = wait(&sh.q_full, 0);
            tc_fence_after();
            auto scores = [&](uint32_t t) -> bool {
                const uint32_t slot = t % C::slots, b = t & 1;
                if (!wait(&sh.k_full[slot], (t / C::slots) & 1)) return false;
                tc_fence_after();
                const uint64_t desc = smem_desc_sw128(ks + slot * C::slot);
                const uint32_t d = tm + C::s0 + b * kTcKeys;
                if (leader) {
#pragma unroll
                    for (int x = 0; x < 3; ++x) {  // lo hi, hi lo, hi hi
#pragma unroll
                        for (int j = 0; j < HD / 16; ++j)
                            mma_f16_ta(d, tm + (x == 0 ? C::q_lo : C::q_hi) + 8 * j,
                                       desc + (((x == 1 ? C::half : 0) + (j >> 2) * (kTcKeys * 128)) >> 4) + 2 * (j & 3),
                                       C::idesc_s, (x | j) != 0);
                    }
                    mma_commit(&sh.k_empty[slot]);
                    mma_commit(&sh.s_full[b]);
                    mbar_arrive(&sh.s_full[b]);
                }
                __syncwarp();
                return true;
            };
            ok = ok && scores(0);
            for (uint32_t t = 0; ok && t < nt; ++t) {
                // S(t + 1) goes where P(t - 1) was: its product was issued before
                if (t + 1 < nt && !scores(t + 1)) {
                    ok = false;
                    break;
                }
                const uint32_t slot = t % C::slots, b = t & 1;
                ok = wait(&sh.v_full[slot], (t / C::slots) & 1) && wait(&sh.p_full[b], (t >> 1) & 1) &&
                     (t < 2 || wait(&sh.o_empty[b], ((t >> 1) - 1) & 1));
                if (!ok) break;
                tc_fence_after();
                const uint64_t desc = smem_desc_sw128_mn(vs + slot * C::slot, kTcKeys * 128);
                const uint32_t pa = tm + C::s0 + b * kTcKeys, d = tm + C::o0 + b * 128;
                if (leader) {
#pragma unroll
                    for (int x = 0; x < 3; ++x) {
#pragma unroll
                        for (int j = 0; j < (int)kTcKeys / 16; ++j)
                            mma_f16_ta(d, pa + (x == 0 ? 32 : 0) + 8 * j,
                                       desc + (((x == 1 ? C::half : 0) + j * 2048) >> 4), C::idesc_pv, (x | j) != 0);
                    }
                    mma_commit(&sh.v_empty[slot]);
                    mma_commit(&sh.o_full[b]);
                    mbar_arrive(&sh.o_full[b]);
                }
                __syncwarp();
            }
            // tensor memory is freed only after every MMA has completed
            if (leader) mma_commit(&sh.done);
            __syncwarp();
            ok = mbar_wait_soon(&sh.done, 0) && ok;
        } else if (warp < 27 && lane == 0) {
            const uint32_t op = warp - 25;
            const float* rows_src = (op ? a.vcache : a.kcache) + (size_t)g * a.max_ctx * HD;
            const uint32_t sent = min(nt, op ? v_first : C::slots);
            ok = !op || nt == sent || mbar_wait_soon(&sh.q_full, 0);
            if (!ok) tc_landed<HD>(sent, sh.raw_full[op]);
            else ok = tc_copy<HD>(rows_src, p.n, t0, sent, nt, op ? vs : ks, sh.raw_full[op],
                                  op ? sh.v_empty : sh.k_empty) && tc_landed<HD>(nt, sh.raw_full[op]);
        }
    }
    if (!ok) atomicOr(p.err, kErrTreeWait);
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (warp == 24) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tm), "r"(512u) : "memory");
    }
}

// ---- joining -------------------------------------------------------------------

// Join the splits' partials: a CTA per (KV head, row), its threads 4 columns of
// every (threads * 4 / HD)-th split each, so that all loads are in flight at
// once (one warp walking the splits took 13 to 57 us of dependent loads).
constexpr int kMergeThreads = 256;
template <int HD>
__device__ __forceinline__ void merge_row(const TreeParams& p, size_t row) {
    constexpr int L4 = HD / 4, PARTS = kMergeThreads / L4;
    __shared__ float4 acc[PARTS][L4];
    __shared__ float red[32], redl[32];
    const TreeArgs& a = p.a;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, c = tid % L4, part = tid / L4;
    const size_t rows = (size_t)a.n_kv * p.R;
    // the first splits of each part leave with the maxima (past the last split
    // the loads repeat it and are dropped)
    constexpr int PRE = 4;
    float2 ml[PRE];
    float4 v[PRE];
#pragma unroll
    for (int k = 0; k < PRE; ++k) {
        const uint32_t s = min((uint32_t)(part + k * PARTS), p.n_split - 1);
        ml[k] = p.part_ml[s * rows + row];
        v[k] = reinterpret_cast<const float4*>(p.part_o + (s * rows + row) * HD)[c];
    }
    float M = -INFINITY;
    for (uint32_t s = tid; s < p.n_split; s += kMergeThreads) M = fmaxf(M, p.part_ml[s * rows + row].x);
    M = warp_max(M);
    if (lane == 0) red[warp] = M;
    __syncthreads();
    M = red[0];
#pragma unroll
    for (int w = 1; w < kMergeThreads / 32; ++w) M = fmaxf(M, red[w]);
    const float ref = M == -INFINITY ? 0.f : M;
    float L = 0.f;
    float4 O = make_float4(0.f, 0.f, 0.f, 0.f);
    auto add = [&](float2 s, float4 x) {
        const float f = exp2f(s.x - ref);
        L = fmaf(f, s.y, L);
        O.x = fmaf(f, x.x, O.x), O.y = fmaf(f, x.y, O.y), O.z = fmaf(f, x.z, O.z), O.w = fmaf(f, x.w, O.w);
    };
#pragma unroll
    for (int k = 0; k < PRE; ++k)
        if (part + k * PARTS < p.n_split) add(ml[k], v[k]);
#pragma unroll 4
    for (uint32_t s = part + PRE * PARTS; s < p.n_split; s += PARTS)
        add(p.part_ml[s * rows + row], reinterpret_cast<const float4*>(p.part_o + (s * rows + row) * HD)[c]);
    acc[part][c] = O;
    if (c == 0) redl[part] = L;
    __syncthreads();
    if (part) return;
    L = redl[0];
#pragma unroll
    for (int k = 1; k < PARTS; ++k) {
        const float4 v = acc[k][c];
        O.x += v.x, O.y += v.y, O.z += v.z, O.w += v.w;
        L += redl[k];
    }
    const float inv = row_inverse(M, L);
    const float up = inv * p.head_up;
    const uint32_t g = (uint32_t)(row / p.R), r = (uint32_t)(row % p.R);
    float* o = a.out + (size_t)(r / p.G) * a.out_stride + ((size_t)g * p.G + r % p.G) * HD;
    reinterpret_cast<float4*>(o)[c] = make_float4(O.x * up, O.y * up, O.z * up, O.w * up);
    if (c == 0 && p.sc_rows && p.scores) p.stats[row] = make_float2(ref, inv);
}

template <int HD>
__global__ void __launch_bounds__(kMergeThreads) smallm_tree_merge_kernel(const TreeParams p) {
    pdl_wait();
    merge_row<HD>(p, blockIdx.x);
}

// weights[g][k] += sum_r 2^(s c - mc_r) / sum_r, in a fixed order, so that the
// total does not depend on the launch.  Scores of up to kFewRows rows run along
// the keys: a lane has a key and walks the rows; the CTAs behind the n_join
// that join the splits find mc and sum of the rows from the splits themselves,
// so that neither waits for the other (a kernel after the joining one: 8% longer
// for one token over 16384 rows).  More rows run along
// themselves, four keys of a row together: the lanes of a warp have the rows of 8
// keys, and their sums meet by shuffles.  31 tokens over 12300 rows, 12 heads of
// 128: 27.3 us, 19.7 us of them without the totals; 29.2 us with 16 keys a warp,
// 29.1 us with a key's scores each 4 bytes of their own in its rows' stores, 36 us
// with mc and sum from the splits as well.
constexpr int kWeightKeys = 8, kWeightWarps = 8, kWeightRows = 2;
constexpr uint32_t kFewRows = 16;
static_assert(kTcKeys % (kWeightWarps * kWeightKeys) == 0 && kWeightKeys % 4 == 0, "a CTA's keys lie in a tile");
// ROWS: R at most (half of kFewRows where that does: 2% of one token's call)
template <int HD, uint32_t ROWS>
__global__ void __launch_bounds__(kMergeThreads) smallm_tree_weights_few_kernel(const TreeParams p, uint32_t n_join) {
    __shared__ float2 stats[ROWS];
    pdl_wait();
    if (blockIdx.x < n_join) {
        merge_row<HD>(p, blockIdx.x);
        return;
    }
    const uint32_t blocks = (p.n + kMergeThreads - 1) / kMergeThreads, at = blockIdx.x - n_join;
    const uint32_t g = at / blocks, key = at % blocks * kMergeThreads + threadIdx.x, lane = threadIdx.x & 31;
    // (loads past the last row or key repeat it and are dropped)
    float* w = p.a.weights + (size_t)g * p.a.max_ctx + min(key, p.n - 1);
    const float* s = p.scores + (size_t)g * p.R * p.sc_keys + min(key, p.n - 1);
    const float old = *w;
    float v[ROWS];
#pragma unroll
    for (uint32_t r = 0; r < ROWS; ++r) v[r] = __ldg(s + (size_t)min(r, p.R - 1) * p.sc_keys);
    for (uint32_t r = threadIdx.x >> 5; r < p.R; r += kMergeThreads / 32) {
        const size_t row = (size_t)g * p.R + r, rows = (size_t)p.a.n_kv * p.R;
        if (p.n_split == 1) {
            if (lane == 0) stats[r] = p.stats[row];
            continue;
        }
        float m = -INFINITY, l = 0.f;
        for (uint32_t i = lane; i < p.n_split; i += 32) {
            const float2 ml = p.part_ml[i * rows + row];
            const float top = fmaxf(m, ml.x), ref = top == -INFINITY ? 0.f : top;
            l = fmaf(l, exp2f(m - ref), ml.y * exp2f(ml.x - ref));
            m = top;
        }
        const float top = warp_max(m), ref = top == -INFINITY ? 0.f : top;
        l = warp_sum(l * exp2f(m - ref));
        if (lane == 0) stats[r] = make_float2(ref, row_inverse(top, l));
    }
    __syncthreads();
    if (key >= p.n) return;
    float acc = 0.f;
#pragma unroll
    for (uint32_t r = 0; r < ROWS; ++r)
        if (r < p.R)
            acc = row_plain(stats[r]) ? add_weight<true>(acc, v[r], p.c, stats[r]) : add_weight<false>(acc, v[r], p.c, stats[r]);
    *w = old + acc;
}
__global__ void __launch_bounds__(32 * kWeightWarps) smallm_tree_weights_kernel(const TreeParams p) {
    const uint32_t lane = threadIdx.x & 31, g = blockIdx.y;
    const uint32_t key = (blockIdx.x * kWeightWarps + (threadIdx.x >> 5)) * kWeightKeys;
    pdl_wait();
    float acc[kWeightKeys];
#pragma unroll
    for (int k = 0; k < kWeightKeys; ++k) acc[k] = 0.f;
    // (loads without conditions, so that all are in flight: past the last row they
    // read it again and it is dropped; the keys' scores are stored to a tile's end)
    float* w = p.a.weights + (size_t)g * p.a.max_ctx;
    const float4* s = reinterpret_cast<const float4*>(p.scores + ((size_t)g * p.sc_keys + key) * p.sc_rows);
    const float old = w[min(key + lane % kWeightKeys, p.n - 1)];
    const float2* stats = p.stats + (size_t)g * p.R;
    for (uint32_t r = lane; r - lane < p.R; r += 32 * kWeightRows) {
        float2 st[kWeightRows];
        float4 v[kWeightRows][kWeightKeys / 4];
#pragma unroll
        for (int j = 0; j < kWeightRows; ++j) {
            const uint32_t rj = min(r + 32 * j, p.R - 1);
            st[j] = stats[rj];
#pragma unroll
            for (int k = 0; k < kWeightKeys / 4; ++k) v[j][k] = __ldg(s + k * p.sc_rows + rj);
        }
#pragma unroll
        for (int j = 0; j < kWeightRows; ++j) {
            if (r + 32 * j >= p.R) break;
            auto add = [&](auto plain) {
#pragma unroll
                for (int k = 0; k < kWeightKeys / 4; ++k) {
                    const float4 x = v[j][k];
                    constexpr bool P = decltype(plain)::value;
                    acc[4 * k] = add_weight<P>(acc[4 * k], x.x, p.c, st[j]);
                    acc[4 * k + 1] = add_weight<P>(acc[4 * k + 1], x.y, p.c, st[j]);
                    acc[4 * k + 2] = add_weight<P>(acc[4 * k + 2], x.z, p.c, st[j]);
                    acc[4 * k + 3] = add_weight<P>(acc[4 * k + 3], x.w, p.c, st[j]);
                }
            };
            if (row_plain(st[j])) add(std::true_type{});
            else add(std::false_type{});
        }
    }
    float mine = 0.f;  // lane k: key k
#pragma unroll
    for (int k = 0; k < kWeightKeys; ++k) {
        const float sum = warp_sum(acc[k]);
        if (lane == (uint32_t)k) mine = sum;
    }
    if (lane < kWeightKeys && key + lane < p.n) w[key + lane] = old + mine;
}

size_t align256(size_t x) { return (x + 255) & ~(size_t)255; }

// Split of the keys and the workspace's layout, from sizes alone.
struct TreePlan {
    uint32_t n_split, tiles_per_split, sc_rows, sc_keys;
    size_t off_ml, off_scores, off_stats, bytes;
};

TreePlan tree_plan(uint32_t n_heads, uint32_t n_kv, uint32_t hd, uint32_t n_past, uint32_t n_tokens, bool weights) {
    TreePlan t{};
    const uint32_t R = n_tokens * (n_heads / n_kv), n = n_past + n_tokens;
    const uint32_t blocks = n_kv * ((R + kTcRows - 1) / kTcRows), tiles = (n + kTcKeys - 1) / kTcKeys;
    // one CTA per SM in all; two tiles cost a CTA less than the joining kernel
    t.n_split = tiles <= 2 ? 1 : std::min(std::max(1u, (uint32_t)device_sm_count() / blocks), tiles);
    t.tiles_per_split = (tiles + t.n_split - 1) / t.n_split;
    t.n_split = (tiles + t.tiles_per_split - 1) / t.tiles_per_split;
    const size_t rows = (size_t)n_kv * R;
    size_t at = t.n_split > 1 ? align256(4 * rows * t.n_split * hd) : 0;
    t.off_ml = at;
    if (t.n_split > 1) at += align256(8 * rows * t.n_split);
    t.off_scores = at;
    t.sc_rows = R > kFewRows ? (R + 31) / 32 * 32 : 0;
    t.sc_keys = tiles * kTcKeys;
    if (weights) at += align256(4 * (size_t)n_kv * (t.sc_rows ? t.sc_rows : R) * t.sc_keys);
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
    const void* fn = !p.scores   ? (const void*)smallm_tree_kernel<HD, 0>
                     : p.sc_rows ? (const void*)smallm_tree_kernel<HD, 2>
                                 : (const void*)smallm_tree_kernel<HD, 1>;
    set_smem_limit_once(fn, (int)TcTree<HD>::smem);
    const dim3 grid((p.R + kTcRows - 1) / kTcRows, p.n_split, p.a.n_kv);
    TreeParams pp = p;
    void* args[] = {&pp};
    launch_kernel_ex(fn, grid, dim3(kTcThreads), TcTree<HD>::smem, stream, true, args);
    const uint32_t n_join = p.n_split > 1 ? p.a.n_kv * p.R : 0;
    if (p.a.weights && !p.sc_rows) {
        uint32_t join = n_join;
        void* few[] = {&pp, &join};
        const uint32_t blocks = (p.n + kMergeThreads - 1) / kMergeThreads;
        const void* sums = p.R <= kFewRows / 2 ? (const void*)smallm_tree_weights_few_kernel<HD, kFewRows / 2>
                                               : (const void*)smallm_tree_weights_few_kernel<HD, kFewRows>;
        launch_kernel_ex(sums, dim3(n_join + blocks * p.a.n_kv),
                         dim3(kMergeThreads), 0, stream, true, few);
        return;
    }
    if (n_join)
        launch_kernel_ex((const void*)smallm_tree_merge_kernel<HD>, dim3(n_join), dim3(kMergeThreads), 0, stream, true,
                         args);
    if (p.a.weights) {
        const uint32_t keys = kWeightWarps * kWeightKeys;
        launch_kernel_ex((const void*)smallm_tree_weights_kernel, dim3((p.n + keys - 1) / keys, p.a.n_kv),
                         dim3(32 * kWeightWarps), 0, stream, true, args);
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
    p.n_split = t.n_split;
    p.tiles_per_split = t.tiles_per_split;
    p.sc_rows = t.sc_rows;
    p.sc_keys = t.sc_keys;
    p.c = (float)(1.4426950408889634 / sqrt((double)a.hd));
    uint32_t head = 1;  // the weights' sum is below n, and rounded up once more by what P and V round
    while (p.n >> (head - 1)) ++head;
    p.o_below = kPShift + (float)head;
    p.head_up = ldexpf(1.f, (int)head);
    p.err = device_error_flag();
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
