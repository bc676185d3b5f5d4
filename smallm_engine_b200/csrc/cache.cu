// Keeping a KV cache within its budget: which rows of each KV head to keep,
// and the in-place move that closes the gaps.
//
// select: of rows 0..n-1 of a KV head keep the first n_first, the last n_last
// and, of those between, the n_keep - n_first - n_last with the largest totals
// (equal totals: the lower row; NaN below everything).  A cluster of up to 16
// CTAs owns a head, each a contiguous range of its keys in shared memory.  The
// k-th largest key is found digit by digit (9, 8, 8 and 7 bits, most
// significant first): histograms of the keys that match the digits so far,
// summed over the cluster's shared memory, then the bin that holds the rank.
// (Digits of 11, 11 and 10 bits save a barrier, but then every CTA reads 8 KB
// from each of 15 others for each digit: 37 us for 8 x 131072 keys where this
// takes 20 us.  Histograms read by more threads, fewer reads each: 21 us.)
// Every larger key is kept, and of the equal ones the first few in row order;
// rows come out ascending.  Bound by latency: one read of the totals, five
// cluster barriers and four rounds of remote reads.
//
// move: row dst + i of K and V (and the totals) becomes row rows[i], for a
// strictly ascending list with rows[i] >= dst + i.  In place: a cluster owns a
// slice of columns of one head's K or V and walks the list in waves, a part of
// a wave for each CTA, its rows in registers between load and store.  A store
// may only overwrite rows that have been read.  Row dst + j is read by entries
// <= j alone, so a CTA may store its part of a wave once the others have loaded
// every wave whose first source lies below the part's end; each tells the
// others how many waves it has loaded.  The distance rows[i] - (dst + i) never
// shrinks along the list, so beyond the first few waves of an eviction that
// has long been the case and nobody waits.  Bound by the bytes moved.
// 8 heads x 16384 of 32768 rows of 128: 63 us (77 us without the streaming
// hints); with a cluster barrier for each wave 166 us, and rows by bulk copies
// through shared memory, whatever the buffers, 88 us at best: copies of a row
// or two are too small for them.  Half a wave, with the next one's loads sent
// before its stores: 74 us; reads and writes do better apart.
#include <cooperative_groups.h>

#include <algorithm>
#include <map>
#include <mutex>
#include <tuple>

#include "common.cuh"
#include "engine.h"
#include "smallm_cuda.h"

namespace smallm {
namespace {

namespace cg = cooperative_groups;

constexpr int kSelThreads = 512;  // (two CTAs fit an SM: 14 clusters of 16 at once instead of 7)
constexpr int kSelWarps = kSelThreads / 32;
constexpr int kSelPasses = 4;
constexpr uint32_t kSelBins = 512;
constexpr uint32_t kSelCached = 20480;  // keys of a CTA that fit shared memory
constexpr uint32_t kSelMaxCluster = 16;
constexpr uint32_t kCacheMaxRows = 1u << 30;  // keeps 32-bit row numbers from wrapping

// Order-preserving key, NaN lowest, -0 equal to +0.
__device__ __forceinline__ uint32_t total_key(float x) { return x == x ? float_order_key(x + 0.f) : 0u; }

struct SelShared {
    alignas(16) uint32_t hist[kSelPasses][kSelBins];
    uint32_t warp[kSelWarps], warp_own[kSelWarps];
    uint32_t digit, rank, above;
    uint2 counts[kSelMaxCluster];  // every CTA's keys above / equal to the k-th largest
};

__global__ void __launch_bounds__(kSelThreads, 2)
    smallm_cache_select_kernel(const float* __restrict__ weights, uint32_t stride, uint32_t n, uint32_t n_keep,
                               uint32_t n_first, uint32_t n_last, uint32_t per_cta, uint32_t cached,
                               uint32_t* __restrict__ rows) {
    extern __shared__ uint32_t cache[];
    __shared__ SelShared sh;
    cg::cluster_group cluster = cg::this_cluster();
    const uint32_t C = cluster.num_blocks(), cr = cluster.block_rank(), head = blockIdx.x / C;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uint32_t m = n - n_first - n_last, k = n_keep - n_first - n_last;
    const uint32_t b0 = min(m, cr * per_cta), len = min(m, b0 + per_cta) - b0;
    const float* w = weights + (size_t)head * stride + n_first + b0;
    uint32_t* out = rows + (size_t)head * n_keep;
    for (uint32_t i = tid; i < kSelPasses * kSelBins; i += kSelThreads) (&sh.hist[0][0])[i] = 0;
    __syncthreads();
    pdl_wait();
    if (cr == 0) {
        for (uint32_t i = tid; i < n_first; i += kSelThreads) out[i] = i;
        for (uint32_t i = tid; i < n_last; i += kSelThreads) out[n_first + k + i] = n - n_last + i;
    }
    if (!k) return;
    // keys from the totals, counted by their first digit on the way (eight loads in
    // flight; past the range they repeat its last total)
    for (uint32_t i = tid; i < len; i += 8 * kSelThreads) {
        float v[8];
#pragma unroll
        for (uint32_t j = 0; j < 8; ++j) v[j] = __ldg(w + min(i + j * kSelThreads, len - 1));
#pragma unroll
        for (uint32_t j = 0; j < 8; ++j) {
            const uint32_t key = total_key(v[j]);
            if (i + j * kSelThreads >= len) continue;
            if (cached) cache[i + j * kSelThreads] = key;
            atomicAdd(&sh.hist[0][key >> 23], 1u);
        }
    }
    // (past the range: its last key)
    auto key_of = [&](uint32_t i) {
        i = min(i, len - 1);
        return cached ? cache[i] : total_key(w[i]);
    };
    __syncthreads();
    uint32_t prefix = 0, want = k, my_gt = 0;
#pragma unroll 1
    for (int pass = 0; pass < kSelPasses; ++pass) {
        const int shift = pass == 0 ? 23 : (pass == 1 ? 15 : (pass == 2 ? 7 : 0));
        const uint32_t bins = pass == 0 ? 512u : (pass == 3 ? 128u : 256u);
        const uint32_t high = ~(bins * (1u << shift) - 1u);
        uint32_t* hist = sh.hist[pass];
        // (the first digit has been counted; four keys of a lane at a time; plain
        // shared-memory adds, even where all keys share a bin: counting a warp's
        // equal bins first cost more)
        for (uint32_t i0 = tid; pass && i0 - lane < len; i0 += 4 * kSelThreads) {
            uint32_t bin[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t i = i0 + j * kSelThreads;
                const uint32_t key = key_of(i);
                bin[j] = i < len && (key & high) == prefix ? key >> shift & (bins - 1) : kSelBins;
            }
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (bin[j] != kSelBins) atomicAdd(&hist[bin[j]], 1u);
        }
        if (C > 1) cluster.sync();
        else __syncthreads();
        // thread t: four bins, counted from the top
        const uint32_t top = bins - 4 - 4 * tid;
        uint4 sum = make_uint4(0, 0, 0, 0), own = sum;
        if (4u * tid < bins) {
            own = *reinterpret_cast<const uint4*>(&hist[top]);
            sum = own;
            // the peers' reads in flight together (past the last one the loads
            // repeat it and are dropped)
            for (uint32_t r = 1; r < C; r += 5) {
                uint4 v[5];
#pragma unroll
                for (uint32_t j = 0; j < 5; ++j) {
                    const uint32_t d = cr + min(r + j, C - 1), peer = d < C ? d : d - C;
                    v[j] = *reinterpret_cast<const uint4*>(cluster.map_shared_rank(&hist[top], peer));
                }
#pragma unroll
                for (uint32_t j = 0; j < 5; ++j) {
                    const uint32_t on = r + j < C ? 0xFFFFFFFFu : 0u;
                    sum.x += v[j].x & on, sum.y += v[j].y & on, sum.z += v[j].z & on, sum.w += v[j].w & on;
                }
            }
        }
        // inclusive scan from the top: keys in these bins or above, of the head and of this CTA
        const uint32_t all = sum.x + sum.y + sum.z + sum.w, mine = own.x + own.y + own.z + own.w;
        uint32_t incl = all, iown = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t y = __shfl_up_sync(0xffffffffu, incl, o), z = __shfl_up_sync(0xffffffffu, iown, o);
            if (lane >= o) incl += y, iown += z;
        }
        if (lane == 31) {
            sh.warp[warp] = incl;
            sh.warp_own[warp] = iown;
        }
        __syncthreads();
        uint32_t before = incl - all, obefore = iown - mine;
        before += __reduce_add_sync(0xffffffffu, lane < warp ? sh.warp[lane] : 0u);
        obefore += __reduce_add_sync(0xffffffffu, lane < warp ? sh.warp_own[lane] : 0u);
        // the bin where the count from the top reaches `want`
        if (before < want && want <= before + all) {
            uint32_t digit = top + 3, c = sum.w, o = own.w;
            if (want > before + c) before += c, obefore += o, --digit, c = sum.z, o = own.z;
            if (want > before + c) before += c, obefore += o, --digit, c = sum.y, o = own.y;
            if (want > before + c) before += c, obefore += o, --digit;
            sh.digit = digit;
            sh.rank = want - before;
            sh.above = obefore;
        }
        __syncthreads();
        prefix |= sh.digit << shift;
        want = sh.rank;
        my_gt += sh.above;  // this CTA's keys in higher bins
    }
    // keys above `prefix` are kept, and the first `want` of the head that equal
    // it; every CTA tells the others how many it has of each
    if ((uint32_t)tid < C)
        *cluster.map_shared_rank(&sh.counts[cr], tid) = make_uint2(my_gt, sh.hist[kSelPasses - 1][prefix & 127u]);
    if (C > 1) cluster.sync();
    else __syncthreads();
    uint2 prior = (uint32_t)lane < cr ? sh.counts[lane] : make_uint2(0, 0);
    uint32_t gt0 = __reduce_add_sync(0xffffffffu, prior.x), eq0 = __reduce_add_sync(0xffffffffu, prior.y);
    // each warp owns a contiguous run of the range
    const uint32_t run = (len + kSelThreads - 1) / kSelThreads * 32;
    const uint32_t wb = min(len, warp * run), we = min(len, wb + run);
    uint32_t cg_ = 0, ce = 0;
#pragma unroll 4
    for (uint32_t i = wb + lane; i - lane < we; i += 32) {
        const uint32_t key = key_of(i);
        cg_ += __popc(__ballot_sync(0xffffffffu, i < we && key > prefix));
        ce += __popc(__ballot_sync(0xffffffffu, i < we && key == prefix));
    }
    if (lane == 0) {
        sh.warp[warp] = cg_;
        sh.warp_own[warp] = ce;
    }
    __syncthreads();
    gt0 += __reduce_add_sync(0xffffffffu, lane < warp ? sh.warp[lane] : 0u);
    eq0 += __reduce_add_sync(0xffffffffu, lane < warp ? sh.warp_own[lane] : 0u);
    const uint32_t lt = (1u << lane) - 1u;
#pragma unroll 4
    for (uint32_t i = wb + lane; i - lane < we; i += 32) {
        const uint32_t key = key_of(i);
        const bool gt = i < we && key > prefix, eq = i < we && key == prefix;
        const uint32_t bg = __ballot_sync(0xffffffffu, gt), be = __ballot_sync(0xffffffffu, eq);
        const uint32_t g = gt0 + __popc(bg & lt), e = eq0 + __popc(be & lt);
        if (gt || (eq && e < want)) out[n_first + g + min(e, want)] = n_first + b0 + i;
        gt0 += __popc(bg);
        eq0 += __popc(be);
    }
}

constexpr int kMoveThreads = 512;
constexpr int kMoveUnroll = 8;
constexpr uint32_t kMoveWave = kMoveThreads * kMoveUnroll;  // vectors of a CTA per wave in registers
constexpr uint32_t kMoveMaxCluster = 8;

struct MoveArgs {
    const uint32_t* rows;
    uint32_t n_rows, dst, max_ctx;
    unsigned int* err;
};

// Source row of entry i (< n_rows); dst + i, no move, where the entry breaks the
// list's rules, which raises bit 7 of the error word.
__device__ __forceinline__ uint32_t move_source(const MoveArgs& a, uint32_t i) {
    const uint32_t src = __ldg(a.rows + i);
    const bool ok = src < a.max_ctx && src >= a.dst + i && (i == 0 || __ldg(a.rows + i - 1) < src);
    if (!ok) atomicOr(a.err, kErrMoveList);
    return ok ? src : a.dst + i;
}

// base[(dst + i) * width + c] = base[rows[i] * width + c] for c < width (vectors
// of type V) of a list that fits one wave of a CTA.
template <typename V>
__device__ __forceinline__ void move_rows(V* base, uint32_t width, const MoveArgs& a) {
    const uint32_t c = threadIdx.x % width, r0 = threadIdx.x / width, step = kMoveThreads / width;
    V v[kMoveUnroll];
    uint32_t go = 0;
#pragma unroll
    for (int u = 0; u < kMoveUnroll; ++u) {
        const uint32_t i = r0 + u * step;
        if (i >= a.n_rows) continue;
        const uint32_t src = move_source(a, i);
        if (src == a.dst + i) continue;
        v[u] = base[(size_t)src * width + c];
        go |= 1u << u;
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < kMoveUnroll; ++u)
        if (go >> u & 1) base[(size_t)(a.dst + r0 + u * step) * width + c] = v[u];
}

// grid.y: head, grid.z: K, V, totals; a list of at most kMoveWave vectors, one CTA each
__global__ void __launch_bounds__(kMoveThreads, 1)
    smallm_cache_move_short_kernel(float* kc, float* vc, float* totals, uint32_t hd, MoveArgs a, uint32_t list_stride) {
    a.rows += (size_t)blockIdx.y * list_stride;
    pdl_wait();
    if (blockIdx.z == 2) {
        move_rows<float>(totals + (size_t)blockIdx.y * a.max_ctx, 1, a);
    } else {
        float* base = (blockIdx.z ? vc : kc) + (size_t)blockIdx.y * a.max_ctx * hd;
        move_rows<float4>(reinterpret_cast<float4*>(base), hd / 4, a);
    }
}

constexpr uint32_t kMoveTotals = kMoveWave / 4 / kMoveThreads;  // rows of a thread in a wave of the narrowest slice
constexpr uint32_t kMoveStarts = 2048;  // waves whose first sources are kept at hand

__device__ __forceinline__ uint32_t ld_acquire_cluster(const uint32_t* p) {
    uint32_t v;
    asm volatile("ld.acquire.cluster.shared::cta.u32 %0, [%1];" : "=r"(v) : "r"(smem_u32(p)) : "memory");
    return v;
}
// *p of CTA `rank` = v
__device__ __forceinline__ void st_release_cluster(const uint32_t* p, uint32_t rank, uint32_t v) {
    uint32_t at;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(p)), "r"(rank));
    asm volatile("st.release.cluster.shared::cluster.u32 [%0], %1;" ::"r"(at), "r"(v) : "memory");
}

// grid.x: (slice of columns) x cluster, grid.y: head, grid.z: K, V; `slice`
// float4s of a row.  The first slice of K takes the totals along.
__global__ void __launch_bounds__(kMoveThreads, 2)
    smallm_cache_move_kernel(float* kc, float* vc, float* totals, uint32_t hd, uint32_t slice, MoveArgs a,
                             uint32_t list_stride) {
    __shared__ uint32_t start[kMoveStarts];
    __shared__ uint32_t loaded[kMoveMaxCluster];  // waves that each CTA has loaded
    __shared__ uint32_t stuck;
    cg::cluster_group cluster = cg::this_cluster();
    const uint32_t C = cluster.num_blocks(), cr = cluster.block_rank(), tid = threadIdx.x;
    a.rows += (size_t)blockIdx.y * list_stride;
    const uint32_t per = kMoveWave / slice, wave = per * C;  // rows of a CTA and of the cluster in a wave
    const uint32_t waves = (a.n_rows + wave - 1) / wave;
    pdl_wait();
    for (uint32_t w = tid; w < min(waves, kMoveStarts); w += kMoveThreads) start[w] = __ldg(a.rows + w * wave);
    if (tid < kMoveMaxCluster) loaded[tid] = 0;
    if (tid == 0) stuck = 0;
    float4* base = reinterpret_cast<float4*>((blockIdx.z ? vc : kc) + (size_t)blockIdx.y * a.max_ctx * hd) +
                   blockIdx.x / C * slice + tid % slice;
    const uint32_t pitch = hd / 4, step = kMoveThreads / slice, own = tid / slice;
    totals = totals && blockIdx.z == 0 && blockIdx.x < C ? totals + (size_t)blockIdx.y * a.max_ctx : nullptr;
    // the next wave's source rows, and which of them move (for the others the
    // list's last row, which is never overwritten, is read and dropped: loads
    // without conditions)
    const uint32_t end_row = move_source(a, a.n_rows - 1);
    uint32_t src[kMoveUnroll], next = 0;
    auto sources = [&](uint32_t w) {
        const uint32_t first = w * wave + cr * per;
        next = 0;
#pragma unroll
        for (int u = 0; u < kMoveUnroll; ++u) {
            const uint32_t i = first + own + u * step;
            src[u] = move_source(a, min(i, a.n_rows - 1));
            if (i < a.n_rows && src[u] != a.dst + i) next |= 1u << u;
            else src[u] = end_row;
        }
    };
    sources(0);
    cluster.sync();
    uint32_t need = 0;  // the last wave with a source below this part's end
    for (uint32_t w = 0; w < waves; ++w) {
        const uint32_t first = w * wave + cr * per;
        float4 v[kMoveUnroll];
        const uint32_t go = next;
        uint32_t seen = 0;
#pragma unroll
        for (int u = 0; u < kMoveUnroll; ++u) v[u] = __ldcs(&base[(size_t)src[u] * pitch]);
        float total[kMoveTotals] = {};
        if (totals) {
#pragma unroll
            for (int u = 0; u < (int)kMoveTotals; ++u) {
                const uint32_t j = tid + u * kMoveThreads;
                if (j < per && first + j < a.n_rows) {
                    total[u] = totals[move_source(a, first + j)];
                    seen |= __float_as_uint(total[u]);
                }
            }
        }
        if (w + 1 < waves) sources(w + 1);
#pragma unroll
        for (int u = 0; u < kMoveUnroll; ++u)
            seen |= __float_as_uint(v[u].x) | __float_as_uint(v[u].y) | __float_as_uint(v[u].z) | __float_as_uint(v[u].w);
        // every thread's loads have returned (their values are in `seen`)
        asm volatile(
            "{\n .reg .pred p, q;\n setp.ne.u32 p, %0, 0;\n barrier.cta.red.or.pred q, 0, p;\n}" ::"r"(seen) : "memory");
        if (tid < 32) {
            if (tid < C) st_release_cluster(&loaded[cr], tid, w + 1);
            const uint32_t end = a.dst + min(a.n_rows, first + per);
            while (need < w && (need + 1 >= kMoveStarts || start[need + 1] < end)) ++need;
            const long long t0 = clock64();
            for (;;) {
                const bool behind = tid < C && ld_acquire_cluster(&loaded[tid]) <= need;
                if (!__any_sync(0xffffffffu, behind)) break;
                if (__any_sync(0xffffffffu, clock64() - t0 > (1ll << 31))) {
                    if (tid == 0) stuck = 1;
                    break;
                }
            }
        }
        __syncthreads();
        if (stuck) continue;
#pragma unroll
        for (int u = 0; u < kMoveUnroll; ++u)
            if (go >> u & 1) __stcs(&base[(size_t)(a.dst + first + own + u * step) * pitch], v[u]);
        if (totals) {
#pragma unroll
            for (int u = 0; u < (int)kMoveTotals; ++u) {
                const uint32_t j = tid + u * kMoveThreads;
                if (j < per && first + j < a.n_rows) totals[a.dst + first + j] = total[u];
            }
        }
    }
    if (tid == 0 && stuck) atomicOr(a.err, kErrMoveWait);
    cluster.sync();  // peers may still write here
}

// Clusters of C CTAs that run at once on the current device (asked once for
// each kernel, size and device).
uint32_t clusters_at_once(const void* fn, uint32_t C, uint32_t threads, size_t smem) {
    static std::mutex mu;
    static std::map<std::tuple<int, const void*, uint32_t, size_t>, uint32_t> known;
    int dev = 0;
    SM_CUDA(cudaGetDevice(&dev));
    std::lock_guard<std::mutex> g(mu);
    const auto key = std::make_tuple(dev, fn, C, smem);
    const auto it = known.find(key);
    if (it != known.end()) return it->second;
    if (C > 8) allow_large_clusters_once(fn);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(C);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = C;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    int n = 0;
    SM_CUDA(cudaOccupancyMaxActiveClusters(&n, fn, &cfg));
    return known[key] = (uint32_t)n;
}

}  // namespace

void launch_cache_select(const float* weights, uint32_t n_kv, uint32_t max_ctx, uint32_t n, uint32_t n_keep,
                         uint32_t n_first, uint32_t n_last, uint32_t* rows, cudaStream_t stream) {
    if (n > max_ctx) throw Error(SMALLM_ERR_RANGE, "cache_select: n must not pass max_ctx");
    if (n_keep > n || (uint64_t)n_first + n_last > n_keep)
        throw Error(SMALLM_ERR_INVALID, "cache_select: needs n_first + n_last <= n_keep <= n");
    if (n_kv > 65535) throw Error(SMALLM_ERR_RANGE, "cache_select: at most 65535 KV heads");
    if (n > kCacheMaxRows) throw Error(SMALLM_ERR_RANGE, "cache_select: at most 2^30 rows");
    if ((reinterpret_cast<uintptr_t>(weights) | reinterpret_cast<uintptr_t>(rows)) & 3u)
        throw Error(SMALLM_ERR_INVALID, "cache_select: weights and rows must be 4-byte aligned");
    if (!n_kv || !n_keep) return;
    // CTAs per head: one up to 8 keys a thread (4 x 2500 keys 6.7 us, two CTAs
    // 8.4 us), then clusters of 4 to 16 with as many a thread (8 x 8192: 8.5 us by
    // four CTAs, 9.8 by two, 10.1 by one; 8 x 32768: 11.0 us by 8, 14.0 by 16);
    // two CTAs per SM in all, and no cluster left waiting for another to end
    // (64 x 8192: 11.5 us by four CTAs, 23.9 by eight in two rounds; where a
    // CTA's keys then do not fit shared memory two rounds would be better:
    // 64 x 131072 80 us by four CTAs, 62 us by eight)
    const uint32_t m = n - n_first - n_last, sms = (uint32_t)device_sm_count();
    const void* fn = (const void*)smallm_cache_select_kernel;
    set_smem_limit_once(fn, (int)(4 * kSelCached));
    uint32_t C = 1;
    while (C < kSelMaxCluster && m > C * 8 * kSelThreads && n_kv * C <= sms) C *= C == 1 ? 4 : 2;
    while (C > 1 && clusters_at_once(fn, C, kSelThreads, 4 * kSelCached) < n_kv) C /= 2;
    uint32_t per_cta = (m + C - 1) / C, cached = per_cta <= kSelCached;
    void* args[] = {&weights, &max_ctx, &n, &n_keep, &n_first, &n_last, &per_cta, &cached, &rows};
    launch_cluster_ex(fn, dim3(n_kv * C), dim3(kSelThreads), cached ? 4ull * per_cta : 0, C, stream, args);
}

void launch_cache_move(float* kcache, float* vcache, float* weights, uint32_t n_kv, uint32_t hd, uint32_t max_ctx,
                       const uint32_t* rows, bool per_head, uint32_t n_rows, uint32_t dst, cudaStream_t stream) {
    if (hd != 32 && hd != 64 && hd != 128)
        throw Error(SMALLM_ERR_INVALID, "cache_move: head_dim must be 32, 64 or 128");
    if ((uint64_t)dst + n_rows > max_ctx)
        throw Error(SMALLM_ERR_RANGE, "cache_move: dst + n_rows must not pass max_ctx");
    if (n_kv > 65535) throw Error(SMALLM_ERR_RANGE, "cache_move: at most 65535 KV heads");
    if (n_rows > kCacheMaxRows) throw Error(SMALLM_ERR_RANGE, "cache_move: at most 2^30 rows");
    if ((reinterpret_cast<uintptr_t>(kcache) | reinterpret_cast<uintptr_t>(vcache)) & 15u)
        throw Error(SMALLM_ERR_INVALID, "cache_move: kcache and vcache must be 16-byte aligned");
    if ((reinterpret_cast<uintptr_t>(weights) | reinterpret_cast<uintptr_t>(rows)) & 3u)
        throw Error(SMALLM_ERR_INVALID, "cache_move: weights and rows must be 4-byte aligned");
    if (!n_kv || !n_rows) return;
    MoveArgs a{rows, n_rows, dst, max_ctx, device_error_flag()};
    uint32_t stride = per_head ? n_rows : 0;
    if ((uint64_t)n_rows * hd / 4 <= kMoveWave) {
        void* args[] = {&kcache, &vcache, &weights, &hd, &a, &stride};
        launch_kernel_ex((const void*)smallm_cache_move_short_kernel, dim3(1, n_kv, weights ? 3 : 2),
                         dim3(kMoveThreads), 0, stream, true, args);
        return;
    }
    // CTAs of a cluster: a wave's part each at least; then slices of columns (64
    // bytes at least) until there are two CTAs per SM; no cluster left waiting
    // for another to end
    const uint32_t sms = (uint32_t)device_sm_count();
    const void* fn = (const void*)smallm_cache_move_kernel;
    uint32_t C = 1, slices = 1;
    while (C < kMoveMaxCluster && (uint64_t)n_rows * hd / 4 > (uint64_t)C * kMoveWave && n_kv * 4 * C <= 2 * sms) C *= 2;
    while (hd / slices > 16 && n_kv * 4 * C * slices <= 2 * sms) slices *= 2;
    while (C > 1 && clusters_at_once(fn, C, kMoveThreads, 0) < 2 * n_kv * slices) C /= 2;
    uint32_t slice = hd / 4 / slices;
    void* args[] = {&kcache, &vcache, &weights, &hd, &slice, &a, &stride};
    launch_cluster_ex(fn, dim3(slices * C, n_kv, 2), dim3(kMoveThreads), 0, C, stream, args);
}

}  // namespace smallm
