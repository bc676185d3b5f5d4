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
// takes %SEL_US%.)  Every larger key is kept, and of the equal ones the first few
// in row order; rows come out ascending.  Bound by latency: one read of the
// totals and five cluster barriers.
//
// move: row dst + i of K and V (and the totals) becomes row rows[i], for a
// strictly ascending list with rows[i] >= dst + i.  In place: a cluster owns
// one head's K or V and walks the list in waves, all of a wave's rows read
// before any is written, by a cluster barrier.  A later wave's source rows[j],
// j >= i, is at least dst + j, so no store of an earlier wave can have
// overwritten it, and its reads run while the wave before is written.
//   - up to a wave of one CTA (an accepted path): rows pass through registers;
//   - longer lists: rows arrive in shared memory by bulk copies, one for each
//     run of neighbours, and leave, being neighbours now, by one bulk copy of a
//     buffer.  One warp per CTA, four buffers of 16 KB, three of them on their
//     way in while the barrier of the wave before is waited for.  Bound by the
//     bytes moved.  8 heads x 16384 of 32768 rows of 128: %MOVE_US%; two buffers
//     of 48 KB and 512 threads 88 us, through registers 166 us.
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
    if (cr == 0) {
        for (uint32_t i = tid; i < n_first; i += kSelThreads) out[i] = i;
        for (uint32_t i = tid; i < n_last; i += kSelThreads) out[n_first + k + i] = n - n_last + i;
    }
    if (!k) return;
    for (uint32_t i = tid; i < kSelPasses * kSelBins; i += kSelThreads) (&sh.hist[0][0])[i] = 0;
    if (cached) {
#pragma unroll 16
        for (uint32_t i = tid; i < len; i += kSelThreads) cache[i] = total_key(__ldg(w + i));
    }
    auto key_of = [&](uint32_t i) { return cached ? cache[i] : total_key(w[i]); };
    __syncthreads();
    uint32_t prefix = 0, want = k, my_gt = 0;
    for (int pass = 0; pass < kSelPasses; ++pass) {
        const int shift = pass == 0 ? 23 : (pass == 1 ? 15 : (pass == 2 ? 7 : 0));
        const uint32_t bins = pass == 0 ? 512u : (pass == 3 ? 128u : 256u);
        const uint32_t high = pass == 0 ? 0u : ~(bins * (1u << shift) - 1u);
        uint32_t* hist = sh.hist[pass];
        for (uint32_t i = tid; i - lane < len; i += kSelThreads) {
            const uint32_t key = i < len ? key_of(i) : 0u;
            const bool in = i < len && (key & high) == prefix;
            const uint32_t bin = key >> shift & (bins - 1);
            const uint32_t act = __ballot_sync(0xffffffffu, in);
            if (!act) continue;
            // a warp whose keys share a bin (like totals) counts once
            const uint32_t lead = __shfl_sync(0xffffffffu, bin, __ffs(act) - 1);
            if (__all_sync(0xffffffffu, !in || bin == lead)) {
                if (lane == 0) atomicAdd(&hist[lead], __popc(act));
            } else if (in) {
                atomicAdd(&hist[bin], 1u);
            }
        }
        if (C > 1) cluster.sync();
        else __syncthreads();
        // thread t: four bins, counted from the top
        const uint32_t top = bins - 4 - 4 * tid;
        uint4 sum = make_uint4(0, 0, 0, 0), own = sum;
        if (4u * tid < bins) {
            own = *reinterpret_cast<const uint4*>(&hist[top]);
            sum = own;
            // all peers' reads in flight at once
#pragma unroll
            for (uint32_t r = 1; r < kSelMaxCluster; ++r)
                if (r < C) {
                    const uint32_t peer = cr + r < C ? cr + r : cr + r - C;
                    const uint4 v = *reinterpret_cast<const uint4*>(cluster.map_shared_rank(&hist[top], peer));
                    sum.x += v.x, sum.y += v.y, sum.z += v.z, sum.w += v.w;
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
        const uint32_t key = i < we ? key_of(i) : 0u;
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
        const uint32_t key = i < we ? key_of(i) : 0u;
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
constexpr uint32_t kMoveMaxCluster = 16;
constexpr unsigned kErrMoveList = 128u, kErrMoveWait = 512u;

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
// of type V), by a cluster of C CTAs that take consecutive parts of a wave.
template <typename V>
__device__ __forceinline__ void move_rows(V* base, uint32_t width, const MoveArgs& a, uint32_t C, uint32_t cr) {
    const uint32_t wave = kMoveWave * C / width;  // rows per wave (width divides kMoveThreads)
    const uint32_t c = threadIdx.x % width, r0 = (cr * kMoveWave + threadIdx.x) / width, step = kMoveThreads / width;
    for (uint32_t first = 0; first < a.n_rows; first += wave) {
        V v[kMoveUnroll];
        uint32_t go = 0;
#pragma unroll
        for (int u = 0; u < kMoveUnroll; ++u) {
            const uint32_t i = first + r0 + u * step;
            if (i >= a.n_rows) continue;
            const uint32_t src = move_source(a, i);
            if (src == a.dst + i) continue;
            v[u] = base[(size_t)src * width + c];
            go |= 1u << u;
        }
        if (C > 1) cg::this_cluster().sync();
        else __syncthreads();
#pragma unroll
        for (int u = 0; u < kMoveUnroll; ++u)
            if (go >> u & 1) base[(size_t)(a.dst + first + r0 + u * step) * width + c] = v[u];
    }
}

// grid.y: head, grid.z: K, V, totals; a list of at most kMoveWave vectors, one CTA each
__global__ void __launch_bounds__(kMoveThreads, 1)
    smallm_cache_move_short_kernel(float* kc, float* vc, float* totals, uint32_t hd, MoveArgs a, uint32_t list_stride) {
    a.rows += (size_t)blockIdx.y * list_stride;
    if (blockIdx.z == 2) {
        move_rows<float>(totals + (size_t)blockIdx.y * a.max_ctx, 1, a, 1, 0);
    } else {
        float* base = (blockIdx.z ? vc : kc) + (size_t)blockIdx.y * a.max_ctx * hd;
        move_rows<float4>(reinterpret_cast<float4*>(base), hd / 4, a, 1, 0);
    }
}

// The totals of a longer list: a cluster per head.
__global__ void __launch_bounds__(kMoveThreads)
    smallm_cache_move_totals_kernel(float* totals, MoveArgs a, uint32_t list_stride) {
    pdl_launch_dependents();  // K and V do not wait for the totals
    cg::cluster_group cluster = cg::this_cluster();
    a.rows += (size_t)blockIdx.y * list_stride;
    move_rows<float>(totals + (size_t)blockIdx.y * a.max_ctx, 1, a, cluster.num_blocks(), cluster.block_rank());
}

constexpr uint32_t kMoveBuf = 16 * 1024;  // bytes of one of a CTA's buffers
constexpr uint32_t kMoveBufs = 4;         // (three CTAs fit an SM)

// grid.x: the cluster's CTAs (one warp each), grid.y: head, grid.z: K, V
__global__ void __launch_bounds__(32) smallm_cache_move_kernel(float* kc, float* vc, uint32_t hd, MoveArgs a,
                                                             uint32_t list_stride) {
    extern __shared__ __align__(128) uint8_t buf[];
    __shared__ __align__(8) uint64_t full[kMoveBufs];
    cg::cluster_group cluster = cg::this_cluster();
    const uint32_t C = cluster.num_blocks(), cr = cluster.block_rank(), lane = threadIdx.x;
    a.rows += (size_t)blockIdx.y * list_stride;
    if (lane == 0) {
        for (uint32_t b = 0; b < kMoveBufs; ++b) mbar_init(&full[b], 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncwarp();
    float* base = (blockIdx.z ? vc : kc) + (size_t)blockIdx.y * a.max_ctx * hd;
    const uint32_t row = hd * 4, per = kMoveBuf / row;  // bytes of a row; rows of a CTA per wave (32, 64 or 128)
    const uint32_t waves = (a.n_rows + per * C - 1) / (per * C);
    // this CTA's entries of wave w
    auto range = [&](uint32_t w, uint32_t& first, uint32_t& count) {
        first = min(a.n_rows, (w * C + cr) * per);
        count = min(a.n_rows - first, per);
    };
    uint32_t src[4];  // the lane's entries of the wave that is fetched next
    auto sources = [&](uint32_t w) {
        uint32_t first, count;
        range(w, first, count);
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (32 * j + lane < count) src[j] = move_source(a, first + 32 * j + lane);
    };
    auto fetch = [&](uint32_t w) {
        uint32_t first, count;
        range(w, first, count);
        uint64_t* bar = &full[w % kMoveBufs];
        if (lane == 0) {
            if (count) mbar_arrive_expect_tx(bar, count * row);
            else mbar_arrive(bar);
        }
        __syncwarp();
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (32 * j >= count) break;
            // neighbours travel in one copy
            const bool in = 32 * j + lane < count;
            const uint32_t left = __shfl_up_sync(0xffffffffu, src[j], 1);
            const uint32_t heads = __ballot_sync(0xffffffffu, in && (lane == 0 || src[j] != left + 1));
            if (!(heads >> lane & 1)) continue;
            const uint32_t more = heads & ~((2u << lane) - 1u);  // the next run's first lane
            const uint32_t len = min(more ? __ffs(more) - 1 - lane : 32u - lane, count - 32 * j - lane);
            bulk_g2s(buf + (w % kMoveBufs) * kMoveBuf + (32 * j + lane) * row, base + (size_t)src[j] * hd, len * row, bar);
        }
        __syncwarp();
    };
    for (uint32_t w = 0; w < min(waves, kMoveBufs - 1); ++w) {
        sources(w);
        fetch(w);
    }
    if (kMoveBufs - 1 < waves) sources(kMoveBufs - 1);
    bool ok = true;
    for (uint32_t w = 0; w < waves; ++w) {
        // (a second wait after one that gave up: no copy lands in a CTA that has left)
        uint64_t* bar = &full[w % kMoveBufs];
        const uint32_t parity = w / kMoveBufs & 1;
        ok = (mbar_wait(bar, parity) || (mbar_wait(bar, parity), false)) && ok;
        ok = __all_sync(0xffffffffu, ok);
        cluster_arrive_release();  // this CTA's rows of the wave have been read
        const uint32_t next = w + kMoveBufs - 1;
        if (next < waves) {
            // the buffer's rows of wave w - 1 have left
            if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
            __syncwarp();
            fetch(next);
            if (next + 1 < waves) sources(next + 1);
        }
        cluster_wait();  // everybody's have
        uint32_t first, count;
        range(w, first, count);
        if (ok && count && lane == 0) {
            asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(
                             base + (size_t)(a.dst + first) * hd),
                         "r"(smem_u32(buf + (w % kMoveBufs) * kMoveBuf)), "r"(count * row)
                         : "memory");
            asm volatile("cp.async.bulk.commit_group;" ::: "memory");
        }
        __syncwarp();
    }
    if (lane == 0) {
        asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
        if (!ok) atomicOr(a.err, kErrMoveWait);
    }
    pdl_wait();  // this kernel ends after the totals' (where there is one before it)
}

void launch_cluster(const void* fn, dim3 grid, uint32_t threads, size_t smem, uint32_t C, cudaStream_t stream,
                    void** args, bool pdl = false) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = C;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl ? 2 : 1;
    SM_CUDA(cudaLaunchKernelExC(&cfg, fn, args));
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
    if (C > 8) SM_CUDA(cudaFuncSetAttribute(fn, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
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
    if (!n_kv || !n_keep) return;
    // CTAs per head: a couple of keys per thread at least, two CTAs per SM in
    // all, and no cluster left waiting for another to end
    const uint32_t m = n - n_first - n_last, sms = (uint32_t)device_sm_count();
    const void* fn = (const void*)smallm_cache_select_kernel;
    set_smem_limit_once(fn, (int)(4 * kSelCached));
    uint32_t C = 1;
    while (C < kSelMaxCluster && m > C * 2 * kSelThreads && n_kv * C <= sms) C *= 2;
    while (C > 1 && clusters_at_once(fn, C, kSelThreads, 4 * kSelCached) < n_kv) C /= 2;
    uint32_t per_cta = (m + C - 1) / C, cached = per_cta <= kSelCached;
    void* args[] = {&weights, &max_ctx, &n, &n_keep, &n_first, &n_last, &per_cta, &cached, &rows};
    launch_cluster(fn, dim3(n_kv * C), kSelThreads, cached ? 4ull * per_cta : 0, C, stream, args);
}

void launch_cache_move(float* kcache, float* vcache, float* weights, uint32_t n_kv, uint32_t hd, uint32_t max_ctx,
                       const uint32_t* rows, bool per_head, uint32_t n_rows, uint32_t dst, cudaStream_t stream) {
    if (hd != 32 && hd != 64 && hd != 128)
        throw Error(SMALLM_ERR_INVALID, "cache_move: head_dim must be 32, 64 or 128");
    if ((uint64_t)dst + n_rows > max_ctx)
        throw Error(SMALLM_ERR_RANGE, "cache_move: dst + n_rows must not pass max_ctx");
    if (n_kv > 65535) throw Error(SMALLM_ERR_RANGE, "cache_move: at most 65535 KV heads");
    if ((reinterpret_cast<uintptr_t>(kcache) | reinterpret_cast<uintptr_t>(vcache)) & 15u)
        throw Error(SMALLM_ERR_INVALID, "cache_move: kcache and vcache must be 16-byte aligned");
    if (!n_kv || !n_rows) return;
    MoveArgs a{rows, n_rows, dst, max_ctx, device_error_flag()};
    uint32_t stride = per_head ? n_rows : 0;
    if ((uint64_t)n_rows * hd / 4 <= kMoveWave) {
        void* args[] = {&kcache, &vcache, &weights, &hd, &a, &stride};
        launch_kernel_ex((const void*)smallm_cache_move_short_kernel, dim3(1, n_kv, weights ? 3 : 2),
                         dim3(kMoveThreads), 0, stream, false, args);
        return;
    }
    if (weights) {
        uint32_t C = 1;
        while (C < 8 && n_rows > C * kMoveWave) C *= 2;
        void* args[] = {&weights, &a, &stride};
        launch_cluster((const void*)smallm_cache_move_totals_kernel, dim3(C, n_kv), kMoveThreads, 0, C, stream, args);
    }
    // CTAs of a cluster: a buffer each at least, two CTAs per SM in all, and no
    // cluster left waiting for another to end
    const uint32_t sms = (uint32_t)device_sm_count();
    const void* fn = (const void*)smallm_cache_move_kernel;
    set_smem_limit_once(fn, (int)(kMoveBufs * kMoveBuf));
    uint32_t C = 1;
    while (C < kMoveMaxCluster && (uint64_t)n_rows * hd * 4 > (uint64_t)C * kMoveBuf && n_kv * 2 * C <= 2 * sms) C *= 2;
    while (C > 1 && clusters_at_once(fn, C, 32, kMoveBufs * kMoveBuf) < 2 * n_kv) C /= 2;
    void* args[] = {&kcache, &vcache, &hd, &a, &stride};
    launch_cluster(fn, dim3(C, n_kv, 2), 32, kMoveBufs * kMoveBuf, C, stream, args, weights != nullptr);
}

}  // namespace smallm
