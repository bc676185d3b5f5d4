// Keeping a KV cache within its budget: which rows of each KV head to keep,
// and the in-place move that closes the gaps.
//
// select: of rows 0..n-1 of a KV head keep the first n_first, the last n_last
// and, of those between, the n_keep - n_first - n_last with the largest totals
// (equal totals: the lower row; NaN below everything).  A cluster of up to 16
// CTAs owns a head, each a contiguous range of its keys in shared memory.  The
// k-th largest key is found digit by digit (11, 11 and 10 bits, most
// significant first): histograms of the keys that match the digits so far,
// summed over the cluster's shared memory, then the bin that holds the rank.
// 11 bits take in two of the mantissa, so that totals within a few powers of
// two do not all count into the same bins.  Every larger key is kept, and of
// the equal ones the first few in row order; rows come out ascending.  Bound by
// latency: one read of the totals and four cluster barriers.
//
// move: row dst + i of K and V (and the totals) becomes row rows[i], for a
// strictly ascending list with rows[i] >= dst + i.  In place: a cluster owns
// one head's K or V and walks the list in waves, all of a wave's rows read
// before any is written, by a cluster barrier.  A later wave's source rows[j],
// j >= i, is at least dst + j, so no store of an earlier wave can have
// overwritten it, and its reads run while the wave before is written.
//   - up to a wave of one CTA (an accepted path): rows pass through registers;
//   - longer lists: rows arrive in two shared-memory buffers by a bulk copy
//     each, and leave, being neighbours now, by one bulk copy of the buffer.
//     Bound by the bytes moved (registers instead of bulk copies: %MOVE_REG%).
#include <cooperative_groups.h>

#include <algorithm>

#include "common.cuh"
#include "engine.h"
#include "smallm_cuda.h"

namespace smallm {
namespace {

namespace cg = cooperative_groups;

constexpr int kSelThreads = 1024;
constexpr int kSelWarps = kSelThreads / 32;
constexpr uint32_t kSelBins = 2048;
constexpr uint32_t kSelCached = 40960;  // keys of a CTA that fit shared memory
constexpr uint32_t kSelMaxCluster = 16;

// Order-preserving key, NaN lowest, -0 equal to +0.
__device__ __forceinline__ uint32_t total_key(float x) { return x == x ? float_order_key(x + 0.f) : 0u; }

struct SelShared {
    uint32_t hist[3][kSelBins];
    uint32_t warp[kSelWarps];
    uint32_t warp_eq[kSelWarps];
    uint32_t digit, rank, above;
    uint32_t gt, eq;  // this CTA's keys above / equal to the k-th largest
};

__global__ void __launch_bounds__(kSelThreads, 1)
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
    for (uint32_t i = tid; i < 3 * kSelBins; i += kSelThreads) (&sh.hist[0][0])[i] = 0;
    if (cached) {
#pragma unroll 8
        for (uint32_t i = tid; i < len; i += kSelThreads) cache[i] = total_key(w[i]);
    }
    auto key_of = [&](uint32_t i) { return cached ? cache[i] : total_key(w[i]); };
    __syncthreads();
    uint32_t prefix = 0, want = k, my_gt = 0;
    for (int pass = 0; pass < 3; ++pass) {
        const int shift = pass == 0 ? 21 : (pass == 1 ? 10 : 0);
        const uint32_t bins = pass == 2 ? 1024u : 2048u;
        const uint32_t high = pass == 0 ? 0u : (pass == 1 ? 0xFFFFFFFFu << 21 : 0xFFFFFFFFu << 10);
        uint32_t* hist = sh.hist[pass];
#pragma unroll 4
        for (uint32_t i = tid; i < len; i += kSelThreads) {
            const uint32_t key = key_of(i);
            if ((key & high) == prefix) atomicAdd(&hist[(key >> shift) & (bins - 1)], 1u);
        }
        if (C > 1) cluster.sync();
        else __syncthreads();
        // thread t: bins 2t', 2t'+1 counted from the top
        const uint32_t top = bins - 2 - 2 * tid;
        uint2 sum = make_uint2(0, 0), own = make_uint2(0, 0);
        if (2u * tid < bins) {
            own = *reinterpret_cast<const uint2*>(&hist[top]);
            sum = own;
            // all peers' reads in flight at once
#pragma unroll
            for (uint32_t r = 1; r < kSelMaxCluster; ++r)
                if (r < C) {
                    const uint32_t peer = cr + r < C ? cr + r : cr + r - C;
                    const uint2 v = *reinterpret_cast<const uint2*>(cluster.map_shared_rank(&hist[top], peer));
                    sum.x += v.x;
                    sum.y += v.y;
                }
        }
        // inclusive scan of the pairs from the top: keys in this pair's bins or above
        uint32_t incl = sum.x + sum.y, iown = own.x + own.y;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t y = __shfl_up_sync(0xffffffffu, incl, o), z = __shfl_up_sync(0xffffffffu, iown, o);
            if (lane >= o) incl += y, iown += z;
        }
        if (lane == 31) {
            sh.warp[warp] = incl;
            sh.warp_eq[warp] = iown;
        }
        __syncthreads();
        uint32_t before = incl - sum.x - sum.y, obefore = iown - own.x - own.y;
        before += __reduce_add_sync(0xffffffffu, lane < warp ? sh.warp[lane] : 0u);
        obefore += __reduce_add_sync(0xffffffffu, lane < warp ? sh.warp_eq[lane] : 0u);
        // the bin where the count from the top reaches `want`
        if (before < want && want <= before + sum.x + sum.y) {
            const bool up = want <= before + sum.y;  // the higher bin of the pair
            sh.digit = top + (up ? 1 : 0);
            sh.rank = want - before - (up ? 0 : sum.y);
            sh.above = obefore + (up ? 0 : own.y);
        }
        __syncthreads();
        prefix |= sh.digit << shift;
        want = sh.rank;
        my_gt += sh.above;  // this CTA's keys in higher bins
    }
    // keys above `prefix` are kept, and the first `want` of the head that equal it
    if (tid == 0) {
        sh.gt = my_gt;
        sh.eq = sh.hist[2][prefix & 1023u];
    }
    if (C > 1) cluster.sync();
    else __syncthreads();
    // keys of the ranges before this one (lane r: CTA r)
    uint32_t gt0 = 0, eq0 = 0;
    if ((uint32_t)lane < cr) {
        const SelShared* o = cluster.map_shared_rank(&sh, lane);
        gt0 = o->gt;
        eq0 = o->eq;
    }
    gt0 = __reduce_add_sync(0xffffffffu, gt0);
    eq0 = __reduce_add_sync(0xffffffffu, eq0);
    // each warp owns a contiguous run of the range
    const uint32_t run = (len + kSelThreads - 1) / kSelThreads * 32;
    const uint32_t wb = min(len, warp * run), we = min(len, wb + run);
    uint32_t cg_ = 0, ce = 0;
    for (uint32_t i = wb + lane; i - lane < we; i += 32) {
        const uint32_t key = i < we ? key_of(i) : 0u;
        cg_ += __popc(__ballot_sync(0xffffffffu, i < we && key > prefix));
        ce += __popc(__ballot_sync(0xffffffffu, i < we && key == prefix));
    }
    if (lane == 0) {
        sh.warp[warp] = cg_;
        sh.warp_eq[warp] = ce;
    }
    __syncthreads();
    gt0 += __reduce_add_sync(0xffffffffu, lane < warp ? sh.warp[lane] : 0u);
    eq0 += __reduce_add_sync(0xffffffffu, lane < warp ? sh.warp_eq[lane] : 0u);
    const uint32_t lt = (1u << lane) - 1u;
    for (uint32_t i = wb + lane; i - lane < we; i += 32) {
        const uint32_t key = i < we ? key_of(i) : 0u;
        const bool gt = i < we && key > prefix, eq = i < we && key == prefix;
        const uint32_t bg = __ballot_sync(0xffffffffu, gt), be = __ballot_sync(0xffffffffu, eq);
        const uint32_t g = gt0 + __popc(bg & lt), e = eq0 + __popc(be & lt);
        if (gt || (eq && e < want)) out[n_first + g + min(e, want)] = n_first + b0 + i;
        gt0 += __popc(bg);
        eq0 += __popc(be);
    }
    if (C > 1) cluster.sync();  // a peer may still read this CTA's counts
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

constexpr uint32_t kMoveBuf = 96 * 1024;  // bytes of one of a CTA's two buffers

// grid.x: the cluster's CTAs, grid.y: head, grid.z: K, V
__global__ void __launch_bounds__(kMoveThreads, 1)
    smallm_cache_move_kernel(float* kc, float* vc, uint32_t hd, MoveArgs a, uint32_t list_stride) {
    extern __shared__ __align__(128) uint8_t buf[];
    __shared__ __align__(8) uint64_t full[2];
    cg::cluster_group cluster = cg::this_cluster();
    const uint32_t C = cluster.num_blocks(), cr = cluster.block_rank();
    const int tid = threadIdx.x;
    a.rows += (size_t)blockIdx.y * list_stride;
    if (tid == 0) {
        mbar_init(&full[0], 1);
        mbar_init(&full[1], 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    float* base = (blockIdx.z ? vc : kc) + (size_t)blockIdx.y * a.max_ctx * hd;
    const uint32_t row = hd * 4, per = kMoveBuf / row;  // bytes of a row; rows of a CTA per wave
    const uint32_t waves = (a.n_rows + per * C - 1) / (per * C);
    // this CTA's entries of wave w
    auto range = [&](uint32_t w, uint32_t& first, uint32_t& count) {
        first = min(a.n_rows, (w * C + cr) * per);
        count = min(a.n_rows - first, per);
    };
    auto fetch = [&](uint32_t w) {
        uint32_t first, count;
        range(w, first, count);
        uint64_t* bar = &full[w & 1];
        if (tid == 0) {
            if (count) mbar_arrive_expect_tx(bar, count * row);
            else mbar_arrive(bar);
        }
        for (uint32_t i = tid; i < count; i += kMoveThreads)
            bulk_g2s(buf + (w & 1) * kMoveBuf + i * row, base + (size_t)move_source(a, first + i) * hd, row, bar);
    };
    fetch(0);
    bool ok = true;
    for (uint32_t w = 0; w < waves; ++w) {
        if (w + 1 < waves) {
            // the other buffer's rows have left
            if (w && tid == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
            __syncthreads();
            fetch(w + 1);
        }
        // (a second wait after one that gave up: no copy lands in a CTA that has left)
        ok = (mbar_wait(&full[w & 1], w >> 1 & 1) || (mbar_wait(&full[w & 1], w >> 1 & 1), false)) && ok;
        ok = !__syncthreads_or(!ok);
        if (C > 1) cluster.sync();  // every row of the wave has been read
        else __syncthreads();
        uint32_t first, count;
        range(w, first, count);
        if (ok && count && tid == 0) {
            asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(
                             base + (size_t)(a.dst + first) * hd),
                         "r"(smem_u32(buf + (w & 1) * kMoveBuf)), "r"(count * row)
                         : "memory");
            asm volatile("cp.async.bulk.commit_group;" ::: "memory");
        }
    }
    if (tid == 0) {
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

}  // namespace

void launch_cache_select(const float* weights, uint32_t n_kv, uint32_t max_ctx, uint32_t n, uint32_t n_keep,
                         uint32_t n_first, uint32_t n_last, uint32_t* rows, cudaStream_t stream) {
    if (n > max_ctx) throw Error(SMALLM_ERR_RANGE, "cache_select: n must not pass max_ctx");
    if (n_keep > n || (uint64_t)n_first + n_last > n_keep)
        throw Error(SMALLM_ERR_INVALID, "cache_select: needs n_first + n_last <= n_keep <= n");
    if (n_kv > 65535) throw Error(SMALLM_ERR_RANGE, "cache_select: at most 65535 KV heads");
    if (!n_kv || !n_keep) return;
    // CTAs per head: a couple of keys per thread at least, one CTA per SM in all
    const uint32_t m = n - n_first - n_last, sms = (uint32_t)device_sm_count();
    uint32_t C = 1;
    while (C < kSelMaxCluster && m > C * 2 * kSelThreads && n_kv * C * 2 <= sms) C *= 2;
    uint32_t per_cta = (m + C - 1) / C, cached = per_cta <= kSelCached;
    const void* fn = (const void*)smallm_cache_select_kernel;
    set_smem_limit_once(fn, (int)(4 * kSelCached));
    if (C > 8) SM_CUDA(cudaFuncSetAttribute(fn, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
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
    // CTAs of a cluster: a buffer each at least, one CTA per SM in all
    const uint32_t sms = (uint32_t)device_sm_count();
    uint32_t C = 1;
    while (C < kMoveMaxCluster && (uint64_t)n_rows * hd * 4 > (uint64_t)C * kMoveBuf && n_kv * 2 * C * 2 <= sms) C *= 2;
    const void* fn = (const void*)smallm_cache_move_kernel;
    set_smem_limit_once(fn, (int)(2 * kMoveBuf));
    if (C > 8) SM_CUDA(cudaFuncSetAttribute(fn, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    void* args[] = {&kcache, &vcache, &hd, &a, &stride};
    launch_cluster(fn, dim3(C, n_kv, 2), kMoveThreads, 2 * kMoveBuf, C, stream, args, weights != nullptr);
}

}  // namespace smallm
