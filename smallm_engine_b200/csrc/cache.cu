// Keeping a KV cache within its budget: which rows of each KV head to keep,
// and the in-place move that closes the gaps.
//
// select: of rows 0..n-1 of a KV head keep the first n_first, the last n_last
// and, of those between, the n_keep - n_first - n_last with the largest totals
// (equal totals: the lower row; NaN below everything).  The k-th largest key
// is found digit by digit (8 bits, most significant first, a histogram of the
// keys that match the digits so far); every larger key is kept, and of the
// equal ones the first few in row order.  Rows come out ascending.
//
// move: row dst + i of K and V (and the totals) becomes row rows[i], for a
// strictly ascending list with rows[i] >= dst + i.  In place: a CTA owns a
// slice of columns of one head and walks the list in chunks, all of a chunk's
// loads before any of its stores.  A later chunk's source rows[j], j >= i, is
// at least dst + j, so no store of an earlier chunk can have overwritten it.
#include "common.cuh"
#include "engine.h"
#include "smallm_cuda.h"

namespace smallm {
namespace {

constexpr int kSelThreads = 1024;

// Order-preserving key, NaN lowest, -0 equal to +0.
__device__ __forceinline__ uint32_t total_key(float x) { return x == x ? float_order_key(x + 0.f) : 0u; }

__global__ void __launch_bounds__(kSelThreads)
    smallm_cache_select_kernel(const float* __restrict__ weights, uint32_t stride, uint32_t n, uint32_t n_keep,
                               uint32_t n_first, uint32_t n_last, uint32_t* __restrict__ rows) {
    __shared__ uint32_t hist[256];
    __shared__ uint32_t sh_digit, sh_rank;
    __shared__ uint32_t wsum[2][32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const float* w = weights + (size_t)blockIdx.x * stride + n_first;
    uint32_t* out = rows + (size_t)blockIdx.x * n_keep;
    const uint32_t m = n - n_first - n_last, k = n_keep - n_first - n_last;
    for (uint32_t i = tid; i < n_first; i += kSelThreads) out[i] = i;
    for (uint32_t i = tid; i < n_last; i += kSelThreads) out[n_first + k + i] = n - n_last + i;
    if (!k) return;
    uint32_t prefix = 0, want = k;  // the want-th largest of the keys that match the prefix
    for (int shift = 24; shift >= 0; shift -= 8) {
        for (int i = tid; i < 256; i += kSelThreads) hist[i] = 0;
        __syncthreads();
        const uint32_t high = shift == 24 ? 0u : 0xFFFFFFFFu << (shift + 8);
        for (uint32_t i = tid; i < m; i += kSelThreads) {
            const uint32_t key = total_key(w[i]);
            if ((key & high) == prefix) atomicAdd(&hist[(key >> shift) & 255], 1u);
        }
        __syncthreads();
        if (tid == 0) {
            uint32_t left = want;
            int d = 255;
            for (; d > 0 && hist[d] < left; --d) left -= hist[d];
            sh_digit = (uint32_t)d;
            sh_rank = left;
        }
        __syncthreads();
        prefix |= sh_digit << shift;
        want = sh_rank;
    }
    // keys above `prefix` are kept, and the first `want` that equal it
    uint32_t done_gt = 0, done_eq = 0;
    for (uint32_t b = 0; b < m; b += kSelThreads) {
        const uint32_t i = b + tid;
        const uint32_t key = i < m ? total_key(w[i]) : 0u;
        const bool gt = i < m && key > prefix, eq = i < m && key == prefix;
        const uint32_t bg = __ballot_sync(0xffffffffu, gt), be = __ballot_sync(0xffffffffu, eq);
        if (lane == 0) {
            wsum[0][warp] = __popc(bg);
            wsum[1][warp] = __popc(be);
        }
        __syncthreads();
        uint32_t g0 = done_gt, e0 = done_eq, tg = 0, te = 0;
        for (int v = 0; v < kSelThreads / 32; ++v) {
            if (v < warp) {
                g0 += wsum[0][v];
                e0 += wsum[1][v];
            }
            tg += wsum[0][v];
            te += wsum[1][v];
        }
        const uint32_t lt = (1u << lane) - 1u;
        g0 += __popc(bg & lt);
        e0 += __popc(be & lt);
        if (gt || (eq && e0 < want)) out[n_first + g0 + min(e0, want)] = n_first + i;
        done_gt += tg;
        done_eq += te;
        __syncthreads();
    }
}

constexpr int kMoveThreads = 256;
constexpr int kMoveUnroll = 4;
constexpr unsigned kErrMoveList = 128u;

// Whether entry i of the list may be moved; raises bit 7 of the error word if not.
__device__ __forceinline__ bool move_entry(const uint32_t* rows, uint32_t i, uint32_t dst, uint32_t max_ctx,
                                           unsigned int* err, uint32_t& src) {
    src = __ldg(rows + i);
    const bool ok = src < max_ctx && src >= dst + i && (i == 0 || __ldg(rows + i - 1) < src);
    if (!ok) atomicOr(err, kErrMoveList);
    return ok && src != dst + i;
}

// grid (hd / 16, n_kv, 2): 16 columns of one head of K or V
__global__ void __launch_bounds__(kMoveThreads)
    smallm_cache_move_kernel(float* kc, float* vc, uint32_t hd, uint32_t max_ctx, const uint32_t* __restrict__ lists,
                             uint32_t list_stride, uint32_t n_rows, uint32_t dst, unsigned int* err) {
    const uint32_t* rows = lists + (size_t)blockIdx.y * list_stride;
    float* base = (blockIdx.z ? vc : kc) + (size_t)blockIdx.y * max_ctx * hd + blockIdx.x * 16 + (threadIdx.x & 3) * 4;
    constexpr uint32_t kStep = kMoveThreads / 4;
    for (uint32_t b = 0; b < n_rows; b += kStep * kMoveUnroll) {
        float4 v[kMoveUnroll];
        bool go[kMoveUnroll];
#pragma unroll
        for (int u = 0; u < kMoveUnroll; ++u) {
            const uint32_t i = b + u * kStep + (threadIdx.x >> 2);
            uint32_t src = 0;
            go[u] = i < n_rows && move_entry(rows, i, dst, max_ctx, err, src);
            if (go[u]) v[u] = *reinterpret_cast<const float4*>(base + (size_t)src * hd);
        }
        __syncthreads();
#pragma unroll
        for (int u = 0; u < kMoveUnroll; ++u) {
            const uint32_t i = b + u * kStep + (threadIdx.x >> 2);
            if (go[u]) *reinterpret_cast<float4*>(base + (size_t)(dst + i) * hd) = v[u];
        }
        __syncthreads();
    }
}

__global__ void __launch_bounds__(1024)
    smallm_cache_move_totals_kernel(float* weights, uint32_t max_ctx, const uint32_t* __restrict__ lists,
                                    uint32_t list_stride, uint32_t n_rows, uint32_t dst, unsigned int* err) {
    const uint32_t* rows = lists + (size_t)blockIdx.x * list_stride;
    float* w = weights + (size_t)blockIdx.x * max_ctx;
    for (uint32_t b = 0; b < n_rows; b += 1024) {
        const uint32_t i = b + threadIdx.x;
        uint32_t src = 0;
        const bool go = i < n_rows && move_entry(rows, i, dst, max_ctx, err, src);
        const float v = go ? w[src] : 0.f;
        __syncthreads();
        if (go) w[dst + i] = v;
        __syncthreads();
    }
}

}  // namespace

void launch_cache_select(const float* weights, uint32_t n_kv, uint32_t max_ctx, uint32_t n, uint32_t n_keep,
                         uint32_t n_first, uint32_t n_last, uint32_t* rows, cudaStream_t stream) {
    if (n > max_ctx) throw Error(SMALLM_ERR_RANGE, "cache_select: n must not pass max_ctx");
    if (n_keep > n || (uint64_t)n_first + n_last > n_keep)
        throw Error(SMALLM_ERR_INVALID, "cache_select: needs n_first + n_last <= n_keep <= n");
    if (n_kv > 65535) throw Error(SMALLM_ERR_RANGE, "cache_select: at most 65535 KV heads");
    if (!n_kv || !n_keep) return;
    smallm_cache_select_kernel<<<n_kv, kSelThreads, 0, stream>>>(weights, max_ctx, n, n_keep, n_first, n_last, rows);
    SM_CUDA(cudaGetLastError());
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
    unsigned int* err = device_error_flag();
    const uint32_t stride = per_head ? n_rows : 0;
    smallm_cache_move_kernel<<<dim3(hd / 16, n_kv, 2), kMoveThreads, 0, stream>>>(kcache, vcache, hd, max_ctx, rows,
                                                                                stride, n_rows, dst, err);
    SM_CUDA(cudaGetLastError());
    if (weights) {
        smallm_cache_move_totals_kernel<<<n_kv, 1024, 0, stream>>>(weights, max_ctx, rows, stride, n_rows, dst, err);
        SM_CUDA(cudaGetLastError());
    }
}

}  // namespace smallm
