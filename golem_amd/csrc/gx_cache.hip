// gx_cache.hip - a conversation's cache entries moved as a whole: a kept path's
// draft entries into the caches, and a conversation's first positions into
// other slots.  Every layer in one launch: the layers' addresses are kernel
// arguments.  Bytes alone, read once.
#include "gx_device.hpp"
#include "gx_internal.hpp"

namespace gx {
namespace {

struct CommitLayers {
    uint16_t *kc[kCacheLayers], *vc[kCacheLayers];
    const uint16_t *kd[kCacheLayers], *vd[kCacheLayers];
};

// grid (kv_heads, trees, layers): node path[b][j] of tree b, draft row first[b]
// + that, becomes position prefix[b] + j of its conversation.  A node or a
// position out of range is left out.
__global__ __launch_bounds__(256) void cache_commit_kernel(const CommitLayers at, int M, int max_nodes,
                                                           const int32_t *__restrict__ first,
                                                           const int32_t *__restrict__ path,
                                                           const int32_t *__restrict__ counts,
                                                           const int32_t *__restrict__ prefix, int hd, int context,
                                                           int draft_context, const int32_t *__restrict__ slots,
                                                           int nslots) {
    __shared__ int from[kTreeNodes];
    const int tid = threadIdx.x, kvh = blockIdx.x, kv_heads = gridDim.x, b = blockIdx.y, layer = blockIdx.z;
    const int f0 = min(max(first[b], 0), M), T = min(min(max(first[b + 1], f0), M) - f0, max_nodes);
    const int count = min(max(counts[b], 0), max_nodes), p0 = prefix[b], slot = slots ? slots[b] : 0;
    if (slot < 0 || slot >= nslots || p0 < 0 || p0 >= context)
        return;
    for (int j = tid; j < count; j += 256) {
        const int node = path[(size_t)b * max_nodes + j];
        from[j] = node >= 0 && node < T && p0 < context - j ? f0 + node : -1;
    }
    __syncthreads();
    const size_t to = ((size_t)slot * kv_heads + kvh) * hd * context, src = (size_t)kvh * hd * draft_context;
    // Consecutive threads take consecutive positions of an element (or of a piece
    // of the keys), whose bytes lie together on both sides; all of a thread's
    // loads before its stores, the values' past the caches (kept there, sixteen
    // paths of twelve through 36 layers take 45 us where this takes 37; the keys'
    // past them too 42).  Of the 37 us the bytes are 15 at a large copy's rate (30
    // MB read and 42 written by the counters where 22 each are wanted: 24 bytes of
    // values and 192 of keys lie together), and the vector instructions, most of
    // them index arithmetic, 11 (5900 a SIMD); the wavefronts spend 44 % of their
    // time waiting for memory and 49 % for their turn to issue.  (An element's
    // positions a thread: each store on a line of its own, 74 us; two positions a
    // word a thread: 46.)
    v4u_stream *kc = (v4u_stream *)(at.kc[layer] + to);
    const v4u_stream *kd = (const v4u_stream *)(at.kd[layer] + src);
    uint16_t *vc = at.vc[layer] + to;
    const uint16_t *vd = at.vd[layer] + src;
    const int keys = hd / 8 * count, values = hd * count;
    for (int k0 = tid, i0 = tid; i0 < values; k0 += 256, i0 += 8 * 256) {
        v4u_stream k;
        uint16_t v[8];
        size_t kpos, vpos[8];
        int krow, vrow[8];
        {
            const int i = min(k0, keys - 1), e = i / count, j = i - e * count;
            krow = k0 < keys ? from[j] : -1;
            kpos = (size_t)e * context + p0 + j;
            k = kd[(size_t)e * draft_context + max(krow, 0)];
        }
#pragma unroll
        for (int u = 0; u < 8; u++) {
            const int i = min(i0 + u * 256, values - 1), e = i / count, j = i - e * count;
            vrow[u] = i0 + u * 256 < values ? from[j] : -1;
            vpos[u] = (size_t)e * context + p0 + j;
            v[u] = vd[(size_t)e * draft_context + max(vrow[u], 0)];
        }
        if (krow >= 0)
            kc[kpos] = k;
#pragma unroll
        for (int u = 0; u < 8; u++)
            if (vrow[u] >= 0)
                __builtin_nontemporal_store(v[u], vc + vpos[u]);
    }
}

struct ForkLayers {
    uint16_t *kc[kCacheLayers], *vc[kCacheLayers];
    int dsts[kForkSlots];
};

// grid (kv_heads * hd / 8, 2, layers): a piece row of the keys (y 0, 16 bytes a
// position) or eight element rows of the values (32 threads each).  Four loads
// a thread before their stores, and one read for all the copies.  At the rate of
// a large copy (4.8 TB/s): 301 positions of 36 layers, 89 MB, in 16 us and four
// copies of 1999, 1.47 GB, in 310.
__global__ __launch_bounds__(256) void cache_fork_kernel(const ForkLayers at, int kv_heads, int hd, int context,
                                                         int src, int n, int len) {
    const int tid = threadIdx.x, layer = blockIdx.z;
    const size_t slot = (size_t)kv_heads * hd * context / 8;  // 16-byte pieces
    const bool keys = blockIdx.y == 0;
    const int row = tid >> 5;
    v4u_stream *base = (v4u_stream *)(keys ? at.kc[layer] + (size_t)blockIdx.x * 8 * context
                                           : at.vc[layer] + ((size_t)blockIdx.x * 8 + row) * context);
    const int count = keys ? len : len / 8, step = keys ? 256 : 32;
    const v4u_stream *from = base + src * slot;
    for (int i0 = keys ? tid : tid & 31; i0 < count; i0 += 4 * step) {
        v4u_stream v[4];
#pragma unroll
        for (int u = 0; u < 4; u++)
            v[u] = from[min(i0 + u * step, count - 1)];
        for (int d = 0; d < n; d++) {
            v4u_stream *to = base + at.dsts[d] * slot;
#pragma unroll
            for (int u = 0; u < 4; u++)
                if (i0 + u * step < count)
                    to[i0 + u * step] = v[u];
        }
    }
    // positions from len on stay the slot's own
    const int i = len / 8 * 8 + (tid & 31);
    if (!keys && i < len) {
        const uint16_t v = ((const uint16_t *)from)[i];
        for (int d = 0; d < n; d++)
            ((uint16_t *)(base + at.dsts[d] * slot))[i] = v;
    }
}

}  // namespace

int launch_cache_commit(gx_ctx *ctx, int layers, uint16_t *const *kcaches, uint16_t *const *vcaches,
                        const uint16_t *const *kdrafts, const uint16_t *const *vdrafts, int n, int M, int max_nodes,
                        const int32_t *first, const int32_t *path, const int32_t *counts, const int32_t *prefix,
                        int kv_heads, int hd, int context, int draft_context, const int32_t *slots, int nslots) {
    for (int l0 = 0; l0 < layers; l0 += kCacheLayers) {
        const int here = layers - l0 < kCacheLayers ? layers - l0 : kCacheLayers;
        CommitLayers at{};
        for (int l = 0; l < here; l++) {
            at.kc[l] = kcaches[l0 + l];
            at.vc[l] = vcaches[l0 + l];
            at.kd[l] = kdrafts[l0 + l];
            at.vd[l] = vdrafts[l0 + l];
        }
        cache_commit_kernel<<<dim3((unsigned)kv_heads, (unsigned)n, (unsigned)here), 256, 0, ctx->stream>>>(
            at, M, max_nodes, first, path, counts, prefix, hd, context, draft_context, slots, nslots);
        if (int rc = check_launch("commit of drafted entries"))
            return rc;
    }
    return GX_OK;
}

int launch_cache_fork(gx_ctx *ctx, int layers, uint16_t *const *kcaches, uint16_t *const *vcaches, int kv_heads,
                      int hd, int context, int src, const int32_t *dsts, int n, int len) {
    for (int l0 = 0; l0 < layers; l0 += kCacheLayers)
        for (int d0 = 0; d0 < n; d0 += kForkSlots) {
            const int here = layers - l0 < kCacheLayers ? layers - l0 : kCacheLayers;
            const int slots = n - d0 < kForkSlots ? n - d0 : kForkSlots;
            ForkLayers at{};
            for (int l = 0; l < here; l++) {
                at.kc[l] = kcaches[l0 + l];
                at.vc[l] = vcaches[l0 + l];
            }
            for (int d = 0; d < slots; d++)
                at.dsts[d] = dsts[d0 + d];
            cache_fork_kernel<<<dim3((unsigned)(kv_heads * hd / 8), 2, (unsigned)here), 256, 0, ctx->stream>>>(
                at, kv_heads, hd, context, src, slots, len);
            if (int rc = check_launch("fork of a conversation"))
                return rc;
        }
    return GX_OK;
}

}  // namespace gx
