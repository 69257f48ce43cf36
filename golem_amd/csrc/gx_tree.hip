// gx_tree.hip - a tree of drafted tokens: its plan (what every layer of a pass
// reads) and its verification against the target model's logits.
#include "gx_device.hpp"
#include "gx_internal.hpp"

namespace gx {
namespace {

// ---- the plan ----------------------------------------------------------------
//
// A node's depth and ancestors by doubling the step up the tree: after round k
// a node's bits hold its first 2^k ancestors, itself included, `up` is the
// next one above them, and depth counts them; nine rounds reach 512.  A node
// whose parent is no earlier node has no place, and so have the nodes below.
// grid n + 1: a workgroup a tree, the last one for the tokens behind the trees.
constexpr int kPlanThreads = 256;

__global__ __launch_bounds__(kPlanThreads) void tree_plan_kernel(
    int n, int M, int max_nodes, int words, const int32_t *__restrict__ first, const int32_t *__restrict__ parents,
    const int32_t *__restrict__ prefix, const float *__restrict__ rope_cos, const float *__restrict__ rope_sin,
    int half, int context, int32_t *__restrict__ rows, int32_t *__restrict__ positions, uint32_t *__restrict__ mask,
    float *__restrict__ cos, float *__restrict__ sin) {
    constexpr int kMine = kTreeNodes / kPlanThreads;
    constexpr int kBits = kTreeNodes * (kTreeNodes / 32) / kPlanThreads;
    __shared__ uint32_t bits[kTreeNodes * (kTreeNodes / 32)];
    __shared__ int16_t up[kTreeNodes], depth[kTreeNodes];  // up: -1 above a root, -2 no place
    __shared__ int place[kTreeNodes];                      // a node's position, or -1
    const int tid = threadIdx.x, b = blockIdx.x;
    const bool tail = b == n;
    const int f0 = min(max(first[tail ? n : b], 0), M), f1 = tail ? M : min(max(first[b + 1], f0), M);
    const int T = tail ? 0 : min(f1 - f0, max_nodes);
    for (int i = tid; i < T; i += kPlanThreads) {
        const int p = parents[f0 + i];
        up[i] = (int16_t)(p == -1 ? -1 : p >= 0 && p < i ? p : -2);
        depth[i] = 1;
    }
    for (int i = tid; i < T * words; i += kPlanThreads) {
        const int node = i / words, w = i - node * words;
        bits[i] = node >> 5 == w ? 1u << (node & 31) : 0u;
    }
    __syncthreads();
    for (int span = 1; span < T; span <<= 1) {
        int16_t u[kMine], d[kMine];
        uint32_t w[kBits];
#pragma unroll
        for (int k = 0; k < kMine; k++) {
            const int i = tid + k * kPlanThreads;
            if (i < T) {
                u[k] = up[i] < 0 ? up[i] : up[up[i]];
                d[k] = up[i] < 0 ? depth[i] : (int16_t)(depth[i] + depth[up[i]]);
            }
        }
#pragma unroll
        for (int k = 0; k < kBits; k++) {
            const int i = tid + k * kPlanThreads;
            if (i < T * words) {
                const int node = i / words;
                w[k] = bits[i] | (up[node] < 0 ? 0u : bits[up[node] * words + i - node * words]);
            }
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < kMine; k++) {
            const int i = tid + k * kPlanThreads;
            if (i < T) {
                up[i] = u[k];
                depth[i] = d[k];
            }
        }
#pragma unroll
        for (int k = 0; k < kBits; k++) {
            const int i = tid + k * kPlanThreads;
            if (i < T * words)
                bits[i] = w[k];
        }
        __syncthreads();
    }
    const int base = tail ? -1 : prefix[b];
    for (int i = tid; i < f1 - f0; i += kPlanThreads) {
        const int64_t p = i < T && up[i] == -1 && base >= 0 ? (int64_t)base + depth[i] - 1 : -1;
        const int at = p < context ? (int)p : -1;
        if (i < T)
            place[i] = at;
        rows[f0 + i] = at < 0 ? -1 : f0 + i;
        positions[f0 + i] = at;
    }
    __syncthreads();
    for (int i = tid; i < (f1 - f0) * words; i += kPlanThreads)
        mask[(size_t)f0 * words + i] = i < T * words && place[i / words] >= 0 ? bits[i] : 0u;
    for (int i = tid; i < (f1 - f0) * half; i += kPlanThreads) {
        const int node = i / half, k = i - node * half, at = node < T ? place[node] : -1;
        cos[(size_t)f0 * half + i] = at < 0 ? 0.0f : rope_cos[(size_t)at * half + k];
        sin[(size_t)f0 * half + i] = at < 0 ? 0.0f : rope_sin[(size_t)at * half + k];
    }
}

// ---- verification --------------------------------------------------------------
//
// p = softmax(logits / T) of a node's row, q = softmax(draft / Td).  The walk
// starts at node 0 and tries a node's children in index order; x the child's
// token, u its random number.  With s the drafts' mass tried so far and
// P(x) = max(p(x) - c q(x), 0) what is left of the target, N its sum,
//     x is taken where u N q(x) < P(x) (1 - s);
// otherwise c += N / (1 - s), s += q(x), N = sum P.  That is rejection
// sampling with the residual max(p_i - q_i, 0) / N_i a child, q_i being q
// without the tokens tried: the residuals' scales only ever add up in c, so
// one row of p and one of q give every one of them.  Without draft logits a
// child is a token of its own: taken where u N < p(x), else p loses x.  Where
// no child is taken the last token is the least x whose running sum of P
// passes u_0 sum P, u_0 node 0's number.
//
// Everything is float64, and so is the exponential: the answers are whole
// numbers, and a running sum over 150,000 tokens in float32 would move a
// border past one draw in thirty.

constexpr int kStatThreads = 256;
constexpr int kStatChunk = 8192;  // tokens a workgroup of the row sums takes
constexpr int kWalkThreads = 1024;
constexpr int kPickChunk = 2048;  // tokens a running sum is kept for

struct RowStat {
    double top, sum;  // the row's largest logit, the sum of e^((l - top) / T)
};

// e^d for d <= 0: exp_neg's steps, the float64 left as it is (within an ulp).
__device__ __forceinline__ double exp64(double d) {
    const double n = __builtin_rint(d * 0x1.71547652b82fep+6);
    double r = __builtin_fma(-n, 0x1.62e42fefa38p-7, d);
    r = __builtin_fma(-n, 0x1.ef358p-51, r);
    double p = 1.0 / 720.0;
    p = __builtin_fma(p, r, 1.0 / 120.0);
    p = __builtin_fma(p, r, 1.0 / 24.0);
    p = __builtin_fma(p, r, 1.0 / 6.0);
    p = __builtin_fma(p, r, 0.5);
    p = __builtin_fma(p, r, 1.0);
    p = p * r;
    const int ni = (int)n;
    const double t = kExp2Sixtyfourths[ni & 63];
    const double out = __builtin_ldexp(__builtin_fma(t, p, t), ni >> 6);
    return d < -740.0 ? 0.0 : out;
}

__device__ __forceinline__ double wave_sum64(double v) {
    for (int d = 32; d > 0; d >>= 1)
        v += __shfl_xor(v, d);
    return v;
}

// grid (chunks, M, 1 or 2): a chunk's largest logit and sum of exponentials,
// of the target's rows (z 0) and the draft's.  A logit of -inf has no chance;
// a NaN or +inf makes the sum NaN.
__global__ __launch_bounds__(kStatThreads) void verify_stats_kernel(const float *__restrict__ logits, int ldl,
                                                                    const float *__restrict__ draft, int ldd,
                                                                    int vocab, double it, double itd,
                                                                    float *__restrict__ tops,
                                                                    double *__restrict__ sums) {
    constexpr int kMine = kStatChunk / kStatThreads;
    __shared__ float wt[kStatThreads / 64];
    __shared__ double wsum[kStatThreads / 64];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int row = blockIdx.y, c0 = blockIdx.x * kStatChunk;
    const float *x = blockIdx.z ? draft + (size_t)row * ldd : logits + (size_t)row * ldl;
    const double inv = blockIdx.z ? itd : it;
    float v[kMine];
    float top = -INFINITY;
#pragma unroll
    for (int k = 0; k < kMine; k++) {
        const int i = c0 + tid + k * kStatThreads;
        v[k] = i < vocab ? x[i] : -INFINITY;
    }
#pragma unroll
    for (int k = 0; k < kMine; k++)
        top = fmaxf(top, v[k]);
    top = wave_max(top);
    if (lane == 0)
        wt[wave] = top;
    __syncthreads();
    for (int w = 0; w < kStatThreads / 64; w++)
        top = fmaxf(top, wt[w]);
    double sum = 0.0;
#pragma unroll
    for (int k = 0; k < kMine; k++)
        if (v[k] != -INFINITY)
            sum += exp64(((double)v[k] - (double)top) * inv);
    sum = wave_sum64(sum);
    if (lane == 0)
        wsum[wave] = sum;
    __syncthreads();
    if (tid == 0) {
        for (int w = 1; w < kStatThreads / 64; w++)
            sum += wsum[w];
        const size_t at = ((size_t)blockIdx.z * gridDim.y + row) * gridDim.x + blockIdx.x;
        tops[at] = top;
        sums[at] = sum;
    }
}

struct WalkArgs {
    const float *logits, *draft, *uniforms;
    int ldl, ldd, M, max_nodes, vocab, chunks;
    const int32_t *first, *parents, *tokens, *picks;
    double it, itd;
    const float *tops;
    const double *sums;
    int32_t *path, *counts, *next;
};

// A row's statistics from its chunks' (every lane of the wavefront).
__device__ __forceinline__ RowStat row_stat(const float *tops, const double *sums, int chunks, double inv) {
    const int lane = threadIdx.x & 63;
    float top = -INFINITY;
    for (int i = lane; i < chunks; i += 64)
        top = fmaxf(top, tops[i]);
    top = wave_max(top);
    double sum = 0.0;
    for (int i = lane; i < chunks; i += 64)
        if (sums[i] != 0.0)  // (a chunk without a chance has no largest logit either)
            sum += sums[i] * exp64(((double)tops[i] - (double)top) * inv);
    return {(double)top, wave_sum64(sum)};
}

// grid n: a workgroup a tree.
__global__ __launch_bounds__(kWalkThreads) void verify_walk_kernel(const WalkArgs a) {
    __shared__ int par[kTreeNodes], tok[kTreeNodes];
    __shared__ double part[kWalkThreads / 64];
    __shared__ double run[kVocabMax / kPickChunk];
    __shared__ int gone[kTreeNodes];  // the tokens turned down at this node
    __shared__ int found;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, b = blockIdx.x;
    const int f0 = min(max(a.first[b], 0), a.M), T = min(min(max(a.first[b + 1], f0), a.M) - f0, a.max_nodes);
    int32_t *path = a.path + (size_t)b * a.max_nodes;
    for (int i = tid; i < a.max_nodes; i += kWalkThreads)
        path[i] = -1;
    for (int i = tid; i < T; i += kWalkThreads) {
        par[i] = a.parents[f0 + i];
        tok[i] = a.tokens[f0 + i];
    }
    __syncthreads();
    if (T <= 0) {
        if (tid == 0) {
            a.counts[b] = 0;
            a.next[b] = -1;
        }
        return;
    }
    if (tid == 0)
        path[0] = 0;
    int v = 0, kept = 1;
    if (a.picks) {  // greedy
        for (int m = 1; m < T; m++)
            if (par[m] == v && tok[m] == a.picks[f0 + v]) {
                if (tid == 0)
                    path[kept] = m;
                v = m;
                kept++;
            }
        if (tid == 0) {
            a.counts[b] = kept;
            a.next[b] = a.picks[f0 + v];
        }
        return;
    }
    const float *lr = nullptr, *dr = nullptr;
    RowStat st{}, sd{};
    double c = 0.0, tried = 0.0, mass = 1.0;
    int turned = 0;
    auto enter = [&]() {
        const size_t row = f0 + v;
        lr = a.logits + row * a.ldl;
        st = row_stat(a.tops + row * a.chunks, a.sums + row * a.chunks, a.chunks, a.it);
        if (a.draft) {
            dr = a.draft + row * a.ldd;
            sd = row_stat(a.tops + (a.M + row) * a.chunks, a.sums + (a.M + row) * a.chunks, a.chunks, a.itd);
        }
        c = tried = 0.0;
        mass = 1.0;
        turned = 0;
    };
    auto pt = [&](int x) { return lr[x] == -INFINITY ? 0.0 : exp64(((double)lr[x] - st.top) * a.it) / st.sum; };
    auto qd = [&](int x) { return dr[x] == -INFINITY ? 0.0 : exp64(((double)dr[x] - sd.top) * a.itd) / sd.sum; };
    auto was = [&](int x) {
        for (int i = 0; i < turned; i++)
            if (gone[i] == x)
                return true;
        return false;
    };
    // what is left of token x's chance
    auto left = [&](int x) {
        const double p = pt(x);
        if (a.draft) {
            const double r = c > 0.0 ? p - c * qd(x) : p;
            return r < 0.0 ? 0.0 : r;
        }
        return was(x) ? 0.0 : p;
    };
    // the sum of left() in chunks of kPickChunk, a wavefront a chunk, then in order
    const int parts = (a.vocab + kPickChunk - 1) / kPickChunk;
    auto total = [&]() {
        __syncthreads();
        for (int k = wave; k < parts; k += kWalkThreads / 64) {
            double s = 0.0;
            for (int i = lane; i < kPickChunk; i += 64)
                if (k * kPickChunk + i < a.vocab)
                    s += left(k * kPickChunk + i);
            s = wave_sum64(s);
            if (lane == 0)
                run[k] = s;
        }
        __syncthreads();
        double s = 0.0;
        for (int k = 0; k < parts; k++)
            s += run[k];
        return s;
    };
    enter();
    for (int m = 1; m < T; m++) {
        if (par[m] != v)
            continue;
        const int x = tok[m];
        if (x < 0 || x >= a.vocab || was(x))
            continue;  // no token, or one turned down already: passed over
        const double u = (double)a.uniforms[f0 + m];
        bool take;
        const double px = left(x);
        if (a.draft) {
            const double rest = 1.0 - tried, qx = qd(x);
            if (!(rest > 0.0) || !(mass > 0.0))
                continue;  // nothing a draft could have come from is left
            take = u * mass * qx < px * rest;
            if (!take) {
                c += mass / rest;
                tried += qx;
                mass = total();
            }
        } else {
            take = u * mass < px;
            if (!take)
                mass -= px;
        }
        if (take) {
            if (tid == 0)
                path[kept] = m;
            v = m;
            kept++;
            __syncthreads();
            enter();
        } else {
            __syncthreads();
            if (tid == 0)
                gone[turned] = x;
            turned++;
            __syncthreads();
        }
    }
    double sum = total();
    if (!(sum > 0.0) && sum == 0.0) {  // rounding left nothing: the row as it was
        c = 0.0;
        turned = 0;
        sum = total();
    }
    int token = -1;
    if (sum > 0.0 && sum - sum == 0.0) {
        const double aim = (double)a.uniforms[f0] * sum;
        double s = 0.0;
        int k = 0, last = 0;
        for (int i = 0; i < parts; i++)
            if (run[i] > 0.0)
                last = i;
        for (; k < last && s + run[k] <= aim; k++)
            s += run[k];
        // within the chunk, 1,024 tokens a round: a running sum over the wavefronts
        if (tid == 0)
            found = 0x7fffffff;
        int fallback = -1;
        for (int i0 = 0; i0 < kPickChunk; i0 += kWalkThreads) {
            const int x = k * kPickChunk + i0 + tid;
            const double w = i0 + tid < kPickChunk && x < a.vocab ? left(x) : 0.0;
            double up = w;
            for (int d = 1; d < 64; d <<= 1) {
                const double o = __shfl_up(up, d);
                if (lane >= d)
                    up += o;
            }
            __syncthreads();
            if (lane == 63)
                part[wave] = up;
            __syncthreads();
            double before = s;
            for (int i = 0; i < wave; i++)
                before += part[i];
            if (w > 0.0 && before + up > aim)
                atomicMin(&found, x);
            for (int i = 0; i < kWalkThreads / 64; i++)
                s += part[i];
            if (w > 0.0)
                fallback = x;
            __syncthreads();
            if (found != 0x7fffffff)
                break;
        }
        if (found == 0x7fffffff) {  // the running sum's rounding passed the aim by: the last token with a chance
            __syncthreads();
            if (tid == 0)
                found = -1;
            __syncthreads();
            atomicMax(&found, fallback);
            __syncthreads();
        }
        token = found;
    }
    if (tid == 0) {
        a.counts[b] = kept;
        a.next[b] = token;
    }
}

size_t up256(size_t n) { return (n + 255) & ~(size_t)255; }
int stat_chunks(int vocab) { return (vocab + kStatChunk - 1) / kStatChunk; }

}  // namespace

int launch_tree_plan(gx_ctx *ctx, int n, int M, int max_nodes, const int32_t *first, const int32_t *parents,
                     const int32_t *prefix, const float *rope_cos, const float *rope_sin, int half, int context,
                     int32_t *rows, int32_t *positions, uint32_t *mask, float *cos, float *sin) {
    tree_plan_kernel<<<n + 1, kPlanThreads, 0, ctx->stream>>>(n, M, max_nodes, (max_nodes + 31) / 32, first, parents,
                                                              prefix, rope_cos, rope_sin, half, context, rows,
                                                              positions, mask, cos, sin);
    return check_launch("plan of drafted trees");
}

// Target and draft chunk sums, chunk maxima, and the greedy picks.
size_t tree_verify_workspace(int n, int M, int vocab) {
    const size_t cells = (size_t)2 * M * stat_chunks(vocab);
    return up256(cells * 8) + up256(cells * 4) + up256((size_t)M * 4);
}

int launch_tree_verify(gx_ctx *ctx, const float *logits, int ldl, int n, int M, int max_nodes, int vocab,
                       const int32_t *first, const int32_t *parents, const int32_t *tokens, const float *draft,
                       int ldd, float temperature, float draft_temperature, const float *uniforms, int32_t *path,
                       int32_t *counts, int32_t *next, uint8_t *workspace) {
    const int chunks = stat_chunks(vocab);
    const size_t cells = (size_t)2 * M * chunks;
    double *sums = (double *)workspace;
    float *tops = (float *)(workspace + up256(cells * 8));
    int32_t *picks = (int32_t *)(workspace + up256(cells * 8) + up256(cells * 4));
    const bool greedy = temperature == 0.0f;
    WalkArgs a{logits, greedy ? nullptr : draft, uniforms, ldl,  ldd,  M,    max_nodes, vocab, chunks,
               first,  parents, tokens, greedy ? picks : nullptr, greedy ? 0.0 : 1.0 / (double)temperature,
               greedy || !draft ? 0.0 : 1.0 / (double)draft_temperature, tops, sums, path, counts, next};
    if (M == 0) {  // empty trees only
    } else if (greedy) {
        if (int rc = launch_argmax(ctx, logits, ldl, M, vocab, picks, nullptr, 0, nullptr, nullptr))
            return rc;
    } else {
        verify_stats_kernel<<<dim3((unsigned)chunks, (unsigned)M, draft ? 2u : 1u), kStatThreads, 0, ctx->stream>>>(
            logits, ldl, draft, ldd, vocab, a.it, a.itd, tops, sums);
        if (int rc = check_launch("chances of drafted tokens"))
            return rc;
    }
    verify_walk_kernel<<<n, kWalkThreads, 0, ctx->stream>>>(a);
    return check_launch("verification of drafted trees");
}

}  // namespace gx
