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
// A tree of at most 64 nodes is a wavefront's: a lane a node, two words of bits,
// a step up one exchange; larger ones take the workgroup and LDS.
// grid (n + 1, pieces): workgroups a tree, each with every pieces-th of the
// rotation rows; the last tree stands for the tokens behind the trees.  Bound by
// its launch and three loads in a row: 2.4 us for six nodes, 4.2 for sixteen
// trees of 63, whose 0.8 MB would take 0.2 (LDS and barriers for those too: 9).
constexpr int kPlanThreads = 256;

__global__ __launch_bounds__(kPlanThreads) void tree_plan_kernel(
    int n, int M, int max_nodes, int words, const int32_t *__restrict__ first, const int32_t *__restrict__ parents,
    const int32_t *__restrict__ prefix, const float *__restrict__ rope_cos, const float *__restrict__ rope_sin,
    int half, int context, bool wide, int32_t *__restrict__ rows, int32_t *__restrict__ positions,
    uint32_t *__restrict__ mask, float *__restrict__ cos, float *__restrict__ sin) {
    constexpr int kMine = kTreeNodes / kPlanThreads;
    constexpr int kBits = kTreeNodes * (kTreeNodes / 32) / kPlanThreads;
    __shared__ uint32_t bits[kTreeNodes * (kTreeNodes / 32)];
    __shared__ int16_t up[kTreeNodes], depth[kTreeNodes];  // up: -1 above a root, -2 no place
    __shared__ int place[kTreeNodes];                      // a node's position, or -1
    const int tid = threadIdx.x, b = blockIdx.x, lane = tid & 63;
    const bool tail = b == n, writes = blockIdx.y == 0;
    const int f0 = min(max(first[tail ? n : b], 0), M), f1 = tail ? M : min(max(first[b + 1], f0), M);
    const int T = tail ? 0 : min(f1 - f0, max_nodes);
    const int base = tail ? -1 : prefix[b];
    if (T <= 64) {
        if (tid < 64) {
            const int p = lane < T ? parents[f0 + lane] : -2;
            int u = p == -1 ? -1 : p >= 0 && p < lane ? p : -2, d = 1;
            uint32_t w0 = lane < 32 ? 1u << lane : 0u, w1 = lane < 32 ? 0u : 1u << (lane - 32);
            for (int span = 1; span < T; span <<= 1) {
                const int at = max(u, 0), uu = __shfl(u, at), dd = __shfl(d, at);
                const uint32_t x0 = __shfl(w0, at), x1 = __shfl(w1, at);
                if (u >= 0) {
                    u = uu;
                    d += dd;
                    w0 |= x0;
                    w1 |= x1;
                }
            }
            const int64_t at = u == -1 && base >= 0 ? (int64_t)base + d - 1 : -1;
            const int pos = at < context ? (int)at : -1;
            place[lane] = lane < T ? pos : -1;
            if (lane < T && writes) {
                rows[f0 + lane] = pos < 0 ? -1 : f0 + lane;
                positions[f0 + lane] = pos;
                uint32_t *to = mask + (size_t)(f0 + lane) * words;
                for (int w = 0; w < words; w++)
                    to[w] = pos < 0 || w > 1 ? 0u : w ? w1 : w0;
            }
        }
        __syncthreads();
    } else {
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
        for (int i = tid; i < T; i += kPlanThreads) {
            const int64_t at = up[i] == -1 && base >= 0 ? (int64_t)base + depth[i] - 1 : -1;
            const int pos = at < context ? (int)at : -1;
            place[i] = pos;
            if (writes) {
                rows[f0 + i] = pos < 0 ? -1 : f0 + i;
                positions[f0 + i] = pos;
            }
        }
        __syncthreads();
        if (writes)
            for (int i = tid; i < T * words; i += kPlanThreads)
                mask[(size_t)f0 * words + i] = place[i / words] >= 0 ? bits[i] : 0u;
    }
    if (writes)  // the tokens past a tree's nodes, or past every tree
        for (int i = T + tid; i < f1 - f0; i += kPlanThreads) {
            rows[f0 + i] = positions[f0 + i] = -1;
            for (int w = 0; w < words; w++)
                mask[(size_t)(f0 + i) * words + w] = 0u;
        }
    const int start = blockIdx.y * kPlanThreads + tid, step = gridDim.y * kPlanThreads;
    if (wide) {  // 16 bytes at a time
        typedef float v4f __attribute__((ext_vector_type(4)));
        const int pieces = half >> 2, items = (f1 - f0) * pieces;
        for (int i0 = start; i0 < items; i0 += 2 * step) {
            v4f c[2], s[2];
#pragma unroll
            for (int u = 0; u < 2; u++) {
                const int i = min(i0 + u * step, items - 1), node = i / pieces, at = node < T ? place[node] : -1;
                const size_t src = (size_t)max(at, 0) * half + 4 * (i - node * pieces);
                c[u] = *(const v4f *)(rope_cos + src);
                s[u] = *(const v4f *)(rope_sin + src);
                if (at < 0)
                    c[u] = s[u] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
            }
#pragma unroll
            for (int u = 0; u < 2; u++)
                if (i0 + u * step < items) {
                    *((v4f *)(cos + (size_t)f0 * half) + i0 + u * step) = c[u];
                    *((v4f *)(sin + (size_t)f0 * half) + i0 + u * step) = s[u];
                }
        }
        return;
    }
    for (int i = start; i < (f1 - f0) * half; i += step) {
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
// Two launches: the rows' maxima and sums of exponentials, every logit read
// once, then the walks.  Sampling reads again the rows where a walk turns a child
// down or ends, and those alone; what is left of a row is never written.
//
// Everything is float64, and so is the exponential: the answers are whole
// numbers, and a running sum over 150,000 tokens in float32 would move a
// border past one draw in thirty.

constexpr int kStatThreads = 256;
constexpr int kStatChunk = 8192;  // tokens a workgroup of the row sums takes
constexpr int kWalkThreads = 256;
constexpr int kPart = 2048;       // tokens a part of a running sum, eight a thread
constexpr int kParts = kVocabMax / kPart;
constexpr int kCells = 1536;      // chunks' statistics a walk stages at a time
constexpr int kWalkGroups = 640;  // workgroups of a walk, over all its trees (three fit a CU)

// e^((x - top) / T) as 2^(y / 64), y = (x - top) 64 / (T ln 2): n = y rounded
// by adding 1.5 * 2^52, whose low bits are then n's; 2^((y - n) / 64) by its
// Taylor series to the fourth power (4e-14 off), times 2^(n mod 64 / 64) from a
// table in LDS whose high words lack their index times 2^14, so that n times
// 2^14 added puts n div 64 into the exponent: eleven float64 operations, none
// of the slow kinds (rounding, ldexp and int conversions), and three others.
// y is held at -1023 * 64, where that gives the bits of zero: a chance below
// 2^-1022 is none, and so is that of -inf.  NaN and +inf are not told apart
// here: their row's sum is NaN.
struct Exp64 {
    double A, top, least;
    const double *table;
    __device__ Exp64(const double *lds, double inv, double t)
        : A(inv * 0x1.71547652b82fep+6), top(t == -INFINITY ? 0.0 : t), table(lds) {
        least = -65472.0 / A;
    }
    __device__ __forceinline__ double operator()(float x) const {
        const double d = fmax((double)x - top, least);
        const double z = __builtin_fma(d, A, 0x1.8p+52);
        const double f = __builtin_fma(d, A, 0x1.8p+52 - z);
        double p = 0x1.3b2ab6fba4e77p-31;  // ln2^4 / 24 / 64^4, and so down
        p = __builtin_fma(p, f, 0x1.c6b08d704a0bfp-23);
        p = __builtin_fma(p, f, 0x1.ebfbdff82c58ep-15);
        p = __builtin_fma(p, f, 0x1.62e42fefa39efp-7);
        const uint32_t n = (uint32_t)__double2loint(z);
        const double t = table[n & 63];
        const double s = __hiloint2double((int)((n << 14) + (uint32_t)__double2hiint(t)), __double2loint(t));
        return __builtin_fma(s * f, p, s);
    }
};

constexpr int kTable = 64;
__device__ __forceinline__ void exp64_table(double *lds) {
    if (threadIdx.x < kTable) {
        const double t = kExp2Sixtyfourths[threadIdx.x];
        lds[threadIdx.x] = __hiloint2double((int)((uint32_t)__double2hiint(t) - (threadIdx.x << 14)), __double2loint(t));
    }
}

__device__ __forceinline__ double wave_sum64(double v) {
    for (int d = 32; d > 0; d >>= 1)
        v += __shfl_xor(v, d);
    return v;
}

// What a walk's workgroups share, one a tree.  The first of them walks; the
// others, once they have seen it walk, join it under a number each.  Where it
// needs a sum over a row it says which in `what`, and how many had joined: they
// and it take every so many-th of the row's parts, and it waits for theirs, so
// only ever for a workgroup that runs and stays until the walk has ended.  The
// others wait only for one that walks: a workgroup that finds none walking
// after a while ends.
struct Share {
    unsigned long long begun;                // 1 while the first walks
    alignas(128) unsigned long long joined;  // the others that have joined
    // the open sum: words that name it in their high 16 bits each, so that they need
    // no order among them (one load and one store of a wavefront's lanes)
    alignas(128) unsigned long long what[8];
    // the parts' sums, kNone until they are there; odd and even sums apart, so that
    // the next one's can be cleared while this one's are on their way
    alignas(128) unsigned long long part[2][kParts];
    int gone[kTreeNodes];
};
constexpr unsigned long long kNone = ~0ull;  // (the bits of no sum: a logit's NaN has low bits of zero)
constexpr int kWalked = 0xFFFF;              // what[0]'s name behind the last sum (0 before the first)

template <typename T>
__device__ __forceinline__ T share_load(const T *p) {
    return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
template <typename T>
__device__ __forceinline__ void share_store(T *p, T v) {
    __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

template <typename T>
__device__ __forceinline__ T share_add(T *p, T v) {
    return __hip_atomic_fetch_add(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
// Everything before it done, for every XCD, before anything after: all that the
// workgroups share goes through the two calls above, past the caches that are
// not coherent, so waiting for them is enough.  (Agent-scope release and acquire
// would write back and drop the XCD's L2 each time: 20 us a sum in place of 7.)
__device__ __forceinline__ void share_order() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// grid (chunks, M, 1 or 2): a chunk's largest logit and sum of exponentials,
// of the target's rows (z 0) and the draft's; and the walks' shares cleared.
// A chunk stays in registers between the two; the loads stay in the caches, for
// the walks (past them: 30 us become 32 for eight chains, 54 become 55 for four
// trees).  204 rows of 151936 (124 MB and 31
// million exponentials of twelve float64 operations and five others): 25 us,
// where the loads alone would take 18 and the operations about 13; 72 rows 12.
__global__ __launch_bounds__(kStatThreads) void verify_stats_kernel(const float *__restrict__ logits, int ldl,
                                                                    const float *__restrict__ draft, int ldd,
                                                                    int vocab, double it, double itd,
                                                                    float *__restrict__ tops,
                                                                    double *__restrict__ sums, Share *share, int n) {
    constexpr int kMine = kStatChunk / kStatThreads;
    __shared__ float wt[kStatThreads / 64];
    __shared__ double wsum[kStatThreads / 64];
    __shared__ double table[kTable];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int row = blockIdx.y, c0 = blockIdx.x * kStatChunk;
    const float *x = blockIdx.z ? draft + (size_t)row * ldd : logits + (size_t)row * ldl;
    exp64_table(table);
    float v[kMine];
    float top = -INFINITY;
    if (c0 + kStatChunk <= vocab && ((uintptr_t)x & 15) == 0) {
        typedef float v4f __attribute__((ext_vector_type(4)));
#pragma unroll
        for (int k = 0; k < kMine / 4; k++) {
            const v4f w = *((const v4f *)(x + c0) + tid + k * kStatThreads);
#pragma unroll
            for (int i = 0; i < 4; i++)
                v[4 * k + i] = w[i];
        }
    } else {
#pragma unroll
        for (int k = 0; k < kMine; k++) {
            const int i = c0 + tid + k * kStatThreads;
            const float w = x[min(i, vocab - 1)];
            v[k] = i < vocab ? w : -INFINITY;
        }
    }
    // (a maximum that a NaN goes through: one instruction for two tokens tells of
    // NaN and +inf too)
#pragma unroll
    for (int k = 0; k < kMine; k++)
        top = __builtin_elementwise_maximum(top, v[k]);
    const bool bad = __ballot(!(top < INFINITY)) != 0;
    top = wave_max(top);
    if (lane == 0)
        wt[wave] = top;
    __syncthreads();
    for (int w = 0; w < kStatThreads / 64; w++)
        top = fmaxf(top, wt[w]);
    const Exp64 e(table, blockIdx.z ? itd : it, top);
    double sum = 0.0;
#pragma unroll
    for (int k = 0; k < kMine; k++)
        sum += e(v[k]);
    if (bad)
        sum = NAN;
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
    if (blockIdx.x == 0 && blockIdx.y == 0 && blockIdx.z == 0)
        for (int b = tid; b < n; b += kStatThreads)
            share[b].begun = share[b].joined = 0;
}

// grid (chunks, M): a chunk's largest logit and the lowest index that has it, by
// gx_argmax's rule (a NaN never wins here; one at index 0 is the walk's affair).
// Eight rows of 151936: 3.3 us, most of it the launch.
__global__ __launch_bounds__(kStatThreads) void verify_best_kernel(const float *__restrict__ logits, int ldl,
                                                                   int vocab, float *__restrict__ tops,
                                                                   int32_t *__restrict__ ids) {
    constexpr int kMine = kStatChunk / kStatThreads;
    __shared__ float wt[kStatThreads / 64];
    __shared__ int wi[kStatThreads / 64];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int row = blockIdx.y, c0 = blockIdx.x * kStatChunk;
    const float *x = logits + (size_t)row * ldl;
    float v[kMine], top = -INFINITY;
#pragma unroll
    for (int k = 0; k < kMine; k++) {
        const int i = c0 + tid + k * kStatThreads;
        const float w = x[min(i, vocab - 1)];
        v[k] = i < vocab ? w : -INFINITY;
    }
#pragma unroll
    for (int k = 0; k < kMine; k++)
        top = fmaxf(top, v[k]);
    top = wave_max(top);
    if (lane == 0)
        wt[wave] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kStatThreads / 64; w++)
        top = fmaxf(top, wt[w]);
    int at = 0x7fffffff;
#pragma unroll
    for (int k = kMine - 1; k >= 0; k--)
        at = v[k] == top ? c0 + tid + k * kStatThreads : at;
    at = wave_min_i32(at);
    if (lane == 0)
        wi[wave] = at;
    __syncthreads();
    if (tid == 0) {
        for (int w = 1; w < kStatThreads / 64; w++)
            at = min(at, wi[w]);
        tops[(size_t)row * gridDim.x + blockIdx.x] = top;
        ids[(size_t)row * gridDim.x + blockIdx.x] = at;
    }
}

struct WalkArgs {
    const float *logits, *draft, *uniforms;
    int ldl, ldd, M, max_nodes, vocab, chunks, groups;
    const int32_t *first, *parents, *tokens, *picks;
    double it, itd;
    const float *tops;
    const double *sums;
    Share *share;
    int32_t *path, *counts, *next;
};

// The chance left to tokens of a row, from both rows' logits.
struct Left {
    const float *lr, *dr;  // dr NULL: nothing of the draft's to take off
    Exp64 p, q;
    double scale, dscale;
    const int *gone;
    int turned, vocab;
    // eight tokens x0, x0 + step, ..; none past the vocabulary
    __device__ __forceinline__ void load(const float *from, int x0, int step, float v[8]) const {
#pragma unroll
        for (int i = 0; i < 8; i++)
            v[i] = from[min(x0 + i * step, vocab - 1)];
    }
    __device__ __forceinline__ void eight(int x0, int step, double w[8]) const {
        float l[8], d[8];
        load(lr, x0, step, l);
        if (dr)
            load(dr, x0, step, d);
        chances(x0, step, l, d, w);
    }
    __device__ __forceinline__ void chances(int x0, int step, const float l[8], const float d[8], double w[8]) const {
#pragma unroll
        for (int i = 0; i < 8; i++) {
            double r = p(l[i]) * scale;
            if (dr)
                r -= q(d[i]) * dscale;
            w[i] = r < 0.0 || x0 + i * step >= vocab ? 0.0 : r;
        }
        for (int k = 0; k < turned; k++)
#pragma unroll
            for (int i = 0; i < 8; i++)
                w[i] = gone[k] == x0 + i * step ? 0.0 : w[i];
    }
};

// A workgroup's parts of the sums of its tree.
struct Parts {
    const WalkArgs &a;
    const double *table;
    double *wsum;
    // the part that was loaded last, and its logits: a row's next sum is often of the
    // same row, its chances scaled anew
    float l[8], d[8];
    int part = -1, target = -1, draft = -1;
    __device__ __forceinline__ Left left(int row, int listed, const int *gone, double top, double dtop, double scale,
                                         double dscale) const {
        return Left{a.logits + (size_t)row * a.ldl,
                    dscale > 0.0 ? a.draft + (size_t)row * a.ldd : nullptr,
                    Exp64(table, a.it, top),
                    Exp64(table, a.itd, dtop),
                    scale,
                    dscale,
                    gone,
                    listed,
                    a.vocab};
    }
    // Part k's sum, by the whole workgroup (every thread gets it): eight tokens a
    // thread, a wavefront's 64 tokens in a row.
    __device__ __forceinline__ double sum(const Left &of, int row, int k) {
        const int tid = threadIdx.x, x0 = k * kPart + tid;
        if (part != k || target != row)
            of.load(of.lr, x0, kWalkThreads, l);
        if (of.dr && (part != k || draft != row)) {
            of.load(of.dr, x0, kWalkThreads, d);
            draft = row;
        } else if (part != k) {
            draft = -1;
        }
        part = k;
        target = row;
        double w[8];
        of.chances(x0, kWalkThreads, l, d, w);
        double s = ((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7]));
        s = wave_sum64(s);
        __syncthreads();
        if ((tid & 63) == 0)
            wsum[tid >> 6] = s;
        __syncthreads();
        s = wsum[0];
        for (int i = 1; i < kWalkThreads / 64; i++)
            s += wsum[i];
        return s;
    }
};

// The least of the workgroup's `hit`s, or where there is none the largest of
// its `some`s (in every thread).
__device__ __forceinline__ int first_of(int hit, int some, int *wmin) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    // (one minimum for both: hits as they are, the others behind them, largest first)
    const int key = wave_min_i32(hit != 0x7fffffff ? hit : 0x7ffffffe - some);
    __syncthreads();
    if (lane == 0)
        wmin[wave] = key;
    __syncthreads();
    int least = wmin[0];
    for (int w = 1; w < kWalkThreads / 64; w++)
        least = min(least, wmin[w]);
    return least <= kVocabMax ? least : 0x7ffffffe - least;
}

constexpr int kPolls = 400;  // looks for a walk that has begun, before a workgroup ends
constexpr int kLooks = 16;   // looks of the walk for workgroups that have not joined it yet

// grid (groups, n): a tree's first workgroup walks, the others help.
//
// Bound by round trips to memory shared among the XCDs.  Eight chains of up to six
// nodes over 151936 tokens take 18 us, four trees of up to 33 take 35 to 38: some 10 us to
// begin (the tree, its rows' sums, the children's chances, the others joining),
// about 4 a sum, two loads and a scan to draw the last token.  A workgroup a tree
// alone takes 360 and 590; parts handed out by a claim of each workgroup 20
// and 43.  The greedy walk of eight nodes takes 3.6.
__global__ __launch_bounds__(kWalkThreads) void verify_walk_kernel(const WalkArgs a) {
    __shared__ int par[kTreeNodes], tok[kTreeNodes], gone[kTreeNodes];
    __shared__ double px[kTreeNodes], qx[kTreeNodes];                        // a node's token by its parent's rows
    __shared__ double top[kTreeNodes], sum[kTreeNodes], dtop[kTreeNodes], dsum[kTreeNodes];  // a node's own rows
    // (the chunks' statistics are read before the first running sum is written:
    // with them apart two workgroups fit a CU, and not three)
    __shared__ __align__(16) uint8_t both[kCells * 12];
    static_assert(kCells * 12 >= kParts * 16, "the running sums fit");
    double *const csum = (double *)both, *const run = (double *)both, *const own = run + kParts;
    float *const ctop = (float *)(both + kCells * 8);
    __shared__ double table[kTable], wsum[kWalkThreads / 64];
    __shared__ int wmin[kWalkThreads / 64];
    __shared__ float un[kTreeNodes];
    __shared__ unsigned long long got, what[8];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, b = blockIdx.y;
    const int f0 = min(max(a.first[b], 0), a.M), T = min(min(max(a.first[b + 1], f0), a.M) - f0, a.max_nodes);
    const int parts = (a.vocab + kPart - 1) / kPart;
    Share &sh = a.share[b];
    Parts mine{a, table, wsum};
    if (blockIdx.x > 0) {
        if (T <= 0)
            return;
        exp64_table(table);
        if (tid == 0) {
            got = 0;
            for (int spent = 0; spent < kPolls; spent++) {
                if (share_load(&sh.begun) != 0) {
                    got = share_add(&sh.joined, 1ull) + 1;
                    break;
                }
                __builtin_amdgcn_s_sleep(8);
            }
        }
        __syncthreads();
        const int number = (int)got;
        if (number == 0)
            return;
        for (int seen = 0;;) {
            if (wave == 0) {
                unsigned long long w;
                for (;;) {
                    w = share_load(&sh.what[lane & 7]);
                    const int name = (int)(w >> 48), first = __builtin_amdgcn_readfirstlane(name);
                    if (first == kWalked || (first != seen && __ballot(name != first) == 0))
                        break;
                    __builtin_amdgcn_s_sleep(4);
                }
                if (lane < 8)
                    what[lane] = w;
            }
            __syncthreads();
            const unsigned long long w0 = what[0];
            seen = (int)(w0 >> 48);
            if (seen == kWalked)
                return;
            const int row = (int)(w0 & 0xFFFF), listed = (int)(w0 >> 16 & 0x3FF), workers = (int)(w0 >> 26 & 0x3FF);
            const Left left = mine.left(row, listed, gone, __uint_as_float((uint32_t)what[1]),
                                        __uint_as_float((uint32_t)what[2]),
                                        __hiloint2double((int)(uint32_t)what[4], (int)(uint32_t)what[3]),
                                        __hiloint2double((int)(uint32_t)what[6], (int)(uint32_t)what[5]));
            for (int i = tid; i < listed; i += kWalkThreads)
                gone[i] = share_load(&sh.gone[i]);
            __syncthreads();  // (and `what` has been read)
            if (number < workers)
                for (int k = number; k < parts; k += workers) {
                    const double s = mine.sum(left, row, k);
                    if (tid == 0)
                        share_store(&sh.part[seen & 1][k], (unsigned long long)__double_as_longlong(s));
                }
        }
    }
    int32_t *path = a.path + (size_t)b * a.max_nodes;
    for (int i = tid; i < a.max_nodes; i += kWalkThreads)
        path[i] = -1;
    if (T <= 0) {
        if (tid == 0) {
            a.counts[b] = 0;
            a.next[b] = -1;
        }
        return;
    }
    // the parts' sums of a parity, none of them there
    auto clear = [&](int parity) __attribute__((always_inline)) {
        for (int i = tid; i < parts; i += kWalkThreads)
            share_store(&sh.part[parity][i], kNone);
    };
    // what hangs on nothing but the tree's place, asked for together: its nodes, and
    // the chunks' statistics that are staged first
    constexpr int kMine = kTreeNodes / kWalkThreads, kCell = kCells / kWalkThreads;
    const int rows = a.draft ? 2 * T : T, batch = max(1, kCells / a.chunks);
    float ct[kCell];
    double cs[kCell];
    auto load_cells = [&](int r0) __attribute__((always_inline)) {
        // (the target's rows of a tree follow one another, and so do the draft's)
        const int c0 = r0 * a.chunks, split = T * a.chunks, last = min(r0 + batch, rows) * a.chunks - 1;
#pragma unroll
        for (int k = 0; k < kCell; k++) {
            const int i = min(c0 + tid + k * kWalkThreads, last);
            const size_t at = i < split ? (size_t)f0 * a.chunks + i : (size_t)(a.M + f0) * a.chunks + (i - split);
            ct[k] = a.tops[at];
            cs[k] = a.sums[at];
        }
    };
    int up[kMine], id[kMine];
    float number[kMine];
#pragma unroll
    for (int k = 0; k < kMine; k++) {
        const int i = f0 + min(tid + k * kWalkThreads, T - 1);
        up[k] = a.parents[i];
        id[k] = a.tokens[i];
        number[k] = a.picks ? 0.0f : a.uniforms[i];
    }
    if (!a.picks) {
        load_cells(0);
        clear(1);
        if (tid < 8)
            share_store(&sh.what[tid], 0ull);
    }
    exp64_table(table);
#pragma unroll
    for (int k = 0; k < kMine; k++)
        if (tid + k * kWalkThreads < T) {
            par[tid + k * kWalkThreads] = up[k];
            tok[tid + k * kWalkThreads] = id[k];
            un[tid + k * kWalkThreads] = number[k];
        }
    share_order();
    __syncthreads();  // (and the path's -1s are written)
    if (!a.picks && tid == 0)
        share_store(&sh.begun, 1ull);
    if (tid == 0)
        path[0] = 0;
    int v = 0, kept = 1;
    if (a.picks) {  // greedy: each row's best chunk, a wavefront a row
        for (int i = wave; i < T; i += kWalkThreads / 64) {
            const size_t row = f0 + i;
            float best = -INFINITY;
            int id = 0;
            const float zero = a.logits[row * a.ldl];
            for (int c = lane; c < a.chunks; c += 64) {
                const float v = a.tops[row * a.chunks + c];
                const int pick = a.picks[row * a.chunks + c];
                id = v > best ? pick : id;
                best = fmaxf(best, v);
            }
            const float mx = wave_max(best);
            id = wave_min_i32(best == mx && mx > -INFINITY ? id : 0x7fffffff);
            if (lane == 0)
                gone[i] = zero != zero || id == 0x7fffffff ? 0 : id;
        }
        __syncthreads();
        for (int m = 1; m < T; m++)
            if (par[m] == v && tok[m] == gone[v]) {
                if (tid == 0)
                    path[kept] = m;
                v = m;
                kept++;
            }
        if (tid == 0) {
            a.counts[b] = kept;
            a.next[b] = gone[v];
        }
        return;
    }
    // a child's logits in its parent's rows, and every row's statistics from its
    // chunks' (staged in LDS, so many rows' at a time); then every child's chances
    float lx[kMine], dx[kMine];
#pragma unroll
    for (int k = 0; k < kMine; k++) {
        const int m = min(tid + k * kWalkThreads, T - 1), p = min(max(par[m], 0), T - 1);
        const int x = min(max(tok[m], 0), a.vocab - 1);
        lx[k] = a.logits[(size_t)(f0 + p) * a.ldl + x];
        dx[k] = a.draft ? a.draft[(size_t)(f0 + p) * a.ldd + x] : 0.0f;
    }
    for (int r0 = 0; r0 < rows; r0 += batch) {
        const int here = min(batch, rows - r0);
        if (r0 > 0)
            load_cells(r0);
#pragma unroll
        for (int k = 0; k < kCell; k++) {
            ctop[tid + k * kWalkThreads] = ct[k];
            csum[tid + k * kWalkThreads] = cs[k];
        }
        __syncthreads();
        for (int i = tid; i < here; i += kWalkThreads) {
            const int row = r0 + i, z = row >= T, node = z ? row - T : row;
            float mx = -INFINITY;
#pragma unroll 4
            for (int c = 0; c < a.chunks; c++)
                mx = fmaxf(mx, ctop[i * a.chunks + c]);
            const Exp64 e(table, z ? a.itd : a.it, mx);
            double s = 0.0;
#pragma unroll 4
            for (int c = 0; c < a.chunks; c++) {
                const double cs = csum[i * a.chunks + c];
                const double w = cs * e(ctop[i * a.chunks + c]);
                s += cs == 0.0 ? 0.0 : cs - cs == 0.0 ? w : cs;
            }
            (z ? dtop : top)[node] = mx;
            (z ? dsum : sum)[node] = s;
        }
        __syncthreads();
    }
    if (tid == 0)
        got = share_load(&sh.joined);
#pragma unroll
    for (int k = 0; k < kMine; k++) {
        const int m = tid + k * kWalkThreads, p = m < T ? par[m] : -1;
        if (p < 0 || p >= m || tok[m] < 0 || tok[m] >= a.vocab)
            continue;
        px[m] = Exp64(table, a.it, top[p])(lx[k]) / sum[p];
        if (a.draft)
            qx[m] = Exp64(table, a.itd, dtop[p])(dx[k]) / dsum[p];
    }
    __syncthreads();
    // those that have joined, and this one (the others had time to since it began;
    // what is left of them is waited for a little)
    int workers = (int)got + 1;
    for (int looks = 0; looks < kLooks && workers < a.groups; looks++) {
        __syncthreads();
        if (tid == 0)
            got = share_load(&sh.joined);
        __syncthreads();
        workers = (int)got + 1;
    }
    double c = 0.0, tried = 0.0, mass = 1.0, all = 0.0;
    int turned = 0, m = 1;
    unsigned sums = 0;
    bool known = true;    // mass is up to date
    bool summed = false;  // run[] holds the parts of what is left
    // the factor of the draft's exponentials in what is left (a row of q that is
    // none takes nothing off)
    auto off = [&]() __attribute__((always_inline)) {
        const double d = a.draft ? c / dsum[v] : 0.0;
        return d > 0.0 && d - d == 0.0 ? d : 0.0;
    };
    for (;;) {
        // down the tree, until a sum is wanted or the nodes are at their end
        while (m < T) {
            const int x = tok[m];
            bool over = par[m] != v || x < 0 || x >= a.vocab;  // no child, or no token
            for (int i = 0; !over && i < turned; i++)
                over = gone[i] == x;  // one turned down already
            if (over) {
                m++;
                continue;
            }
            const double u = (double)un[m];
            bool take;
            if (a.draft) {
                if (!known)
                    break;
                const double rest = 1.0 - tried;
                if (!(rest > 0.0) || !(mass > 0.0)) {  // nothing a draft could have come from is left
                    m++;
                    continue;
                }
                const double r = px[m] - c * qx[m];
                take = u * mass * qx[m] < (r < 0.0 ? 0.0 : r) * rest;
                if (!take) {
                    c += mass / rest;
                    tried += qx[m];
                    known = summed = false;
                }
            } else {
                take = u * mass < px[m];
                if (!take)
                    mass -= px[m];
            }
            __syncthreads();
            if (take) {
                if (tid == 0)
                    path[kept] = m;
                v = m;
                kept++;
                c = tried = 0.0;
                mass = 1.0;
                turned = 0;
                known = true;
                summed = false;
            } else {
                if (tid == 0)
                    gone[turned] = x;
                turned++;
            }
            __syncthreads();
            m++;
        }
        const bool ending = m >= T;
        if (!summed) {
            // the sum of what is left of v's row, handed out
            const int listed = a.draft ? 0 : turned;
            sums++;
            for (int i = tid; i < listed; i += kWalkThreads)
                share_store(&sh.gone[i], gone[i]);
            if (tid == 0 && workers < a.groups)  // (more of them may have joined)
                got = share_load(&sh.joined);
            share_order();  // (and the parts' sums are cleared)
            __syncthreads();
            if (workers < a.groups)
                workers = (int)got + 1;
            const double scale = 1.0 / sum[v], dscale = off(), tv = top[v], dv = a.draft ? dtop[v] : 0.0;
            if (tid < 8) {
                const uint32_t words[8] = {0u,
                                           __float_as_uint((float)tv),
                                           __float_as_uint((float)dv),
                                           (uint32_t)__double2loint(scale),
                                           (uint32_t)__double2hiint(scale),
                                           (uint32_t)__double2loint(dscale),
                                           (uint32_t)__double2hiint(dscale),
                                           0u};
                unsigned long long mine = (unsigned long long)(f0 + v) | (unsigned long long)listed << 16 |
                                          (unsigned long long)workers << 26;
#pragma unroll
                for (int i = 1; i < 8; i++)
                    mine = tid == i ? words[i] : mine;
                share_store(&sh.what[tid], mine | (unsigned long long)sums << 48);
            }
            clear((sums + 1) & 1);
            const Left left = mine.left(f0 + v, listed, gone, tv, dv, scale, dscale);
            for (int k = 0; k < parts; k += workers) {
                const double s = mine.sum(left, f0 + v, k);
                if (tid == 0)
                    own[k] = s;
            }
            __syncthreads();
            // the parts' sums, two of them a thread, as they come
            static_assert(kParts == 2 * kWalkThreads, "two parts a thread");
            const unsigned long long *from = sh.part[sums & 1] + 2 * tid;
            auto at_hand = [&](int k) __attribute__((always_inline)) {
                return k >= parts ? 0ull : k % workers ? kNone : (unsigned long long)__double_as_longlong(own[k]);
            };
            unsigned long long w1 = at_hand(2 * tid), w2 = at_hand(2 * tid + 1);
            do {
                if (w1 == kNone)
                    w1 = share_load(from);
                if (w2 == kNone)
                    w2 = share_load(from + 1);
            } while (__syncthreads_or(w1 == kNone || w2 == kNone));
            const double one = __longlong_as_double((long long)w1), two = __longlong_as_double((long long)w2);
            double up = one + two;
            for (int d = 1; d < 64; d <<= 1) {
                const double o = __shfl_up(up, d);
                if (lane >= d)
                    up += o;
            }
            if (lane == 63)
                wsum[wave] = up;
            __syncthreads();
            double at = 0.0;
            for (int i = 0; i < wave; i++)
                at += wsum[i];
            run[2 * tid] = at + (up - two);
            run[2 * tid + 1] = at + up;
            own[2 * tid] = one;
            own[2 * tid + 1] = two;
            __syncthreads();
            summed = known = true;
        }
        all = run[parts - 1];
        mass = all;
        if (!ending)
            continue;
        if (all == 0.0 && (c > 0.0 || turned > 0)) {  // rounding left nothing: the row as it was
            c = 0.0;
            turned = 0;
            summed = false;
            continue;
        }
        break;
    }
    if (tid == 0)
        share_store(&sh.what[0], (unsigned long long)kWalked << 48);
    int token = -1;
    if (all > 0.0 && all - all == 0.0) {
        const double aim = (double)un[0] * all;
        // the first part that adds to the running sum and at whose end it is past
        // the aim, or the last that adds to it
        int k = 0x7fffffff, some = -1;
        for (int i = tid; i < parts; i += kWalkThreads)
            if (own[i] > 0.0) {
                some = i;
                if (run[i] > aim)
                    k = min(k, i);
            }
        k = first_of(k, some, wmin);
        const double s = k > 0 ? run[k - 1] : 0.0;
        // the part's running sum: eight tokens in a row a thread
        constexpr int kEach = kPart / kWalkThreads;
        static_assert(kEach == 8, "Left::eight");
        const Left left = mine.left(f0 + v, a.draft ? 0 : turned, gone, top[v], a.draft ? dtop[v] : 0.0, 1.0 / sum[v], off());
        const int x0 = k * kPart + tid * kEach;
        double w[kEach], mine = 0.0;
        left.eight(x0, 1, w);
#pragma unroll
        for (int i = 0; i < kEach; i++)
            mine += w[i];
        double up = mine;
        for (int d = 1; d < 64; d <<= 1) {
            const double o = __shfl_up(up, d);
            if (lane >= d)
                up += o;
        }
        if (lane == 63)
            wsum[wave] = up;
        __syncthreads();
        double at = s + (up - mine);
        for (int i = 0; i < wave; i++)
            at += wsum[i];
        int hit = 0x7fffffff;
        some = -1;  // (where rounding passed the aim by: the last token with a chance)
#pragma unroll
        for (int i = 0; i < kEach; i++) {
            at += w[i];
            if (w[i] > 0.0) {
                some = x0 + i;
                if (at > aim && hit == 0x7fffffff)
                    hit = x0 + i;
            }
        }
        token = first_of(hit, some, wmin);
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
    const bool wide =
        half % 4 == 0 &&
        (((uintptr_t)rope_cos | (uintptr_t)rope_sin | (uintptr_t)cos | (uintptr_t)sin) & 15) == 0;
    // a round of the rotation rows a workgroup
    const int64_t items = (int64_t)max_nodes * (wide ? half / 4 : half);
    const int pieces = (int)(items <= 2 * kPlanThreads ? 1 : items >= 8 * 2 * kPlanThreads ? 8 : items / (2 * kPlanThreads));
    tree_plan_kernel<<<dim3((unsigned)n + 1, (unsigned)pieces), kPlanThreads, 0, ctx->stream>>>(
        n, M, max_nodes, (max_nodes + 31) / 32, first, parents, prefix, rope_cos, rope_sin, half, context, wide, rows,
        positions, mask, cos, sin);
    return check_launch("plan of drafted trees");
}

// The walks' shares, target and draft chunk sums and chunk maxima (the greedy
// walk: the chunks' best tokens and their logits).
size_t tree_verify_workspace(int n, int M, int vocab) {
    const size_t cells = (size_t)2 * M * stat_chunks(vocab);
    return up256((size_t)n * sizeof(Share)) + up256(cells * 8) + up256(cells * 4);
}

int launch_tree_verify(gx_ctx *ctx, const float *logits, int ldl, int n, int M, int max_nodes, int vocab,
                       const int32_t *first, const int32_t *parents, const int32_t *tokens, const float *draft,
                       int ldd, float temperature, float draft_temperature, const float *uniforms, int32_t *path,
                       int32_t *counts, int32_t *next, uint8_t *workspace) {
    const int chunks = stat_chunks(vocab);
    const size_t cells = (size_t)2 * M * chunks;
    Share *share = (Share *)workspace;
    double *sums = (double *)(workspace + up256((size_t)n * sizeof(Share)));
    float *tops = (float *)((uint8_t *)sums + up256(cells * 8));
    int32_t *picks = (int32_t *)sums;
    const bool greedy = temperature == 0.0f;
    const int parts = (vocab + kPart - 1) / kPart, each = kWalkGroups / n;
    const int groups = greedy || M == 0 ? 1 : parts < each ? parts : each > 0 ? each : 1;
    const WalkArgs a{logits,
                     greedy ? nullptr : draft,
                     uniforms,
                     ldl,
                     ldd,
                     M,
                     max_nodes,
                     vocab,
                     chunks,
                     groups,
                     first,
                     parents,
                     tokens,
                     greedy ? picks : nullptr,
                     greedy ? 0.0 : 1.0 / (double)temperature,
                     greedy || !draft ? 0.0 : 1.0 / (double)draft_temperature,
                     tops,
                     sums,
                     share,
                     path,
                     counts,
                     next};
    if (M == 0) {  // empty trees only
    } else if (greedy) {
        verify_best_kernel<<<dim3((unsigned)chunks, (unsigned)M), kStatThreads, 0, ctx->stream>>>(logits, ldl, vocab, tops,
                                                                                                  picks);
        if (int rc = check_launch("best tokens of drafted trees"))
            return rc;
    } else {
        verify_stats_kernel<<<dim3((unsigned)chunks, (unsigned)M, draft ? 2u : 1u), kStatThreads, 0, ctx->stream>>>(
            logits, ldl, draft, ldd, vocab, a.it, a.itd, tops, sums, share, n);
        if (int rc = check_launch("chances of drafted tokens"))
            return rc;
    }
    verify_walk_kernel<<<dim3((unsigned)groups, (unsigned)n), kWalkThreads, 0, ctx->stream>>>(a);
    return check_launch("verification of drafted trees");
}

}  // namespace gx
