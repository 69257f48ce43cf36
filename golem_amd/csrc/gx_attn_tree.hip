// gx_attn_tree.hip - attention of drafted tokens: every node of a tree against
// its conversation's cached prefix and the draft entries of its ancestors.
//
// For node i of tree b, query head h and the keys j it sees (positions 0 ..
// prefix - 1 of the cache, then the tree's nodes named by its mask bits):
//   o = sum_j e^(s_j - m) v_j / sum_j e^(s_j - m),   s_j = q . k_j / sqrt(hd)
// in one pass with the running maximum m.
//
// The matrix cores take 32 keys against 32 rows (a row: a node and a query
// head of the key-value head's group) a step.  S^T = K Q^T puts a row's scores
// down one lane's registers, so the maximum and the sum stay in the lane (the
// wavefront's halves hold 16 keys each), and with key piece m of a step read
// from position swap23(m) (bits 2 and 3 exchanged) registers 8t .. 8t + 7 of
// half h are the keys 16t + 8h .. + 7: the second operand of O^T = V^T P^T as
// it stands, beside value rows read 16 bytes a lane.  Neither product passes
// through LDS.
//
// A probability enters the second product as two fp16 values, its leading 11
// bits and the rest (about 22 bits together): rounded to one, the head
// outputs would be 2e-4 off, which the float output could not hide.  Sums,
// maxima and outputs are float32.
#include <algorithm>

#include "gx_device.hpp"
#include "gx_internal.hpp"

namespace gx {
namespace {

typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef float v16f __attribute__((ext_vector_type(16)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));

constexpr int kWaves = 4;        // wavefronts a workgroup, each with a share of its tiles
constexpr int kTile = 32;        // keys a step
constexpr int kMaxSplits = 64;   // shares of the keys, over workgroups
constexpr float kShift = 10.0f;  // probabilities are held times 2^10, their low parts clear of fp16's subnormals

struct Args {
    const uint16_t *qh;
    const int32_t *first;
    const uint32_t *mask;
    const int32_t *prefix;
    const int32_t *slots;
    const uint16_t *kc, *vc, *kd, *vd;
    int n, M, max_nodes, words, max_prefix, heads, kv_heads, context, draft_context, nslots, S;
    float c;       // 1 / sqrt(hd) in the exponent's base 2
    float *po;     // [S][M][heads][hd] unnormalised outputs
    float *pml;    // [S][M][heads][2] maximum (base 2) and sum
};

// A tree's tokens, cached positions and steps, the same for every kernel.
struct Tree {
    int f0, T, P, a, np, total, per;
    __device__ Tree(const Args &x, int b) {
        f0 = min(max(x.first[b], 0), x.M);
        T = min(min(max(x.first[b + 1], f0), x.M) - f0, x.max_nodes);
        P = min(max(x.prefix[b], 0), min(x.max_prefix, x.context));
        a = f0 & 7;  // draft rows are read from a multiple of 8
        np = (P + kTile - 1) / kTile;
        total = np + (T > 0 ? (a + T + kTile - 1) / kTile : 0);
        per = max(1, (total + x.S - 1) / x.S);
    }
};

__device__ __forceinline__ float other_half(float v) { return __shfl_xor(v, 32); }

// Elements lo .. hi - 1 of eight, the rest zero.
__device__ __forceinline__ v8h keep(v8h v, int lo, int hi) {
    v8h r;
#pragma unroll
    for (int j = 0; j < 8; j++)
        r[j] = j >= lo && j < hi ? v[j] : (_Float16)0.0f;
    return r;
}

// grid (kv_heads, 32-row tiles, trees * S): key-value heads fastest, so that
// with eight of them every workgroup of a head is on one XCD and shares its L2.
template <int HD>
__global__ __launch_bounds__(64 * kWaves) void attn_tree_kernel(const Args x) {
    constexpr int KS = HD / 16, ET = HD / 32;
    __shared__ float ms[kWaves][kTile], ls[kWaves][kTile];
    __shared__ float os[kTile][HD + 1];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int li = lane & 31, h = lane >> 5;
    const int kvh = blockIdx.x, b = blockIdx.z / x.S, sp = blockIdx.z % x.S;
    const Tree t(x, b);
    const int g = x.heads / x.kv_heads, R = t.T * g, r0 = blockIdx.y * kTile;
    const int t0 = sp * t.per, t1 = min(t.total, t0 + t.per);
    if (r0 >= R || t0 >= t1)
        return;
    const int slot = x.slots ? min(max(x.slots[b], 0), x.nslots - 1) : 0;
    const size_t cache = ((size_t)slot * x.kv_heads + kvh) * HD * x.context;
    const uint16_t *kc = x.kc + cache, *vc = x.vc + cache;
    const uint16_t *kd = x.kd + (size_t)kvh * HD * x.draft_context, *vd = x.vd + (size_t)kvh * HD * x.draft_context;

    const int r = min(r0 + li, R - 1), node = r / g;
    const uint16_t *qr = x.qh + ((size_t)(t.f0 + node) * x.heads + kvh * g + (r - node * g)) * HD + 8 * h;
    v8h q[KS];
#pragma unroll
    for (int s = 0; s < KS; s++)
        q[s] = *(const v8h *)(qr + 16 * s);
    const uint32_t *mrow = x.mask + (size_t)(t.f0 + node) * x.words;
    const int lis = (li & ~12) | ((li & 4) << 1) | ((li & 8) >> 1);

    v16f o[ET] = {};
    float m = -INFINITY, l = 0.0f;
    for (int j = t0 + wave; j < t1; j += kWaves) {
        const bool draft = j >= t.np;
        const int d = j - t.np;
        // the tile's first row and its rows' range, in the cache or the draft buffers
        const int p0 = draft ? t.f0 - t.a + kTile * d : kTile * j;
        const int lo = draft ? t.f0 : 0, hi = draft ? t.f0 + t.T : t.P;
        const uint16_t *kb = draft ? kd : kc, *vb = draft ? vd : vc;
        const int rows = draft ? x.draft_context : x.context;
        const int kp = min(max(p0 + lis, lo), hi - 1);
        v16f s = {};
#pragma unroll
        for (int k = 0; k < KS; k++) {
            const v8h a = *(const v8h *)(kb + ((size_t)(2 * k + h) * rows + kp) * 8);
            s = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, q[k], s, 0, 0, 0);
        }
        v8h v[ET][2];
#pragma unroll
        for (int et = 0; et < ET; et++)
#pragma unroll
            for (int u = 0; u < 2; u++)
                v[et][u] = *(const v8h *)(vb + (size_t)(32 * et + li) * rows + min(p0 + 16 * u + 8 * h, rows - 8));
        uint32_t sees = ~0u;
        if (draft) {
            const uint32_t w = d < x.words ? mrow[d] : 0u;
            sees = t.a ? (w << t.a) | (d > 0 ? mrow[d - 1] >> (32 - t.a) : 0u) : w;
        }
        if (p0 < lo || p0 + kTile > hi) {  // the tile's rows outside the range: not seen, their values zero
#pragma unroll
            for (int u = 0; u < 2; u++) {
                const int pv = p0 + 16 * u + 8 * h;
#pragma unroll
                for (int et = 0; et < ET; et++)
                    v[et][u] = keep(v[et][u], lo - pv, hi - pv);
            }
            const int below = max(lo - p0, 0), above = min(hi - p0, kTile);
            sees &= (above >= 32 ? ~0u : (1u << above) - 1) & ~((1u << below) - 1);
        }
        float mx = -INFINITY;
#pragma unroll
        for (int i = 0; i < 16; i++) {
            const int k = 16 * (i >> 3) + 8 * h + (i & 7);
            s[i] = sees >> k & 1 ? s[i] * x.c : -INFINITY;
            mx = fmaxf(mx, s[i]);
        }
        const float mn = fmaxf(m, fmaxf(mx, other_half(mx)));
        const float base = mn == -INFINITY ? 0.0f : mn - kShift;
        const float corr = mn == -INFINITY ? 1.0f : exp2f(m - mn);
        m = mn;
        v8h ph[2], pl[2];
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < 16; i++) {
            const float p = exp2f(s[i] - base);
            sum += p;
            const _Float16 hp = (_Float16)p;
            ph[i >> 3][i & 7] = hp;
            pl[i >> 3][i & 7] = (_Float16)(p - (float)hp);
        }
        l = l * corr + sum;
#pragma unroll
        for (int et = 0; et < ET; et++) {
#pragma unroll
            for (int i = 0; i < 16; i++)
                o[et][i] *= corr;
#pragma unroll
            for (int u = 0; u < 2; u++) {
                o[et] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v[et][u], ph[u], o[et], 0, 0, 0);
                o[et] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v[et][u], pl[u], o[et], 0, 0, 0);
            }
        }
    }
    // the wavefronts' parts, in their order
    l += other_half(l);
    if (h == 0) {
        ms[wave][li] = m;
        ls[wave][li] = l;
    }
    __syncthreads();
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWaves; w++)
        top = fmaxf(top, ms[w][li]);
    const float corr = m == -INFINITY ? 0.0f : exp2f(m - top);
    for (int w = 0; w < kWaves; w++) {
        if (wave == w) {
#pragma unroll
            for (int et = 0; et < ET; et++)
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    float *to = &os[li][32 * et + 8 * (i >> 2) + 4 * h + (i & 3)];
                    const float v = m == -INFINITY ? 0.0f : o[et][i] * corr;
                    *to = w == 0 ? v : *to + v;
                }
        }
        __syncthreads();
    }
    for (int i = tid; i < kTile * HD; i += 64 * kWaves) {
        const int rr = i / HD, e = i - rr * HD;
        if (r0 + rr < R) {
            const int nd = (r0 + rr) / g, hh = kvh * g + (r0 + rr - nd * g);
            x.po[(((size_t)sp * x.M + t.f0 + nd) * x.heads + hh) * HD + e] = os[rr][e];
        }
    }
    if (tid < kTile && r0 + tid < R) {
        float sum = 0.0f;
#pragma unroll
        for (int w = 0; w < kWaves; w++)
            sum += ms[w][tid] == -INFINITY ? ls[w][tid] : ls[w][tid] * exp2f(ms[w][tid] - top);
        const int nd = (r0 + tid) / g, hh = kvh * g + (r0 + tid - nd * g);
        float *to = x.pml + (((size_t)sp * x.M + t.f0 + nd) * x.heads + hh) * 2;
        to[0] = top;
        to[1] = sum;
    }
}

// One head element a lane: the shares of a row joined in order, and the Q8_0
// of 32 elements.  grid (heads * HD / 64, M), 64 threads.
//
// An infinite or NaN value that a row's mask hides still makes 0 * inf in its
// tile: a row whose sum is a number and whose output is none is computed
// again here, key by key over what it sees alone.
template <int HD>
__global__ __launch_bounds__(64) void attn_tree_join_kernel(const Args x, float *__restrict__ out,
                                                            int8_t *__restrict__ q8, float *__restrict__ scales,
                                                            int32_t *__restrict__ qsum) {
    const int lane = threadIdx.x, tok = blockIdx.y, width = x.heads * HD;
    int b = 0, hi = x.n;  // the tree: the last whose first token is not past this one
    while (hi - b > 1) {
        const int mid = (b + hi) >> 1;
        if (x.first[mid] <= tok)
            b = mid;
        else
            hi = mid;
    }
    const Tree t(x, b);
    if (tok < t.f0 || tok >= t.f0 + t.T)
        return;
    const int col = min((int)blockIdx.x * 64 + lane, width - 1), head = col / HD, e = col - head * HD;
    const int live = (t.total + t.per - 1) / t.per;
    const size_t row = (size_t)tok * x.heads + head, step = (size_t)x.M * x.heads;
    float top = -INFINITY;
    for (int s = 0; s < live; s++)
        top = fmaxf(top, x.pml[(s * step + row) * 2]);
    float l = 0.0f, o = 0.0f;
    for (int s = 0; s < live; s++) {
        const float m = x.pml[(s * step + row) * 2];
        const float corr = m == -INFINITY ? (top == -INFINITY ? 1.0f : 0.0f) : exp2f(m - top);
        const float sl = x.pml[(s * step + row) * 2 + 1], so = x.po[(s * step + row) * HD + e];
        l += m == -INFINITY ? sl : sl * corr;
        o += m == -INFINITY ? 0.0f : so * corr;
    }
    const uint32_t *mrow = x.mask + (size_t)tok * x.words;
    bool any = t.P > 0;
    for (int w = 0; 32 * w < t.T; w++)
        any |= (mrow[w] & (t.T - 32 * w >= 32 ? ~0u : (1u << (t.T - 32 * w)) - 1)) != 0;
    if (any && l - l == 0.0f && o - o != 0.0f) {
        const int g = x.heads / x.kv_heads, kvh = head / g;
        const int slot = x.slots ? min(max(x.slots[b], 0), x.nslots - 1) : 0;
        const size_t cache = ((size_t)slot * x.kv_heads + kvh) * HD * x.context;
        const uint16_t *qr = x.qh + row * HD;
        o = 0.0f;
        for (int part = 0; part < 2; part++) {
            const int rows = part ? x.draft_context : x.context, base = part ? t.f0 : 0, count = part ? t.T : t.P;
            const uint16_t *kb = part ? x.kd + (size_t)kvh * HD * rows : x.kc + cache;
            const uint16_t *vb = (part ? x.vd + (size_t)kvh * HD * rows : x.vc + cache) + (size_t)e * rows + base;
            for (int j = 0; j < count; j++) {
                if (part && !(mrow[j >> 5] >> (j & 31) & 1))
                    continue;
                float s = 0.0f;
                for (int k = 0; k < HD; k++)
                    s = fmaf(half_bits_to_float(qr[k]),
                             half_bits_to_float(kb[((size_t)(k >> 3) * rows + base + j) * 8 + (k & 7)]), s);
                o = fmaf(exp2f(s * x.c - top + kShift), half_bits_to_float(vb[j]), o);
            }
        }
    }
    const float y = any ? o / l : 0.0f;
    const bool in = (int)blockIdx.x * 64 + lane < width;
    if (out && in)
        out[(size_t)tok * width + col] = y;
    if (q8) {
        float stored;
        int32_t sm;
        const int32_t nq = q8_0_lane(in ? y : 0.0f, &stored, &sm);
        if (in) {
            q8[(size_t)tok * width + col] = (int8_t)nq;
            if ((lane & 31) == 0) {
                scales[(size_t)tok * (width >> 5) + (col >> 5)] = stored;
                qsum[(size_t)tok * (width >> 5) + (col >> 5)] = sm;
            }
        }
    }
}

// Workgroups for two rounds of the CUs, each share at least eight steps a
// wavefront.
int splits(int n, int max_nodes, int heads, int kv_heads, int max_prefix) {
    const int tiles = (max_nodes * (heads / kv_heads) + kTile - 1) / kTile;
    const int steps = (max_prefix + kTile - 1) / kTile + (max_nodes + 7 + kTile - 1) / kTile;
    const int most = std::max(1, steps / (4 * kWaves));
    return (int)std::max<int64_t>(1, std::min<int64_t>({most, kMaxSplits, 1024 / ((int64_t)std::max(n, 1) * kv_heads * tiles) + 1}));
}

template <int HD>
int launch_hd(gx_ctx *ctx, const Args &x, float *out, int8_t *q, float *scales, int32_t *qsum) {
    const int tiles = (x.max_nodes * (x.heads / x.kv_heads) + kTile - 1) / kTile;
    const dim3 grid((unsigned)x.kv_heads, (unsigned)tiles, (unsigned)(x.n * x.S));
    attn_tree_kernel<HD><<<grid, 64 * kWaves, 0, ctx->stream>>>(x);
    if (int rc = check_launch("attention of drafted trees"))
        return rc;
    const dim3 join((unsigned)((x.heads * HD + 63) / 64), (unsigned)x.M);
    attn_tree_join_kernel<HD><<<join, 64, 0, ctx->stream>>>(x, out, q, scales, qsum);
    return check_launch("attention of drafted trees, joined");
}

}  // namespace

size_t attn_tree_workspace(int n, int M, int max_nodes, int heads, int kv_heads, int hd, int max_prefix) {
    const size_t rows = (size_t)splits(n, max_nodes, heads, kv_heads, max_prefix) * M * heads;
    return ((rows * (hd + 2) * 4) + 255) & ~(size_t)255;
}

int launch_attn_tree(gx_ctx *ctx, const TreeAttention &y, float *out, int8_t *q, float *scales, int32_t *qsum,
                     uint8_t *workspace) {
    const int S = splits(y.n, y.max_nodes, y.heads, y.kv_heads, y.max_prefix);
    float *po = (float *)workspace;
    const Args x{y.qh,      y.first,   y.mask,      y.prefix,  y.slots,
                 y.kcache,  y.vcache,  y.kdraft,    y.vdraft,  y.n,
                 y.M,       y.max_nodes, (y.max_nodes + 31) / 32, y.max_prefix, y.heads,
                 y.kv_heads, y.context, y.draft_context, y.nslots, S,
                 (float)(1.4426950408889634 / sqrt((double)y.hd)), po, po + (size_t)S * y.M * y.heads * y.hd};
    switch (y.hd) {
    case 32:
        return launch_hd<32>(ctx, x, out, q, scales, qsum);
    case 64:
        return launch_hd<64>(ctx, x, out, q, scales, qsum);
    case 96:
        return launch_hd<96>(ctx, x, out, q, scales, qsum);
    case 128:
        return launch_hd<128>(ctx, x, out, q, scales, qsum);
    default:
        return fail(GX_ERR_UNSUPPORTED, "gx: attention supports head widths 32, 64, 96 and 128");
    }
}

}  // namespace gx
