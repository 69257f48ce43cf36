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
// it stands, beside value rows read 16 bytes a lane.  Scores and probabilities
// never leave the registers.
//
// A probability enters the second product as two fp16 values, its leading 11
// bits and the next 11, cut off: together within 2^-21 of it, or within 2^-32 of
// the row's largest where that is more (the second then below fp16's normal
// numbers).  The leading bits alone would leave a head's outputs 3.5e-4 short,
// which the float output could not hide.  Sums, maxima and outputs are float32.
//
// Two kernels and a join of the keys' shares.  Trees of one tile of rows (eight
// nodes of four query heads a key-value head, say) move bytes more than they
// compute and take attn_tree_narrow_kernel, and so do larger ones over short
// prefixes; the shortest need no join.  The others take attn_tree_kernel.
#include <algorithm>
#include <type_traits>

#include "gx_device.hpp"
#include "gx_internal.hpp"

namespace gx {
namespace {

typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef float v16f __attribute__((ext_vector_type(16)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));

constexpr int kTile = 32;        // rows a wavefront
constexpr int kStage = 64;       // keys a step
constexpr int kNarrow = 32;      // keys a step of the kernel for one tile
constexpr int kMaxWaves = 8;     // wavefronts a workgroup: a tile of rows each, the keys shared
constexpr int kMaxSplits = 64;   // shares of the keys, over workgroups
// Probabilities are held times 2^8, their low parts clear of fp16's
// subnormals, and the reference the exponent is taken from follows the maximum
// only when that has risen by 2^7: still below fp16's largest.
constexpr float kShift = 8.0f, kRise = 7.0f;

struct Args {
    const uint16_t *qh;
    const int32_t *first;
    const uint32_t *mask;
    const int32_t *prefix;
    const int32_t *slots;
    const uint16_t *kc, *vc, *kd, *vd;
    int n, M, max_nodes, words, max_prefix, heads, kv_heads, context, draft_context, nslots, S, stage, halves;
    float c;       // 1 / sqrt(hd) in the exponent's base 2
    float *po;     // [S][M][heads][hd] unnormalised outputs
    float *pml;    // [S][M][heads][2] maximum (base 2) and sum
    float *out;    // the results, each optional
    int8_t *q8;
    float *scales;
    int32_t *qsum;
};

// A tree's tokens, cached positions and steps, the same for every kernel.
struct Tree {
    int f0, T, P, a, np, total, per;  // (total and per: steps)
    __device__ Tree(const Args &x, int b, int stage) : Tree(x, x.first[b], x.first[b + 1], x.prefix[b], stage) {}
    __device__ Tree(const Args &x, int from, int to, int prefix, int stage) {
        f0 = __builtin_amdgcn_readfirstlane(min(max(from, 0), x.M));
        T = __builtin_amdgcn_readfirstlane(min(min(max(to, f0), x.M) - f0, x.max_nodes));
        P = __builtin_amdgcn_readfirstlane(min(max(prefix, 0), min(x.max_prefix, x.context)));
        a = f0 & 7;  // draft rows are read from a multiple of 8
        np = (P + stage - 1) / stage;
        total = np + (T > 0 ? (a + T + stage - 1) / stage : 0);
        per = max(1, (total + x.S - 1) / x.S);
    }
};

// The larger of a lane's value and the other half's.
__device__ __forceinline__ float halves_max(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
// LDS reads asked for before this are asked for here, not where they are used.
__device__ __forceinline__ void reads_first() { asm volatile("" ::: "memory"); }

// Elements lo .. hi - 1 of eight, the rest zero.
__device__ __forceinline__ v8h keep(v8h v, int lo, int hi) {
    v8h r;
#pragma unroll
    for (int j = 0; j < 8; j++)
        r[j] = j >= lo && j < hi ? v[j] : (_Float16)0.0f;
    return r;
}

// lo/hi(a) * lo/hi(b) + c for fp16 pairs a and b, as one v_fma_mix.
__device__ __forceinline__ float fma_mix_lo(uint32_t a, uint32_t b, float c) {
    float r;
    asm("v_fma_mix_f32 %0, %1, %2, %3 op_sel_hi:[1,1,0]" : "=v"(r) : "v"(a), "v"(b), "v"(c));
    return r;
}
__device__ __forceinline__ float fma_mix_hi(uint32_t a, uint32_t b, float c) {
    float r;
    asm("v_fma_mix_f32 %0, %1, %2, %3 op_sel:[1,1,0] op_sel_hi:[1,1,0]" : "=v"(r) : "v"(a), "v"(b), "v"(c));
    return r;
}

__device__ __forceinline__ uint32_t pack_rtz(float a, float b) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(a, b));
}

// Eight keys' chances (w: which of a step's scores s), their leading 11 bits
// and the rest, added to l.
__device__ __forceinline__ void chances(const v16f &s, int w, float c, float base, v8h &ph, v8h &pl, float &l) {
    uint32_t hb[4], lb[4];
    float part = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float p = __builtin_amdgcn_exp2f(fmaf(s[8 * w + 2 * i], c, base));
        const float p1 = __builtin_amdgcn_exp2f(fmaf(s[8 * w + 2 * i + 1], c, base));
        part += p + p1;
        hb[i] = pack_rtz(p, p1);
        lb[i] = pack_rtz(fma_mix_lo(hb[i], 0xBC00BC00u, p), fma_mix_hi(hb[i], 0xBC00BC00u, p1));
    }
    l += part;
    const v4u hv = {hb[0], hb[1], hb[2], hb[3]}, lv = {lb[0], lb[1], lb[2], lb[3]};
    ph = __builtin_bit_cast(v8h, hv);
    pl = __builtin_bit_cast(v8h, lv);
}

// grid (kv_heads, row groups, trees * S), 64 threads a 32-row tile of the
// group: key-value heads fastest, so that with eight of them every workgroup
// of a head is on one XCD and shares its L2.
//
// 64 nodes of 32 heads over 8, 128 wide, and 32000 positions take 60 us, 2.2
// TB/s of keys and values; the join 8 us.  Some 45 of the 60 are matrix
// instructions: 1500 a SIMD (48 a step and wavefront) at 30 ns each, where a
// large fp16 product of a library reaches 28; they keep the matrix units busy
// for 47 % of the kernel's cycles by the counters.  What is left was not taken
// apart: the launch, the first step's loads, and the shares' outputs, 34 MB
// that all workgroups write at the end.  A second wavefront a SIMD adds nothing
// to a step's rate, nor did scores and products of neighbouring steps side by
// side (65 us), a longer ring, or an order of the instructions laid down by
// hand.  Eight trees of up to 33 nodes over 1500 positions take 23.5 us: 15 of
// matrix instructions on the SIMDs that have one and a half tiles of a 33-node
// tree (every tree gets the same shares, so that the average SIMD has half of
// that).
//
// A step's 64 keys and values come into LDS by direct loads, one step ahead of
// the products, for every tile of the group: the keys as 1 KiB pieces of 64
// positions, a value row's 128 bytes with its eight 16-byte chunks exchanged
// by the row's low bits, so that both the loads (eight whole rows each) and
// the operand reads (a chunk of 32 rows) go round the banks (two cycles of
// conflict an LDS instruction by the counters).
template <int HD>
__global__ __launch_bounds__(64 * kMaxWaves) void attn_tree_kernel(const Args x) {
    constexpr int KS = HD / 16, ET = HD / 32, kSlot = HD * 256;
    extern __shared__ __align__(16) uint8_t lds[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int nw = blockDim.x >> 6, li = lane & 31, h = lane >> 5;
    const int kvh = blockIdx.x, b = blockIdx.z / x.S, sp = blockIdx.z % x.S;
    const Tree t(x, b, kStage);
    // Five or six tiles: the first four a wavefront each, the others two, one of
    // a step's halves each, so that no SIMD has two whole tiles (eight trees of
    // 33 nodes over 4000 positions 46 us, and 51 with five whole ones; of 80, 81 and 91).
    const int tiles = x.halves ? nw / 2 + 2 : nw, whole = x.halves ? 4 : nw;
    const int half = wave < whole ? 0 : (wave - whole) & 1, tile = wave < whole ? wave : whole + (wave - whole) / 2;
    const int g = x.heads / x.kv_heads, R = t.T * g, g0 = blockIdx.y * tiles * kTile, r0 = g0 + tile * kTile;
    const int t0 = sp * t.per, t1 = min(t.total, t0 + t.per);
    if (g0 >= R || t0 >= t1)
        return;
    const int slot = __builtin_amdgcn_readfirstlane(x.slots ? min(max(x.slots[b], 0), x.nslots - 1) : 0);
    const size_t cache = ((size_t)slot * x.kv_heads + kvh) * HD * x.context;
    const uint16_t *kc = x.kc + cache, *vc = x.vc + cache;
    const uint16_t *kd = x.kd + (size_t)kvh * HD * x.draft_context, *vd = x.vd + (size_t)kvh * HD * x.draft_context;

    // step j's rows: where they begin, and which of them there are
    auto rows_of = [&](int j, int &p0, int &lo, int &hi) __attribute__((always_inline)) {
        const bool draft = j >= t.np;
        p0 = draft ? t.f0 - t.a + kStage * (j - t.np) : kStage * j;
        lo = draft ? t.f0 : 0;
        hi = draft ? t.f0 + t.T : t.P;
        return draft;
    };
    auto load = [&](int j, uint8_t *to) __attribute__((always_inline)) {
        int p0, lo, hi;
        const bool draft = rows_of(j, p0, lo, hi);
        const int rows = draft ? x.draft_context : x.context;
        const char *kb = (const char *)(draft ? kd : kc), *vb = (const char *)(draft ? vd : vc);
        const uint32_t kp = (uint32_t)min(max(p0 + lane, lo), hi - 1) * 16;
        const int pv = min(max(p0 + 8 * ((lane & 7) ^ (lane >> 3)), lo & ~7), (hi - 1) & ~7);
        const uint32_t vp = ((uint32_t)(lane >> 3) * rows + pv) * 2;
        // (a uniform base and the lane's 32-bit offset: no vector instruction a load)
        for (int i = wave; i < HD / 8; i += nw) {
            const char *src = kb + (size_t)i * rows * 16;
            asm("" : "+s"(src));
            __builtin_amdgcn_global_load_lds(src + kp, (lds_ptr)(to + i * 1024), 16, 0, 0);
        }
        for (int i = wave; i < HD / 8; i += nw) {
            const char *src = vb + (size_t)i * rows * 16;
            asm("" : "+s"(src));
            __builtin_amdgcn_global_load_lds(src + vp, (lds_ptr)(to + HD * 128 + i * 1024), 16, 0, 0);
        }
    };
    load(t0, lds);

    const int r = min(r0 + li, R - 1), node = r / g;
    const uint16_t *qr = x.qh + ((size_t)(t.f0 + node) * x.heads + kvh * g + (r - node * g)) * HD + 8 * h;
    v8h q[KS];
#pragma unroll
    for (int s = 0; s < KS; s++)
        q[s] = *(const v8h *)(qr + 16 * s);
    const uint32_t *mrow = x.mask + (size_t)(t.f0 + node) * x.words;
    uint32_t mw[3] = {0u, mrow[0], x.words > 1 ? mrow[1] : 0u};  // the words before, at and after a draft step's first
    const uint32_t klane = h * 1024 + ((li & ~12) | ((li & 4) << 1) | ((li & 8) >> 1)) * 16;
    const uint32_t vlane = HD * 128 + li * 128, vx = h ^ (li & 7);

    // the first four wavefronts go first: the others' matrix products then run
    // beside their exponentials (up to 3 us of 60, as the clock allows)
    if (wave < 4)
        __builtin_amdgcn_s_setprio(1);
    v16f o[ET] = {};
    float m = -INFINITY, l = 0.0f;  // m: in the scores' own units
    int at = 0;
    // the steps, 32 U keys of each from the u0-th half on
    auto steps = [&](auto count, int u0) __attribute__((always_inline)) {
        constexpr int U = decltype(count)::value;
        for (int j = t0; j < t1; j++, at = kSlot - at) {
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            lds_barrier();
            if (j + 1 < t1)
                load(j + 1, lds + (kSlot - at));
            uint8_t *st = lds + at;
            int p0, lo, hi;
            const bool draft = rows_of(j, p0, lo, hi);
            // Keys and chunks of values past the rows that there are repeat one that is
            // (its chance will be zero).  The rows beside those become zero, in the
            // chunk with the first and in the chunk with the last and every copy of it:
            // a NaN there would make 0 * NaN in every row's sums.
            const int cl = p0 < lo ? 0 : 8, ch = p0 + kStage > hi && (hi & 7) ? (hi - p0) >> 3 : 8;
            if (cl < 8 || ch < 8) {
                for (int i = tid; i < 8 * HD; i += 64 * nw) {
                    const int e = i >> 3, c = i & 7;
                    if (c == cl || c >= ch) {
                        v8h *to = (v8h *)(st + HD * 128 + e * 128 + ((c ^ (e & 7)) << 4));
                        *to = keep(*to, lo - (p0 + 8 * c), hi - (p0 + 8 * c));
                    }
                }
                lds_barrier();
            }
            if (r0 >= R)
                continue;
            v8h a[KS][U];
#pragma unroll
            for (int k = 0; k < KS; k++)
#pragma unroll
                for (int u = 0; u < U; u++)
                    a[k][u] = *(const v8h *)(st + klane + 2048 * k + 512 * (u0 + u));
            reads_first();
            v16f s[U] = {};
#pragma unroll
            for (int k = 0; k < KS; k++)
#pragma unroll
                for (int u = 0; u < U; u++)
                    s[u] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[k][u], q[k], s[u], 0, 0, 0);
            v8h v[2 * U][ET];
            auto values = [&](int w) __attribute__((always_inline)) {
#pragma unroll
                for (int et = 0; et < ET; et++)
                    v[w][et] = *(const v8h *)(st + vlane + 4096 * et + (((uint32_t)(2 * (2 * u0 + w)) ^ vx) << 4));
            };
            values(0);
            values(1);
            reads_first();
            if (draft || p0 + kStage > hi) {
                // bit k of sees[u]: key 32 (u0 + u) + k of the step
                const int above = hi - p0, below = max(lo - p0, 0);
                uint32_t sees[U];
#pragma unroll
                for (int u = 0; u < U; u++) {
                    const int n = min(max(above - 32 * (u0 + u), 0), 32), z = min(max(below - 32 * (u0 + u), 0), 32);
                    sees[u] = (uint32_t)((1ull << n) - (1ull << z)) & (n > z ? ~0u : 0u);
                }
                if (draft) {
                    const int w0 = 2 * (j - t.np);  // bits from node 32 w0 - a on
                    if (w0 > 0) {
#pragma unroll
                        for (int i = 0; i < 3; i++)
                            mw[i] = w0 + i <= x.words ? mrow[w0 + i - 1] : 0u;
                    }
#pragma unroll
                    for (int u = 0; u < U; u++) {
                        const uint32_t here = U == 1 && u0 ? mw[2] : mw[u + 1], last = U == 1 && u0 ? mw[1] : mw[u];
                        sees[u] &= t.a ? (here << t.a) | (last >> (32 - t.a)) : here;
                    }
                }
#pragma unroll
                for (int u = 0; u < U; u++) {
                    const uint32_t bits = sees[u] >> (8 * h);
#pragma unroll
                    for (int i = 0; i < 16; i++)
                        s[u][i] = bits >> (16 * (i >> 3) + (i & 7)) & 1 ? s[u][i] : -INFINITY;
                }
            }
            float mx = -INFINITY;
#pragma unroll
            for (int u = 0; u < U; u++)
#pragma unroll
                for (int i = 0; i < 16; i++)
                    mx = fmaxf(mx, s[u][i]);
            mx = halves_max(mx);
            // (a row that sees nothing yet, or whose maximum has risen past what the
            // reference allows: the reference becomes the maximum)
            if (__ballot(mx * x.c > m * x.c + kRise || (m == -INFINITY && mx > m))) {
                const float mn = fmaxf(m, mx);
                const float corr = mn == m ? 1.0f : __builtin_amdgcn_exp2f((m - mn) * x.c);
                m = mn;
                l *= corr;
#pragma unroll
                for (int et = 0; et < ET; et++)
#pragma unroll
                    for (int i = 0; i < 16; i++)
                        o[et][i] *= corr;
            }
            const float base = kShift - (m == -INFINITY ? 0.0f : m * x.c);
            v8h ph[2 * U], pl[2 * U];
            chances(s[0], 0, x.c, base, ph[0], pl[0], l);
#pragma unroll
            for (int w = 0; w < 2 * U; w++) {
#pragma unroll
                for (int et = 0; et < ET; et++)
                    o[et] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v[w][et], ph[w], o[et], 0, 0, 0);
#pragma unroll
                for (int et = 0; et < ET; et++)
                    o[et] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v[w][et], pl[w], o[et], 0, 0, 0);
                if (w + 2 < 2 * U)
                    values(w + 2);
                if (w + 1 < 2 * U)
                    chances(s[(w + 1) >> 1], (w + 1) & 1, x.c, base, ph[w + 1], pl[w + 1], l);
            }
        }
    };
    // (the loops meet at the same barriers)
    if (x.halves && wave >= whole)
        steps(std::integral_constant<int, 1>(), half);
    else
        steps(std::integral_constant<int, 2>(), 0);
    l += __shfl_xor(l, 32);
    if (x.halves) {  // a tile's second half joins its first
        lds_barrier();
        v4f *to = (v4f *)lds + (wave - whole) / 2 * (ET * 4 * 64) + lane;
        float *const ml = (float *)(lds + kSlot) + (wave - whole) / 2 * 128 + lane;
        if (wave >= whole && half) {
#pragma unroll
            for (int k = 0; k < 4 * ET; k++)
                to[64 * k] = v4f{o[k / 4][4 * (k % 4)], o[k / 4][4 * (k % 4) + 1], o[k / 4][4 * (k % 4) + 2],
                                 o[k / 4][4 * (k % 4) + 3]};
            ml[0] = m;
            ml[64] = l;
        }
        lds_barrier();
        if (half)
            return;
        if (wave >= whole) {
            const float m2 = ml[0], l2 = ml[64], mn = fmaxf(m, m2);
            const float c1 = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((m - mn) * x.c);
            const float c2 = m2 == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((m2 - mn) * x.c);
            // (a half that saw nothing, or nothing but NaN, has no maximum)
            l = (m == -INFINITY ? l : l * c1) + (m2 == -INFINITY ? l2 : l2 * c2);
            m = mn;
#pragma unroll
            for (int k = 0; k < 4 * ET; k++) {
                const v4f z = to[64 * k];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float y = o[k / 4][4 * (k % 4) + i];
                    o[k / 4][4 * (k % 4) + i] = (c1 == 0.0f ? 0.0f : y * c1) + (c2 == 0.0f ? 0.0f : z[i] * c2);
                }
            }
        }
    }
    if (r0 + li >= R)
        return;
    const size_t row = ((size_t)sp * x.M + t.f0 + node) * x.heads + kvh * g + (r - node * g);
    float *po = x.po + row * HD + 4 * h;
#pragma unroll
    for (int et = 0; et < ET; et++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const v4f w = {o[et][4 * i], o[et][4 * i + 1], o[et][4 * i + 2], o[et][4 * i + 3]};
            *(v4f *)(po + 32 * et + 8 * i) = w;
        }
    if (h == 0) {
        x.pml[2 * row] = m == -INFINITY ? m : m * x.c;
        x.pml[2 * row + 1] = l;
    }
}

// The elements of a row that a masked value has spoilt (an infinite or NaN
// value that the mask hides makes 0 * inf in its step), summed again over what
// the node sees alone: 64 keys at a time, a key a lane, the spoilt elements in
// turn.  o: four of the row's outputs, from element e on; spoilt: which of them.
template <int HD>
__device__ __forceinline__ v4f attn_tree_again(const Args &x, const Tree &t, int b, int tok, int head, float top, v4f o,
                                               int e, uint32_t spoilt) {
    const int lane = threadIdx.x & 63, kvh = head / (x.heads / x.kv_heads);
    const int slot = x.slots ? min(max(x.slots[b], 0), x.nslots - 1) : 0;
    const size_t cache = ((size_t)slot * x.kv_heads + kvh) * HD * x.context;
    const uint16_t *qr = x.qh + ((size_t)tok * x.heads + head) * HD;
    const uint32_t *mrow = x.mask + (size_t)tok * x.words;
#pragma unroll
    for (int i = 0; i < 4; i++)
        o[i] = spoilt >> i & 1 ? 0.0f : o[i];
    for (int part = 0; part < 2; part++) {
        const int rows = part ? x.draft_context : x.context, base = part ? t.f0 : 0, count = part ? t.T : t.P;
        const uint16_t *kb = part ? x.kd + (size_t)kvh * HD * rows : x.kc + cache;
        const uint16_t *vb = part ? x.vd + (size_t)kvh * HD * rows : x.vc + cache;
        for (int j0 = 0; j0 < count; j0 += 64) {
            const int j = min(j0 + lane, count - 1);
            const bool sees = j0 + lane < count && (!part || (mrow[j >> 5] >> (j & 31) & 1));
            float s = 0.0f;
            for (int k = 0; k < HD; k++)
                s = fmaf(half_bits_to_float(qr[k]), half_bits_to_float(kb[((size_t)(k >> 3) * rows + base + j) * 8 + (k & 7)]),
                         s);
            const float p = exp2f(s * x.c - top + kShift);
#pragma unroll
            for (int i = 0; i < 4; i++)
                for (unsigned long long who = __ballot(spoilt >> i & 1); who; who &= who - 1) {
                    const int l = __builtin_ctzll(who);
                    const float v = half_bits_to_float(vb[(size_t)(__shfl(e, l) + i) * rows + base + j]);
                    const float sum = wave_pairwise_sum(sees ? p * v : 0.0f);
                    if (lane == l)
                        o[i] += sum;
                }
        }
    }
    return o;
}

// Four elements' results at `at`: the quotients, and the Q8_0 of 32 elements by
// the eight lanes that hold them.
__device__ __forceinline__ void attn_tree_store(const Args &x, v4f o, bool any, float l, size_t at) {
    float y[4];
#pragma unroll
    for (int i = 0; i < 4; i++)
        y[i] = any ? o[i] / l : 0.0f;
    if (x.out && ((uintptr_t)x.out & 15) == 0)
        *(v4f *)(x.out + at) = v4f{y[0], y[1], y[2], y[3]};
    else if (x.out)
        for (int i = 0; i < 4; i++)
            x.out[at + i] = y[i];
    if (x.q8) {
        float stored;
        int32_t sm;
        const uint32_t packed = q8_0_quad(y, &stored, &sm);
        if (((uintptr_t)x.q8 & 3) == 0)
            *(uint32_t *)(x.q8 + at) = packed;
        else
            for (int i = 0; i < 4; i++)
                x.q8[at + i] = (int8_t)(packed >> (8 * i));
        if ((threadIdx.x & 7) == 0) {
            x.scales[at >> 5] = stored;
            x.qsum[at >> 5] = sm;
        }
    }
}

// A tile of a tree's rows: eight wavefronts of a workgroup take steps of 32 keys
// in turn, each with its own maximum and sum, keys and values straight into
// registers: the next step's keys asked for before this one's products, its
// values as soon as this one's are used.  The wavefronts' results are added in
// LDS.  Where one workgroup covers the keys (S 1) it writes the results itself,
// and there is no join.  grid (kv_heads, tiles, trees * S).
//
// Bound by the loads: 64 trees of five nodes over 2000 positions (8 key-value
// heads, 128 wide) read 524 MB in 103 us, 5.1 TB/s; one tree over 32000 takes
// 38 us with its join, eight over 1500 take 17 where the kernel for more tiles
// takes 21, 32 over 500 take 16 where it takes 23, and one over 60 takes 7
// where it and the join take 10.
template <int HD>
__global__ __launch_bounds__(512) void attn_tree_narrow_kernel(const Args x) {
    constexpr int KS = HD / 16, ET = HD / 32, W = 8;
    __shared__ __align__(16) float lds[W * kTile * 64];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int li = lane & 31, h = lane >> 5;
    const int kvh = blockIdx.x, b = blockIdx.z / x.S, sp = blockIdx.z % x.S;
    const Tree t(x, b, kNarrow);
    const int g = x.heads / x.kv_heads, R = t.T * g, r0 = blockIdx.y * kTile;
    const int t0 = sp * t.per, t1 = min(t.total, t0 + t.per);
    if (r0 >= R || t0 >= t1)
        return;
    const int slot = __builtin_amdgcn_readfirstlane(x.slots ? min(max(x.slots[b], 0), x.nslots - 1) : 0);
    const size_t cache = ((size_t)slot * x.kv_heads + kvh) * HD * x.context;
    const uint16_t *kc = x.kc + cache, *vc = x.vc + cache;
    const uint16_t *kd = x.kd + (size_t)kvh * HD * x.draft_context, *vd = x.vd + (size_t)kvh * HD * x.draft_context;
    const int swapped = (li & ~12) | ((li & 4) << 1) | ((li & 8) >> 1);

    // step j's rows: where they begin, and which of them there are
    auto rows_of = [&](int j, int &p0, int &lo, int &hi) __attribute__((always_inline)) {
        const bool draft = j >= t.np;
        p0 = draft ? t.f0 - t.a + kNarrow * (j - t.np) : kNarrow * j;
        lo = draft ? t.f0 : 0;
        hi = draft ? t.f0 + t.T : t.P;
        return draft;
    };
    v8h a0[KS], a1[KS], v[2][ET];
    auto load_keys = [&](int j, v8h *a) __attribute__((always_inline)) {
        int p0, lo, hi;
        const bool draft = rows_of(j, p0, lo, hi);
        const int rows = draft ? x.draft_context : x.context;
        const char *kb = (const char *)(draft ? kd : kc);
        const uint32_t at = ((uint32_t)h * rows + min(max(p0 + swapped, lo), hi - 1)) * 16;
#pragma unroll
        for (int k = 0; k < KS; k++)
            a[k] = *(const v8h *)(kb + (size_t)(2 * k) * rows * 16 + at);
    };
    auto load_values = [&](int j) __attribute__((always_inline)) {
        int p0, lo, hi;
        const bool draft = rows_of(j, p0, lo, hi);
        const int rows = draft ? x.draft_context : x.context;
        const char *vb = (const char *)(draft ? vd : vc);
#pragma unroll
        for (int w = 0; w < 2; w++) {
            const int c = min(max(p0 + 16 * w + 8 * h, lo & ~7), (hi - 1) & ~7);
            const uint32_t at = ((uint32_t)li * rows + c) * 2;
#pragma unroll
            for (int et = 0; et < ET; et++)
                v[w][et] = *(const v8h *)(vb + (size_t)(32 * et) * rows * 2 + at);
        }
    };
    const int r = min(r0 + li, R - 1), node = r / g;
    v16f o[ET] = {};
    float m = -INFINITY, l = 0.0f;  // m: in the scores' own units
    int j = t0 + wave;
    if (j < t1) {
        load_keys(j, a0);
        const uint16_t *qr = x.qh + ((size_t)(t.f0 + node) * x.heads + kvh * g + (r - node * g)) * HD + 8 * h;
        v8h q[KS];
#pragma unroll
        for (int s = 0; s < KS; s++)
            q[s] = *(const v8h *)(qr + 16 * s);
        const uint32_t *mrow = x.mask + (size_t)(t.f0 + node) * x.words;
        const uint32_t first = mrow[0];
        load_values(j);
        reads_first();
        auto step = [&](v8h *a, v8h *an) __attribute__((always_inline)) {
            const bool more = j + W < t1;
            if (more)
                load_keys(j + W, an);
            reads_first();
            v16f s = {}, s1 = {};
#pragma unroll
            for (int k = 0; k < KS; k += 2) {
                s = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[k], q[k], s, 0, 0, 0);
                s1 = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[k + 1], q[k + 1], s1, 0, 0, 0);
            }
            s += s1;
            int p0, lo, hi;
            const bool draft = rows_of(j, p0, lo, hi);
            if (draft || p0 + kNarrow > hi) {
                // bit k of sees: key k of the step; values past the rows there are become zero
                uint32_t sees = hi - p0 >= kNarrow ? ~0u : (1u << (hi - p0)) - 1;
                if (draft) {
                    const int w = j - t.np;
                    const uint32_t here = w == 0 ? first : w < x.words ? mrow[w] : 0u;
                    const uint32_t last = w == 0 ? 0u : w == 1 ? first : mrow[w - 1];
                    sees &= t.a ? (here << t.a) | (last >> (32 - t.a)) : here;
                }
                const uint32_t bits = sees >> (8 * h);
#pragma unroll
                for (int i = 0; i < 16; i++)
                    s[i] = bits >> (16 * (i >> 3) + (i & 7)) & 1 ? s[i] : -INFINITY;
#pragma unroll
                for (int w = 0; w < 2; w++) {
                    const int c = min(max(p0 + 16 * w + 8 * h, lo & ~7), (hi - 1) & ~7);
#pragma unroll
                    for (int et = 0; et < ET; et++)
                        v[w][et] = keep(v[w][et], lo - c, hi - c);
                }
            }
            float mx = -INFINITY;
#pragma unroll
            for (int i = 0; i < 16; i++)
                mx = fmaxf(mx, s[i]);
            mx = halves_max(mx);
            if (__ballot(mx * x.c > m * x.c + kRise || (m == -INFINITY && mx > m))) {
                const float mn = fmaxf(m, mx);
                const float corr = mn == m ? 1.0f : __builtin_amdgcn_exp2f((m - mn) * x.c);
                m = mn;
                l *= corr;
#pragma unroll
                for (int et = 0; et < ET; et++)
#pragma unroll
                    for (int i = 0; i < 16; i++)
                        o[et][i] *= corr;
            }
            const float base = kShift - (m == -INFINITY ? 0.0f : m * x.c);
#pragma unroll
            for (int w = 0; w < 2; w++) {
                v8h ph, pl;
                chances(s, w, x.c, base, ph, pl, l);
#pragma unroll
                for (int et = 0; et < ET; et++)
                    o[et] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v[w][et], ph, o[et], 0, 0, 0);
#pragma unroll
                for (int et = 0; et < ET; et++)
                    o[et] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v[w][et], pl, o[et], 0, 0, 0);
            }
            if (more)
                load_values(j + W);
            reads_first();
        };
        for (;;) {
            step(a0, a1);
            if ((j += W) >= t1)
                break;
            step(a1, a0);
            if ((j += W) >= t1)
                break;
        }
        l += __shfl_xor(l, 32);
    }
    // the wavefronts' maxima and sums, then their outputs times their weights, 64
    // elements a round: a row's sixteen pieces exchanged by its low bits, without
    // conflicts both ways
    if (h == 0) {
        lds[wave * kTile + li] = m;
        lds[(W + wave) * kTile + li] = l;
    }
    __syncthreads();
    const int row = tid >> 4, piece = tid & 15;  // what this thread adds up
    const int had = min(W, t1 - t0);             // wavefronts that had a step
    float top = -INFINITY, mine = -INFINITY, sum = 0.0f;
#pragma unroll
    for (int w = 0; w < W; w++) {
        top = fmaxf(top, lds[w * kTile + row]);
        mine = fmaxf(mine, lds[w * kTile + li]);
    }
#pragma unroll
    for (int w = 0; w < W; w++) {
        // (a wavefront that saw nothing, or nothing but NaN, has no maximum)
        const float mw = lds[w * kTile + row], lw = lds[(W + w) * kTile + row];
        sum += mw == -INFINITY ? lw : lw * __builtin_amdgcn_exp2f((mw - top) * x.c);
    }
    const float weight = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((m - mine) * x.c);
    constexpr int kRounds = (ET + 1) / 2;
    v4f y[kRounds];
#pragma unroll
    for (int k = 0; k < kRounds; k++) {
        __syncthreads();
        float *to = lds + (wave * kTile + li) * 64;
        if (wave < had)
#pragma unroll
            for (int e2 = 0; e2 < 2 && 2 * k + e2 < ET; e2++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    v4f z;
#pragma unroll
                    for (int u = 0; u < 4; u++)
                        z[u] = weight == 0.0f ? 0.0f : o[2 * k + e2][4 * i + u] * weight;
                    *(v4f *)(to + 4 * ((8 * e2 + 2 * i + h) ^ (li & 15))) = z;
                }
        __syncthreads();
        y[k] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
        if (64 * k + 4 * piece < HD)
#pragma unroll
            for (int w = 0; w < W; w++) {
                const v4f z = *(const v4f *)(lds + (w * kTile + row) * 64 + 4 * (piece ^ (row & 15)));
                y[k] += w < had ? z : v4f{0.0f, 0.0f, 0.0f, 0.0f};
            }
    }
    const bool there = r0 + row < R;
    const int rr = min(r0 + row, R - 1), tn = rr / g, tok = t.f0 + tn, head = kvh * g + (rr - tn * g);
    if (x.S > 1) {
        const size_t part = ((size_t)sp * x.M + tok) * x.heads + head;
#pragma unroll
        for (int k = 0; k < kRounds; k++)
            if (there && 64 * k + 4 * piece < HD)
                *(v4f *)(x.po + part * HD + 64 * k + 4 * piece) = y[k];
        if (there && piece == 0) {
            x.pml[2 * part] = top == -INFINITY ? top : top * x.c;
            x.pml[2 * part + 1] = sum;
        }
        return;
    }
    bool any = t.P > 0;
    for (int w = 0; !any && 32 * w < t.T; w++)
        any = (x.mask[(size_t)tok * x.words + w] & (t.T - 32 * w >= 32 ? ~0u : (1u << (t.T - 32 * w)) - 1)) != 0;
#pragma unroll
    for (int k = 0; k < kRounds; k++) {
        const int e = 64 * k + 4 * piece;
        uint32_t spoilt = 0;
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (there && e < HD && any && sum - sum == 0.0f && y[k][i] - y[k][i] != 0.0f)
                spoilt |= 1u << i;
        for (unsigned long long who = __ballot(spoilt != 0); who;) {  // a row after another
            const int first = __builtin_ctzll(who) & ~15;
            const uint32_t here = (lane & ~15) == first ? spoilt : 0u;
            y[k] = attn_tree_again<HD>(x, t, b, __builtin_amdgcn_readlane(tok, first),
                                       __builtin_amdgcn_readlane(head, first),
                                       __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(top), first)) * x.c,
                                       y[k], e, here);
            who &= ~(0xFFFFull << first);
        }
        if (there && e < HD)
            attn_tree_store(x, y[k], any, sum, ((size_t)tok * x.heads + head) * HD + e);
    }
}

// A row (a node's head) a wavefront: its shares' maxima and sums a lane each,
// its outputs four elements a lane, several shares side by side, added in a
// fixed order; and the Q8_0 of 32 elements.  grid (heads / 4, M), 256 threads.
// Bound by its launch and loads for few rows (4.1 us for five nodes
// of 32 heads in nine shares), by the shares' bytes for more (8.2 for 64 nodes in
// 32 shares, 34 MB).
template <int HD>
__global__ __launch_bounds__(256) void attn_tree_join_kernel(const Args x) {
    constexpr int L = HD / 4, SP = 64 / L;  // lanes a share, shares side by side
    const int lane = threadIdx.x & 63, tok = blockIdx.y;
    const int head = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (head >= x.heads)
        return;
    // All that hangs on the token alone is asked for together, whichever of the
    // shares there are.
    const size_t row = (size_t)tok * x.heads + head, step = (size_t)x.M * x.heads;
    const int g = lane / L, e = 4 * (lane - g * L);
    typedef float v2f __attribute__((ext_vector_type(2)));
    const v2f ml = *(const v2f *)(x.pml + (min(lane, x.S - 1) * step + row) * 2);
    const float *po = x.po + row * HD + e;
    auto shares = [&](int s0, v4f *p) __attribute__((always_inline)) {
#pragma unroll
        for (int k = 0; k < 4; k++)
            p[k] = *(const v4f *)(po + (size_t)min(s0 + k * SP + g, x.S - 1) * step * HD);
    };
    v4f p[4];
    shares(0, p);
    const uint32_t seen = x.mask[(size_t)tok * x.words + min(lane, x.words - 1)];
    int b = -1, from = 0, to = 0, prefix = 0;  // the tree: the last whose first token is not past this one
    for (int i = 0; i < x.n; i += 64) {
        const int k = min(i + lane, x.n - 1), f0 = x.first[k], f1 = x.first[k + 1], before = x.prefix[k];
        reads_first();
        const int count = __popcll(__ballot(i + lane < x.n && f0 <= tok));
        if (count > 0) {
            b = i + count - 1;
            from = __builtin_amdgcn_readlane(f0, count - 1);
            to = __builtin_amdgcn_readlane(f1, count - 1);
            prefix = __builtin_amdgcn_readlane(before, count - 1);
        }
    }
    const Tree t(x, from, to, prefix, x.stage);
    if (b < 0 || tok < t.f0 || tok >= t.f0 + t.T)
        return;
    const int live = (t.total + t.per - 1) / t.per;  // at most S
    const int bits = t.T - 32 * lane;                // nodes that this lane's mask word speaks of
    const uint32_t word = bits > 0 ? seen & (bits >= 32 ? ~0u : (1u << bits) - 1) : 0u;
    const bool any = t.P > 0 || __ballot(word != 0) != 0;
    const float m = lane < live ? ml.x : -INFINITY, top = wave_max(m);
    const float weight = m == -INFINITY ? 0.0f : exp2f(m - top);
    // (a share that saw nothing, or nothing but NaN, has no maximum)
    const float l = wave_pairwise_sum(lane < live ? (m == -INFINITY ? ml.y : ml.y * weight) : 0.0f);
    v4f o = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int s0 = 0; s0 < live; s0 += 4 * SP) {
        if (s0 > 0)
            shares(s0, p);
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const int s = s0 + k * SP + g;
            const float w = __shfl(weight, s & 63);
            if (s < live && w != 0.0f && g < SP)
                o += p[k] * w;
        }
    }
    for (int k = 1; k < SP; k++) {
        v4f p;
#pragma unroll
        for (int i = 0; i < 4; i++)
            p[i] = __shfl(o[i], (lane + k * L) & 63);
        if (lane < L)
            o += p;
    }
    uint32_t spoilt = 0;
#pragma unroll
    for (int i = 0; i < 4; i++)
        if (lane < L && any && l - l == 0.0f && o[i] - o[i] != 0.0f)
            spoilt |= 1u << i;
    if (__ballot(spoilt != 0))
        o = attn_tree_again<HD>(x, t, b, tok, head, top, o, e, spoilt);
    if (lane >= L)
        return;
    attn_tree_store(x, o, any, l, (size_t)tok * x.heads * HD + head * HD + e);
}

// Wavefronts a workgroup: a group's tiles of rows, the groups alike.
struct Groups {
    int waves, groups, halves;
    Groups(int max_nodes, int heads, int kv_heads) {
        const int tiles = (max_nodes * (heads / kv_heads) + kTile - 1) / kTile;
        groups = (tiles + kMaxWaves - 1) / kMaxWaves;
        waves = (tiles + groups - 1) / groups;
        halves = waves == 5 || waves == 6;  // (the kernel's `tiles` from its wavefronts)
        if (halves)
            waves = 2 * waves - 4;
    }
};

// How a call's rows and keys are shared out.
struct Shares {
    bool narrow;  // attn_tree_narrow_kernel's
    int tiles;    // of rows a tree
    int S;        // shares of the keys
};

// A tile a workgroup (narrow): one share, and no join, up to two steps a
// wavefront (five nodes over 250 positions 9.4 us, and 9.8 in shares; 64 over 300
// 10.1 and 11.5; five over 500 11.8 and 10.0); past that two steps a share while
// there are CUs (four: 10.5 for the 10.0; sixteen: 12.2; two workgroups a CU 46 us
// over 32000 positions where one takes 38).  Trees of more tiles read the keys
// again for each, from the caches, which costs less than the other kernel's
// workgroups of several tiles up to seven steps a wavefront: 64 nodes over 20
// positions 7.6 us for 14.1, over 2000 15.8 for 20.1; eight trees of 30 over 800
// 16.4 for 21.9; at seven twelve of 20 over 800 16.7 for 21.8 and one of 33 over
// 10000 28.2 for 27.0; at eight twelve of twelve over 2000 40.4 for 29.4.
// That kernel: as many workgroups as run at once (two wavefronts a SIMD by their
// registers, two workgroups a CU by their LDS), so that the last round is whole
// (512 of more than four wavefronts: 82 us where 256 take 70).
Shares shares(int n, int max_nodes, int heads, int kv_heads, int max_prefix) {
    const int tiles = (max_nodes * (heads / kv_heads) + kTile - 1) / kTile;
    const int64_t trees = (int64_t)std::max(n, 1) * kv_heads, all = trees * tiles;
    const int few = (max_prefix + kNarrow - 1) / kNarrow + (max_nodes + 7 + kNarrow - 1) / kNarrow;
    const int64_t S = few <= 16 ? 1 : std::max<int64_t>(1, std::min<int64_t>({(few + 1) / 2, kMaxSplits, 256 / all}));
    if (tiles == 1 || (all * S + 255) / 256 * few <= 7 * 8 * S)
        return {true, tiles, (int)S};
    const Groups w(max_nodes, heads, kv_heads);
    const int steps = (max_prefix + kStage - 1) / kStage + (max_nodes + 7 + kStage - 1) / kStage;
    const int64_t one = trees * w.groups, most = w.waves > 4 ? 256 : 512;
    return {false, tiles, (int)std::max<int64_t>(1, std::min<int64_t>({steps, kMaxSplits, most / one}))};
}

template <int HD>
int launch_hd(gx_ctx *ctx, const Args &x, const Shares &y) {
    if (y.narrow) {
        const dim3 grid((unsigned)x.kv_heads, (unsigned)y.tiles, (unsigned)(x.n * x.S));
        attn_tree_narrow_kernel<HD><<<grid, 512, 0, ctx->stream>>>(x);
    } else {
        const Groups w(x.max_nodes, x.heads, x.kv_heads);
        const dim3 grid((unsigned)x.kv_heads, (unsigned)w.groups, (unsigned)(x.n * x.S));
        attn_tree_kernel<HD><<<grid, 64 * w.waves, 2 * 256 * HD, ctx->stream>>>(x);
    }
    if (int rc = check_launch("attention of drafted trees"))
        return rc;
    if (y.narrow && x.S == 1)
        return GX_OK;
    const dim3 join((unsigned)((x.heads + 3) / 4), (unsigned)x.M);
    attn_tree_join_kernel<HD><<<join, 256, 0, ctx->stream>>>(x);
    return check_launch("attention of drafted trees, joined");
}

}  // namespace

size_t attn_tree_workspace(int n, int M, int max_nodes, int heads, int kv_heads, int hd, int max_prefix) {
    const size_t rows = (size_t)shares(n, max_nodes, heads, kv_heads, max_prefix).S * M * heads;
    return ((rows * (hd + 2) * 4) + 255) & ~(size_t)255;
}

int launch_attn_tree(gx_ctx *ctx, const TreeAttention &y, float *out, int8_t *q, float *scales, int32_t *qsum,
                     uint8_t *workspace) {
    const Shares how = shares(y.n, y.max_nodes, y.heads, y.kv_heads, y.max_prefix);
    const int S = how.S;
    float *po = (float *)workspace;
    const Args x{y.qh,      y.first,   y.mask,      y.prefix,  y.slots,
                 y.kcache,  y.vcache,  y.kdraft,    y.vdraft,  y.n,
                 y.M,       y.max_nodes, (y.max_nodes + 31) / 32, y.max_prefix, y.heads,
                 y.kv_heads, y.context, y.draft_context, y.nslots, S,
                 how.narrow ? kNarrow : kStage,
                 Groups(y.max_nodes, y.heads, y.kv_heads).halves,
                 (float)(1.4426950408889634 / sqrt((double)y.hd)), po, po + (size_t)S * y.M * y.heads * y.hd,
                 out,       q,         scales,      qsum};
    switch (y.hd) {
    case 32:
        return launch_hd<32>(ctx, x, how);
    case 64:
        return launch_hd<64>(ctx, x, how);
    case 96:
        return launch_hd<96>(ctx, x, how);
    case 128:
        return launch_hd<128>(ctx, x, how);
    default:
        return fail(GX_ERR_UNSUPPORTED, "gx: attention supports head widths 32, 64, 96 and 128");
    }
}

}  // namespace gx
