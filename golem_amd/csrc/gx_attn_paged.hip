// gx_attn_paged.hip - attention of each conversation's newest tokens over its
// pages.
//
// For token i of conversation b, which stands at position p = length - tokens +
// i, query head h and the positions j = 0 .. p:
//   o = sum_j e^(s_j - m) v_j / sum_j e^(s_j - m),   s_j = q . k_j / sqrt(hd)
// in one pass with the running maximum m.  Sums, maxima and outputs are float32.
//
// A row is a token and a query head of a key-value head's group.  The matrix
// cores take 32 keys against 16 rows a step.  S^T = K Q^T puts a row's scores
// down one lane's registers: with key 8 (i / 4) + 4 a + i % 4 as row i of the
// a-th of a step's two products, lane group g (of four) holds keys 8g .. 8g + 7
// in order, the second operand of O^T = V^T P^T as it stands.  The first, eight
// positions of one element a lane, is made from value rows as the pages hold
// them, hd / 16 elements of eight positions a lane, by exchanging 16-bit (8-bit)
// pieces between registers: no lane needs another's, and an append writes whole
// rows.  Lane li's elements are hd / 16 li + d for the d-th product.
//
// A probability enters the second product as two fp16 values, its leading 11
// bits and the next 11, cut off: together within 2^-21 of it, or within 2^-32 of
// the row's largest where that is more (the second then below fp16's normal
// numbers).  The leading bits alone would leave a head's outputs 3.5e-4 short,
// which the float output could not hide.
//
// 8-bit pages enter as fp16 integers, which are exact; a key's scale multiplies
// its score, a value's its probability, each in float32.  What is cut in two is then
// that product: within 2^-21 of it, or 2^-29 of the row's largest.
#include <algorithm>
#include <type_traits>

#include "gx_device.hpp"
#include "gx_internal.hpp"

namespace gx {
namespace {

typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef short v4s __attribute__((ext_vector_type(4)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v16f __attribute__((ext_vector_type(16)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));

constexpr int kRows = 16;       // rows a tile, and
constexpr int kKeys = 32;       // keys a step, of the kernel for few rows
constexpr int kWide = 32;       // rows a wavefront,
constexpr int kWideWaves = 4;   // wavefronts a tile, and
constexpr int kStage = 64;      // keys a step, of the kernel for many
constexpr int kMaxSplits = 64;  // shares of the keys, over workgroups
constexpr int kWaves = 8;       // wavefronts a workgroup, steps in turn
// Probabilities are held times 2^8, their low parts clear of fp16's subnormals,
// and the reference the exponent is taken from follows the maximum only when
// that has risen by 2^7: still below fp16's largest.
constexpr float kShift = 8.0f, kRise = 7.0f;

struct Args {
    PagedAttention y;
    Pages at;
    float c;     // 1 / sqrt(hd) in the exponent's base 2
    int S;       // shares (the kernel for many rows)
    int G, least;  // workgroups a key-value head that the steps are spread over, and a workgroup's least steps
    int32_t *plan;  // [1 + n]: a workgroup's steps, and where each conversation's begin
    float *po;   // unnormalised outputs: [S][M][heads][hd], or [kv_heads][2 G][kRows][hd]
    float *pml;  // their maxima (base 2) and sums, two floats a row
};

// Conversation b's rows of qh and its positions, within the call's bounds.
struct Conversation {
    int f0, T, L;
    __device__ Conversation(const PagedAttention &y, int from, int to, int length) {
        f0 = __builtin_amdgcn_readfirstlane(min(max(from, 0), y.M));
        T = __builtin_amdgcn_readfirstlane(min(min(max(to, f0), y.M) - f0, y.max_tokens));
        L = __builtin_amdgcn_readfirstlane(min(max(length, 0), y.max_length));
    }
    // Positions that row r sees, and that any of the rows of r's tile does.
    __device__ int sees(int r, int group) const { return L - T + r / group + 1; }
    __device__ int tile_sees(int r, int tile, int group) const {
        return max(0, sees(min(r / tile * tile + tile, T * group) - 1, group));
    }
};
// A tile's steps by its conversation's length (where they are spread; the causal
// ones are at most that many), and a share of a tile's steps.
__device__ __forceinline__ int spread_steps(int length) { return max(1, (length + kKeys - 1) / kKeys); }
__device__ __forceinline__ int share_of(int steps, int S) { return max(1, (steps + S - 1) / S); }

// Loads asked for before this are asked for here, not where they are used.
__device__ __forceinline__ void loads_first() { asm volatile("" ::: "memory"); }

// lo/hi(a) * -1 + c for an fp16 pair a, as one v_fma_mix.
__device__ __forceinline__ float less_lo(uint32_t a, float c) {
    float r;
    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(r) : "v"(a), "v"(c));
    return r;
}
__device__ __forceinline__ float less_hi(uint32_t a, float c) {
    float r;
    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(r) : "v"(a), "v"(c));
    return r;
}
__device__ __forceinline__ uint32_t pack_rtz(float a, float b) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(a, b));
}
// What two fp16 values (h) leave of the floats a and b they were cut from.
__device__ __forceinline__ uint32_t rest_of(uint32_t h, float a, float b) { return pack_rtz(less_lo(h, a), less_hi(h, b)); }

// The maximum and the sum over the four lanes that share a row.
__device__ __forceinline__ float groups_max(float v) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float groups_sum(float v) {
    v += __shfl_xor(v, 16);
    return v + __shfl_xor(v, 32);
}
// The larger of a lane's value and the other half's.
__device__ __forceinline__ float halves_max(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
// What is added to a score in base 2, the reference m being in the scores' own units.
__device__ __forceinline__ float base_of(float m, float c) { return kShift - (m == -INFINITY ? 0.0f : m * c); }

// 8-bit values' scales go with the probabilities, z = p * scale, and those enter the
// products as z / cap: cap is a power of two of a row's own, 2^-8 of its largest z,
// and follows that as the maximum's reference does, when it rises past 2^15 cap or
// the reference moves (so that a large scale with little weight, or one whose weight
// has become little, takes no bits from the others).
//
// May a step's z pass 2^15 cap?  (r: its largest scale / cap, p: its largest
// probability.  Nor may r itself come near float's largest, as p may be zero.)
__device__ __forceinline__ bool cap_short(float r, float p) { return p * r > 0x1p15f || r > 0x1p100f; }
// 2^-16 z, which float holds whatever the scale.
__device__ __forceinline__ float scaled_down(float p, float scale) { return p * (fabsf(scale) * 0x1p-16f); }
// A power of two above (at most 2^127), and one not above.
__device__ __forceinline__ float power_above(float v) {
    return __uint_as_float(min((__float_as_uint(v) & 0x7F800000u) + 0x00800000u, 0x7F000000u));
}
__device__ __forceinline__ float power_within(float v) { return __uint_as_float(__float_as_uint(v) & 0x7F800000u); }
// A row's cap and its inverse, its sums being multiplied by corr for a reference that
// moved; z: 2^-16 of the step's largest, or up to four times as much,
// top: its largest scale.  Returns what the outputs, held divided by cap, are
// multiplied by.
__device__ __forceinline__ float cap_to(float &cap, float &by, float corr, bool moved, float z, float top) {
    if (!moved && !(z > 0.5f * cap) && !(top * by > 0x1p100f))
        return corr;
    const float had = cap * corr;
    cap = fminf(fmaxf(fmaxf(power_above(z) * 0x1p8f, power_within(had)), power_above(top) * 0x1p-100f), 0x1p126f);
    by = __uint_as_float(0x7F000000u - __float_as_uint(cap));  // 1 / cap
    return had * by;
}

// Two of eight bytes (w's four, then v's), integers, as fp16: set in the low bits of
// 1024 with their sign bit turned, less 1152.
__device__ __forceinline__ uint32_t half_of(uint32_t turned) {
    const v2h r = __builtin_bit_cast(v2h, turned) - (v2h){1152.0f, 1152.0f};
    return __builtin_bit_cast(uint32_t, r);
}
template <int I, int J>
__device__ __forceinline__ uint32_t bytes_to_half(uint32_t turned) {
    return half_of(__builtin_amdgcn_perm(0x64646464u, turned, 0x04000400u | I | J << 16));
}

// A step's keys as they come from the pages, 1 KiB an instruction in whole lines,
// and through a wavefront's own LDS to the lanes that want them: a product's
// sixteen keys read where they lie are 64 bytes each of sixteen lines (one token
// after 500 positions 9.9 us so, 7.0 by LDS).  Pieces of 16 bytes are exchanged by
// the key, or rows padded where they are no power of two, so that sixteen keys'
// pieces go round the banks.
template <int HD, int KIND>
struct Keys {
    static constexpr int RB = HD * (KIND == GX_PAGES_F16 ? 2 : 1), CH = RB / 16, N = CH / 2, KS = HD / 32;
    static constexpr bool even = (CH & (CH - 1)) == 0;
    static constexpr int SC = even ? CH : CH + 1, bytes = kKeys * SC * 16;
    v4u x[N];
    static __device__ __forceinline__ int at(int key, int c) {
        const int z = CH == 16  ? (key & 3) | (key >> 3) << 2
                      : CH == 8 ? (key >> 1 & 1) | (key >> 3) << 1
                      : CH == 4 ? key >> 3
                      : CH == 2 ? key >> 3 & 1
                                : 0;
        return (key * SC + (c ^ z)) * 16;
    }
    // the step's first and second sixteen keys
    __device__ void load(const char *a, const char *b, int lane) {
#pragma unroll
        for (int i = 0; i < N; i++) {
            const uint32_t p = (64 * i + lane) * 16;
            x[i] = *(const v4u *)(64 * (i + 1) <= 16 * CH ? a + p
                                  : 64 * i >= 16 * CH     ? b + (p - 16 * RB)
                                  : p < 16 * RB           ? a + p
                                                          : b + (p - 16 * RB));
        }
    }
    __device__ void store(uint8_t *lds, int lane) const {
#pragma unroll
        for (int i = 0; i < N; i++)
            *(v4u *)(lds + at((64 * i + lane) / CH, (64 * i + lane) % CH)) = x[i];
    }
    // the element that slab s of lane group g begins at (8 bits: two slabs are one
    // read of 16 bytes, an odd last one 8 bytes)
    static __device__ int slab(int s, int g) {
        return KIND == GX_PAGES_F16 || (s | 1) >= KS ? 32 * s + 8 * g : 64 * (s / 2) + 16 * g + 8 * (s & 1);
    }
    // slab s of key `key` as it lies, and as the product's operand
    typedef typename std::conditional<KIND == GX_PAGES_F16, v8h, uint2>::type Slab;
    static __device__ __forceinline__ Slab read(const uint8_t *lds, int key, int s, int g) {
        const int e = slab(s, g) * RB / HD;
        return *(const Slab *)(lds + at(key, e / 16) + e % 16);
    }
    static __device__ __forceinline__ v8h operand(const Slab &w) {
        if constexpr (KIND == GX_PAGES_F16) {
            return w;
        } else {
            const uint32_t u[2] = {w.x ^ 0x80808080u, w.y ^ 0x80808080u};
            const v4u r = {bytes_to_half<0, 1>(u[0]), bytes_to_half<2, 3>(u[0]), bytes_to_half<0, 1>(u[1]),
                           bytes_to_half<2, 3>(u[1])};
            return __builtin_bit_cast(v8h, r);
        }
    }
};

// A step's values, D = HD / 16 products.
template <int HD, int KIND>
struct Values;
template <int HD>
struct Values<HD, GX_PAGES_F16> {
    static constexpr int D = HD / 16;
    struct __attribute__((packed, aligned(4))) Row {
        uint32_t w[D / 2];
    } x[8];
    __device__ void load(const char *p, int li, bool once) {
        if (D == 8 && once) {  // (read by no other tile: past the caches)
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const v4u z = __builtin_nontemporal_load((const v4u *)(p + j * HD * 2 + li * 16));
#pragma unroll
                for (int w = 0; w < D / 2; w++)
                    x[j].w[w] = z[w & 3];
            }
        } else {
#pragma unroll
            for (int j = 0; j < 8; j++)
                x[j] = *(const Row *)(p + j * HD * 2 + li * D * 2);
        }
    }
    // rows from `count` on become zero
    __device__ void clear(int count) {
#pragma unroll
        for (int j = 0; j < 8; j++)
#pragma unroll
            for (int w = 0; w < D / 2; w++)
                x[j].w[w] = j < count ? x[j].w[w] : 0u;
    }
    __device__ v8h operand(int d) const {
        const uint32_t sel = d & 1 ? 0x07060302u : 0x05040100u;
        v4u r;
#pragma unroll
        for (int i = 0; i < 4; i++)
            r[i] = __builtin_amdgcn_perm(x[2 * i + 1].w[d / 2], x[2 * i].w[d / 2], sel);
        return __builtin_bit_cast(v8h, r);
    }
};
template <int HD>
struct Values<HD, GX_PAGES_I8> {
    static constexpr int D = HD / 16;
    struct __attribute__((packed, aligned(2))) Row {
        uint16_t w[D / 2];
    };
    uint32_t x[8][(D + 3) / 4];
    __device__ void load(const char *p, int li, bool) {
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const Row r = *(const Row *)(p + j * HD + li * D);
            x[j][(D - 1) / 4] = 0;
            __builtin_memcpy(x[j], &r, D);
        }
    }
    __device__ void clear(int count) {}  // (integers: a probability of zero clears them)
    // (two positions' bytes side by side first, two elements of them at a time)
    __device__ v8h operand(int d) const {
        v4u r;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t pair = __builtin_amdgcn_perm(x[2 * i + 1][d / 4], x[2 * i][d / 4], d & 2 ? 0x07030602u : 0x05010400u) ^
                                  0x80808080u;
            r[i] = d & 1 ? bytes_to_half<2, 3>(pair) : bytes_to_half<0, 1>(pair);
        }
        return __builtin_bit_cast(v8h, r);
    }
};

template <int KIND>
__device__ __forceinline__ float page_value(const void *pool, int64_t i) {
    return KIND == GX_PAGES_F16 ? half_bits_to_float(((const uint16_t *)pool)[i]) : (float)((const int8_t *)pool)[i];
}

// The elements of a row that a hidden value has spoilt (an infinite or NaN value
// of a later token makes 0 * inf in its step), summed again over what the row
// sees alone: 64 keys at a time, a key a lane, the spoilt elements in turn.  o:
// four of the row's outputs, from element e on; spoilt: which of them; top: the
// row's reference in base 2, from which its other sums were taken.
template <int HD>
__device__ __forceinline__ v4f attn_paged_again(const Args &x, int b, int tok, int head, int sees, float top, v4f o, int e,
                                                uint32_t spoilt) {
    const int lane = threadIdx.x & 63, kvh = head / (x.y.heads / x.y.kv_heads);
    const uint16_t *q = x.y.qh + ((size_t)tok * x.y.heads + head) * HD;
#pragma unroll
    for (int i = 0; i < 4; i++)
        o[i] = spoilt >> i & 1 ? 0.0f : o[i];
    for (int j0 = 0; j0 < sees; j0 += 64) {
        const int j = min(j0 + lane, sees - 1), page = x.at.table[(size_t)b * x.at.width + (j >> x.at.shift)];
        const bool there = page >= 0 && page < x.at.count;
        const int64_t at = ((((int64_t)(there ? page : 0) * x.y.kv_heads + kvh) << x.at.shift) +
                            (j & ((1 << x.at.shift) - 1))) * HD;
        float s = 0.0f;
        for (int k = 0; k < HD; k++)
            s = fmaf(half_bits_to_float(q[k]), page_value<GX_PAGES_F16>(x.at.k, at + k), s);
        const float p = there ? exp2f(s * x.c - top + kShift) : __uint_as_float(0x7FC00000u);
#pragma unroll
        for (int i = 0; i < 4; i++)
            for (unsigned long long who = __ballot(spoilt >> i & 1); who; who &= who - 1) {
                const int l = __builtin_ctzll(who);
                const float v = page_value<GX_PAGES_F16>(x.at.v, at + __shfl(e, l) + i);
                const float sum = wave_pairwise_sum(j0 + lane < sees ? p * v : 0.0f);
                if (lane == l)
                    o[i] += sum;
            }
    }
    return o;
}

// Four elements' results at `at`, and the Q8_0 of 32 elements by the eight lanes
// that hold them.
__device__ __forceinline__ void attn_paged_store(const PagedAttention &x, v4f o, size_t at) {
    const float y[4] = {o[0], o[1], o[2], o[3]};
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

// A tile of a conversation's rows: the wavefronts of a workgroup take steps of 32
// keys in turn, each with its own maximum and sum, keys and values straight into
// registers: the next step's keys asked for before this one's products, its values
// as soon as this one's are used, its pages' numbers a step before both.  The
// wavefronts' results are added in LDS.
//
// One tile a workgroup, which writes its results: grid (kv_heads, tiles,
// conversations).  Or SPREAD: the steps of all tiles of a key-value head, one
// after another, in even parts over G workgroups, however long each conversation
// is: grid (kv_heads, G).  A part may end one tile, take others whole and begin a
// last one; what it has of the first and the last goes to the join.
template <int HD, int KIND, bool SPREAD>
__global__ __launch_bounds__(64 * kWaves) void attn_paged_tile_kernel(const Args x) {
    using K = Keys<HD, KIND>;
    constexpr int KS = HD / 32, D = HD / 16, W = kWaves, kPad = HD + 4;
    // a wavefront's keys, later its outputs
    constexpr int kOwn = K::bytes / 4 > kRows * kPad ? K::bytes / 4 : kRows * kPad;
    __shared__ __align__(16) float lds[W * kOwn];
    __shared__ float mls[2 * W * kRows];
    __shared__ int found[W + 2];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int li = lane & 15, g = lane >> 4, kvh = SPREAD ? blockIdx.y : blockIdx.x, group = x.y.heads / x.y.kv_heads;
    const int own = blockIdx.x;  // SPREAD: which of the G
    // the conversation, the step among its tiles', the step among the head's, steps to go
    int b = blockIdx.z, at_step = 0, here = 0, left = 1;
    if constexpr (SPREAD) {
        auto cost = [&](int i) __attribute__((always_inline)) {
            const int f0 = min(max(x.y.first[i], 0), x.y.M), f1 = min(max(x.y.first[i + 1], f0), x.y.M);
            const int tiles = (min(f1 - f0, x.y.max_tokens) * group + kRows - 1) / kRows;
            return tiles * spread_steps(min(max(x.y.lengths[i], 0), x.y.max_length));
        };
        auto running = [&](int c) __attribute__((always_inline)) {
            for (int w = 1; w < 64; w <<= 1) {
                const int z = __shfl_up(c, w);
                c += lane >= w ? z : 0;
            }
            return c;
        };
        // up to 64 conversations every wavefront adds up by itself, a lane each
        const bool few = x.y.n <= 64;
        int mine = 0, up = 0, total = 0;
        if (few) {
            mine = lane < x.y.n ? cost(lane) : 0;
            up = running(mine);
            total = __builtin_amdgcn_readlane(up, 63);
        } else {
            int sum = 0;
            for (int i = tid; i < x.y.n; i += 64 * W)
                sum += cost(i);
            for (int w = 32; w > 0; w >>= 1)
                sum += __shfl_xor(sum, w);
            if (lane == 0)
                found[wave] = sum;
            __syncthreads();
            for (int w = 0; w < W; w++)
                total += found[w];
        }
        const int each = max(x.least, (total + x.G - 1) / x.G);
        here = __builtin_amdgcn_readfirstlane(min((int64_t)own * each, (int64_t)INT32_MAX));
        if (own == 0 && kvh == 0 && tid == 0)
            x.plan[0] = each;
        left = __builtin_amdgcn_readfirstlane(min(each, total - here));
        if (left <= 0)
            return;
        // the conversation whose step that is: by the running sums, a chunk after another
        if (few) {
            b = __builtin_ctzll(__ballot(up > here && up - mine <= here));
            at_step = here - __builtin_amdgcn_readlane(up - mine, b);
        } else {
            int before = 0;
            for (int i0 = 0; i0 < x.y.n; i0 += 64 * W) {
                const int c = i0 + tid < x.y.n ? cost(i0 + tid) : 0;
                int up = running(c);
                __syncthreads();
                if (lane == 63)
                    found[wave] = up;
                __syncthreads();
                int all = 0;
                for (int w = 0; w < W; w++) {
                    up += w < wave ? found[w] : 0;
                    all += found[w];
                }
                up += before;
                if (up > here && up - c <= here) {
                    found[W] = i0 + tid;
                    found[W + 1] = here - (up - c);
                }
                before += all;
            }
            __syncthreads();
            b = __builtin_amdgcn_readfirstlane(found[W]);
            at_step = __builtin_amdgcn_readfirstlane(found[W + 1]);
        }
    }
    while (left > 0 && b < x.y.n) {
        const Conversation t(x.y, x.y.first[b], x.y.first[b + 1], x.y.lengths[b]);
        const int R = t.T * group;
        int tile = blockIdx.y, t0 = 0, t1 = INT32_MAX;
        if constexpr (SPREAD) {
            const int steps = spread_steps(t.L), all = (R + kRows - 1) / kRows * steps;
            if (at_step >= all) {
                b++;
                at_step = 0;
                continue;
            }
            if (at_step == 0 && kvh == 0 && tid == 0)
                x.plan[1 + b] = here;
            tile = at_step / steps;
            t0 = at_step - tile * steps;
            const int take = min(left, steps - t0);
            t1 = t0 + take;
            here += take;
            left -= take;
            at_step += take;
        } else {
            left = 0;
            if (tile * kRows >= R)
                return;
        }
        const int r0 = tile * kRows, most = t.tile_sees(r0, kRows, group), total = (most + kKeys - 1) / kKeys;
        const bool begins = t0 == 0, whole = begins && t1 >= total;
        t1 = min(t1, total);
        if (t0 >= t1 && !whole)
            continue;
        const int32_t *row = x.at.table + (size_t)b * x.at.width;
        const int shift = x.at.shift, in_page = (1 << shift) - 1, last = max(most - 1, 0) >> shift;

        // the pages of a step's two runs of sixteen positions, in lanes 0 and 1 (and the
        // others like them), and the pool's row that run y begins at
        auto pages_of = [&](int j) __attribute__((always_inline)) {
            return row[min((kKeys * j + 16 * (lane & 1)) >> shift, last)];
        };
        auto place = [&](int ids, int j, int y) __attribute__((always_inline)) {
            const int id = __builtin_amdgcn_readlane(ids, y);
            return (((int64_t)((uint32_t)id < (uint32_t)x.at.count ? id : 0) * x.y.kv_heads + kvh) << shift) +
                   ((kKeys * j + 16 * y) & in_page);
        };
        const int r = min(r0 + li, R - 1), node = r / group, sees = t.sees(r, group);
        v4f o[D] = {};
        float m = -INFINITY, l = 0.0f;  // m: in the scores' own units
        float cap = 0.0f, by = 0.0f;    // 8-bit values' outputs are held divided by cap (by: 1 / cap)
        int j = t0 + wave;
        if (j < t1) {
            K k;
            Values<HD, KIND> v;
            float sv[8], sk[8];
            uint8_t *const mine = (uint8_t *)(lds + wave * kOwn);
            // (a step's pages' numbers are asked for before the loads of the step before
            // it: loads come back in order)
            int ids = pages_of(j), next_ids = pages_of(j + W);
            auto load_keys = [&](int ids, int at) __attribute__((always_inline)) {
                const char *a = (const char *)x.at.k + place(ids, at, 0) * K::RB, *b = (const char *)x.at.k + place(ids, at, 1) * K::RB;
                k.load(a, b, lane);
            };
            auto load_values = [&](int ids, int at) __attribute__((always_inline)) {
                const int64_t a = place(ids, at, 0), b = place(ids, at, 1), from = (g < 2 ? a : b) + 8 * (g & 1);
                v.load((const char *)x.at.v + from * K::RB, li, R <= kRows);
                if constexpr (KIND == GX_PAGES_I8) {
                    *(v4f *)sk = *(const v4f *)(x.at.ks + from), *(v4f *)(sk + 4) = *(const v4f *)(x.at.ks + from + 4);
                    *(v4f *)sv = *(const v4f *)(x.at.vs + from), *(v4f *)(sv + 4) = *(const v4f *)(x.at.vs + from + 4);
                }
            };
            load_keys(ids, j);
            const uint16_t *qr = x.y.qh + ((size_t)(t.f0 + node) * x.y.heads + kvh * group + (r - node * group)) * HD;
            v8h q[KS];
#pragma unroll
            for (int s = 0; s < KS; s++)
                q[s] = *(const v8h *)(qr + K::slab(s, g));
            load_values(ids, j);
            loads_first();
            const int key = 8 * (li >> 2) + (li & 3);  // a lane's key of the first product, four more: of the second
            for (; j < t1; j += W) {
                const bool more = j + W < t1;
                const int last_ids = pages_of(j + 2 * W);
                k.store(mine, lane);
                // (a wavefront's LDS operations are done in order)
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
                __builtin_amdgcn_wave_barrier();
                loads_first();
                // (past the last step this one's again: the loads in flight are then the
                // same on every path, and none is waited for with another)
                load_keys(more ? next_ids : ids, more ? j + W : j);
                typename K::Slab w[KS][2];
#pragma unroll
                for (int i = 0; i < KS; i++)
#pragma unroll
                    for (int a = 0; a < 2; a++)
                        w[i][a] = K::read(mine, key + 4 * a, i, g);
                __builtin_amdgcn_sched_barrier(0);
                v4f s[2] = {};
#pragma unroll
                for (int i = 0; i < KS; i++)
#pragma unroll
                    for (int a = 0; a < 2; a++)
                        s[a] = __builtin_amdgcn_mfma_f32_16x16x32_f16(K::operand(w[i][a]), q[i], s[a], 0, 0, 0);
                // (the reads before the next step's stores)
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
                __builtin_amdgcn_wave_barrier();
                if constexpr (KIND == GX_PAGES_I8)
#pragma unroll
                    for (int i = 0; i < 8; i++)
                        s[i >> 2][i & 3] *= sk[i];
                const int p0 = kKeys * j + 8 * g;
                const bool gone_a = (uint32_t)__builtin_amdgcn_readlane(ids, 0) >= (uint32_t)x.at.count;
                const bool gone_b = (uint32_t)__builtin_amdgcn_readlane(ids, 1) >= (uint32_t)x.at.count;
                if (gone_a || gone_b) {  // keys of a page that is not there
                    asm volatile("" ::: "memory");  // (a branch)
                    if (g < 2 ? gone_a : gone_b)
                        s[0] = s[1] = v4f{} + __uint_as_float(0x7FC00000u);
                }
                const bool edge = kKeys * (j + 1) > t.L - t.T + 1;  // some row may not see all of the step
                if (edge) {
#pragma unroll
                    for (int i = 0; i < 8; i++)
                        s[i >> 2][i & 3] = p0 + i < sees ? s[i >> 2][i & 3] : -INFINITY;
                    if constexpr (KIND == GX_PAGES_I8)
#pragma unroll
                        for (int i = 0; i < 8; i++)
                            sv[i] = p0 + i < sees ? sv[i] : 0.0f;
                    v.clear(t.L - p0);
                }
                float mx = s[0][0];
#pragma unroll
                for (int i = 1; i < 8; i++)
                    mx = fmaxf(mx, s[i >> 2][i & 3]);
                // (the reference of a row that sees nothing yet, or whose maximum has risen
                // past what it allows, becomes the maximum; the others' stay: a row's bits
                // hang on its own keys alone)
                auto rises = [&](float to) __attribute__((always_inline)) {
                    return to * x.c > m * x.c + kRise || (m == -INFINITY && to > m);
                };
                float top = 0.0f;
                bool grows = false;
                if constexpr (KIND == GX_PAGES_I8) {
#pragma unroll
                    for (int i = 0; i < 8; i++)
                        top = fmaxf(top, fabsf(sv[i]));  // (NaN falls out)
                    grows = cap_short(top * by, __builtin_amdgcn_exp2f(fmaf(mx, x.c, base_of(m, x.c))));
                }
                if (__ballot(rises(mx) || grows)) {
                    const float most = groups_max(mx), mn = rises(most) ? most : m;
                    float corr = mn == m ? 1.0f : __builtin_amdgcn_exp2f((m - mn) * x.c);
                    l *= corr;
                    if constexpr (KIND == GX_PAGES_I8) {
                        float base = base_of(mn, x.c);
                        asm volatile("" : "+v"(base));  // (the branch's own probabilities)
                        float z = 0.0f;
#pragma unroll
                        for (int i = 0; i < 8; i++)
                            z = fmaxf(z, scaled_down(__builtin_amdgcn_exp2f(fmaf(s[i >> 2][i & 3], x.c, base)), sv[i]));
                        corr = cap_to(cap, by, corr, mn != m, groups_max(z), groups_max(top));
                    }
                    m = mn;
#pragma unroll
                    for (int d = 0; d < D; d++)
                        o[d] *= corr;
                }
                const float base = base_of(m, x.c);
                float part = 0.0f, p[8];
                uint32_t hb[4], lb[4];
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    p[i] = __builtin_amdgcn_exp2f(fmaf(s[i >> 2][i & 3], x.c, base));
                    part += p[i];
                    if constexpr (KIND == GX_PAGES_I8)
                        p[i] *= sv[i] * by;
                }
                l += part;
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    hb[i] = pack_rtz(p[2 * i], p[2 * i + 1]);
                    lb[i] = rest_of(hb[i], p[2 * i], p[2 * i + 1]);
                }
                const v8h ph = __builtin_bit_cast(v8h, (v4u){hb[0], hb[1], hb[2], hb[3]});
                const v8h pl = __builtin_bit_cast(v8h, (v4u){lb[0], lb[1], lb[2], lb[3]});
#pragma unroll
                for (int d = 0; d < D; d++) {
                    const v8h a = v.operand(d);
                    o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, ph, o[d], 0, 0, 0);
                    o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, pl, o[d], 0, 0, 0);
                }
                load_values(more ? next_ids : ids, more ? j + W : j);
                ids = next_ids;
                next_ids = last_ids;
                loads_first();
            }
            l = groups_sum(l);
            if constexpr (KIND == GX_PAGES_I8)
#pragma unroll
                for (int d = 0; d < D; d++)
                    o[d] *= cap;
        }
        // the wavefronts' maxima and sums, then their outputs times their weights
        if (g == 0) {
            mls[wave * kRows + li] = m;
            mls[(W + wave) * kRows + li] = l;
        }
        __syncthreads();
        const int had = min(W, t1 - t0);  // wavefronts that had a step
        if (wave < had) {
            float top = -INFINITY;
#pragma unroll
            for (int w = 0; w < W; w++)
                top = fmaxf(top, mls[w * kRows + li]);
            const float weight = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((m - top) * x.c);
            float *to = lds + wave * kOwn + li * kPad;
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int d = 0; d < D; d++)
                    to[D * (4 * g + i) + d] = weight == 0.0f ? 0.0f : o[d][i] * weight;
        }
        __syncthreads();
        const int rows = min(kRows, R - r0);
        for (int it = tid; it < (rows * (HD / 4) + 63) / 64 * 64; it += 64 * W) {
            const int rr = min(it / (HD / 4), rows - 1), e = 4 * (it % (HD / 4));
            const bool there = it / (HD / 4) < rows;
            float top = -INFINITY, sum = 0.0f;
#pragma unroll
            for (int w = 0; w < W; w++)
                top = fmaxf(top, mls[w * kRows + rr]);
            v4f y = {0.0f, 0.0f, 0.0f, 0.0f};
            for (int w = 0; w < had; w++) {
                // (a wavefront that saw nothing, or nothing but NaN, has no maximum)
                const float mw = mls[w * kRows + rr], lw = mls[(W + w) * kRows + rr];
                sum += mw == -INFINITY ? lw : lw * __builtin_amdgcn_exp2f((mw - top) * x.c);
                y += *(const v4f *)(lds + w * kOwn + rr * kPad + e);
            }
            const int rt = (r0 + rr) / group, tok = t.f0 + rt, head = kvh * group + (r0 + rr - rt * group);
            if (SPREAD && !whole) {
                const size_t part = (((size_t)kvh * x.G + own) * 2 + begins) * kRows + rr;
                if (there) {
                    *(v4f *)(x.po + part * HD + e) = y;
                    if (e == 0) {
                        x.pml[2 * part] = top == -INFINITY ? top : top * x.c;
                        x.pml[2 * part + 1] = sum;
                    }
                }
                continue;
            }
            const int seen = t.sees(r0 + rr, group);
            if (KIND == GX_PAGES_F16 && t.T > 1) {
                uint32_t spoilt = 0;
#pragma unroll
                for (int i = 0; i < 4; i++)
                    if (there && seen > 0 && sum - sum == 0.0f && y[i] - y[i] != 0.0f)
                        spoilt |= 1u << i;
                for (unsigned long long who = __ballot(spoilt != 0); who;) {  // a row after another
                    const int one = __builtin_ctzll(who), its = __builtin_amdgcn_readlane(rr, one);
                    const bool mine = rr == its;
                    y = attn_paged_again<HD>(x, b, __builtin_amdgcn_readlane(tok, one), __builtin_amdgcn_readlane(head, one),
                                             __builtin_amdgcn_readlane(seen, one),
                                             __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(top), one)) * x.c, y, e,
                                             mine ? spoilt : 0u);
                    who &= ~__ballot(mine);
                }
            }
            if (there)
                attn_paged_store(x.y, seen > 0 ? y / sum : v4f{0.0f, 0.0f, 0.0f, 0.0f}, ((size_t)tok * x.y.heads + head) * HD + e);
        }
        if (SPREAD)
            __syncthreads();
    }
}

// Many rows: 32 rows a wavefront, four wavefronts a workgroup, 64 keys a step
// through a ring of two in LDS.  The matrix cores take 32 keys against 32 rows, a
// step's halves u: S^T = K Q^T with key piece i read from position swap23(i)
// (bits 2 and 3 exchanged), so that registers 8t .. 8t + 7 of lane half h are the
// keys 32u + 16t + 8h .. + 7, the second operand of O^T = V^T P^T; the first comes
// out of value rows by transposing reads of 4 x 16 elements.
//
// Keys and values lie in LDS a position a row, their 16-byte pieces exchanged by
// the position's low bits: sixteen keys' pieces, and four positions' 64 bytes, go
// round the banks.  fp16 pages come in by direct loads, one step ahead of the
// products; 8-bit ones through registers, two steps ahead, made fp16 on the way.
// Tiles that see most come first, and then those that see least: with two
// workgroups a CU the long ones lie beside the short ones (a prompt of 2048 65 us;
// long and short in turn 77).
//
// A prompt of 2048 tokens of 32 heads over 8 of 128 takes 64 to 69 us by card, 34 GFLOP:
// the longest tile's 32 steps after each other, 2 us each on a CU of its own; two
// workgroups a CU take 3.5 us for a step of each, where the matrix instructions
// alone (96 a SIMD, a third of them for the probabilities' second part) take 2.1 at
// the clock that they leave on this card (21.6 ns each beside four vector
// instructions; a library's large product takes 28).  By the counters the matrix
// units are busy 32 % of the cycles, the vector units 35, LDS 12, and the CUs'
// average is 72 % of the longest.  Tried and dropped: wave priorities around the
// products or for every second workgroup (1 %), scheduling the exponentials between
// the products (kept, 1 %), the probabilities' rests by v_fma_mixlo (the compiler
// widens them: 2 us more).
template <int HD, int KIND>
__global__ __launch_bounds__(64 * kWideWaves, 2) void attn_paged_wide_kernel(const Args x) {
    constexpr int KS = HD / 16, ET = HD / 32, W = kWideWaves, RB = HD * 2, CH = HD / 8, kTileRows = kWide * W;
    constexpr int kValues = kStage * RB, kSlot = 2 * kValues;
    constexpr bool f16 = KIND == GX_PAGES_F16;
    static_assert(HD == 64 || HD == 128, "rows of whole swizzles");
    // (dynamic, so that the order of its reads can be laid down)
    extern __shared__ __align__(16) uint8_t lds[];
    float *const scales = (float *)(lds + 2 * kSlot);  // 8 bits: a slot's keys', then its values'
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int li = lane & 31, h = lane >> 5;
    const int kvh = blockIdx.x, b = blockIdx.z / x.S, sp = blockIdx.z % x.S;
    const Conversation t(x.y, x.y.first[b], x.y.first[b + 1], x.y.lengths[b]);
    const int group = x.y.heads / x.y.kv_heads, R = t.T * group, tiles = (R + kTileRows - 1) / kTileRows;
    const int turn = (tiles + 1) / 2, tile = (int)blockIdx.y < turn ? tiles - 1 - (int)blockIdx.y : (int)blockIdx.y - turn;
    if ((int)blockIdx.y >= tiles)
        return;
    const int g0 = tile * kTileRows, r0 = g0 + wave * kWide;
    const int most = t.tile_sees(g0, kTileRows, group), total = (most + kStage - 1) / kStage, per = share_of(total, x.S);
    const int t0 = sp * per, t1 = min(total, t0 + per);
    if (t0 >= t1 && x.S > 1)
        return;
    const int32_t *row = x.at.table + (size_t)b * x.at.width;
    const int shift = x.at.shift, in_page = (1 << shift) - 1, last = max(most - 1, 0) >> shift;

    // the pages of a step's four runs of sixteen positions, in lanes 0 .. 3
    auto pages_of = [&](int j) __attribute__((always_inline)) {
        return row[min((kStage * j + 16 * (lane & 3)) >> shift, last)];
    };
    // the pool's row of a step's position p, whose page is run p / 16's
    auto place = [&](int ids, int j, int p) __attribute__((always_inline)) {
        const int id = __builtin_amdgcn_readlane(ids, p >> 4);
        return (((int64_t)((uint32_t)id < (uint32_t)x.at.count ? id : 0) * x.y.kv_heads + kvh) << shift) +
               ((kStage * j + p) & in_page);
    };
    auto swizzle_k = [](int p) __attribute__((always_inline)) { return HD == 128 ? p & 15 : (p >> 1) & 7; };
    auto swizzle_v = [](int p) __attribute__((always_inline)) { return HD == 128 ? 4 * (p & 3) : 4 * ((p >> 1) & 1); };
    // fp16: 1 KiB an instruction, whole rows
    constexpr int RI = 1024 / RB;
    const int dr = lane / CH;
    const uint32_t dk = dr * RB + ((lane % CH) ^ swizzle_k(wave * RI + dr)) * 16;
    const uint32_t dv = dr * RB + ((lane % CH) ^ swizzle_v(dr)) * 16;
    auto load_direct = [&](int j, int ids, uint8_t *to) __attribute__((always_inline)) {
        // (the four runs' places, a run a lane)
        const int id = (uint32_t)ids < (uint32_t)x.at.count ? ids : 0, p = kStage * j + 16 * (lane & 3);
        const uint64_t run = (((uint64_t)((uint32_t)id * (uint64_t)x.y.kv_heads + kvh) << shift) + (p & in_page)) * RB;
#pragma unroll
        for (int i = 0; i < kStage / RI; i += W) {
            const int first = (i + wave) * RI;
            const uint64_t at = ((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(run >> 32), first >> 4) << 32 |
                                 (uint32_t)__builtin_amdgcn_readlane((int)run, first >> 4)) + (first & 15) * RB;
            const char *ks = (const char *)x.at.k + at, *vs = (const char *)x.at.v + at;
            asm("" : "+s"(ks), "+s"(vs));
            __builtin_amdgcn_global_load_lds(ks + dk, (lds_ptr)(to + (i + wave) * 1024), 16, 0, 0);
            __builtin_amdgcn_global_load_lds(vs + dv, (lds_ptr)(to + kValues + (i + wave) * 1024), 16, 0, 0);
        }
    };
    // 8 bits: sixteen elements a thread
    constexpr int PR = 64 * W * 16 / HD, PM = kStage / PR;  // rows a pass, passes
    const int pr = tid / (HD / 16), pc = tid % (HD / 16);
    uint4 rk[f16 ? 1 : PM], rv[f16 ? 1 : PM];
    float rs = 0.0f;
    auto load_raw = [&](int j, int ids) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < PM; i++) {
            const int first = i * PR + wave * (PR / W);  // the wavefront's rows, of one run of sixteen
            const int64_t at = (place(ids, j, first) + (pr - wave * (PR / W))) * HD + 16 * pc;
            rk[i] = *(const uint4 *)((const char *)x.at.k + at);
            rv[i] = *(const uint4 *)((const char *)x.at.v + at);
        }
        if (wave < 2) {
            const int id = __shfl(ids, lane >> 4);
            const int64_t at = (((int64_t)((uint32_t)id < (uint32_t)x.at.count ? id : 0) * x.y.kv_heads + kvh) << shift) +
                               ((kStage * j + lane) & in_page);
            rs = (wave ? x.at.vs : x.at.ks)[at];
        }
    };
    auto store_raw = [&](int slot) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < PM; i++) {
            const int p = i * PR + pr;
            const uint32_t w[2][4] = {{rk[i].x, rk[i].y, rk[i].z, rk[i].w}, {rv[i].x, rv[i].y, rv[i].z, rv[i].w}};
#pragma unroll
            for (int y = 0; y < 2; y++) {
                uint8_t *to = lds + slot * kSlot + y * kValues + p * RB;
                const int z = y ? swizzle_v(p) : swizzle_k(p);
#pragma unroll
                for (int c = 0; c < 2; c++) {
                    v4u o;
#pragma unroll
                    for (int u = 0; u < 2; u++) {
                        const uint32_t q = w[y][2 * c + u] ^ 0x80808080u;
                        o[2 * u] = bytes_to_half<0, 1>(q);
                        o[2 * u + 1] = bytes_to_half<2, 3>(q);
                    }
                    *(v4u *)(to + (((2 * pc + c) ^ z) << 4)) = o;
                }
            }
        }
        if (wave < 2)
            scales[(2 * slot + wave) * kStage + lane] = rs;
    };

    const int r = max(0, min(r0 + li, R - 1)), node = r / group, sees = t.sees(r, group);
    const int wave_least = t.sees(min(r0, R - 1), group);
    int ids = t0 < t1 ? pages_of(t0) : 0, next_ids = ids, raw_ids = ids;
    v8h q[KS];
    const uint16_t *qr = x.y.qh + ((size_t)(t.f0 + node) * x.y.heads + kvh * group + (r - node * group)) * HD + 8 * h;
    if (t0 < t1) {
        if constexpr (f16) {
            load_direct(t0, ids, lds);
            next_ids = pages_of(t0 + 1);
        } else {
            load_raw(t0, ids);
            next_ids = pages_of(t0 + 1);
            store_raw(0);
            load_raw(t0 + 1, next_ids);
            raw_ids = pages_of(t0 + 2);
        }
#pragma unroll
        for (int s = 0; s < KS; s++)
            q[s] = *(const v8h *)(qr + 16 * s);
    }
    // where a lane's operands begin: its key's piece 0 (piece k is k << 5 exchanged),
    // its four positions' elements (those of et are et << 6 exchanged)
    const int key = (li & ~12) | ((li & 4) << 1) | ((li & 8) >> 1), i16 = lane & 15, vr = i16 >> 2;
    const uint32_t ka = key * RB + ((h ^ swizzle_k(key)) << 4);
    const uint32_t va = kValues + (8 * h + vr) * RB + (((2 * ((lane >> 4) & 1) + ((i16 & 3) >> 1)) ^ swizzle_v(vr)) << 4) +
                        8 * (i16 & 1);

    v16f o[ET] = {};
    float m = -INFINITY, l = 0.0f;  // m: in the scores' own units
    float cap = 0.0f, by = 0.0f;    // as in the kernel for few rows
    // a step begins: its keys and values are there, the next ones' loads go out
    // (fp16: after the reads of this step's values, by load_next: a transposing
    // read waits for every direct load asked for before it)
    int here = ids;
    auto begin = [&](int j) __attribute__((always_inline)) {
        const int slot = (j - t0) & 1;
        if constexpr (f16)
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        lds_barrier();
        here = ids;
        ids = next_ids;
        if constexpr (f16) {
            if (kStage * (j + 1) > t.L) {
                // values behind the last position become zero: a NaN there would make 0 * NaN
                for (int i = tid; i < kValues / 16; i += 64 * W)
                    if (kStage * j + i / CH >= t.L)
                        *(v4u *)(lds + slot * kSlot + kValues + 16 * i) = v4u{0u, 0u, 0u, 0u};
                lds_barrier();
            }
        }
    };
    auto load_next = [&](int j) __attribute__((always_inline)) {
        const int other = 1 - ((j - t0) & 1);
        if constexpr (f16) {
            if (j + 1 < t1)
                load_direct(j + 1, ids, lds + other * kSlot);
            next_ids = pages_of(j + 2);
        } else {
            if (j + 1 < t1)
                store_raw(other);
            if (j + 2 < t1)
                load_raw(j + 2, raw_ids);
            next_ids = raw_ids;
            raw_ids = pages_of(j + 3);
        }
    };
    // edge: some row may not see all of the step.  8 bits: the next step's keys and
    // values are made fp16 between this one's products (8-bit prompt of 2048 91 us
    // before the first, 86 here; one loop for steps of either kind 104); with half of
    // the values read as far ahead, for want of registers, 84.
    auto step = [&](int j, bool edge) __attribute__((always_inline)) {
        begin(j);
        const int slot = (j - t0) & 1, p0 = kStage * j;
        const uint32_t kb = ka + slot * kSlot, vb = va + slot * kSlot;
        // keys' reads half of the products ahead of them
        constexpr int kAhead = KS / 2;
        v8h a[KS][2];
        auto keys = [&](int k) __attribute__((always_inline)) {
#pragma unroll
            for (int u = 0; u < 2; u++)
                a[k][u] = *(const v8h *)(lds + (kb ^ (k << 5)) + 32 * RB * u);
            __builtin_amdgcn_sched_barrier(0);
        };
#pragma unroll
        for (int k = 0; k < kAhead; k++)
            keys(k);
        // the values' reads between the products of the scores
        v16f s[2] = {};
        v8h v[4][ET];
        auto value = [&](int i) __attribute__((always_inline)) {
            typedef __attribute__((address_space(3))) v4s *tr;
            union {
                v4s half[2];
                v8h all;
            } z;
#pragma unroll
            for (int y = 0; y < 2; y++)
                z.half[y] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((tr)(lds + (vb ^ ((i % ET) << 6)) + (16 * (i / ET) + 4 * y) * RB));
            v[i / ET][i % ET] = z.all;
        };
#pragma unroll
        for (int k = 0; k < KS; k++) {
#pragma unroll
            for (int u = 0; u < 2; u++)
                s[u] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[k][u], q[k], s[u], 0, 0, 0);
            if (k + kAhead < KS)
                keys(k + kAhead);
            if (f16 || k < KS / 4) {  // (8 bits: no direct loads, and no room for all)
                value(2 * k);
                value(2 * k + 1);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        load_next(j);
        const float *ks = scales + 2 * slot * kStage + 8 * h, *vs = ks + kStage;  // (8 bits)
        if constexpr (!f16)
#pragma unroll
            for (int i = 0; i < 32; i++)
                s[i >> 4][i & 15] *= ks[16 * (i >> 3) + (i & 7)];
        const uint32_t gone = (uint32_t)__ballot(lane < 4 && (uint32_t)here >= (uint32_t)x.at.count);
        if (gone) {  // keys of a page that is not there
            asm volatile("" ::: "memory");  // (a branch)
#pragma unroll
            for (int i = 0; i < 32; i++)
                s[i >> 4][i & 15] = gone >> (i >> 3) & 1 ? __uint_as_float(0x7FC00000u) : s[i >> 4][i & 15];
        }
        const int lim = sees - p0 - 8 * h;
        if (edge)
#pragma unroll
            for (int i = 0; i < 32; i++)
                s[i >> 4][i & 15] = 16 * (i >> 3) + (i & 7) < lim ? s[i >> 4][i & 15] : -INFINITY;
        float mx = s[0][0];
#pragma unroll
        for (int i = 1; i < 32; i++)
            mx = fmaxf(mx, s[i >> 4][i & 15]);
        mx = halves_max(mx);
        // (as in the kernel for few rows)
        const bool rises = mx * x.c > m * x.c + kRise || (m == -INFINITY && mx > m);
        float top = 0.0f, scale = 0.0f;
        bool grows = false;
        if constexpr (!f16) {
            if (edge) {
#pragma unroll
                for (int i = 0; i < 32; i++) {
                    const float z = vs[16 * (i >> 3) + (i & 7)];
                    top = fmaxf(top, 16 * (i >> 3) + (i & 7) < lim ? fabsf(z) : 0.0f);  // (NaN falls out)
                }
                top = halves_max(top);
            } else {
                scale = fabsf(scales[(2 * slot + 1) * kStage + lane]);
                top = fmaxf(0.0f, wave_max(scale));
            }
            grows = cap_short(top * by, __builtin_amdgcn_exp2f(fmaf(mx, x.c, base_of(m, x.c))));
        }
        if (__ballot(rises || grows)) {
            const float mn = rises ? mx : m;
            float corr = mn == m ? 1.0f : __builtin_amdgcn_exp2f((m - mn) * x.c);
            l *= corr;
            if constexpr (!f16) {
                // z by the largest probability and the largest scale where the step's scales
                // are within four of each other, or else key by key (for all: an 8-bit
                // prompt of 2048 96 us, so 84)
                float base = base_of(mn, x.c);
                asm volatile("" : "+v"(base)::"memory");  // (the branch's own: no room to hold the step's over it)
                float z = scaled_down(__builtin_amdgcn_exp2f(fmaf(mx, x.c, base)), top);
                if (edge || !(-wave_max(-scale) * 4.0f >= top)) {
                    asm volatile("" ::: "memory");  // (a branch)
                    z = 0.0f;
#pragma unroll
                    for (int i = 0; i < 32; i++) {
                        const float y = scaled_down(__builtin_amdgcn_exp2f(fmaf(s[i >> 4][i & 15], x.c, base)),
                                                    vs[16 * (i >> 3) + (i & 7)]);
                        z = fmaxf(z, edge && 16 * (i >> 3) + (i & 7) >= lim ? 0.0f : y);
                    }
                    z = halves_max(z);
                }
                asm volatile("" ::: "memory");
                corr = cap_to(cap, by, corr, mn != m, z, top);
            }
            m = mn;
#pragma unroll
            for (int et = 0; et < ET; et++)
                o[et] *= corr;
        }
        const float base = base_of(m, x.c);
        v8h ph[4], pl[4];
        // eight keys' probabilities (times their values' scales), their leading 11 bits and the rest
        auto chances = [&](int w) __attribute__((always_inline)) {
            v4u hb, lb;
            float part = 0.0f;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                float p[2];
#pragma unroll
                for (int y = 0; y < 2; y++) {
                    p[y] = __builtin_amdgcn_exp2f(fmaf(s[w >> 1][8 * (w & 1) + 2 * i + y], x.c, base));
                    part += p[y];
                    if constexpr (!f16) {
                        const float z = vs[16 * w + 2 * i + y] * by;
                        p[y] *= edge && 16 * w + 2 * i + y >= lim ? 0.0f : z;
                    }
                }
                hb[i] = pack_rtz(p[0], p[1]);
                lb[i] = rest_of(hb[i], p[0], p[1]);
            }
            l += part;
            ph[w] = __builtin_bit_cast(v8h, hb);
            pl[w] = __builtin_bit_cast(v8h, lb);
        };
        chances(0);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int w = 0; w < 4; w++) {
#pragma unroll
            for (int et = 0; et < ET; et++) {
                if (!f16 && w < 3)
                    value((w + 1) * ET + et);
                o[et] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v[w][et], ph[w], o[et], 0, 0, 0);
            }
#pragma unroll
            for (int et = 0; et < ET; et++)
                o[et] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v[w][et], pl[w], o[et], 0, 0, 0);
            // the next keys' probabilities between the products of these
            if (w + 1 < 4) {
                chances(w + 1);
#pragma unroll
                for (int et = 0; et < 2 * ET; et++) {
                    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                    __builtin_amdgcn_sched_group_barrier(0x402, 40 / (2 * ET), 0);
                }
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    if (r0 >= R) {  // a wavefront of no rows
        for (int j = t0; j < t1; j++) {
            begin(j);
            load_next(j);
        }
    } else if constexpr (f16) {
        for (int j = t0; j < t1; j++)
            step(j, kStage * (j + 1) > wave_least);
    } else {  // (two loops: an edge costs every value's scale a comparison)
        int j = t0;
        for (; j < t1 && kStage * (j + 1) <= wave_least; j++)
            step(j, false);
        for (; j < t1; j++)
            step(j, true);
    }
    l += __shfl_xor(l, 32);
    if constexpr (!f16)
#pragma unroll
        for (int et = 0; et < ET; et++)
            o[et] *= cap;
    // a wavefront's outputs through its quarter of LDS, so that rows are stored whole
    lds_barrier();
    if (r0 >= R)
        return;
    v4f *const mine = (v4f *)(lds + wave * (2 * kSlot / W));
#pragma unroll
    for (int k = 0; k < 4 * ET; k++)
        mine[li * (HD / 4) + ((2 * k + h) ^ (li & 15))] =
            v4f{o[k / 4][4 * (k % 4)], o[k / 4][4 * (k % 4) + 1], o[k / 4][4 * (k % 4) + 2], o[k / 4][4 * (k % 4) + 3]};
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    const int own = (t.f0 + node) * x.y.heads + kvh * group + (r - node * group);  // a lane's row of the output
    const float whole = x.S > 1 ? 1.0f : sees > 0 ? 1.0f / l : 0.0f;
    if (x.S > 1 && h == 0 && r0 + li < R) {
        const size_t part = (size_t)sp * x.y.M * x.y.heads + own;
        x.pml[2 * part] = m == -INFINITY ? m : m * x.c;
        x.pml[2 * part + 1] = l;
    }
    for (int it = lane; it < kWide * (HD / 4); it += 64) {
        const int rr = it / (HD / 4), c4 = it % (HD / 4), e = 4 * c4;
        v4f y = mine[rr * (HD / 4) + (c4 ^ (rr & 15))];
        const int at = __shfl(own, rr);
        const float by_sum = __shfl(whole, rr);
        const bool there = r0 + rr < R;
        if (x.S > 1) {
            if (there)
                *(v4f *)(x.po + ((size_t)sp * x.y.M * x.y.heads + at) * HD + e) = y;
            continue;
        }
        y = by_sum == 0.0f ? v4f{0.0f, 0.0f, 0.0f, 0.0f} : y * by_sum;
        if constexpr (f16) {
            uint32_t spoilt = 0;
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (there && by_sum - by_sum == 0.0f && y[i] - y[i] != 0.0f)
                    spoilt |= 1u << i;
            for (unsigned long long who = __ballot(spoilt != 0); who;) {  // a row after another
                const int one = __builtin_ctzll(who), its = __builtin_amdgcn_readlane(rr, one);
                const int out = __builtin_amdgcn_readlane(at, one);
                const float top = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(m), its));
                const v4f z = attn_paged_again<HD>(x, b, out / x.y.heads, out % x.y.heads, __builtin_amdgcn_readlane(sees, its),
                                                   top * x.c, y, e, rr == its ? spoilt : 0u);
                if (rr == its)
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        y[i] = spoilt >> i & 1 ? z[i] * by_sum : y[i];
                who &= ~__ballot(rr == its);
            }
        }
        if (there)
            attn_paged_store(x.y, y, (size_t)at * HD + e);
    }
}

// A row a wavefront: its parts' maxima and sums a lane each, its outputs four
// elements a lane, several parts side by side, added in a fixed order; and the
// Q8_0 of 32 elements.  A row that one workgroup had whole is written already.
// grid (heads / 4, M), 256 threads.  Bound by its loads, one after another's answer,
// for one token (5.6 us for 32 parts), by the parts' bytes for more (7.5 for 230
// tokens in five shares, 19 MB).
template <int HD, int KIND, bool SPREAD>
__global__ __launch_bounds__(256) void attn_paged_join_kernel(const Args x) {
    constexpr int L = HD / 4, SP = 64 / L;  // lanes a part, parts side by side
    const int lane = threadIdx.x & 63, tok = blockIdx.y;
    const int head = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (head >= x.y.heads)
        return;
    const int each = SPREAD ? x.plan[0] : 1;
    // the last conversation whose first token is not past this one (and its first step)
    int b = -1, from = 0, to = 0, length = 0, begin = 0;
    for (int i = 0; i < x.y.n; i += 64) {
        const int k = min(i + lane, x.y.n - 1), f0 = x.y.first[k], f1 = x.y.first[k + 1], n = x.y.lengths[k];
        const int begins = SPREAD ? x.plan[1 + k] : 0;  // (of one that has no steps, as it was)
        loads_first();
        const int count = __popcll(__ballot(i + lane < x.y.n && f0 <= tok));
        if (count > 0) {
            b = i + count - 1;
            from = __builtin_amdgcn_readlane(f0, count - 1);
            to = __builtin_amdgcn_readlane(f1, count - 1);
            length = __builtin_amdgcn_readlane(n, count - 1);
            begin = __builtin_amdgcn_readlane(begins, count - 1);
        }
    }
    const Conversation t(x.y, from, to, length);
    if (b < 0 || tok < t.f0 || tok >= t.f0 + t.T)
        return;
    const int group = x.y.heads / x.y.kv_heads, kvh = head / group, r = (tok - t.f0) * group + head % group;
    const int sees = t.sees(r, group);
    const size_t row = (size_t)tok * x.y.heads + head;
    // part s of the row, and how many there are (at most 64)
    size_t first, next;
    int live;
    if constexpr (SPREAD) {
        const int steps = (t.tile_sees(r, kRows, group) + kKeys - 1) / kKeys;
        const int at = begin + r / kRows * spread_steps(t.L);
        const int w0 = at / each, w1 = (at + steps - 1) / each;
        if (steps == 0 || w0 == w1)
            return;
        live = w1 - w0 + 1;
        next = (((size_t)kvh * x.G + w0) * 2) * kRows + r % kRows;  // what a workgroup has of its first tile
        first = next + kRows;                                        // and of its last
    } else {
        const int total = (t.tile_sees(r, kWide * kWideWaves, group) + kStage - 1) / kStage;
        const int per = share_of(total, x.S);
        live = (total + per - 1) / per;
        first = next = row;
    }
    const size_t step = SPREAD ? 2 * kRows : (size_t)x.y.M * x.y.heads;
    auto part = [&](int s) __attribute__((always_inline)) { return (s == 0 ? first : next) + s * step; };
    const int g = lane / L, e = 4 * (lane - g * L);
    typedef float v2f __attribute__((ext_vector_type(2)));
    const v2f ml = live > 0 ? *(const v2f *)(x.pml + 2 * part(min(lane, live - 1))) : v2f{-INFINITY, 0.0f};
    auto shares = [&](int s0, v4f *p) __attribute__((always_inline)) {
#pragma unroll
        for (int k = 0; k < 4; k++)
            p[k] = *(const v4f *)(x.po + part(min(s0 + k * SP + g, live - 1)) * HD + e);
    };
    v4f p[4];
    if (live > 0)
        shares(0, p);
    const float m = lane < live ? ml.x : -INFINITY, top = wave_max(m);
    const float weight = m == -INFINITY ? 0.0f : exp2f(m - top);
    // (a part that saw nothing, or nothing but NaN, has no maximum)
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
    const v4f mine = o;
    for (int k = 1; k < SP; k++) {
        v4f z;
#pragma unroll
        for (int i = 0; i < 4; i++)
            z[i] = __shfl(mine[i], (lane + k * L) & 63);
        if (lane < L)
            o += z;
    }
    if (KIND == GX_PAGES_F16 && t.T > 1) {
        uint32_t spoilt = 0;
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (lane < L && sees > 0 && l - l == 0.0f && o[i] - o[i] != 0.0f)
                spoilt |= 1u << i;
        if (__ballot(spoilt != 0))
            o = attn_paged_again<HD>(x, b, tok, head, sees, top, o, e, spoilt);
    }
    if (lane >= L)
        return;
    attn_paged_store(x.y, sees > 0 ? o / l : v4f{0.0f, 0.0f, 0.0f, 0.0f}, row * HD + e);
}

// How a call's rows and keys are shared out.
struct Plan {
    enum Form { kWhole, kSpread, kMany } form;  // the tile kernel's two, and the kernel for many rows
    int64_t tiles;                              // of rows a conversation
    int S, G, least;
};

// Which kernel, and how it is launched.  The times (us) are of 32 query heads over 8
// of 128, fp16, thirty calls over the same pages; over three sets of pages in turn
// they are up to a fifth longer.  The rule goes by these for every width and kind.
//
// Many rows or tiles, by estimates.  A tile of 16 rows a workgroup takes 6 and 1.1 a
// round of eight steps, one of its workgroups a CU (1.7 where the tiles are more than
// the CUs): 9 tokens of one conversation after 500 positions 7.9, 17 of eight after
// 1000 11.5, 33 after 4000 23, a prompt of 1024 56.  The kernel for many rows takes
// 4, 2 a step and, in shares, 6 for the join and its parts' bytes at 4 TB/s: 15, 19,
// 17 and 33 for the same four.  Near the border it misses: a prompt of 512 takes 24
// by tiles, as chosen, and 21 by the other; at 64 wide one of 1024 takes 39, as
// chosen, and 29 by tiles.  Widths 32 and 96 have the tiles alone.
//
// Whole tiles or their steps spread, by thresholds.  Spreading costs the search for a
// workgroup's part and the join, and pays where whole tiles would leave CUs idle for
// long: one token after 1000 positions 9.2 whole and 10.6 spread, after 1600 11.9 and
// 11.5, after 4000 28.6 and 12.1; four after 1000 10.9 and 12.8, after 2000 17.7 and
// 13.8; 12 after 4000 39.4 and 37.7, 16 41.6 and 45.5 (8-bit 31.6 and 29.3), 64 138
// and 137.  Past 256 steps the longest conversation would be alone at the end.
Plan plan_of(int n, int M, int max_tokens, int heads, int kv_heads, int hd, int max_length) {
    const int64_t rows = (int64_t)max_tokens * (heads / kv_heads), all = (int64_t)kv_heads * std::max(n, 1);
    const int64_t tiles = (rows + kRows - 1) / kRows, steps = (max_length + (int64_t)kKeys - 1) / kKeys;
    if (rows > 2 * kRows && (hd == 64 || hd == 128)) {
        const int64_t wide = (rows + kWide * kWideWaves - 1) / (kWide * kWideWaves), stages = (max_length + (int64_t)kStage - 1) / kStage;
        const int64_t most = std::max<int64_t>(1, std::min<int64_t>({(stages + 3) / 4, kMaxSplits, 512 / (all * wide)}));
        double best = 4.0 + 2.0 * stages;
        int S = 1;
        for (int s = 2; s <= most; s++) {
            const double t = 10.0 + 2.0 * stages / s + (double)s * M * heads * hd * 8 / 4e6;
            if (t < best)
                best = t, S = s;
        }
        const double rounds = (double)((all * tiles + 255) / 256) * ((steps + kWaves - 1) / kWaves);
        if (6.0 + (all * tiles > 256 ? 1.7 : 1.1) * rounds > best)
            return {Plan::kMany, wide, S, 0, 0};
    }
    if (steps <= 48 || (steps <= 256 && all * tiles >= 128) || all * tiles > 4096 || (double)n * tiles * steps > 2e9)
        return {Plan::kWhole, tiles, 1, 0, 0};
    // a workgroup a CU, at most 62 of them a tile (the join's 64 parts)
    return {Plan::kSpread, tiles, 1, std::max(1, 256 / kv_heads), (int)std::max<int64_t>(kWaves, (steps + 61) / 62)};
}

template <int HD, int KIND>
int launch_kind(gx_ctx *ctx, const Args &x, const Plan &how) {
    // (at most 65535 tiles: checked; n * S: at most 16384 with one share, else 512)
    const dim3 grid((unsigned)x.y.kv_heads, (unsigned)how.tiles, (unsigned)(x.y.n * x.S));
    if (how.form == Plan::kWhole)
        attn_paged_tile_kernel<HD, KIND, false><<<grid, 64 * kWaves, 0, ctx->stream>>>(x);
    else if (how.form == Plan::kSpread)
        attn_paged_tile_kernel<HD, KIND, true><<<dim3((unsigned)x.G, (unsigned)x.y.kv_heads), 64 * kWaves, 0,
                                                 ctx->stream>>>(x);
    else if constexpr (HD == 64 || HD == 128) {
        const size_t lds = 4 * kStage * HD * 2 + (KIND == GX_PAGES_I8 ? 4 * kStage * sizeof(float) : 0);
        attn_paged_wide_kernel<HD, KIND><<<grid, 64 * kWideWaves, lds, ctx->stream>>>(x);
    }
    if (int rc = check_launch("attention over pages"))
        return rc;
    const dim3 join((unsigned)((x.y.heads + 3) / 4), (unsigned)x.y.M);
    if (how.form == Plan::kSpread)
        attn_paged_join_kernel<HD, KIND, true><<<join, 256, 0, ctx->stream>>>(x);
    else if (x.S > 1)
        attn_paged_join_kernel<HD, KIND, false><<<join, 256, 0, ctx->stream>>>(x);
    return check_launch("attention over pages, joined");
}

template <int HD>
int launch_hd(gx_ctx *ctx, const Args &x, const Plan &how) {
    return x.at.kind == GX_PAGES_F16 ? launch_kind<HD, GX_PAGES_F16>(ctx, x, how)
                                     : launch_kind<HD, GX_PAGES_I8>(ctx, x, how);
}

// Where a plan's workspace holds what: the conversations' first steps, then the
// parts' outputs, then their maxima and sums.
struct Workspace {
    size_t outputs, rest, bytes;
    Workspace(const Plan &how, int n, int M, int heads, int kv_heads, int hd) {
        const size_t rows = how.form == Plan::kSpread ? (size_t)kv_heads * how.G * 2 * kRows
                            : how.S > 1               ? (size_t)how.S * M * heads
                                                      : 0;
        outputs = how.form == Plan::kSpread ? ((size_t)(1 + n) * 4 + 255) & ~(size_t)255 : 0;
        rest = outputs + rows * hd * 4;
        bytes = (rest + rows * 8 + 255) & ~(size_t)255;
    }
};

}  // namespace

size_t attn_paged_workspace(int n, int M, int max_tokens, int heads, int kv_heads, int hd, int max_length) {
    return Workspace(plan_of(n, M, max_tokens, heads, kv_heads, hd, max_length), n, M, heads, kv_heads, hd).bytes;
}

int launch_attn_paged(gx_ctx *ctx, const PagedAttention &y, const Pages &at, uint8_t *workspace) {
    const Plan how = plan_of(y.n, y.M, y.max_tokens, y.heads, y.kv_heads, y.hd, y.max_length);
    const Workspace ws(how, y.n, y.M, y.heads, y.kv_heads, y.hd);
    const Args x{y, at, (float)(1.4426950408889634 / sqrt((double)y.hd)), how.S, how.G, how.least, (int32_t *)workspace,
                 (float *)(workspace + ws.outputs), (float *)(workspace + ws.rest)};
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
        return fail(GX_ERR_UNSUPPORTED, "gx: pages hold head widths 32, 64, 96 and 128");
    }
}

}  // namespace gx
