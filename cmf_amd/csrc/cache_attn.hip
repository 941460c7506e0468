// Attention of b rows (a tree of drafted tokens, or a chain) over a cache,
// whole or through a sliding window with a few first positions that stay
// visible (cmf_attention_dev).
//
// The query rows of one kv head are its queries qi = row * hpk + head (hpk =
// query heads per kv head).  What a block of queries can see is two runs of
// positions, [0, sinks) and [lo, hi); keys are numbered through both, and only
// those are read.
#include <math.h>

#include <algorithm>
#include <mutex>
#include <set>
#include <string>

#include "cache_ops.h"
#include "runtime.h"
#include "wave.h"

namespace cmf {

namespace {

typedef float float2v __attribute__((ext_vector_type(2)));
typedef float float4v __attribute__((ext_vector_type(4)));
typedef float float16v __attribute__((ext_vector_type(16)));
typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef _Float16 half4 __attribute__((ext_vector_type(4)));
typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf2v __attribute__((ext_vector_type(2)));
typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
typedef short short4v __attribute__((ext_vector_type(4)));
typedef uint32_t uint2v __attribute__((ext_vector_type(2)));
typedef uint32_t uint4v __attribute__((ext_vector_type(4)));
typedef unsigned short ushort2v __attribute__((ext_vector_type(2)));

constexpr int HD = CACHE_HD;
constexpr float LOG2E = 1.4426950408889634f;
constexpr long long MAX_ROW_STRIDE = 1 << 22;  // a tile's offsets stay in 32 bits

// the largest of each 16 lanes
__device__ __forceinline__ uint32_t lanes16_max_u32(uint32_t v) {
    auto step = [&](auto ctrl) {
        v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, decltype(ctrl)::value, 0xf, 0xf, true));
    };
    step(std::integral_constant<int, 0xb1>{});   // quad_perm [1,0,3,2]
    step(std::integral_constant<int, 0x4e>{});   // quad_perm [2,3,0,1]
    step(std::integral_constant<int, 0x141>{});  // row_half_mirror
    step(std::integral_constant<int, 0x140>{});  // row_mirror
    return v;
}
// the largest of the wave (the same in every lane)
__device__ __forceinline__ uint32_t wave_max_u32(uint32_t v) {
    v = lanes16_max_u32(v);
    auto a = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = max(a[0], a[1]);
    auto b = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return max(b[0], b[1]);
}

// max / sum over the four lanes l, l ^ 16, l ^ 32, l ^ 48
__device__ __forceinline__ float lanes4_max(float v) {
    auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float lanes4_sum(float v) {
    auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// the larger magnitude; NaN stays
__device__ __forceinline__ float mag(float m, float x) { return __builtin_elementwise_maximum(m, fabsf(x)); }
// the exponent e of a positive finite x in [2^e, 2^(e+1)), 0 for 0
__device__ __forceinline__ int exponent_of(float x) {
    return x == 0.f ? 0 : (int)(__float_as_uint(x) >> 23 & 255) - 127;
}
// The least exponent that a query row is scaled by (to 2^14: f32 holds the factor
// and what undoes it), and the least factor of the scores: not 0, a score that is
// not seen is -inf.
constexpr int QUERY_MIN = -112;
constexpr float LEAST = 1.4e-45f;
// 2^n (what f32 cannot hold ends at its largest power)
__device__ __forceinline__ float pow2(int n) { return ldexpf(1.0f, max(-300, min(n, 127))); }

// A call as the kernels take it.  An item is a block of queries of a kv head
// (the blocks of a head in turn); items from `whole` on are split over their
// keys, and their queries' partial results lie in the items' order.
struct AttnCall {
    cmf_attention_args a;
    int hpk;         // query heads per kv head
    uint32_t inv;    // ceil(2^32 / hpk): query / hpk = high word of query * inv
    int groups, per;  // items of a kv head, queries of an item
    int whole, nsplit;
    float qscale;    // scale * log2(e)
    float *pm, *pl;  // [split items' queries][nsplit] partial maxima (log2 units) and sums
    float* po;       // [split items' queries][nsplit][128], relative to the maximum
};

// row of query qi (exact: queries and hpk multiply to less than 2^32)
__device__ __forceinline__ int row_of(const AttnCall& c, int qi) { return c.hpk == 1 ? qi : (int)__umulhi((uint32_t)qi, c.inv); }

// The keys that the rows [r0, r1] of a block see, numbered [0, nv): positions
// [0, s), then [lo, lo + nv - s).
struct Keys {
    int npos0;  // cached positions
    int s, lo, nv;
    int min_p, max_p;  // the rows' lowest and highest position
    bool tree;
    __device__ __forceinline__ int pos(int v) const { return v < s ? v : v - s + lo; }
};

__device__ __forceinline__ int cached_positions(const cmf_attention_args& a) {
    int n = a.pos0;
    if (a.d_pos0) n = min(n + *a.d_pos0, a.len_bound);
    return max(0, min(n, a.slots));
}

__device__ __forceinline__ Keys keys_of(const cmf_attention_args& a, int r0, int r1) {
    Keys k;
    k.npos0 = cached_positions(a);
    k.tree = a.d_mask != nullptr;
    // a tree's rows lie at most 63 positions past the root: the bound for the
    // range alone (d_depth is looked at row by row)
    k.min_p = k.tree || a.d_depth ? k.npos0 : k.npos0 + r0;
    k.max_p = k.tree || a.d_depth ? 0x3fffffff : k.npos0 + r1;
    const int hi = k.npos0 + (k.tree ? a.b : r1 + 1);
    k.lo = a.window ? max(0, min(k.min_p - a.window + 1, hi)) : 0;
    if (k.tree) k.lo = min(k.lo, k.npos0);  // (new rows are the mask's alone)
    k.s = min(a.sinks, k.lo);
    k.nv = k.s + hi - k.lo;
    return k;
}

// What a query row sees, as tests without branches: new row j (negative: a
// cached position) with j <= lim or bit j of mask, and pos > far, pos < sinks
// or j >= free.
struct Sight {
    int lim, far, free;
    uint64_t mask;
};
// A row's depth and mask bits as read; without them its queries' first bytes,
// not used (no branch: the loads are under way together).
struct SightIn {
    int depth;
    uint64_t mask;
};
__device__ __forceinline__ SightIn sight_in(const cmf_attention_args& a, int row) {
    const float* q = a.q + (size_t)row * a.ldq;
    return SightIn{*(a.d_depth ? a.d_depth + row : (const int*)q),
                   *(a.d_mask ? (const uint64_t*)a.d_mask + row : (const uint64_t*)q)};
}
__device__ __forceinline__ Sight sight_of(const cmf_attention_args& a, const Keys& k, int row, const SightIn& in) {
    const int P = k.npos0 + (a.d_depth ? in.depth : row);
    return Sight{k.tree ? -1 : row, a.window ? P - a.window : -1, k.tree ? 0 : 0x7fffffff, k.tree ? in.mask : 0};
}
__device__ __forceinline__ Sight sight_of(const cmf_attention_args& a, const Keys& k, int row) {
    return sight_of(a, k, row, a.d_mask ? sight_in(a, row) : SightIn{});  // (a depth goes with a mask)
}
__device__ __forceinline__ bool sees(const cmf_attention_args& a, const Keys& k, const Sight& s, int pos) {
    const int j = pos - k.npos0;
    return ((j <= s.lim) | ((s.mask >> (j & 63) & 1) != 0)) & ((pos > s.far) | (pos < a.sinks) | (j >= s.free));
}

// The key and value rows of a kv head, as cached rows and new ones.  The
// addresses are held in registers: chosen among the arguments themselves, a row
// would cost a load of the chosen argument before its own.
template <class T>
struct KvRows {
    uintptr_t k, v, kn, vn;
    uint32_t rs, nrs;  // bytes between rows
    int n0;
    __device__ __forceinline__ KvRows(const cmf_attention_args& a, const Keys& ks, int g) {
        n0 = ks.npos0;
        rs = nrs = (uint32_t)a.row_stride * sizeof(T);
        const uintptr_t o = (uintptr_t)g * a.head_stride * sizeof(T);
        k = (uintptr_t)a.k + o;
        v = (uintptr_t)a.v + o;
        kn = k + (uintptr_t)n0 * rs;
        vn = v + (uintptr_t)n0 * rs;
        if (a.k_new) {
            const uintptr_t p = (uintptr_t)g * a.new_head_stride * sizeof(T);
            kn = (uintptr_t)a.k_new + p;
            vn = (uintptr_t)a.v_new + p;
            nrs = (uint32_t)a.new_row_stride * sizeof(T);
        }
        asm("" : "+s"(k), "+s"(v), "+s"(kn), "+s"(vn), "+s"(rs), "+s"(nrs));
    }
    // (device memory: the global address space lets the loads be global ones)
    static __device__ __forceinline__ const T* ptr(uintptr_t u) {
        return (const T*)(const __attribute__((address_space(1))) T*)u;
    }
    __device__ __forceinline__ uintptr_t offset(int pos) const {
        const bool old = pos < n0;
        return (uintptr_t)(uint32_t)(old ? pos : pos - n0) * (old ? rs : nrs);
    }
    __device__ __forceinline__ const T* key(int pos) const { return ptr((pos < n0 ? k : kn) + offset(pos)); }
    __device__ __forceinline__ const T* value(int pos) const { return ptr((pos < n0 ? v : vn) + offset(pos)); }
};

// N elements as they lie in memory, and as f32
template <class T, int N>
struct Raw {
    typedef uint32_t vec __attribute__((ext_vector_type(N * sizeof(T) / 4)));
    vec v;
    // from element `off` (below 2^30 bytes) on: a wave-uniform base stays in
    // scalar registers
    __device__ __forceinline__ void load(const T* base, uint32_t off) {
        const char* p = (const char*)base + (uint32_t)(off * sizeof(T));
        if constexpr (N * sizeof(T) == 32) {  // two loads of 16 bytes
            const uint4v a = ((const uint4v*)p)[0], b = ((const uint4v*)p)[1];
            v = vec{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
        } else {
            v = *(const vec*)p;
        }
    }
    __device__ __forceinline__ float get(int i) const {
        if constexpr (sizeof(T) == 4) {
            return __uint_as_float(v[i]);
        } else {
            const uint16_t u = (uint16_t)(v[i >> 1] >> (16 * (i & 1)));
            return to_f32(__builtin_bit_cast(T, u));
        }
    }
};
// A 16-bit cache's elements are MFMA operands as they are; the f32 side comes in
// parts of their type that add up to it: two of f16 (22 bits, from values
// scaled into f16's range), three of bf16 (24 bits, f32's range).
template <class T>
struct Part;
template <>
struct Part<_Float16> {
    static constexpr int N = 2;
    static constexpr float SHIFT = 6.f, LAZY = 8.f;  // weights 2^(s - m + SHIFT) <= 2^(SHIFT + LAZY) < 65504
    static constexpr bool SCALED = true;
    static constexpr uint32_t INF = 0x7c00;
    static __device__ __forceinline__ uint32_t pack(float x, float y) {
        return __builtin_bit_cast(uint32_t, __builtin_convertvector((float2v{x, y}), half2v));
    }
    static __device__ __forceinline__ float lo(uint32_t u) { return (float)__builtin_bit_cast(half2v, u)[0]; }
    static __device__ __forceinline__ float hi(uint32_t u) { return (float)__builtin_bit_cast(half2v, u)[1]; }
    static __device__ __forceinline__ float4v mm32(uint4v a, uint4v b, float4v c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8, a), __builtin_bit_cast(half8, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ float4v mm16(uint2v a, uint2v b, float4v c) {
        return __builtin_amdgcn_mfma_f32_16x16x16f16(__builtin_bit_cast(half4, a), __builtin_bit_cast(half4, b), c, 0, 0, 0);
    }
};
template <>
struct Part<bf16_t> {
    static constexpr int N = 3;
    static constexpr float SHIFT = -12.f, LAZY = 12.f;  // weights of at most 1
    static constexpr bool SCALED = false;
    static constexpr uint32_t INF = 0x7f80;
    static __device__ __forceinline__ uint32_t pack(float x, float y) {
        return __builtin_bit_cast(uint32_t, __builtin_convertvector((float2v{x, y}), bf2v));
    }
    static __device__ __forceinline__ float lo(uint32_t u) { return __uint_as_float(u << 16); }
    static __device__ __forceinline__ float hi(uint32_t u) { return __uint_as_float(u & 0xffff0000u); }
    static __device__ __forceinline__ float4v mm32(uint4v a, uint4v b, float4v c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf8, a), __builtin_bit_cast(bf8, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ float4v mm16(uint2v a, uint2v b, float4v c) {
        return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(short4v, a), __builtin_bit_cast(short4v, b), c, 0, 0, 0);
    }
};
template <>
struct Part<float> {
    static constexpr int N = 1;
    static constexpr float SHIFT = -12.f, LAZY = 12.f;  // weights of at most 1
    static constexpr bool SCALED = false;
};
// x as the parts p[0 .. N) of two values
template <class T>
__device__ __forceinline__ void parts2(float x, float y, uint32_t (&p)[Part<T>::N]) {
#pragma unroll
    for (int k = 0; k < Part<T>::N; k++) {
        p[k] = Part<T>::pack(x, y);
        x -= Part<T>::lo(p[k]);
        y -= Part<T>::hi(p[k]);
    }
}

// ---------------------------------------------------------------------------
// Few queries per kv head (decode rows, small trees): the scores and values
// in f32 on the 16x16x4 MFMA, K and V straight from memory into its operands.
//
// A wave takes 16 keys at a time for up to 16 queries, transposed so that
// nothing goes through LDS: S^T = K Q^T (rows keys, columns queries), and the
// weights come out in the lanes and registers that O^T = V^T P^T wants them
// in (lane (n, kq) = query n, keys 4 kq + e in register e; the MFMA's k order
// is free, so step e takes key 4 kq + e from lane group kq).  Lane (m, kq)
// loads 8 consecutive dims 32 j + 8 kq of key m (K) and 16 bytes at a time of
// keys 4 kq + e (V).  Softmax with a running maximum, one column a lane.
// Four waves take a workgroup's 16-key tiles in turn and meet in LDS in wave
// order.  f32 caches: f32 operands, no rounding of the inputs, any range.
// 16-bit caches: K (16x16x32) and V (16x16x16, its four keys per lane packed by
// dim) are operands as they lie in memory, the queries and weights in parts.
//
// Bound by the cache's bytes where that is long (16 KiB of f32 K/V per tile
// against 64 MFMAs of 32 cycles per 16 queries, 8 KiB of f16 against 24 of 16),
// by the chain of round trips where it is short: 5 rows of 32 heads on 8
// through a window of 16000 in f16, 66 MB, 19 us (3.5 TB/s); 9 rows of 16 heads on
// 8 over 2048 f32 keys 11 us, of which about 3 are the first loads and 3 two
// tiles; one row through a window of 1024, 6.2 us.  32 queries a wave read the
// keys half as often, but begin later and take turns at the MFMAs (9 rows of 16
// heads: over 100 keys 10.3 us instead of 8.0, over 2048 15.5 instead of 14.2, over
// 16000 39.9 instead of 42.0).
// grid (nsplit, nkv, ceil(b hpk / 16)), block 256.
// ---------------------------------------------------------------------------
constexpr int RQ = 16;  // queries of a workgroup

template <class T>
__global__ __launch_bounds__(256, 2) void k_attn_rows(AttnCall c) {
    const cmf_attention_args& a = c.a;
    constexpr int NW = 4, OROW = HD + 4;
    constexpr bool F32 = sizeof(T) == 4;
    constexpr float SHIFT = Part<T>::SHIFT, LAZY = Part<T>::LAZY;
    constexpr float up = SHIFT < 0 ? 1.f / (1 << (int)-SHIFT) : 1 << (int)SHIFT;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n = lane & 15, kq = lane >> 4, split = blockIdx.x, g = blockIdx.y, q0 = blockIdx.z * RQ;
    const int nq = a.b * c.hpk;
    const int r0 = row_of(c, q0), r1 = row_of(c, min(q0 + RQ, nq) - 1);
    const Keys ks = keys_of(a, r0, r1);

    const KvRows<T> kv(a, ks, g);
    // this split's keys, whole tiles
    const int per = ((ks.nv + c.nsplit - 1) / c.nsplit + 15) / 16 * 16;
    const int v_lo = min(split * per, ks.nv), v_hi = min(v_lo + per, ks.nv);

    // A tile as it lies in memory: K row n, and V rows 4 kq + e, 16 bytes at a
    // time (component i of lane m is dim 64 (i / 4) + 4 m + i % 4 of f32 rows,
    // 8 m + i of 16-bit ones).  Numbers past the end read the last key.
    constexpr int VP = sizeof(T) == 4 ? 2 : 1;
    Raw<T, 8> kn[4];
    Raw<T, 16 / sizeof(T)> vn[4][VP];
    auto load = [&](int v0) {
        const T* kp = kv.key(ks.pos(min(v0 + n, ks.nv - 1)));
#pragma unroll
        for (int j = 0; j < 4; j++) kn[j].load(kp, 32 * j + 8 * kq);
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const T* vp = kv.value(ks.pos(min(v0 + 4 * kq + e, ks.nv - 1)));
#pragma unroll
            for (int u = 0; u < VP; u++) vn[e][u].load(vp, 64 * u + (VP == 2 ? 4 : 8) * n);
        }
    };
    // the queries: lane (n, kq) holds dims 32 j + 8 kq + c of query n (read
    // before the keys: loads are waited for in order)
    constexpr int QF = F32 ? 32 : 1, QP = F32 ? 1 : 4;
    float qf[QF], cq;  // cq: what the scores are multiplied by, positive
    uint4v qp[QP][Part<T>::N];
    const int qi = min(q0 + n, nq - 1), r = row_of(c, qi), h = g * c.hpk + qi - r * c.hpk;
    const SightIn in = sight_in(a, r);
    const float* q = a.q + (size_t)r * a.ldq + (size_t)h * HD;
    Raw<float, 8> xq[4];
#pragma unroll
    for (int j = 0; j < 4; j++) xq[j].load(q, 32 * j + 8 * kq);
    load(v_lo + 16 * wave);  // (there is a key at least; a wave without a tile reads it in vain)
    const Sight see = sight_of(a, ks, r, in);
    float x[32];
    float f = c.qscale < 0.f ? -1.f : 1.f;
    int eq = 0;
#pragma unroll
    for (int i = 0; i < 32; i++) x[i] = xq[i >> 3].get(i & 7);
    if constexpr (Part<T>::SCALED) {
        float mx = 0.f;
#pragma unroll
        for (int i = 0; i < 32; i++) mx = fmaxf(mx, fabsf(x[i]));
        eq = max(exponent_of(lanes4_max(mx)), QUERY_MIN) - 14;
        f *= pow2(-eq);
    }
    cq = fmaxf(fabsf(ldexpf(c.qscale, eq)), LEAST);
    if constexpr (F32) {
#pragma unroll
        for (int i = 0; i < 32; i++) qf[i] = x[i] * f;
    } else {
#pragma unroll
        for (int i = 0; i < 32; i += 2) {
            uint32_t p[Part<T>::N];
            parts2<T>(x[i] * f, x[i + 1] * f, p);
#pragma unroll
            for (int k = 0; k < Part<T>::N; k++) qp[i >> 3][k][(i & 7) >> 1] = p[k];
        }
    }

    float4v acc[8];
    float m = -INFINITY, l = 0.f;
    int odd_lo = 0, odd_hi = -1;  // the first and last tile left out
#pragma unroll
    for (int i = 0; i < 8; i++) acc[i] = float4v{0.f, 0.f, 0.f, 0.f};

    for (int v0 = v_lo + 16 * wave; v0 < v_hi; v0 += 16 * NW) {
        // a tile with infinities or NaN in V (0 * v is NaN then) is left for the
        // walk at the end
        bool bad;
        if constexpr (F32) {
            float x = 0.f;
#pragma unroll
            for (int e = 0; e < 4; e++)
#pragma unroll
                for (int i = 0; i < 8; i++) x = fmaf(vn[e][i / (8 / VP)].get(i % (8 / VP)), 0.f, x);
            bad = x != x;
        } else {
            ushort2v x = {0, 0};
#pragma unroll
            for (int e = 0; e < 4; e++)
#pragma unroll
                for (int i = 0; i < 4; i++)
                    x = __builtin_elementwise_max(x, __builtin_bit_cast(ushort2v, vn[e][0].v[i] & 0x7fff7fffu));
            bad = max((int)x[0], (int)x[1]) >= (int)Part<std::conditional_t<F32, bf16_t, T>>::INF;
        }
        if (__builtin_amdgcn_ballot_w64(bad) == 0) {
            float4v s = {0.f, 0.f, 0.f, 0.f};
            if constexpr (F32) {
#pragma unroll
                for (int i = 0; i < 32; i++)
                    s = __builtin_amdgcn_mfma_f32_16x16x4f32(kn[i >> 3].get(i & 7), qf[i], s, 0, 0, 0);
            } else {
#pragma unroll
                for (int k = Part<T>::N - 1; k >= 0; k--)  // the small parts first
#pragma unroll
                    for (int j = 0; j < 4; j++)
                        s = Part<T>::mm32(__builtin_bit_cast(uint4v, kn[j].v), qp[j][k], s);
            }
            const bool inside = v0 + 16 <= v_hi;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int v = v0 + 4 * kq + e;
                s[e] = (sees(a, ks, see, ks.pos(v)) & (inside | (v < v_hi))) ? s[e] : -INFINITY;
            }
            // (maximum and differences before the factor: exact near the maximum,
            // however large the scores; 0 for the largest one)
            const float mx = lanes4_max(fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3])));
            if (__builtin_amdgcn_ballot_w64((mx - m) * cq > LAZY)) {
                const float m1 = fmaxf(m, mx), al = exp2f((m - (m1 == -INFINITY ? 0.f : m1)) * cq);
                m = m1;
                l *= al;
#pragma unroll
                for (int i = 0; i < 8; i++) acc[i] *= al;
            }
            // (2^SHIFT as a factor: in the exponent it would cost bits of the score)
            const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                s[e] = __builtin_amdgcn_exp2f((s[e] - ref) * cq) * up;
                l += s[e];
            }
            if constexpr (F32) {
#pragma unroll
                for (int e = 0; e < 4; e++)
#pragma unroll
                    for (int i = 0; i < 8; i++)
                        acc[i] = __builtin_amdgcn_mfma_f32_16x16x4f32(vn[e][i / (8 / VP)].get(i % (8 / VP)), s[e], acc[i], 0, 0, 0);
            } else {
                uint2v w[Part<T>::N];
#pragma unroll
                for (int e = 0; e < 4; e += 2) {
                    uint32_t p[Part<T>::N];
                    parts2<T>(s[e], s[e + 1], p);
#pragma unroll
                    for (int k = 0; k < Part<T>::N; k++) w[k][e >> 1] = p[k];
                }
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    // dim 8 n + i of the lane's four keys
                    const uint32_t sel = i & 1 ? 0x07060302 : 0x05040100;
                    const uint2v x = {__builtin_amdgcn_perm(vn[1][0].v[i >> 1], vn[0][0].v[i >> 1], sel),
                                      __builtin_amdgcn_perm(vn[3][0].v[i >> 1], vn[2][0].v[i >> 1], sel)};
#pragma unroll
                    for (int k = Part<T>::N - 1; k >= 0; k--) acc[i] = Part<T>::mm16(x, w[k], acc[i]);
                }
            }
        } else {
            if (odd_hi < 0) odd_lo = v0;
            odd_hi = v0;
        }
        if (v0 + 16 * NW < v_hi) load(v0 + 16 * NW);
    }

    // the wave's state into LDS
    __shared__ float2 sml[NW][RQ];
    __shared__ __align__(16) float so[NW][RQ][OROW];
    const float un = pow2(-(int)(SHIFT + LAZY));  // (sums of large values stay finite)
    l = lanes4_sum(l) * un;
    m *= cq;  // in log2 units from here on
#pragma unroll
    for (int i = 0; i < 8; i++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const int r = 4 * kq + e;
            so[wave][n][VP == 2 ? 64 * (i >> 2) + 4 * r + (i & 3) : 8 * r + i] = acc[i][e] * un;
        }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    if (odd_hi >= 0) {
        // the tiles left out, key by key; lane (n, kq) has 32 dims of its query
#pragma unroll 1
        for (int v0 = odd_lo; v0 <= odd_hi; v0 += 16 * NW) {
            const T* row = kv.value(ks.pos(min(v0 + n, ks.nv - 1))) + 32 * kq;
            float mv = 0.f;
#pragma unroll
            for (int u = 0; u < 32; u += 8) {
                Raw<T, 8> r;
                r.load(row, u);
#pragma unroll
                for (int i = 0; i < 8; i++) mv = mag(mv, r.get(i));
            }
            if (!__builtin_amdgcn_ballot_w64(!(mv < INFINITY))) continue;
#pragma unroll 1
            for (int k = 0; k < 16; k++) {
                const int v = v0 + k, pos = ks.pos(min(v, ks.nv - 1));
                const bool vis = sees(a, ks, see, pos) & (v < v_hi);
                if (!__builtin_amdgcn_ballot_w64(vis)) continue;
                const T *kp = kv.key(pos), *vp = kv.value(pos);
                float d = 0.f;
#pragma unroll 4
                for (int u = 0; u < 32; u++) d = fmaf(q[32 * kq + u], to_f32(kp[32 * kq + u]), d);
                d = lanes4_sum(d) * c.qscale;
                asm("" : "+v"(d));  // (rounded before the maximum comes off: no fma)
                if (!vis) continue;
                float* o = &so[wave][n][32 * kq];
                const float m1 = fmaxf(m, d), ref = m1 == -INFINITY ? 0.f : m1;
                const float al = exp2f(m - ref), wt = exp2f(d - ref - LAZY);
#pragma unroll 4
                for (int u = 0; u < 32; u++) o[u] = o[u] * al + wt * to_f32(vp[32 * kq + u]);
                l = l * al + wt;
                m = m1;
            }
        }
    }
    if (kq == 0) sml[wave][n] = make_float2(m, l);
    __syncthreads();
    // the four waves meet, in wave order; whole rows out
#pragma unroll
    for (int t = threadIdx.x; t < RQ * 32; t += 256) {
        const int qq = t >> 5, d = (t & 31) * 4, qi = q0 + qq;
        if (qi >= nq) continue;
        float2 e[NW];
        float M = -INFINITY;
#pragma unroll
        for (int w = 0; w < NW; w++) {
            e[w] = sml[w][qq];
            M = fmaxf(M, e[w].x);
        }
        const float ref = M == -INFINITY ? 0.f : M;
        float L = 0.f;
        float4v o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < NW; w++) {
            const float f = exp2f(e[w].x - ref);  // (a wave without keys: 0, and its state is zeros)
            L += e[w].y * f;
            o += *(const float4v*)&so[w][qq][d] * f;
        }
        const int r = row_of(c, qi), h = g * c.hpk + qi - r * c.hpk;
        if (c.nsplit == 1) {
            const float inv = L == 0.f ? 0.f : 1.0f / L;
            *(float4v*)(a.out + (size_t)r * a.ldo + (size_t)h * HD + d) = o * inv;
        } else {
            const size_t at = ((size_t)(g * c.groups + blockIdx.z) * RQ + qq) * c.nsplit + split;
            *(float4v*)(c.po + at * HD + d) = o;
            if (d == 0) {
                c.pm[at] = M;
                c.pl[at] = L;
            }
        }
    }
}

// ---------------------------------------------------------------------------
// Many queries per kv head (prompt chunks, larger trees): tiles of 64 keys in
// LDS as f16 halves, scores and values on the 32x32x16 f16 MFMA: q.k = qh.kh +
// qh.kl + ql.kh and p.v likewise (22-bit operands, f32 sums; a 16-bit cache has
// no kl and vl), three products at 16 times the f32 MFMA's rate.
//
// f16 has 5 exponent bits, so operands of an unusual size are scaled by a power
// of two first (exact): a key row whose largest magnitude is not in [2^-2, 2^6)
// to [2^2, 2^3), a query row always, to [2^14, 2^15), and the values of 8 keys by
// one factor where their rows are alike (within 2^4), else by one a row.  A key's
// factor is undone in its scores, a value's in its weights: they are 2^(s + f - m
// + 6), f the factor's exponent and m, kept per query, at most 8 below the
// largest s + f that the query sees.  What the halves drop is then 2^-23 of an
// element or of its row's largest, and of a query's largest weighted value:
// nothing that a query does not see takes part.
// A block of 32 keys that holds infinities, NaN, keys outside [2^-100, 2^101) or
// values outside [2^-50, 2^61) by their rows' largest (0 is none of these) is
// left for a second walk without MFMAs, so that it reaches only the queries
// that see it.
//
// S^T = K Q^T: a lane (query n = lane % 32, h = lane / 32) ends up with the
// keys 8 a + 4 h + b of a 32-key block in register 4 a + b, which is the B
// operand of O^T = V^T P^T when V's slots hold the same keys: the weights stay
// in registers.  Eight waves: four groups of 32 queries, the two 32-key blocks
// of a tile on different waves, joined at the end.  Two tile buffers: while one
// is multiplied, the next tile, in registers since the tile before, is split
// into the other, and the one after is loaded; one barrier a tile.  The two
// waves of a SIMD (block 0 and 1) go through a tile half a turn apart, one
// multiplies before it splits and loads, the other after, so that the vector
// work of one runs beside the products of the other.
//
// A tile takes a SIMD about 7800 cycles at f32 and 6600 at 16 bits, of which
// the MFMAs of its two waves take 96 and 64 times 32: bound by what each wave does
// one after the other (scores 1550, weights and values 2300, splitting 1850,
// loads 1280, the barrier), and by 26000 cycles a workgroup to read and split
// the queries and to join and write the outputs.  4100 rows of 16 heads on 8
// behind 4000 through a window of 1024, f32: 177 us with the join, 195 TFLOP/s of
// the formula (585 of products), MFMAs busy 33 % of the CUs' cycles; 64 rows of 32
// heads on 8 over 65536 bf16 keys: 183 to 192 us from box to box, 359 TFLOP/s at
// least (717 of products), MFMAs 34 %.  Keys and values of standard deviation
// 0.02, whose rows need factors: 202 and 234 us.
// grid whole + nsplit (items - whole), block 512, LDS Tile<T>::LDS: the items
// (those in one piece, then the splits of the others) in eight runs, one to an
// XCD (workgroups go round them), whose L2 then serves neighbouring blocks the
// same keys.
// ---------------------------------------------------------------------------

constexpr int KT = 64, TQ = 128;     // keys of a tile, queries of a workgroup
constexpr float SHIFT = 6.f, LAZY = 8.f;  // weights are 2^(s - m + SHIFT) <= 2^(SHIFT + LAZY)
constexpr float FAR_SCORE = 4096.f;  // (log2 units: a product's rounding moves a weight by 2^-12 of itself here)
constexpr float UNIT_MIN = -60.f;    // (below the exponents of all values that the tiles take)
constexpr int KFRAG = 528;           // 32 keys x 8 dims (512 B), padded against bank conflicts
constexpr int K_BYTES = 32 * KFRAG;  // one half (hi or lo) of the keys
constexpr int VGROUP = 2048;         // 8 keys x 128 dims: [dim % 2][dim / 2][8 keys]
constexpr int V_BYTES = 8 * VGROUP;
constexpr int OROW = HD + 4;  // f32 rows in LDS: the queries at the start, the eight waves' outputs (32 rows each) at the end
constexpr int END_BYTES = 8 * 32 * (OROW + 2) * 4;
template <class T>
struct Tile {
    static constexpr bool LO = sizeof(T) == 4;
    static constexpr int HALVES = LO ? 2 : 1, BUF = HALVES * (K_BYTES + V_BYTES);
    // and the codes of a block's groups (8 of K, 4 of V in 64 bytes), the key and
    // value rows' factors
    static constexpr int USE = 2 * (BUF + 128 + 8 * KT);
    static constexpr int LDS = (USE > END_BYTES ? USE : END_BYTES) + 64 + 2048;  // (and two numbers a wave, one a lane)
};
static_assert(Tile<float>::LDS <= 160 * 1024, "LDS of a CU");

constexpr int SCHED_MFMA = 8, SCHED_LDS = 0x100;  // of sched_group_barrier: MFMAs, LDS reads
// The scale of a row or group is 2^(PLAIN - e) by its largest magnitude: e =
// PLAIN where f16 halves take it as it is; all zeros; infinities, NaN
constexpr int PLAIN = 2, NO_EXP = -1000, BAD_EXP = 1000;
// What a group of four key rows is: as it stands; rows with factors of their own;
// something that halves and f32 sums cannot hold.  One of eight value rows: its
// exponent, or one of these
enum { ROWS_PLAIN = 0, ROWS_SCALED = 500, ROWS_ODD = BAD_EXP };
constexpr int ALIKE = 4;  // value rows within 2^ALIKE share a factor
constexpr int KEY_RANGE = 100;  // exponents: scores by 2^-14 of a query's stay below 2^25+100, queries' factors normal
// value rows: a sum of weights and the weighted values by one maximum stay within
// f32's range, and so do those of splits by the others' (2^(61 + 50) apart)
constexpr int VALUE_MIN = -50, VALUE_MAX = 60;
__device__ __forceinline__ int exponent_class(uint32_t u) {  // of a magnitude's bits
    const int e = (int)(u >> 23) - 127;
    return u >= 0x7f800000u ? BAD_EXP : u == 0 ? NO_EXP : e >= -2 && e < 6 ? PLAIN : e;
}
// Whether all lanes' magnitudes are below 2^6 and each 16 lanes hold one of
// 2^-2 or more in a and in b (most often all do, which is one comparison).
__device__ __forceinline__ bool each16(uint64_t m) {
    m |= m >> 8;
    m |= m >> 4;
    m |= m >> 2;
    m |= m >> 1;
    return (~m & 0x0001000100010001ull) == 0;
}
__device__ __forceinline__ bool rows16_plain(float a, float b) {
    const bool low = mag(a, b) < 64.f;
    if (!__builtin_amdgcn_ballot_w64(!(low & (fminf(a, b) >= 0.25f)))) return true;
    return !__builtin_amdgcn_ballot_w64(!low) && each16(__builtin_amdgcn_ballot_w64(a >= 0.25f)) &&
           each16(__builtin_amdgcn_ballot_w64(b >= 0.25f));
}
// whether the tiles cannot take a key row whose largest magnitude has class e
__device__ __forceinline__ bool odd_key(int e) { return e == BAD_EXP || (e != NO_EXP && (e > KEY_RANGE || e < -KEY_RANGE)); }
__device__ __forceinline__ bool odd_value(int e) { return e == BAD_EXP || (e != NO_EXP && (e > VALUE_MAX || e < VALUE_MIN)); }
// The largest of each of eight registers over the wave, that of v[lane / 8] in
// every lane.
__device__ __forceinline__ uint32_t rows8_max(const float (&v)[8], int lane) {
    uint32_t a[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(v[i]), __float_as_uint(v[i + 4]), false, false);
        a[i] = max(s[0], s[1]);
    }
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const auto s = __builtin_amdgcn_permlane16_swap(a[i], a[i + 2], false, false);
        a[i] = max(s[0], s[1]);
    }
    auto step = [&](uint32_t x, auto ctrl) {
        return max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, decltype(ctrl)::value, 0xf, 0xf, true));
    };
    const std::integral_constant<int, 0x128> ror8;
    uint32_t r = lane & 8 ? step(a[1], ror8) : step(a[0], ror8);
    r = step(r, std::integral_constant<int, 0xb1>{});      // quad_perm [1,0,3,2]
    r = step(r, std::integral_constant<int, 0x4e>{});      // quad_perm [2,3,0,1]
    return step(r, std::integral_constant<int, 0x141>{});  // row_half_mirror
}
__device__ __forceinline__ bool scaled(int e) { return e != PLAIN && e != NO_EXP; }

struct Split8 {
    half8 hi, lo;
};
// x as f16 halves: hi = f16(x), lo = f16(x - hi)
template <bool LO>
__device__ __forceinline__ Split8 split8(const float (&x)[8]) {
    Split8 r;
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
        const float2v y = {x[i], x[i + 1]};
        const half2v h = __builtin_convertvector(y, half2v);
        r.hi[i] = h[0], r.hi[i + 1] = h[1];
        if constexpr (LO) {
            const float2v d = {y[0] - (float)h[0], y[1] - (float)h[1]};
            const half2v l = __builtin_convertvector(d, half2v);
            r.lo[i] = l[0], r.lo[i + 1] = l[1];
        }
    }
    return r;
}
__device__ __forceinline__ float lanes2_max(float v) {
    auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float lanes2_sum(float v) {
    auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}
// item of workgroup id of n: the eighth of the items that id's XCD takes
__device__ __forceinline__ uint32_t xcd_run(uint32_t id, uint32_t n) {
    const uint32_t x = id & 7, k = n >> 3, r = n & 7;
    return x * k + min(x, r) + (id >> 3);
}

template <class T>
__global__ __launch_bounds__(512, 2) void k_attn_tiles(AttnCall c) {
    const cmf_attention_args& a = c.a;
    constexpr bool LO = Tile<T>::LO;
    constexpr int BUF = Tile<T>::BUF, KL = K_BYTES, VH = Tile<T>::HALVES * K_BYTES, VL = VH + V_BYTES;
    extern __shared__ __align__(16) uint8_t sm[];
    int* code_at = (int*)(sm + 2 * BUF);  // [buffer][block][h][8]: codes of 4 groups of K, 2 of V
    // factors of the rows of groups with ROWS_SCALED: [buffer][key], and [buffer][group][8 values]
    float *kfac = (float*)(code_at + 64), *vfac = kfac + 2 * KT;
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int n = lane & 31, h = lane >> 5, nq = a.b * c.hpk;
    const bool part = (int)blockIdx.x >= c.whole;
    const int nsplit = part ? c.nsplit : 1;
    const uint32_t id = part ? xcd_run(blockIdx.x - c.whole, gridDim.x - c.whole) : xcd_run(blockIdx.x, c.whole);
    const int own = id / (uint32_t)nsplit, split = id - own * nsplit, item = part ? c.whole + own : own;
    const int g = (uint32_t)item / (uint32_t)c.groups, q0 = (item - g * c.groups) * TQ;
    const int r0 = row_of(c, q0), r1 = row_of(c, min(q0 + TQ, nq) - 1);
    const Keys ks = keys_of(a, r0, r1);
    const int per = ((ks.nv + nsplit - 1) / nsplit + KT - 1) / KT * KT;
    const int v_lo = min(split * per, ks.nv), v_hi = min(v_lo + per, ks.nv);
    const KvRows<T> kv(a, ks, g);
    const int qg = wave & 3, kb = wave >> 2;  // the wave's queries and 32-key block

    // the lane, where it is needed: addresses of what is seldom done are not worked
    // out before the loop, which has no registers left for them
    auto lane_here = []() {
        int x;
        asm volatile("v_mbcnt_lo_u32_b32 %0, -1, 0\n\tv_mbcnt_hi_u32_b32 %0, -1, %0" : "=v"(x));
        return x;
    };
    // what thread t stages of a tile: dims 8 kd .. of keys kk and kk + 32, and
    // dims 2 lane, 2 lane + 1 of the keys vk + {0 .. 3, 8 .. 11} (the slots of
    // group (block, 16-key half, h) = wave)
    const int kd = t & 15, kk = t >> 4, vk = 32 * (wave >> 2) + 16 * (wave >> 1 & 1) + 4 * (wave & 1);
    Raw<T, 8> kx[2];
    Raw<T, 2> vx[8];
    // A tile that is one run of the cache needs one address, and a sum a row.
    auto one_run = [&](int v0) { return v0 >= ks.s && v0 + KT <= ks.nv && (ks.pos(v0) + KT <= ks.npos0 || !a.k_new); };
    auto load_k = [&](int v0) {
        if (one_run(v0)) {
            uint32_t rs = kv.rs;
            asm("" : "+s"(rs));  // (the offset is not kept over the loop)
            const uintptr_t k = kv.k + (uintptr_t)(uint32_t)ks.pos(v0) * rs;
            const uint32_t ko = kk * (rs / sizeof(T)) + 8 * kd;
#pragma unroll
            for (int r = 0; r < 2; r++) kx[r].load(kv.ptr(k + 32 * r * rs), ko);
        } else {
#pragma unroll
            for (int r = 0; r < 2; r++) kx[r].load(kv.key(ks.pos(min(v0 + kk + 32 * r, ks.nv - 1))), 8 * kd);
        }
    };
    auto load_v = [&](int v0) {
        if (one_run(v0)) {
            uintptr_t v = kv.v + (uintptr_t)(uint32_t)(ks.pos(v0) + vk) * kv.rs;
#pragma unroll
            for (int i = 0; i < 8; i++) {
                vx[i].load(kv.ptr(v), 2 * lane);
                v += i == 3 ? 5 * kv.rs : kv.rs;
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++)
                vx[i].load(kv.value(ks.pos(min(v0 + vk + 8 * (i >> 2) + (i & 3), ks.nv - 1))), 2 * lane);
        }
    };
    // The queries' rows, whole, on their way to LDS, and behind them the first
    // tile (loads are waited for in order).
    float4v qx[TQ / 16];
#pragma unroll
    for (int k = 0; k < TQ / 16; k++) {
        const int qi = min(q0 + 16 * k + (t >> 5), nq - 1), row = row_of(c, qi), head = g * c.hpk + qi - row * c.hpk;
        qx[k] = *(const float4v*)(a.q + (size_t)row * a.ldq + (size_t)head * HD + 4 * (t & 31));
    }
    if (v_lo < v_hi) {
        load_k(v_lo);
        load_v(v_lo);
    }

    // the wave's queries: lane (n, h) holds dims 16 j + 8 h + i
    // (row and head are worked out where they are needed: the loop has no
    // registers left for them)
    struct Query {
        int row, head;
    };
    auto this_lane = [&]() { return (int)__builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0u)); };
    auto query = [&]() {
        const int qi = min(q0 + 32 * qg + (this_lane() & 31), nq - 1), row = row_of(c, qi);
        return Query{row, g * c.hpk + qi - row * c.hpk};
    };
    half8 qh[8], ql[8];
    float cq;  // the scores' factor: |scale| * log2(e) * 2^(eq - 14)
    {
        float* sq = (float*)sm;
#pragma unroll
        for (int k = 0; k < TQ / 16; k++) *(float4v*)(sq + (16 * k + (t >> 5)) * OROW + 4 * (t & 31)) = qx[k];
        __syncthreads();
        const float* q = sq + (32 * qg + n) * OROW + 8 * h;
        float x[8][8], mx = 0.f;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            load8(q + 16 * j, x[j]);
#pragma unroll
            for (int i = 0; i < 8; i++) mx = fmaxf(mx, fabsf(x[j][i]));
        }
        const int eq = max(exponent_of(lanes2_max(mx)), QUERY_MIN);  // (an infinite or NaN query ends as NaN by itself)
        const float sc = c.qscale < 0.f ? -pow2(14 - eq) : pow2(14 - eq);
        cq = fmaxf(fabsf(ldexpf(c.qscale, eq - 14)), LEAST);
#pragma unroll
        for (int j = 0; j < 8; j++) {
#pragma unroll
            for (int i = 0; i < 8; i++) x[j][i] *= sc;
            const Split8 s = split8<true>(x[j]);
            qh[j] = s.hi;
            ql[j] = s.lo;
        }
        __syncthreads();
    }

    // The tile in registers into buffer `at`.  This wave stages keys 4 wave ..
    // 4 wave + 3 of both blocks (16 lanes a row) and the values of group `wave`.
    auto stage_k = [&](int at) {
        uint8_t* buf = sm + at * BUF;
        int* te = code_at + at * 32 + 8 * (wave & 1) + (wave >> 1);
        float x[2][8], mx[2] = {0.f, 0.f};
#pragma unroll
        for (int r = 0; r < 2; r++)
#pragma unroll
            for (int i = 0; i < 8; i++) {
                x[r][i] = kx[r].get(i);
                mx[r] = mag(mx[r], x[r][i]);
            }
        int code[2] = {ROWS_PLAIN, ROWS_PLAIN};
        if (!rows16_plain(mx[0], mx[1])) {
#pragma unroll
            for (int r = 0; r < 2; r++) {
                const int e = exponent_class(lanes16_max_u32(__float_as_uint(mx[r])));
                const bool sc = scaled(e) && !odd_key(e);
                code[r] = __builtin_amdgcn_ballot_w64(odd_key(e)) ? ROWS_ODD : ROWS_SCALED;
                const float f = sc ? pow2(PLAIN - e) : 1.f;
#pragma unroll
                for (int i = 0; i < 8; i++) x[r][i] *= f;
                const int lane1 = lane_here();
                if (!(lane1 & 15)) kfac[at * KT + 32 * r + 4 * wave + (lane1 >> 4)] = sc ? pow2(e - PLAIN) : 1.f;
            }
        }
#pragma unroll
        for (int r = 0; r < 2; r++) {
            const Split8 s = split8<LO>(x[r]);
            const int o = (r * 16 + kd) * KFRAG + kk * 16;
            *(half8*)(buf + o) = s.hi;
            if (LO) *(half8*)(buf + KL + o) = s.lo;
            te[16 * r] = code[r];  // (all lanes the same)
        }
    };
    auto stage_v = [&](int at) {
        uint8_t* buf = sm + at * BUF;
        // `all`: the largest of the lane's magnitudes; `each`: one that all eight
        // rows reach (in one lane at least, where they are alike)
        float x[2][8], all = 0.f, each = INFINITY;
        auto largest = [&](int i) { return mag(fabsf(x[0][i]), x[1][i]); };
#pragma unroll
        for (int i = 0; i < 8; i++) {
#pragma unroll
            for (int j = 0; j < 2; j++) x[j][i] = vx[i].get(j);
            all = mag(all, largest(i));
            each = fminf(each, largest(i));
        }
        int code = PLAIN;
        if (!__builtin_amdgcn_ballot_w64(each >= 0.25f) || __builtin_amdgcn_ballot_w64(!(all < 64.f))) {
            // one factor by the largest, if every row comes near it
            const uint32_t u = __builtin_amdgcn_readfirstlane(wave_max_u32(__float_as_uint(all)));
            code = u == 0 ? NO_EXP : u >= 0x7f800000u ? BAD_EXP : (int)(u >> 23) - 127;
            bool alike = !odd_value(code);
            const float least = alike ? pow2(code - ALIKE) : 0.f;
            if (!__builtin_amdgcn_ballot_w64(each >= least)) {
#pragma unroll
                for (int i = 0; i < 8; i++) alike &= __builtin_amdgcn_ballot_w64(largest(i) >= least) != 0;
            }
            if (alike) {
                const float f = code == NO_EXP ? 1.f : pow2(PLAIN - code);
#pragma unroll
                for (int i = 0; i < 16; i++) x[i >> 3][i & 7] *= f;
                code = max(code, VALUE_MIN);  // (zeros: the least weight, not to hold others down)
            } else {
                const int lane1 = lane_here();
                float mx[8];
#pragma unroll
                for (int i = 0; i < 8; i++) mx[i] = largest(i);
                const int e = exponent_class(rows8_max(mx, lane1));  // of row lane / 8
                const bool sc = scaled(e) && !odd_value(e);
                code = __builtin_amdgcn_ballot_w64(odd_value(e)) ? ROWS_ODD : ROWS_SCALED;
                const uint32_t f = __float_as_uint(sc ? pow2(PLAIN - e) : 1.f);
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const float fi = __uint_as_float(__builtin_amdgcn_readlane(f, 8 * i));
                    x[0][i] *= fi;
                    x[1][i] *= fi;
                }
                if (!(lane1 & 7))
                    vfac[at * KT + 8 * wave + (lane1 >> 3)] = sc ? pow2(e - PLAIN) : e == NO_EXP ? pow2(VALUE_MIN) : 1.f;
            }
        }
#pragma unroll
        for (int j = 0; j < 2; j++) {
            const Split8 s = split8<LO>(x[j]);
            const int o = wave * VGROUP + j * 1024 + lane * 16;
            *(half8*)(buf + VH + o) = s.hi;
            if (LO) *(half8*)(buf + VL + o) = s.lo;
        }
        code_at[at * 32 + 16 * (wave >> 2) + 8 * (wave & 1) + 4 + (wave >> 1 & 1)] = code;
    };

    float16v acc[4];
#pragma unroll
    for (int d = 0; d < 4; d++)
#pragma unroll
        for (int i = 0; i < 16; i++) acc[d][i] = 0.f;
    float m = -INFINITY, l = 0.f;
    bool odd = false;
    int* odd_at = (int*)(sm + Tile<T>::LDS - 64) + 2 * wave;  // the first and last tile with a block left out
    // Scores far from 0 have no bits for the values' exponents: from the first such
    // block on, m is of the scores alone and acc is in units of 2^unit, a lane's.
    bool far = false;
    float* unit = (float*)(sm + Tile<T>::LDS - 64 - 2048) + 64 * wave;
    unit[lane] = 0.f;

    constexpr int RD = LO ? 2 : 1, MM = LO ? 3 : 2;  // fragments read and products of a step
    float16v s;         // the block's scores, by 1 / cq
    bool kbad = false;  // one of its keys is odd
    // the scores of the wave's block of the tile at v0, in buffer `at`
    auto scores = [&](int v0, int at) {
        const uint8_t* buf = sm + at * BUF;
        const int4 ek = *(const int4*)(code_at + at * 32 + 16 * kb + 8 * h);
        const uint8_t* kp = buf + (kb * 16 + h) * KFRAG + n * 16;
#pragma unroll
        for (int i = 0; i < 16; i++) s[i] = 0.f;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const half8 x = *(const half8*)(kp + 2 * j * KFRAG);
            if constexpr (LO) {
                const half8 y = *(const half8*)(kp + KL + 2 * j * KFRAG);
                s = __builtin_amdgcn_mfma_f32_32x32x16_f16(y, qh[j], s, 0, 0, 0);
            }
            s = __builtin_amdgcn_mfma_f32_32x32x16_f16(x, ql[j], s, 0, 0, 0);
            s = __builtin_amdgcn_mfma_f32_32x32x16_f16(x, qh[j], s, 0, 0, 0);
        }
        // the fragments of three steps are read ahead of the products
        __builtin_amdgcn_sched_group_barrier(SCHED_LDS, 3 * RD + 1, 0);
#pragma unroll
        for (int j = 0; j < 5; j++) {
            __builtin_amdgcn_sched_group_barrier(SCHED_MFMA, MM, 0);
            __builtin_amdgcn_sched_group_barrier(SCHED_LDS, RD, 0);
        }
        __builtin_amdgcn_sched_group_barrier(SCHED_MFMA, 3 * MM, 0);
        kbad = false;
        if (__builtin_amdgcn_ballot_w64((ek.x | ek.y | ek.z | ek.w) != ROWS_PLAIN)) {
            kbad = __builtin_amdgcn_ballot_w64(max(max(ek.x, ek.y), max(ek.z, ek.w)) == ROWS_ODD) != 0;
            const float* kf = kfac + at * KT + 32 * kb + 4 * (lane_here() >> 5);
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
                const int e = i == 0 ? ek.x : i == 4 ? ek.y : i == 8 ? ek.z : ek.w;
                const float4v f = *(const float4v*)(kf + 2 * i);
#pragma unroll
                for (int b = 0; b < 4; b++) s[i + b] *= e == ROWS_SCALED ? f[b] : 1.f;
            }
        }
        // whether every query of the workgroup sees the whole tile
        const int pa = ks.pos(v0), pb = ks.pos(min(v0 + KT - 1, ks.nv - 1));
        const bool all = v0 + KT <= v_hi && pb <= (ks.tree ? ks.npos0 - 1 : ks.min_p) &&
                         (!a.window || (pa >= ks.lo && pa > ks.max_p - a.window) || pb < a.sinks);
        if (!all) {
            const Sight see = sight_of(a, ks, query().row);
#pragma unroll
            for (int i = 0; i < 16; i++) {
                const int v = v0 + 32 * kb + 8 * (i >> 2) + 4 * h + (i & 3);
                s[i] = (sees(a, ks, see, ks.pos(v)) & (v < v_hi)) ? s[i] : -INFINITY;
            }
        }
    };
    // their weights and the values' sum, from buffer `at`
    auto values = [&](int v0, int at) {
        const int2 cv = *(const int2*)(code_at + at * 32 + 16 * kb + 8 * h + 4);
        const bool groups = __builtin_amdgcn_ballot_w64(max(cv.x, cv.y) >= ROWS_SCALED) == 0;
        int left = kbad || (!groups && __builtin_amdgcn_ballot_w64(max(cv.x, cv.y) == ROWS_ODD));
        if (left) {
            if (!odd) odd_at[0] = v0;
            odd_at[1] = v0;
        }
        // (a branch of its own: one for both costs the loop its registers)
        left = __builtin_amdgcn_readfirstlane(left);
        if (left) {
            odd = true;
            return;
        }
        // exponents of the two groups' factors, or of registers 4 a .. 4 a + 3's values
        float e0 = (float)(cv.x - PLAIN), e1 = (float)(cv.y - PLAIN);
        auto exponents = [&](int a) {
            const float4v f = *(const float4v*)(vfac + at * KT + 32 * kb + 8 * (lane_here() >> 5) + 16 * (a >> 1) + 4 * (a & 1));
            float4v e;
#pragma unroll
            for (int b = 0; b < 4; b++) e[b] = (a < 2 ? cv.x : cv.y) == ROWS_SCALED ? (float)exponent_of(f[b]) : a < 2 ? e0 : e1;
            return e;
        };
        // m is the largest score (and exponent) up to 2^LAZY: the sums follow only
        // when one passes that
        float mx;
        if (groups) {
            float a = s[0], b = s[8];
#pragma unroll
            for (int i = 1; i < 8; i++) a = fmaxf(a, s[i]), b = fmaxf(b, s[8 + i]);
            mx = fmaxf(fmaf(a, cq, e0), fmaf(b, cq, e1));
        } else {
            mx = -INFINITY;
#pragma unroll
            for (int a = 0; a < 4; a++) {
                const float4v e = exponents(a);
#pragma unroll
                for (int b = 0; b < 4; b++) mx = fmaxf(mx, fmaf(s[4 * a + b], cq, e[b]));
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        mx = lanes2_max(mx);
        far |= __builtin_amdgcn_ballot_w64((fabsf(mx) > FAR_SCORE) & (mx > -INFINITY)) != 0;
        if (far) {
            mx = s[0];
#pragma unroll
            for (int i = 1; i < 16; i++) mx = fmaxf(mx, s[i]);
            mx = lanes2_max(mx) * cq;
        }
        if (__builtin_amdgcn_ballot_w64(mx > m + LAZY)) {
            const float m1 = fmaxf(m, mx), down = m - (m1 == -INFINITY ? 0.f : m1), al = exp2f(down);
            float f = al;
            if (far) {  // (the unit goes up with m: what acc holds keeps its bits)
                float* at = unit + lane_here();
                const float u0 = *at, u1 = fmaxf(u0 + down, UNIT_MIN);
                f = exp2f(u0 - u1 + down);
                *at = u1;
            }
            l *= al;
#pragma unroll
            for (int d = 0; d < 4; d++) acc[d] *= f;
            m = m1;
        }
        const float m0 = m == -INFINITY ? 0.f : m;
        float f = cq, ref = m0 - SHIFT, own = 1.f;
        if (!groups || far) {
            // A score is rounded as the maximum was before that is taken off: the
            // largest is then 0, and not what the product's rounding left.  The
            // weights without their values' factors are summed here.
            float lu = 0.f;
#pragma unroll
            for (int a = 0; a < 4; a++) {
                const float4v e = exponents(a);
#pragma unroll
                for (int b = 0; b < 4; b++) {
                    float p = s[4 * a + b] * cq;
                    asm("" : "+v"(p));  // (no fma)
                    p -= m0;
                    lu += __builtin_amdgcn_exp2f(p);
                    s[4 * a + b] = p + e[b];
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            l = fmaf(lu, (float)(1 << (int)SHIFT), l);
            if (far) {
                float* at = unit + lane_here();
                float u0 = *at, most = s[0];
#pragma unroll
                for (int i = 1; i < 16; i++) most = fmaxf(most, s[i]);
                most = lanes2_max(most) - u0;
                if (__builtin_amdgcn_ballot_w64(most > LAZY)) {
                    const float up = most > LAZY ? ceilf(most) : 0.f, f1 = exp2f(-up);
#pragma unroll
                    for (int d = 0; d < 4; d++) acc[d] *= f1;
                    u0 += up;
                    *at = u0;
                }
#pragma unroll
                for (int i = 0; i < 16; i++) s[i] -= u0;
            }
            f = 1.f;
            ref = -SHIFT;
            e0 = e1 = own = 0.f;
        }
#pragma unroll
        for (int u = 0; u < 2; u++) {
            // the weights in units of the group's factor, their sum in its own
            const float e = u ? e1 : e0, ru = ref - e;
            float x[8], lu = 0.f;
#pragma unroll
            for (int i = 0; i < 8; i++) {
                x[i] = __builtin_amdgcn_exp2f(fmaf(s[8 * u + i], f, -ru));
                lu += x[i];
            }
            l = fmaf(lu, own * __builtin_amdgcn_exp2f(-e), l);
            const Split8 w = split8<true>(x);
            const uint8_t* vp = sm + at * BUF + VH + (kb * 4 + u * 2 + h) * VGROUP + (n >> 4) * 1024 + (n & 15) * 16;
#pragma unroll
            for (int d = 0; d < 4; d++) {
                const half8 x1 = *(const half8*)(vp + d * 256);
                if constexpr (LO) {
                    const half8 y1 = *(const half8*)(vp + V_BYTES + d * 256);
                    acc[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(y1, w.hi, acc[d], 0, 0, 0);
                }
                acc[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(x1, w.lo, acc[d], 0, 0, 0);
                acc[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(x1, w.hi, acc[d], 0, 0, 0);
            }
        }
        __builtin_amdgcn_sched_group_barrier(SCHED_LDS, 2 * RD, 1);
#pragma unroll
        for (int j = 0; j < 6; j++) {
            __builtin_amdgcn_sched_group_barrier(SCHED_MFMA, MM, 1);
            __builtin_amdgcn_sched_group_barrier(SCHED_LDS, RD, 1);
        }
        __builtin_amdgcn_sched_group_barrier(SCHED_MFMA, 2 * MM, 1);
    };

    if (v_lo < v_hi) {
        stage_k(0);
        stage_v(0);
        if (v_lo + KT < v_hi) {
            load_k(v_lo + KT);
            load_v(v_lo + KT);
        }
    }
    // the tile after v0 into the other buffer, the one after that under way
    auto next = [&](int v0, int at) {
        if (v0 + KT < v_hi) {
            stage_k(at ^ 1);
            stage_v(at ^ 1);
            if (v0 + 2 * KT < v_hi) {
                load_k(v0 + 2 * KT);
                load_v(v0 + 2 * KT);
            }
        }
    };
    if (kb == 0) {
        for (int v0 = v_lo, at = 0; v0 < v_hi; v0 += KT, at ^= 1) {
            __syncthreads();  // this tile is whole, the other buffer free
            scores(v0, at);
            values(v0, at);
            next(v0, at);
        }
    } else {
        for (int v0 = v_lo, at = 0; v0 < v_hi; v0 += KT, at ^= 1) {
            __syncthreads();
            next(v0, at);
            scores(v0, at);
            values(v0, at);
        }
    }

    // The wave's state into LDS (row r = 8 a + 4 h + b of block d is dim 32 d + 16
    // (a % 2) + 8 h + 2 b + a / 2), the weights by 2^-(SHIFT + LAZY) so that sums of
    // large values stay finite.
    __syncthreads();
    float* so = (float*)sm + wave * 32 * OROW;
    float2* ml = (float2*)((float*)sm + 8 * 32 * OROW) + wave * 32;  // (m, l)
    const int lane1 = this_lane(), n1 = lane1 & 31, h1 = lane1 >> 5;
    {
        const float un = pow2(-(int)(SHIFT + LAZY)), uo = un * exp2f(unit[lane1]);
#pragma unroll
        for (int d = 0; d < 4; d++)
#pragma unroll
            for (int i = 0; i < 8; i++)
                *(float2*)(so + n1 * OROW + 32 * d + 16 * (i >> 2) + 8 * h1 + 2 * (i & 3)) =
                    make_float2(acc[d][i] * uo, acc[d][8 + i] * uo);
        l = lanes2_sum(l) * un;  // (m and l: the same in both lanes of a query)
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
    if (odd) {
        // The blocks left out: the wave walks its blocks again, from the first to
        // the last of them, and takes those it left key by key, in f32; lane (n, h)
        // has half the dims of its query.
        const Query w = query();
        const Sight see = sight_of(a, ks, w.row);
        const float* q = a.q + (size_t)w.row * a.ldq + (size_t)w.head * HD + 64 * h1;
        float* o = so + n1 * OROW + 64 * h1;
        const int v1 = __builtin_amdgcn_readfirstlane(odd_at[1]);
#pragma unroll 1
        for (int v0 = __builtin_amdgcn_readfirstlane(odd_at[0]); v0 <= v1; v0 += KT) {
            const int at_n = ks.pos(min(v0 + 32 * kb + n1, ks.nv - 1));
            const T* row = h1 ? kv.value(at_n) : kv.key(at_n);
            float mx = 0.f;  // the largest of key or value row n of the block
#pragma unroll 4
            for (int u = 0; u < HD; u += 8) {
                Raw<T, 8> r;
                r.load(row, u);
#pragma unroll
                for (int i = 0; i < 8; i++) mx = mag(mx, r.get(i));
            }
            const int e = exponent_class(__float_as_uint(mx));
            if (!__builtin_amdgcn_ballot_w64(h1 ? odd_value(e) : odd_key(e))) continue;
#pragma unroll 1
            for (int kn = 0; kn < 32; kn++) {
                const int v = v0 + 32 * kb + kn, pos = ks.pos(min(v, ks.nv - 1));
                const bool vis = sees(a, ks, see, pos) & (v < v_hi);
                if (!__builtin_amdgcn_ballot_w64(vis)) continue;
                const T *kp = kv.key(pos), *vp = kv.value(pos);
                float d = 0.f;
#pragma unroll 4
                for (int u = 0; u < 64; u++) d = fmaf(q[u], to_f32(kp[64 * h1 + u]), d);
                d = lanes2_sum(d) * c.qscale;
                asm("" : "+v"(d));  // (rounded before the maximum comes off: no fma)
                if (!vis) continue;
                const float m1 = fmaxf(m, d), ref = m1 == -INFINITY ? 0.f : m1, al = exp2f(m - ref), wt = ldexpf(exp2f(d - ref), -(int)LAZY);
#pragma unroll 4
                for (int u = 0; u < 64; u++) o[u] = o[u] * al + wt * to_f32(vp[64 * h1 + u]);
                l = l * al + wt;
                m = m1;
            }
        }
    }
    if (h1 == 0) ml[n1] = make_float2(m, l);
    __syncthreads();
    // The two blocks of every query meet; whole rows out, 32 lanes each.
    const int t1 = wave * 64 + lane1;
#pragma unroll 4
    for (int k = t1 >> 5; k < TQ; k += 16) {
        const int qi = q0 + k;
        if (qi >= nq) continue;
        const float* x = (const float*)sm + k * OROW + 4 * (t1 & 31);
        const float2* e = (const float2*)((const float*)sm + 8 * 32 * OROW) + k;
        const float2 e1 = e[0], e2 = e[TQ];
        const float mx = fmaxf(e1.x, e2.x);
        const float f1 = e1.x == -INFINITY ? 0.f : exp2f(e1.x - mx), f2 = e2.x == -INFINITY ? 0.f : exp2f(e2.x - mx);
        const float lt = e1.y * f1 + e2.y * f2, f = part ? 1.f : lt == 0.f ? 0.f : 1.f / lt;
        const float4v y = (*(const float4v*)x * f1 + *(const float4v*)(x + TQ * OROW) * f2) * f;
        const int row = row_of(c, qi), head = g * c.hpk + qi - row * c.hpk;
        if (part) {
            const size_t at = ((size_t)own * TQ + k) * nsplit + split;
            *(float4v*)(c.po + at * HD + 4 * (t1 & 31)) = y;
            if ((t1 & 31) == 0) {
                c.pm[at] = mx;
                c.pl[at] = lt;
            }
        } else {
            *(float4v*)(a.out + (size_t)row * a.ldo + (size_t)head * HD + 4 * (t1 & 31)) = y;
        }
    }
}

// The splits of one query by one wave: out = sum w_c o_c / sum w_c l_c,
// w_c = 2^(m_c - M); lane = dim pair.  The maxima, the sums and CB splits'
// outputs are requested together, so that up to CB splits take one memory
// round trip.  Bound by latency: 2.8 us for 16 queries of 16 splits, 4.8 for
// 1024 of 32.  grid (per, split items), block 64.
template <int CB>
__global__ __launch_bounds__(64) void k_attn_join(AttnCall c) {
    const cmf_attention_args& a = c.a;
    const int lane = threadIdx.x, ns = c.nsplit, item = c.whole + blockIdx.y;
    const int g = (uint32_t)item / (uint32_t)c.groups, qi = (item - g * c.groups) * c.per + blockIdx.x;
    if (qi >= a.b * c.hpk) return;
    const size_t at = (size_t)blockIdx.y * c.per + blockIdx.x;
    const float* pm = c.pm + at * ns;
    const float* pl = c.pl + at * ns;
    const float2* po = (const float2*)(c.po + at * ns * HD) + lane;
    float M = -INFINITY, L = 0.f;
    float2 o = make_float2(0.f, 0.f);
    for (int j0 = 0; j0 < ns; j0 += CB) {
        float2 x[CB];
#pragma unroll
        for (int u = 0; u < CB; u++) x[u] = po[(size_t)min(j0 + u, ns - 1) * 64];
        const int j = j0 + lane;
        const bool in = lane < CB && j < ns;
        const float mj = in ? pm[min(j, ns - 1)] : -INFINITY, lj = in ? pl[min(j, ns - 1)] : 0.f;
        const float M1 = fmaxf(M, wave_max(mj)), ref = M1 == -INFINITY ? 0.f : M1;
        const float al = exp2f(M - ref), w = exp2f(mj - ref);
        M = M1;
        L = L * al + wave_sum(w * lj);
        o.x *= al;
        o.y *= al;
#pragma unroll
        for (int u = 0; u < CB; u++) {
            const float wu = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(w), u));
            o.x = fmaf(wu, x[u].x, o.x);
            o.y = fmaf(wu, x[u].y, o.y);
        }
    }
    const float inv = L == 0.f ? 0.f : 1.0f / L;
    const int r = row_of(c, qi), h = g * c.hpk + qi - r * c.hpk;
    ((float2*)(a.out + (size_t)r * a.ldo + (size_t)h * HD))[lane] = make_float2(o.x * inv, o.y * inv);
}

// the most keys that a block of rows may have to read
long long keys_bound(const cmf_attention_args& a, int rows) {
    const long long cached = a.d_pos0 ? std::min(a.len_bound, a.slots) : a.pos0;
    long long n = cached + a.b;  // (a chunk's last block sees all of its rows)
    if (a.window) n = std::min(n, (long long)a.sinks + a.window + (a.d_mask || a.d_depth ? a.b : rows));
    return std::max(1ll, n);
}

struct Plan {
    bool tiles = false;  // k_attn_tiles, else k_attn_rows
    int groups = 1, per = 1, items = 1, whole = 1, nsplit = 1;  // as AttnCall's
    size_t bytes = 0;
    double cost = 0;  // in us, roughly: what the two kernels are chosen by
    size_t partial() const { return (size_t)(items - whole) * per * nsplit; }
};

// The items' blocks of `per` queries and the splits over their keys that fill
// `room` workgroups; where whole items may stay (whole), those that fill it
// whole times do, and the rest is split to fill it once more.
void lay_out(const cmf_attention_args& a, long long nq, long long nv, int per, int room, bool whole, long long least, Plan* p) {
    p->per = per;
    p->groups = (int)((nq + per - 1) / per);
    p->items = p->groups * a.nkv;
    p->whole = whole ? p->items / room * room : 0;
    const int rest = p->items - p->whole;
    long long ns = rest ? std::max(1ll, std::min<long long>(room / rest, (nv + least - 1) / least)) : 1;
    const size_t one = (size_t)rest * per * (HD + 2) * sizeof(float);
    while (ns > 1 && one * ns > OP_WS_MAX) ns--;
    p->nsplit = (int)ns;
    if (ns == 1) p->whole = p->items;
    p->bytes = ns > 1 ? one * ns : 0;
}

Plan plan_rows(const cmf_attention_args& a, long long nq) {
    Plan p;
    const long long nv = keys_bound(a, (int)std::min<long long>(a.b, RQ / (a.nh / a.nkv) + 2));
    const bool f32 = a.kv_dtype == CMF_DT_F32;
    // Workgroups a CU: one up to 256 keys each (220 keys f32: 20.5 us, with two
    // 21.7), then two (580 keys f32: 31.8 us with one, 28.4), three for long
    // 16-bit caches (5800 keys f16: 161 with one, 92 with two, 76; f32 of 4600 127
    // with two, 150).  Few keys are not split: a join is 3 us, and another launch
    // (8 rows of 16 heads, f32, 108 keys 8.1 us in one piece and 8.5 in two, 158
    // keys 9.9 and 8.7; f16, 258 keys 8.3 and 7.5, a call 8.6 and 10.0).
    const long long load = nv * ((nq + RQ - 1) / RQ * a.nkv);
    const int room = load <= 256 * 256 ? 256 : !f32 && load > 256 * 4096 ? 768 : 512;
    lay_out(a, nq, nv, RQ, room, false, nv <= (f32 ? 128 : 256) ? nv : 64, &p);
    const double wgs = (double)p.items * p.nsplit, tiles = std::ceil((double)nv / p.nsplit / 64);  // of a wave
    if (wgs <= 256) p.cost = (f32 ? 2.6 + 2.6 * tiles : 3.3 + 1.4 * tiles) + (p.nsplit > 1 ? 3.6 : 0);
    else p.cost = std::max(1.0, wgs / 512) * (f32 ? 5.5 + 3.1 * tiles : 5.5 + 1.5 * tiles) + (p.nsplit > 1 ? f32 ? 6.5 : 4 : 0);
    return p;
}

Plan plan_tiles(const cmf_attention_args& a, long long nq) {
    Plan p;
    p.tiles = true;
    const long long nv = keys_bound(a, (int)std::min<long long>(a.b, TQ / (a.nh / a.nkv) + 2));
    const bool f32 = a.kv_dtype == CMF_DT_F32;
    // One workgroup a CU; a split of 64 keys or more, two tiles stay together
    // (the join costs more than a tile), behind whole items 256 or more.
    const bool fills = (nq + TQ - 1) / TQ * a.nkv >= 256;
    lay_out(a, nq, nv, TQ, 256, true, fills ? 256 : nv <= 128 ? nv : 64, &p);
    const auto time = [&](double wgs, int ns) {
        const double tiles = std::ceil((double)nv / ns / KT);
        return std::ceil(wgs / 256) * (f32 ? 7.8 + 4.3 * tiles : 8.6 + 2.8 * tiles);
    };
    p.cost = time(p.whole, 1);
    if (p.nsplit > 1) p.cost += time((double)(p.items - p.whole) * p.nsplit, p.nsplit) + (f32 ? 3.4 : 4.4);
    return p;
}

// Up to 16 queries a kv head are one item of the rows.  Above, the kernel with
// the lower cost, in us, as fitted to 130 random sizes (mean error 8 %; the
// choice loses 0.4 % to the better one): the tiles take longer to begin, the
// rows longer a key and query.  us of the rows and the tiles:
// trees of 30 rows of 32 heads on 8 over 81 keys f32 8.3 16.5; 22 over 26238 f32
// 144 68; 39 of 16 on 4 over 49610 bf16 98 79; windows of 31, 146 rows bf16 5.0
// 16.4; of 107, 1241 rows f16 12.2 24.7; of 165, 985 rows f32 41 36.
Plan plan_of(const cmf_attention_args& a) {
    const long long nq = (long long)a.b * (a.nh / a.nkv);
    const Plan r = plan_rows(a, nq);
    if (nq <= RQ) return r;
    const Plan t = plan_tiles(a, nq);
    return r.cost <= t.cost && r.groups <= 65535 ? r : t;
}

// Allows kernel f its dynamic LDS (once a kernel).
int allow_lds(const void* f, int bytes) {
    static std::mutex mu;
    static std::set<const void*> done;
    std::lock_guard<std::mutex> lk(mu);
    if (!done.count(f)) {
        CMF_HIP(hipFuncSetAttribute(f, hipFuncAttributeMaxDynamicSharedMemorySize, bytes));
        done.insert(f);
    }
    return CMF_OK;
}

template <class T>
int launch_t(const AttnCall& c, const Plan& p, hipStream_t s) {
    if (!p.tiles) {
        const dim3 grid(c.nsplit, c.a.nkv, p.groups);
        hipLaunchKernelGGL(k_attn_rows<T>, grid, dim3(256), 0, s, c);
        return CMF_OK;
    }
    const void* f = (const void*)k_attn_tiles<T>;
    if (allow_lds(f, Tile<T>::LDS) != CMF_OK) return CMF_ERR;
    AttnCall arg = c;
    void* args[] = {&arg};
    CMF_HIP(hipLaunchKernel(f, dim3((unsigned)(p.whole + p.nsplit * (p.items - p.whole))), dim3(512), args, Tile<T>::LDS, s));
    return CMF_OK;
}

}  // namespace

size_t cache_attention_ws(const cmf_attention_args& a) { return plan_of(a).bytes; }

int launch_cache_attention(const cmf_attention_args& a, hipStream_t s) {
    const Plan p = plan_of(a);
    if (p.bytes > a.ws_bytes || (p.bytes && !a.ws)) return fail("attention: the workspace is too small (cmf_attention_workspace)");
    const uint32_t hpk = a.nh / a.nkv;
    AttnCall c{};
    c.a = a;
    c.hpk = (int)hpk;
    c.inv = (uint32_t)(((1ull << 32) + hpk - 1) / hpk);
    c.groups = p.groups;
    c.per = p.per;
    c.whole = p.whole;
    c.nsplit = p.nsplit;
    c.qscale = (a.scale == 0.f ? 0.08838834764831845f : a.scale) * LOG2E;
    if (p.nsplit > 1) {
        c.po = (float*)a.ws;
        c.pm = c.po + p.partial() * HD;
        c.pl = c.pm + p.partial();
    }
    const int rc = a.kv_dtype == CMF_DT_F32   ? launch_t<float>(c, p, s)
                   : a.kv_dtype == CMF_DT_F16 ? launch_t<_Float16>(c, p, s)
                                              : launch_t<bf16_t>(c, p, s);
    if (rc != CMF_OK) return rc;
    const dim3 rows(p.per, p.items - p.whole);
    if (p.nsplit > 16) hipLaunchKernelGGL(k_attn_join<32>, rows, dim3(64), 0, s, c);
    else if (p.nsplit > 1) hipLaunchKernelGGL(k_attn_join<16>, rows, dim3(64), 0, s, c);
    return CMF_OK;
}

static int check_attention(const cmf_attention_args* p) {
    if (!p) return fail("attention: null argument");
    const auto& a = *p;
    if (a.b < 1 || a.nh < 1 || a.nkv < 1 || a.nh % a.nkv) return fail("attention: b, nh, nkv of at least 1, nh a multiple of nkv");
    if (a.b > (1 << 19) || a.nh > 4096 || a.nh / a.nkv > 64)
        return fail("attention: at most 2^19 rows, 4096 heads, 64 query heads per kv head");
    if (!kv_dtype_ok(a.kv_dtype)) return fail("attention: kv_dtype must be f32, f16 or bf16");
    if (a.pos0 < 0 || a.slots < 0 || a.window < 0 || a.sinks < 0) return fail("attention: pos0, slots, window and sinks of at least 0");
    if (a.slots > (1 << 30) || a.window > (1 << 30) || a.sinks > (1 << 30)) return fail("attention: at most 2^30 positions");
    if (!(a.scale == a.scale) || a.scale - a.scale != 0.f) return fail("attention: scale must be finite");
    if (a.d_mask && a.b > CMF_TREE_MAX) return fail("attention: a tree of at most 64 rows");
    if (a.d_depth && !a.d_mask) return fail("attention: d_depth goes with d_mask");
    if (a.d_mask && a.window && !a.d_depth) return fail("attention: a tree under a window needs d_depth");
    if (!a.k_new != !a.v_new) return fail("attention: k_new and v_new go together");
    if (a.ldq < a.nh * HD || a.ldq % 4 || a.ldo < a.nh * HD || a.ldo % 4) return fail("attention: ldq and ldo must hold the heads, multiples of 4");
    if (a.row_stride < HD || a.row_stride % 8 || a.head_stride < 0 || a.head_stride % 8 ||
        (a.k_new && (a.new_row_stride < HD || a.new_row_stride % 8 || a.new_head_stride < 0 || a.new_head_stride % 8)))
        return fail("attention: strides must be multiples of 8 elements, rows of 128");
    if (a.row_stride > MAX_ROW_STRIDE || (a.k_new && a.new_row_stride > MAX_ROW_STRIDE))
        return fail("attention: row strides of at most 2^22 elements");
    const long long need = (long long)a.pos0 + (a.k_new ? 0 : a.b);
    if (!a.d_pos0 && need > a.slots) return fail("attention: positions past the cache's slots");
    if (a.d_pos0 && (a.len_bound < 0 || (long long)a.len_bound + (a.k_new ? 0 : a.b) > a.slots))
        return fail("attention: len_bound past the cache's slots");
    return CMF_OK;
}

}  // namespace cmf

using namespace cmf;

extern "C" {

size_t cmf_attention_workspace(const cmf_attention_args* a) {
    if (check_attention(a) != CMF_OK) return 0;
    return cache_attention_ws(*a);
}

int cmf_attention_dev(const cmf_attention_args* p) {
    if (check_attention(p) != CMF_OK) return CMF_ERR;
    const auto& a = *p;
    if (!a.q || !a.out || ((!a.k || !a.v) && (a.slots > 0 || !a.k_new))) return fail("attention: null q, out, k or v");
    for (const void* x : {(const void*)a.q, (const void*)a.out, a.k, a.v, a.k_new, a.v_new, (const void*)a.ws})
        if (!aligned16(x)) return fail("attention: 16-byte aligned tensors");
    // (a block of rows may write before another has read)
    if (a.out == a.q && a.ldo != a.ldq) return fail("attention: out may be q with the same row stride (ldo = ldq)");
    OpScope sc;
    if (sc.enter(a.stream, "attention") != CMF_OK) return CMF_ERR;
    if (launch_cache_attention(a, sc.s) != CMF_OK) return CMF_ERR;
    CMF_HIP(hipGetLastError());
    return CMF_OK;
}

}  // extern "C"
