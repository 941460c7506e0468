// Log probabilities of given tokens, the entropy of their distributions and
// the top alternatives of rows of logits (cmf_logprobs_dev).
//
// One pass over the logits.  A workgroup of four waves takes a slice of a row
// in rounds of 4096 logits, 16 a lane, the next round's loads in flight while
// one is worked on.  Every lane keeps a softmax state of its own (running
// maximum, sum of weights, sum of weighted differences), every wave the 64
// largest of its logits, one a lane, in order: a round's logits are compared
// with the k-th of them and only the few that pass wait in LDS to be sorted and
// joined, 64 at a time.  In the first round the k-th of the lanes' own maxima
// bounds them.
// The waves and then the slices of a row meet in a fixed order.
// Bound by the logits' bytes for many rows (400 of 151936, f32, 5 alternatives:
// 51 us, 4.8 TB/s, and 4.8 for the join), by latency for few (5 rows, 8
// alternatives: 6.5 and 5.0 us), by the lists for many alternatives (600 rows of
// 50000: none 26 us in all, 5 alternatives 36, 20 44, 64 62).
#include <math.h>

#include <algorithm>
#include <string>

#include "cache_ops.h"
#include "runtime.h"
#include "wave.h"

namespace cmf {

namespace {

constexpr int LT = 256;            // threads of a workgroup
constexpr int LV = 16;             // logits a lane holds per round
constexpr int LROUND = LT * LV;
constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.6931471805599453f;

// A logit and its id as one number that orders as the lists do: the larger
// value first, then the lower id; NaN below -inf.  The keys of a row differ;
// 0 is no logit's.
__device__ __forceinline__ uint64_t key_of(float x, int id) {
    uint32_t u = __float_as_uint(x == 0.f ? 0.f : x);  // (-0 and 0 are equal)
    u = u & 0x80000000u ? ~u : u | 0x80000000u;
    if (x != x) u = 0;
    return (uint64_t)u << 32 | (uint32_t)~id;
}
__device__ __forceinline__ int key_id(uint64_t k) { return (int)~(uint32_t)k; }
__device__ __forceinline__ float key_val(uint64_t k) {  // (what is below -inf's key: a NaN)
    const uint32_t u = (uint32_t)(k >> 32);
    return __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u);
}
// Lanes' values from the lane ^ O or the lane 63 - lane, without a trip through
// LDS.
template <int CTRL>
__device__ __forceinline__ uint32_t lanes_dpp(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp((int)v, (int)v, CTRL, 0xf, 0xf, false);
}
template <int O>
__device__ __forceinline__ uint32_t lane_xor(uint32_t v, int lane) {
    if constexpr (O == 1) return lanes_dpp<0xb1>(v);                    // quad_perm [1,0,3,2]
    else if constexpr (O == 2) return lanes_dpp<0x4e>(v);               // quad_perm [2,3,0,1]
    else if constexpr (O == 4) return lanes_dpp<0x1b>(lanes_dpp<0x141>(v));  // half-row and quad mirrored
    else if constexpr (O == 8) return lanes_dpp<0x128>(v);              // row_ror 8
    else {
        auto s = O == 16 ? __builtin_amdgcn_permlane16_swap(v, v, false, false)
                         : __builtin_amdgcn_permlane32_swap(v, v, false, false);
        return lane & O ? s[0] : s[1];
    }
}
__device__ __forceinline__ uint32_t lane_mirror(uint32_t v, int lane) {
    return lane_xor<32>(lane_xor<16>(lanes_dpp<0x140>(v), lane), lane);  // (rows mirrored first)
}
__device__ __forceinline__ uint64_t lane64(uint64_t v, int src) {  // src wave-uniform
    return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), src) << 32 |
           (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, src);
}

// one compare-exchange step of a descending bitonic network
template <int O>
__device__ __forceinline__ uint64_t exchange(uint64_t v, int lane, bool keep_max) {
    const uint64_t w = (uint64_t)lane_xor<O>((uint32_t)(v >> 32), lane) << 32 | lane_xor<O>((uint32_t)v, lane);
    return (v > w) == keep_max ? v : w;
}
// blocks of 2 O lanes hold bitonic sequences: sorted, descending in the even
// blocks, ascending in the odd ones
template <int O>
__device__ __forceinline__ uint64_t merge_step(uint64_t v, int lane, bool down) {
    v = exchange<O>(v, lane, !(lane & O) == down);
    if constexpr (O > 1) v = merge_step<O / 2>(v, lane, down);
    return v;
}
__device__ __forceinline__ uint64_t bitonic_merge(uint64_t v, int lane) { return merge_step<32>(v, lane, true); }
// Lanes hold sorted lists of n lanes (a power of two), the even ones descending
// and the odd ones ascending, zeros from lane `used` on: the wave sorted,
// descending.
__device__ __forceinline__ uint64_t merge_lists(uint64_t v, int n, int used, int lane) {
    if (n <= 1 && used > 1) v = merge_step<1>(v, lane, !(lane & 2));
    if (n <= 2 && used > 2) v = merge_step<2>(v, lane, !(lane & 4));
    if (n <= 4 && used > 4) v = merge_step<4>(v, lane, !(lane & 8));
    if (n <= 8 && used > 8) v = merge_step<8>(v, lane, !(lane & 16));
    if (n <= 16 && used > 16) v = merge_step<16>(v, lane, !(lane & 32));
    if (n <= 32 && used > 32) v = merge_step<32>(v, lane, true);
    return v;
}
// the 64 largest of two descending lists
__device__ __forceinline__ uint64_t top_join(uint64_t a, uint64_t b, int lane) {
    const uint64_t r = (uint64_t)lane_mirror((uint32_t)(b >> 32), lane) << 32 | lane_mirror((uint32_t)b, lane);
    return bitonic_merge(a > r ? a : r, lane);
}
// Sums relative to the maximum m: z = sum e^(x - m), h = sum e^(x - m) (x - m)
// log2(e); nothing yet: m = -inf, z = h = 0.
struct Soft {
    float m, z, h;
};
__device__ __forceinline__ Soft soft_join(const Soft& a, const Soft& b) {
    const float m = fmaxf(a.m, b.m), ref = m == -INFINITY ? 0.f : m;
    // (a side with nothing yet: e^-inf = 0, and its h and z are 0)
    const float da = fmaxf((a.m - ref) * LOG2E, -1000.f), db = fmaxf((b.m - ref) * LOG2E, -1000.f);
    const float fa = exp2f(da), fb = exp2f(db);
    return Soft{m, a.z * fa + b.z * fb, (a.h + a.z * da) * fa + (b.h + b.z * db) * fb};
}
__device__ __forceinline__ Soft soft_wave(Soft s) {
    const auto add = [](float a, float b) { return a + b; };
    const float m = wave_reduce_f32(s.m, -INFINITY, [](float a, float b) { return fmaxf(a, b); });
    const float d = fmaxf((s.m - (m == -INFINITY ? 0.f : m)) * LOG2E, -1000.f), f = exp2f(d);
    return Soft{m, wave_reduce_f32(s.z * f, 0.f, add), wave_reduce_f32((s.h + s.z * d) * f, 0.f, add)};
}

struct LpCall {
    cmf_logprobs_args a;
    int nslice, per;  // slices of a row, logits of a slice (whole rounds)
    float* soft;      // [rows][nslice][4]
    uint64_t* top;    // [rows][nslice][top_k]
};

constexpr int LQ = 4 * 64 + 64;  // a wave's queue: what four logits a lane may add to less than 64
struct LpShared {
    Soft soft[LT / 64];
    uint64_t top[LT / 64][64];
};

// The largest of `lists` sorted lists of k keys: list j's key e is at
// src[j * ld + e].  As many lists as fit the wave's lanes are merged at a time,
// starting from list `from` groups in and `step` groups on.
__device__ __forceinline__ uint64_t top_lists(const uint64_t* src, int ld, int lists, int k, int from, int step, int lane) {
    const int n = k <= 1 ? 1 : 1 << (32 - __builtin_clz(k - 1)), each = 64 / n;
    const int j = lane / n, e = j & 1 ? n - 1 - (lane & (n - 1)) : lane & (n - 1);
    auto load = [&](int g) { return g * each + j < lists && e < k ? src[(size_t)(g * each + j) * ld + e] : 0; };
    const int groups = (lists + each - 1) / each;
    uint64_t best = 0, next = from < groups ? load(from) : 0;
    for (int g = from; g < groups; g += step) {
        uint64_t v = next;
        if (g + step < groups) next = load(g + step);
        v = merge_lists(v, n, min(lists - g * each, each) * n, lane);
        best = g == from ? v : top_join(best, v, lane);
    }
    return best;
}

// the row's results from its state and list (wave 0, all lanes hold s)
__device__ __forceinline__ void lp_write(const cmf_logprobs_args& a, int row, const Soft& s, uint64_t best, float xt,
                                         int lane) {
    const float lz = log2f(s.z) * LN2;
    if (lane == 0) {
        if (a.logprob) a.logprob[row] = (xt - s.m) - lz;
        if (a.entropy) a.entropy[row] = lz - s.h / s.z * LN2;
    }
    if (lane < a.top_k) {
        if (a.top_ids) a.top_ids[(size_t)row * a.top_k + lane] = key_id(best);
        if (a.top_lp) a.top_lp[(size_t)row * a.top_k + lane] = (key_val(best) - s.m) - lz;
    }
}

template <class T>
__device__ __forceinline__ float lp_target(const cmf_logprobs_args& a, int row) {
    const int t = a.target ? a.target[row] : -1;
    return t >= 0 && t < a.V ? to_f32(((const T*)a.logits)[(size_t)row * a.ld + t]) : NAN;
}

// grid (nslice, rows), block 256.  TOP: with a list.
template <class T, bool TOP>
__global__ __launch_bounds__(LT) void k_logprobs(LpCall c) {
    const cmf_logprobs_args& a = c.a;
    constexpr int VE = 16 / sizeof(T), NV = LV / VE;  // logits of a load, loads of a round
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, slice = blockIdx.x, row = blockIdx.y;
    const T* x = (const T*)a.logits + (size_t)row * a.ld;
    // ids are counted from the 16-byte boundary at or before the row's start
    const int off = (int)(((uintptr_t)x & 15) / sizeof(T));
    const long long lo = (long long)slice * c.per, hi = min(lo + c.per, (long long)a.V + off);
    __shared__ LpShared sh;
    const float xt = lp_target<T>(a, row);
    Soft s{-INFINITY, 0.f, 0.f};
    // The wave's list, the key that a logit has to pass, and the keys that did
    // since the list was last brought up to date.
    uint64_t best = 0, bound = 0;
    float bv = NAN;
    int waiting = 0;
    bool listed = false;
    __shared__ uint64_t queue[TOP ? LT / 64 : 1][TOP ? LQ : 1];
    auto take = [&]() {  // the last 64 of them into the list
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        const int from = max(waiting - 64, 0);
        const uint64_t key = lane < waiting - from ? queue[wave][from + lane] : 0;
        const uint64_t v = merge_lists(key, 1, waiting - from, lane);
        best = listed ? top_join(best, v, lane) : v;
        listed = true;
        waiting = from;
        const uint64_t last = lane64(best, a.top_k - 1);
        bound = last > bound ? last : bound;
        bv = key_val(bound);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    };

    auto load = [&](long long r0, float (&v)[LV]) {
#pragma unroll
        for (int u = 0; u < NV; u++) {
            const long long p = r0 + (long long)(u * LT + t) * VE;  // number of the load's first logit
            const long long id = p - off;
            if (p < hi && id >= 0 && id + VE <= a.V) {
                union {
                    uint4 q;
                    T e[VE];
                } w;
                w.q = *(const uint4*)(x + id);
#pragma unroll
                for (int i = 0; i < VE; i++) v[u * VE + i] = to_f32(w.e[i]);
            } else {
#pragma unroll
                for (int i = 0; i < VE; i++)
                    v[u * VE + i] = p < hi && id + i >= 0 && id + i < a.V ? to_f32(x[id + i]) : -INFINITY;
            }
        }
    };
    auto id_of = [&](long long r0, int i) { return (int)(r0 + (long long)(i / VE * LT + t) * VE + i % VE - off); };

    float v[LV], nx[LV];
    load(lo, v);
    for (long long r0 = lo; r0 < hi; r0 += LROUND) {
        if (r0 + LROUND < hi) load(r0 + LROUND, nx);
        float mx = s.m;
#pragma unroll
        for (int i = 0; i < LV; i++) mx = fmaxf(mx, v[i]);
        const float ref = mx == -INFINITY ? 0.f : mx;
        // (weights under 2^-1000 are 0 in f32: the bound only keeps 0 * inf out)
        const float dm = fmaxf((s.m - ref) * LOG2E, -1000.f), f = exp2f(dm);
        s.h = (s.h + s.z * dm) * f;
        s.z *= f;
        s.m = mx;
#pragma unroll
        for (int i = 0; i < LV; i++) {
            const float d = (v[i] - ref) * LOG2E, p = __builtin_amdgcn_exp2f(d);  // (what is under 2^-126 adds nothing to 1)
            s.z += p;
            s.h = fmaf(p, fmaxf(d, -1000.f), s.h);
        }
        if constexpr (TOP) {
            if (r0 == lo) {
                // top_k lanes' maxima are at or above this: the upper half of its bits, one by one
                // (a lane whose maximum is -inf may hold no logit, or NaN: not counted)
                const uint32_t u = mx > -INFINITY ? (uint32_t)(key_of(mx, 0) >> 32) : 0;
                uint32_t b = 0;
#pragma unroll
                for (int bit = 31; bit >= 16; bit--) {
                    const uint32_t up = b | 1u << bit;
                    if (__builtin_popcountll(__builtin_amdgcn_ballot_w64(u >= up)) >= a.top_k) b = up;
                }
                bound = (uint64_t)b << 32;
                bv = key_val(bound);
            }
#pragma unroll
            for (int i = 0; i < LV; i++) {
                // (the bound's own value may tie: the keys decide; NaN pass)
                if (__builtin_amdgcn_ballot_w64(!(v[i] < bv))) {
                    const int id = id_of(r0, i);
                    const bool is = id >= 0 && id < a.V && r0 + (long long)(i / VE * LT + t) * VE < hi;
                    const uint64_t key = is ? key_of(v[i], id) : 0, pass = __builtin_amdgcn_ballot_w64(key > bound);
                    if (key > bound)
                        queue[wave][waiting + __builtin_amdgcn_mbcnt_hi((uint32_t)(pass >> 32),
                                                                        __builtin_amdgcn_mbcnt_lo((uint32_t)pass, 0))] = key;
                    waiting += __builtin_popcountll(pass);
                }
                if (i % 4 == 3)
                    while (waiting >= 64) take();
            }
        }
#pragma unroll
        for (int i = 0; i < LV; i++) v[i] = nx[i];
    }

    if (TOP && waiting) take();
    s = soft_wave(s);
    if (lane == 0) sh.soft[wave] = s;
    if (TOP) sh.top[wave][lane] = best;
    __syncthreads();
    if (wave) return;
    s = sh.soft[0];
#pragma unroll
    for (int w = 1; w < LT / 64; w++) s = soft_join(s, sh.soft[w]);
    if constexpr (TOP) best = top_lists(sh.top[0], 64, LT / 64, a.top_k, 0, 1, lane);
    if (c.nslice == 1) {
        lp_write(a, row, s, best, xt, lane);
        return;
    }
    const size_t at = (size_t)row * c.nslice + slice;
    if (lane == 0) *(float4*)(c.soft + at * 4) = make_float4(s.m, s.z, s.h, 0.f);
    if (TOP && lane < a.top_k) c.top[at * a.top_k + lane] = best;
}

// The slices of a row: every wave joins a quarter of them, then the waves
// meet.  Bound by latency (the slices' states, then their lists by ten to twenty
// exchanges of a wave).  grid (rows), block 256.
template <class T, bool TOP>
__global__ __launch_bounds__(LT) void k_logprobs_join(LpCall c) {
    const cmf_logprobs_args& a = c.a;
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, row = blockIdx.x;
    __shared__ LpShared sh;
    const float xt = lp_target<T>(a, row);
    const size_t at = (size_t)row * c.nslice;
    Soft s{-INFINITY, 0.f, 0.f};
    for (int j = t; j < c.nslice; j += LT) {
        const float4 q = *(const float4*)(c.soft + (at + j) * 4);
        s = soft_join(s, Soft{q.x, q.y, q.z});
    }
    s = soft_wave(s);
    if (lane == 0) sh.soft[wave] = s;
    uint64_t best = 0;
    if constexpr (TOP) {
        best = top_lists(c.top + at * a.top_k, a.top_k, c.nslice, a.top_k, wave, LT / 64, lane);
        sh.top[wave][lane] = best;
    }
    __syncthreads();
    if (wave) return;
    s = sh.soft[0];
#pragma unroll
    for (int w = 1; w < LT / 64; w++) s = soft_join(s, sh.soft[w]);
    if constexpr (TOP) best = top_lists(sh.top[0], 64, LT / 64, a.top_k, 0, 1, lane);
    lp_write(a, row, s, best, xt, lane);
}

struct LpPlan {
    int nslice, per;
    size_t bytes;
};
// Slices of whole rounds, about 2048 workgroups in all: one round each for a
// few rows (latency), a row each for many (no second launch).
LpPlan plan_of(int rows, int V, int top_k) {
    const long long rounds = ((long long)V + 7 + LROUND - 1) / LROUND;
    long long ns = std::max(1ll, std::min(rounds, 2048ll / rows));
    const size_t each = 16 + 8 * (size_t)top_k;
    while (ns > 1 && (size_t)rows * ns * each > OP_WS_MAX) ns--;
    const long long per = (rounds + ns - 1) / ns;
    ns = (rounds + per - 1) / per;
    return LpPlan{(int)ns, (int)(per * LROUND), ns > 1 ? (size_t)rows * ns * each : 0};
}

template <class T>
void launch_t(const LpCall& c, hipStream_t s) {
    const dim3 grid(c.nslice, c.a.rows);
    if (c.a.top_k) hipLaunchKernelGGL((k_logprobs<T, true>), grid, dim3(LT), 0, s, c);
    else hipLaunchKernelGGL((k_logprobs<T, false>), grid, dim3(LT), 0, s, c);
    if (c.nslice == 1) return;
    if (c.a.top_k) hipLaunchKernelGGL((k_logprobs_join<T, true>), dim3(c.a.rows), dim3(LT), 0, s, c);
    else hipLaunchKernelGGL((k_logprobs_join<T, false>), dim3(c.a.rows), dim3(LT), 0, s, c);
}

int check_logprobs(const cmf_logprobs_args* p) {
    if (!p) return fail("logprobs: null argument");
    const auto& a = *p;
    if (a.rows < 1 || a.rows > 65535 || a.V < 1 || a.V > (1 << 30)) return fail("logprobs: 1 to 65535 rows of 1 to 2^30 logits");
    if (a.ld < a.V) return fail("logprobs: ld must hold a row");
    if (!kv_dtype_ok(a.dtype)) return fail("logprobs: dtype must be f32, f16 or bf16");
    if (a.top_k < 0 || a.top_k > CMF_TOP_MAX || a.top_k > a.V) return fail("logprobs: top_k of 0 to 64, at most V");
    return CMF_OK;
}

}  // namespace

size_t logprobs_ws(int rows, int V, int top_k) { return plan_of(rows, V, top_k).bytes; }

void launch_logprobs(const cmf_logprobs_args& a, hipStream_t s) {
    const LpPlan p = plan_of(a.rows, a.V, a.top_k);
    LpCall c{a, p.nslice, p.per, (float*)a.ws, (uint64_t*)((char*)a.ws + (size_t)a.rows * p.nslice * 16)};
    if (a.dtype == CMF_DT_F32) launch_t<float>(c, s);
    else if (a.dtype == CMF_DT_F16) launch_t<_Float16>(c, s);
    else launch_t<bf16_t>(c, s);
}

}  // namespace cmf

using namespace cmf;

extern "C" {

size_t cmf_logprobs_workspace(const cmf_logprobs_args* a) {
    if (check_logprobs(a) != CMF_OK) return 0;
    return logprobs_ws(a->rows, a->V, a->top_k);
}

int cmf_logprobs_dev(const cmf_logprobs_args* p) {
    if (check_logprobs(p) != CMF_OK) return CMF_ERR;
    const auto& a = *p;
    if (!a.logits) return fail("logprobs: null logits");
    if (!a.target != !a.logprob) return fail("logprobs: target and logprob go together");
    if ((a.top_ids || a.top_lp) && !a.top_k) return fail("logprobs: top lists need top_k");
    if (a.top_k && !a.top_ids && !a.top_lp) return fail("logprobs: top_k needs a top list");
    const size_t es = a.dtype == CMF_DT_F32 ? 4 : 2;
    if ((uintptr_t)a.logits % es || !aligned16(a.ws)) return fail("logprobs: misaligned logits or workspace");
    const size_t need = logprobs_ws(a.rows, a.V, a.top_k);
    if (need > a.ws_bytes || (need && !a.ws)) return fail("logprobs: the workspace is too small (cmf_logprobs_workspace)");
    OpScope sc;
    if (sc.enter(a.stream, "logprobs") != CMF_OK) return CMF_ERR;
    launch_logprobs(a, sc.s);
    CMF_HIP(hipGetLastError());
    return CMF_OK;
}

}  // extern "C"
