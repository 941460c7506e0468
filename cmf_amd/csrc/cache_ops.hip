// Operators on rows of a cache: the head norms with the position rotation,
// stored into a cache (cmf_qk_rope_dev), copies of rows between caches
// (cmf_kv_copy_dev), and the masks of a token tree (cmf_tree_masks).
#include <string>

#include "cache_ops.h"
#include "runtime.h"
#include "wave.h"

namespace cmf {

int OpScope::enter(void* stream, const char* who) {
    int cur = -1;
    if (hipGetDevice(&cur) != hipSuccess) {
        (void)hipGetLastError();
        cur = -1;
    }
    // (a thread's first call makes the library's device current itself)
    const int rc = ensure_init();
    if (cur >= 0 && cur != device()) back = cur;
    if (rc != CMF_OK) return CMF_ERR;
    if (back >= 0) CMF_HIP(hipSetDevice(device()));
    if (!stream) {
        s = cmf::stream();
    } else if (stream == CMF_STREAM_NULL) {
        s = nullptr;
    } else {
        s = (hipStream_t)stream;
        hipDevice_t d = -1;
        CMF_HIP(hipStreamGetDevice(s, &d));
        if (d != device()) return fail(std::string(who) + ": the stream is not of the library's device");
    }
    return CMF_OK;
}

OpScope::~OpScope() {
    if (back >= 0) (void)hipSetDevice(back);
}

namespace {

// One head row by 16 lanes, lane l holding dims 4 l .. 4 l + 3 and the same 64
// up (the rotation pairs), so that every access is 16 bytes a lane and a wave
// serves four heads.  The mean of squares is summed in f64 as the decode
// layers do (norm_rope); its 16 partials meet by four xor shuffles.  Bound by
// memory: a head is read once and written once (2001 rows of 32 + 16 heads into
// a bf16 cache, 91 MB: 16.3 us, 5.6 TB/s, part of it from and to the caches); one
// row by latency, 2.8 us.
// grid (ceil(b (nh + 2 nkv) / 16)), block 256: 16 heads a workgroup.
template <class T>
__global__ __launch_bounds__(256) void k_qk_rope(cmf_qk_rope_args a) {
    const int hpr = a.nh + 2 * a.nkv;
    const long long item = (long long)blockIdx.x * 16 + (threadIdx.x >> 4);
    const int l = threadIdx.x & 15;
    if (item >= (long long)a.b * hpr) return;  // (whole groups of 16 lanes: the shuffles below stay inside one)
    const int i = (int)(item / hpr), h = (int)(item - (long long)i * hpr);
    const int base = a.pos0 + (a.d_pos0 ? *a.d_pos0 : 0);
    const int pos = base + (a.d_depth ? a.d_depth[i] : i);
    const bool is_q = h < a.nh, is_v = h >= a.nh + a.nkv;
    if (is_q ? !a.q_out : !a.k) return;
    if (pos < 0 || pos >= a.max_pos) return;
    const float* x = a.qkv + (size_t)i * a.ldq + (size_t)h * CACHE_HD;
    float4 lo = ((const float4*)x)[l], hi = ((const float4*)(x + 64))[l];
    if (!is_v) {
        const float* w = is_q ? a.q_norm : a.k_norm;
        const float4* r = (const float4*)(a.rope + ((size_t)pos * 64 + 4 * l) * 2);
        const float4 c0 = r[0], c1 = r[1];
        if (w) {
            const float4 w0 = ((const float4*)w)[l], w1 = ((const float4*)(w + 64))[l];
            double ss = (double)lo.x * lo.x + (double)lo.y * lo.y + (double)lo.z * lo.z + (double)lo.w * lo.w +
                        (double)hi.x * hi.x + (double)hi.y * hi.y + (double)hi.z * hi.z + (double)hi.w * hi.w;
#pragma unroll
            for (int o = 1; o < 16; o <<= 1) ss += __shfl_xor(ss, o);
            const float inv = (float)(1.0 / sqrt(ss / 128.0 + a.eps));
            lo = make_float4(lo.x * inv * w0.x, lo.y * inv * w0.y, lo.z * inv * w0.z, lo.w * inv * w0.w);
            hi = make_float4(hi.x * inv * w1.x, hi.y * inv * w1.y, hi.z * inv * w1.z, hi.w * inv * w1.w);
        }
        const float4 p = lo, q = hi;
        lo = make_float4(p.x * c0.x - q.x * c0.y, p.y * c0.z - q.y * c0.w, p.z * c1.x - q.z * c1.y,
                         p.w * c1.z - q.w * c1.w);
        hi = make_float4(p.x * c0.y + q.x * c0.x, p.y * c0.w + q.y * c0.z, p.z * c1.y + q.z * c1.x,
                         p.w * c1.w + q.w * c1.z);
    }
    if (is_q) {
        float* o = a.q_out + (size_t)i * a.ldo + (size_t)h * CACHE_HD;
        ((float4*)o)[l] = lo;
        ((float4*)(o + 64))[l] = hi;
        return;
    }
    const int slot = a.at_pos ? base + i : i;
    if (slot < 0 || slot >= a.slots) return;
    const int g = is_v ? h - a.nh - a.nkv : h - a.nh;
    T* o = (T*)(is_v ? a.v : a.k) + (size_t)g * a.head_stride + (size_t)slot * a.row_stride;
    if constexpr (sizeof(T) == 4) {
        ((float4*)o)[l] = lo;
        ((float4*)(o + 64))[l] = hi;
    } else {
        union {
            uint2 v;
            T t[4];
        } u0, u1;
        u0.t[0] = from_f32<T>(lo.x), u0.t[1] = from_f32<T>(lo.y), u0.t[2] = from_f32<T>(lo.z), u0.t[3] = from_f32<T>(lo.w);
        u1.t[0] = from_f32<T>(hi.x), u1.t[1] = from_f32<T>(hi.y), u1.t[2] = from_f32<T>(hi.z), u1.t[3] = from_f32<T>(hi.w);
        ((uint2*)o)[l] = u0.v;
        ((uint2*)(o + 64))[l] = u1.v;
    }
}

// Rows of 16 C bytes (C = 32: f32, 16: 16-bit caches) by 16-byte pieces, U
// pieces a thread, all loads before the first store.  Bound by memory: 4001
// rows of 16 caches of 8 heads in f32, 524 MB read and written, 107 us (4.9 TB/s);
// 5 rows of 56 caches by latency, 2.6 us.
// grid (ceil(n C / (256 U)), nbuf * nkv), block 256.
template <int C, int U>
__global__ __launch_bounds__(256) void k_kv_copy(cmf_kv_copy_args a) {
    const int j = blockIdx.y / a.nkv, g = blockIdx.y - j * a.nkv;
    const int n = a.d_n ? min(*a.d_n, a.n) : a.n;
    const int base = a.pos0 + (a.d_pos0 ? *a.d_pos0 : 0);
    constexpr int ES = C == 32 ? 4 : 2;
    const char* src = (const char*)a.d_src[j] + (size_t)g * a.src_head_stride * ES;
    char* dst = (char*)a.d_dst[j] + (size_t)g * a.dst_head_stride * ES;
    uint4 v[U];
    char* to[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
        const long long p = ((long long)blockIdx.x * U + u) * 256 + threadIdx.x;
        const int i = (int)(p / C), c = (int)(p % C);
        to[u] = nullptr;
        if (i < n) {
            const int r = a.d_idx ? a.d_idx[i] : i;
            const long long d = (long long)base + i;
            if (r >= 0 && r < a.src_slots && d >= 0 && d < a.dst_slots) {
                v[u] = *(const uint4*)(src + (size_t)r * a.src_row_stride * ES + c * 16);
                to[u] = dst + (size_t)d * a.dst_row_stride * ES + c * 16;
            }
        }
    }
#pragma unroll
    for (int u = 0; u < U; u++)
        if (to[u]) *(uint4*)to[u] = v[u];
}

}  // namespace

void launch_qk_rope(const cmf_qk_rope_args& a, hipStream_t s) {
    const long long items = (long long)a.b * (a.nh + 2 * a.nkv);
    const dim3 grid((unsigned)((items + 15) / 16));
    if (a.kv_dtype == CMF_DT_F32) hipLaunchKernelGGL(k_qk_rope<float>, grid, dim3(256), 0, s, a);
    else if (a.kv_dtype == CMF_DT_F16) hipLaunchKernelGGL(k_qk_rope<_Float16>, grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL(k_qk_rope<bf16_t>, grid, dim3(256), 0, s, a);
}

void launch_kv_copy(const cmf_kv_copy_args& a, hipStream_t s) {
    const int C = a.kv_dtype == CMF_DT_F32 ? 32 : 16;
    const long long pieces = (long long)a.n * C;
    const unsigned y = (unsigned)(a.nbuf * a.nkv);
    if (pieces <= 256) {
        if (C == 32) hipLaunchKernelGGL((k_kv_copy<32, 1>), dim3(1, y), dim3(256), 0, s, a);
        else hipLaunchKernelGGL((k_kv_copy<16, 1>), dim3(1, y), dim3(256), 0, s, a);
        return;
    }
    const dim3 grid((unsigned)((pieces + 1023) / 1024), y);
    if (C == 32) hipLaunchKernelGGL((k_kv_copy<32, 4>), grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((k_kv_copy<16, 4>), grid, dim3(256), 0, s, a);
}

}  // namespace cmf

using namespace cmf;

extern "C" {

int cmf_qk_rope_dev(const cmf_qk_rope_args* p) {
    if (!p) return fail("qk_rope: null argument");
    const auto& a = *p;
    if (a.b < 1 || a.nh < 1 || a.nkv < 1 || a.nh > 4096 || a.nkv > 4096) return fail("qk_rope: b, nh and nkv of at least 1 (heads at most 4096)");
    if (!a.qkv || !a.rope || (!a.q_out && !a.k)) return fail("qk_rope: null qkv, rope or outputs");
    if (!a.k != !a.v) return fail("qk_rope: k and v go together");
    if (!kv_dtype_ok(a.kv_dtype)) return fail("qk_rope: kv_dtype must be f32, f16 or bf16");
    if (a.max_pos < 1) return fail("qk_rope: max_pos of at least 1");
    if ((long long)a.b * (a.nh + 2 * a.nkv) > (1ll << 34)) return fail("qk_rope: too many heads in one call");
    if (a.ldq < (a.nh + 2 * a.nkv) * CACHE_HD || a.ldq % 4 || !aligned16(a.qkv))
        return fail("qk_rope: ldq must hold all heads, 16-byte aligned");
    if (a.q_out && (a.ldo < a.nh * CACHE_HD || a.ldo % 4 || !aligned16(a.q_out)))
        return fail("qk_rope: ldo must hold the query heads, 16-byte aligned");
    if (!aligned16(a.rope) || !aligned16(a.q_norm) || !aligned16(a.k_norm)) return fail("qk_rope: 16-byte aligned tables");
    if (a.k) {
        if (a.slots < 1) return fail("qk_rope: slots of at least 1");
        if (a.row_stride < CACHE_HD || a.row_stride % 8 || a.head_stride < 0 || a.head_stride % 8 || !aligned16(a.k) || !aligned16(a.v))
            return fail("qk_rope: k / v strides must be multiples of 8 elements, rows of 128, 16-byte aligned");
        if (a.nkv > 1 && a.head_stride < CACHE_HD) return fail("qk_rope: k / v heads overlap");
    }
    if (!a.d_pos0 && (a.pos0 < 0 || (!a.d_depth && (long long)a.pos0 + a.b > a.max_pos)))
        return fail("qk_rope: positions outside the rope table");
    if (a.k && !a.d_pos0 && (a.at_pos ? (long long)a.pos0 + a.b : a.b) > a.slots)
        return fail("qk_rope: rows past the cache's slots");
    OpScope sc;
    if (sc.enter(a.stream, "qk_rope") != CMF_OK) return CMF_ERR;
    launch_qk_rope(a, sc.s);
    CMF_HIP(hipGetLastError());
    return CMF_OK;
}

int cmf_kv_copy_dev(const cmf_kv_copy_args* p) {
    if (!p) return fail("kv_copy: null argument");
    const auto& a = *p;
    if (!a.d_dst || !a.d_src) return fail("kv_copy: null argument");
    if (a.nbuf < 1 || a.nkv < 1 || a.n < 0 || (long long)a.nbuf * a.nkv > 65535)
        return fail("kv_copy: nbuf and nkv of at least 1 (at most 65535 heads in all), n >= 0");
    if (!kv_dtype_ok(a.kv_dtype)) return fail("kv_copy: kv_dtype must be f32, f16 or bf16");
    if (a.dst_slots < 0 || a.src_slots < 0) return fail("kv_copy: negative slots");
    for (long long st : {a.dst_head_stride, a.dst_row_stride, a.src_head_stride, a.src_row_stride})
        if (st < 0 || st % 8) return fail("kv_copy: strides must be multiples of 8 elements");
    if (a.dst_row_stride < CACHE_HD || a.src_row_stride < CACHE_HD) return fail("kv_copy: rows of 128 elements");
    if (a.nkv > 1 && a.dst_head_stride < CACHE_HD) return fail("kv_copy: heads of dst overlap");
    if (!a.d_pos0 && (a.pos0 < 0 || (!a.d_n && (long long)a.pos0 + a.n > a.dst_slots)))
        return fail("kv_copy: rows past the slots of dst");
    if (!a.d_idx && !a.d_n && a.n > a.src_slots) return fail("kv_copy: rows past the slots of src");
    if (a.n == 0) return CMF_OK;
    OpScope sc;
    if (sc.enter(a.stream, "kv_copy") != CMF_OK) return CMF_ERR;
    launch_kv_copy(a, sc.s);
    CMF_HIP(hipGetLastError());
    return CMF_OK;
}

int cmf_tree_masks(const int32_t* parent, int b, int pos0, int window, int sinks, uint64_t* mask, int32_t* depth) {
    if (!parent || !mask || !depth) return fail("tree_masks: null argument");
    if (b < 1 || b > CMF_TREE_MAX) return fail("tree_masks: 1 to 64 rows");
    if (pos0 < 0 || window < 0 || sinks < 0) return fail("tree_masks: pos0, window and sinks of at least 0");
    for (int i = 0; i < b; i++)
        if (parent[i] < -1 || parent[i] >= i) return fail("tree_masks: a row's parent must be an earlier row or -1");
    for (int i = 0; i < b; i++) {
        depth[i] = parent[i] < 0 ? 0 : depth[parent[i]] + 1;
        uint64_t m = 0;
        for (int j = i; j >= 0; j = parent[j])
            if (!window || depth[i] - depth[j] < window || (long long)pos0 + depth[j] < sinks) m |= 1ull << j;
        mask[i] = m;
    }
    return CMF_OK;
}

}  // extern "C"
