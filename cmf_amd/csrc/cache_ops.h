// Launchers and shared helpers of the operators on caches and logits
// (cache_ops.hip, cache_attn.hip, logprobs.hip).
#pragma once

#include "../../include/cmf_hip.h"
#include "common.h"

namespace cmf {

constexpr int CACHE_HD = 128;
constexpr size_t OP_WS_MAX = 64u << 20;  // no operator asks for more scratch

// The stream of an operator call (see CMF_STREAM_NULL) with the library's
// device current on the calling thread while the call runs.
struct OpScope {
    hipStream_t s = nullptr;
    int back = -1;  // the device that was current before, -1: the same
    int enter(void* stream, const char* who);
    ~OpScope();
};

inline bool kv_dtype_ok(int dt) { return dt == CMF_DT_F32 || dt == CMF_DT_F16 || dt == CMF_DT_BF16; }
inline bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

// A 16-bit cache element as f32 and back (round to nearest, ties to even).
struct bf16_t {
    uint16_t u;
};
__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(_Float16 x) { return (float)x; }
__device__ __forceinline__ float to_f32(bf16_t x) { return __uint_as_float((uint32_t)x.u << 16); }
template <class T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) {
    return x;
}
template <>
__device__ __forceinline__ _Float16 from_f32<_Float16>(float x) {
    return (_Float16)x;
}
template <>
__device__ __forceinline__ bf16_t from_f32<bf16_t>(float x) {
    const uint32_t u = __float_as_uint(x);
    if (x != x) return bf16_t{(uint16_t)((u >> 16) | 0x40)};
    return bf16_t{(uint16_t)((u + 0x7fff + ((u >> 16) & 1)) >> 16)};
}

// n elements of T at p (16-byte aligned runs of 8) as f32
template <class T>
__device__ __forceinline__ void load8(const T* p, float (&o)[8]) {
    if constexpr (sizeof(T) == 4) {
        const float4 a = ((const float4*)p)[0], b = ((const float4*)p)[1];
        o[0] = a.x, o[1] = a.y, o[2] = a.z, o[3] = a.w, o[4] = b.x, o[5] = b.y, o[6] = b.z, o[7] = b.w;
    } else {
        union {
            uint4 v;
            T h[8];
        } u;
        u.v = *(const uint4*)p;
#pragma unroll
        for (int i = 0; i < 8; i++) o[i] = to_f32(u.h[i]);
    }
}

// enqueue only: arguments checked by the callers
void launch_qk_rope(const cmf_qk_rope_args& a, hipStream_t s);
int launch_cache_attention(const cmf_attention_args& a, hipStream_t s);
void launch_kv_copy(const cmf_kv_copy_args& a, hipStream_t s);
void launch_logprobs(const cmf_logprobs_args& a, hipStream_t s);
size_t logprobs_ws(int rows, int V, int top_k);
size_t cache_attention_ws(const cmf_attention_args& a);

}  // namespace cmf
