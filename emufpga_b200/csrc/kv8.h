// Shared by the translation units of the paged 8-bit cache.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "abi.h"
#include "device.cuh"

namespace spm {

// The argument checks that every spm_kv8_* call makes.
inline void kv8_check(const spm_kv8* c) {
    if (!c) fail(SPM_E_ARG, "null cache");
    if (c->pages < 0 || c->kv_heads < 1) fail(SPM_E_ARG, "a cache has at least one kv head and no negative page count");
    if (c->page_tokens < 16 || c->page_tokens > 256 || (c->page_tokens & (c->page_tokens - 1)))
        fail(SPM_E_ARG, "page_tokens is 16, 32, 64, 128 or 256");
    const int d = c->head_dim;
    if (d != 64 && d != 96 && d != 128 && d != 192 && d != 256) fail(SPM_E_ARG, "head_dim is 64, 96, 128, 192 or 256");
    if (int64_t(c->pages) * c->page_tokens > INT32_MAX) fail(SPM_E_ARG, "slots are 32-bit: pages * page_tokens must fit");
    if (c->pages && (!c->k_codes || !c->v_codes || !c->k_scales || !c->v_scales)) fail(SPM_E_ARG, "null cache memory");
    if ((reinterpret_cast<uintptr_t>(c->k_codes) | reinterpret_cast<uintptr_t>(c->v_codes)) & 15)
        fail(SPM_E_ARG, "codes must be 16-byte aligned");
}

inline void kv8_check_type(uint32_t dtype) {
    if (dtype != SPM_F32 && dtype != SPM_F16 && dtype != SPM_BF16) fail(SPM_E_ENCODING, "activations are f32, f16 or bf16");
}

namespace dev {

template <class T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32(float v) { return v; }
template <>
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <class T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32(float v) { return __float2bfloat16_rn(v); }

// Four consecutive elements as f32; in one load where `vec` says that they are aligned.
template <class T>
__device__ __forceinline__ void load4(const T* p, bool vec, float (&v)[4]) {
    if (vec) {
        if constexpr (sizeof(T) == 4) {
            const float4 q = *reinterpret_cast<const float4*>(p);
            v[0] = q.x, v[1] = q.y, v[2] = q.z, v[3] = q.w;
        } else {
            const uint2 q = *reinterpret_cast<const uint2*>(p);
            const T* h = reinterpret_cast<const T*>(&q);
#pragma unroll
            for (int j = 0; j < 4; j++) v[j] = to_f32(h[j]);
        }
    } else {
#pragma unroll
        for (int j = 0; j < 4; j++) v[j] = to_f32(p[j]);
    }
}

// 2^e for e clamped to the normal range.
__device__ __forceinline__ float pow2i(int e) { return __int_as_float((min(max(e, -126), 127) + 127) << 23); }

}  // namespace dev
}  // namespace spm
