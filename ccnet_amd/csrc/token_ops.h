// Shared pieces of the token operators (norm_rope.hip, kv_cache.hip, attention_cross.hip, attention_cache.hip): (batch, token,
// head, dim) operands with any strides, and the 8-bit codes of the key/value cache.
#pragma once
#include <math.h>
#include "common.h"

// 16-byte vector access: base and strides in whole groups (a stride of an axis of length 1 is never used)
static inline bool cc_heads_ok(const ccnet_heads& x, int dtype, int B, int T, int H) {
    const int g = 16 / cc_esize(dtype);
    return x.ptr && ((uintptr_t)x.ptr % 16) == 0 && (B == 1 || (x.sb % g) == 0) && (T == 1 || (x.st % g) == 0) && (H == 1 || (x.sh % g) == 0);
}
static inline int cc_code_ok(int f) { return f == CCNET_INT8 || f == CCNET_FP8; }

#ifdef __HIPCC__
// element (b, t, h, 0) of a ccnet_heads operand; the products are 64-bit (long caches pass 2^32 elements)
template <typename T>
__device__ __forceinline__ T* heads_at(const ccnet_heads& x, long long b, long long t, long long h) {
    return (T*)x.ptr + b * x.sb + t * x.st + h * x.sh;
}

// ---- codes: int8 in [-127, 127], or OCP e4m3 (max 448, no infinity).  value = code * scale.
template <int FMT> struct Code;
template <> struct Code<CCNET_INT8> {
    static constexpr float qmax = 127.0f;
    // four values already divided by the scale -> four codes, round to nearest even
    static __device__ __forceinline__ uint32_t enc4(const float* f) {
        uint32_t r = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) r |= ((uint32_t)(int)rintf(fminf(fmaxf(f[i], -127.0f), 127.0f)) & 0xFFu) << (8 * i);
        return r;
    }
    static __device__ __forceinline__ void dec4(uint32_t c, float* f) {
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = (float)(int)(signed char)(c >> (8 * i));
    }
};
template <> struct Code<CCNET_FP8> {
    static constexpr float qmax = 448.0f;
    static __device__ __forceinline__ uint32_t enc4(const float* f) {
        float g[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) g[i] = fminf(fmaxf(f[i], -448.0f), 448.0f);
        int r = __builtin_amdgcn_cvt_pk_fp8_f32(g[0], g[1], 0, false);
        return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(g[2], g[3], r, true);
    }
    static __device__ __forceinline__ void dec4(uint32_t c, float* f) {
        f[0] = __builtin_amdgcn_cvt_f32_fp8(c, 0);
        f[1] = __builtin_amdgcn_cvt_f32_fp8(c, 1);
        f[2] = __builtin_amdgcn_cvt_f32_fp8(c, 2);
        f[3] = __builtin_amdgcn_cvt_f32_fp8(c, 3);
    }
};
#endif  // __HIPCC__
