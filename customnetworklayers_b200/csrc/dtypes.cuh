// Element types of the network operators (fp32, fp16, bf16): conversions to and from fp32 and 16-byte vectors.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.h"

namespace cnl {

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }

template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Two neighbouring elements in one register of a 16-bit type.
__device__ __forceinline__ float2 unpack2(unsigned v, __half) { return __half22float2(*reinterpret_cast<const __half2*>(&v)); }
__device__ __forceinline__ float2 unpack2(unsigned v, __nv_bfloat16) {
    return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
}
template <typename T> __device__ __forceinline__ unsigned pack2(float a, float b);
template <> __device__ __forceinline__ unsigned pack2<__half>(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const unsigned*>(&h);
}
template <> __device__ __forceinline__ unsigned pack2<__nv_bfloat16>(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const unsigned*>(&h);
}

// N consecutive elements at a 16-byte aligned address (N * sizeof(T) a multiple of 16).
template <typename T, int N>
__device__ __forceinline__ void load_vec(const T* __restrict__ p, float (&v)[N]) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < N / 4; ++i) {
            const float4 q = __ldg(reinterpret_cast<const float4*>(p) + i);
            v[4 * i] = q.x; v[4 * i + 1] = q.y; v[4 * i + 2] = q.z; v[4 * i + 3] = q.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < N / 8; ++i) {
            const uint4 q = __ldg(reinterpret_cast<const uint4*>(p) + i);
            const unsigned w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float2 f = unpack2(w[j], T());
                v[8 * i + 2 * j] = f.x; v[8 * i + 2 * j + 1] = f.y;
            }
        }
    }
}

template <typename T, int N>
__device__ __forceinline__ void store_vec(T* __restrict__ p, const float (&v)[N]) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < N / 4; ++i)
            reinterpret_cast<float4*>(p)[i] = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
    } else {
#pragma unroll
        for (int i = 0; i < N / 8; ++i) {
            uint4 q;
            q.x = pack2<T>(v[8 * i], v[8 * i + 1]); q.y = pack2<T>(v[8 * i + 2], v[8 * i + 3]);
            q.z = pack2<T>(v[8 * i + 4], v[8 * i + 5]); q.w = pack2<T>(v[8 * i + 6], v[8 * i + 7]);
            reinterpret_cast<uint4*>(p)[i] = q;
        }
    }
}

// 2^x and 1/x by the special-function unit (2 ulp and 1 ulp), subnormals to zero: the plain intrinsics spend three more
// instructions each on subnormals, which no value here needs.
__device__ __forceinline__ float exp2_approx(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float rcp_approx(float x) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

inline bool aligned16(const void* p) { return (reinterpret_cast<size_t>(p) & 15) == 0; }

inline int check_dtype(int dtype) {
    if (dtype != CNL_F32 && dtype != CNL_F16 && dtype != CNL_BF16) return fail(CNL_ERR_BAD_OPTION, "dtype %d is not CNL_F32, CNL_F16 or CNL_BF16", dtype);
    return CNL_OK;
}

}  // namespace cnl
