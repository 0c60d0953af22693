// 8-bit blocks of activations (device side).  Thirty-two neighbouring elements share a power-of-two scale 2^s kept as
// one byte (s + 127); a code is the element times 2^-s, rounded to nearest even: a whole number in -127..127 (int8) or a
// 4-bit-exponent 3-bit-mantissa float (e4m3).
//
// With a = max |x| over the finite elements and E = floor(log2 a):
//   int8: s = E - 6, one more if a 2^-s would round to 128;   e4m3: s = E - 8, one more if a 2^-s > 448.
// A power of two costs up to one bit of int8's range against a scale of a / 127, but both the product with 2^-s and the
// product back are exact in fp32, so the only rounding is the one to 8 bits: codes are a function of the input alone and
// no quotient can fall on the other side of a tie.  s is held to -126 and up, where 2^s and 2^-s are normal numbers; blocks
// below that lose only values under 2^-126.  Elements that are not finite do not take part in a and get a code of their
// own (int8 -128, e4m3 NaN), which comes back as NaN: a blown-up activation stays visible in the gradient.
#pragma once
#include <cuda_fp8.h>

#include "dtypes.cuh"

namespace cnl {
namespace ckpt8 {

constexpr int kBlock = 32;

// s of a block from the bits of max |x|; sets `odd` when an element is not finite (its bits are the maximum then).
template <int FMT>
__device__ __forceinline__ int exponent_of(unsigned top) {
    const int e = (int)(top >> 23) - 127;                        // -127 for subnormals: held to -126 below either way
    const unsigned m = top & 0x7fffffu;
    const int s = FMT == CNL_CKPT_INT8 ? e - 6 + (m >= 0x7f0000u) : e - 8 + (m > 0x600000u);
    return max(s, -126);
}

__device__ __forceinline__ unsigned magnitude(float v) { return __float_as_uint(v) & 0x7fffffffu; }
__device__ __forceinline__ bool not_finite(unsigned mag) { return mag >= 0x7f800000u; }

// max over the `lanes` (a power of two) neighbouring lanes that hold one block
template <int LANES>
__device__ __forceinline__ unsigned lanes_max(unsigned v) {
#pragma unroll
    for (int o = 1; o < LANES; o <<= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

// Codes of N elements of one block that LANES lanes hold together; returns s (the same in all of them).  N = 1, 4 or 8.
// All lanes of the warp must call it together (v = 0 where a lane has nothing).
template <int FMT, int LANES, int N>
__device__ __forceinline__ int encode(const float (&v)[N], unsigned char (&code)[N]) {
    unsigned top = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) top = max(top, magnitude(v[i]));
    top = lanes_max<LANES>(top);
    const bool odd = not_finite(top);
    if (__any_sync(0xffffffffu, odd)) {                          // the maximum again, over the finite elements (rare)
        unsigned fin = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) fin = max(fin, not_finite(magnitude(v[i])) ? 0u : magnitude(v[i]));
        top = lanes_max<LANES>(fin);
    }
    const int s = exponent_of<FMT>(top);
    const float inv = __uint_as_float((unsigned)(127 - s) << 23);
    if constexpr (FMT == CNL_CKPT_INT8) {
#pragma unroll
        for (int i = 0; i < N; ++i) code[i] = (unsigned char)__float_as_uint(fmaf(v[i], inv, 12582912.0f));   // 1.5 * 2^23: rne in the low byte
    } else {
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            const __nv_fp8x2_storage_t p = __nv_cvt_float2_to_fp8x2(make_float2(v[i] * inv, i + 1 < N ? v[i + (N > 1)] * inv : 0.0f), __NV_SATFINITE, __NV_E4M3);
            code[i] = (unsigned char)p;
            if (i + 1 < N) code[i + (N > 1)] = (unsigned char)(p >> 8);
        }
    }
    if (odd) {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (not_finite(magnitude(v[i]))) code[i] = FMT == CNL_CKPT_INT8 ? 0x80 : 0x7f;
    }
    return s;
}

// The values N codes stand for, in fp32.  word: the codes, four to a word (N a multiple of 4), or one code in the low byte
// (N = 1).  Saturated to fp32's finite range (a code of 64 at s = 122 would be 2^128).
template <int FMT, int N>
__device__ __forceinline__ void decode(const unsigned* word, int s, float (&v)[N]) {
    const float unit = __uint_as_float((unsigned)(s + 127) << 23);
#pragma unroll
    for (int i = 0; i < N; i += (N == 1 ? 1 : 2)) {
        const unsigned w = word[i / 4] >> (8 * (i % 4));
        if constexpr (FMT == CNL_CKPT_INT8) {
#pragma unroll
            for (int j = 0; j < (N == 1 ? 1 : 2); ++j) {
                const unsigned c = (w >> (8 * j)) & 0xffu;
                const float f = __uint_as_float(0x4b000000u | (c ^ 0x80u)) - 8388736.0f;          // 2^23 + (c + 128)
                v[i + j] = (c == 0x80u ? __uint_as_float(0x7fffffffu) : f) * unit;
            }
        } else {
            const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w & 0xffffu), __NV_E4M3);
            const float2 f = __half22float2(__half2(h));
            v[i] = f.x * unit;
            if constexpr (N > 1) v[i + 1] = f.y * unit;
        }
    }
    if (s > 118) {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (fabsf(v[i]) > 3.402823466e38f) v[i] = copysignf(3.402823466e38f, v[i]);
    }
}

// One byte of a byte array into the scale exponent and back.
__device__ __forceinline__ unsigned char scale_byte(int s) { return (unsigned char)(s + 127); }
__device__ __forceinline__ int scale_exponent(unsigned char b) { return (int)b - 127; }

}  // namespace ckpt8
}  // namespace cnl
