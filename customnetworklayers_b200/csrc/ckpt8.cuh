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

// s of a block from the bits of its largest finite |x|.
template <int FMT>
__device__ __forceinline__ int exponent_of(unsigned top) {
    const int e = (int)(top >> 23) - 127;                        // -127 for subnormals: held to -126 below either way
    const unsigned m = top & 0x7fffffu;
    const int s = FMT == CNL_CKPT_INT8 ? e - 6 + (m >= 0x7f0000u) : e - 8 + (m > 0x600000u);
    return max(s, -126);
}

__device__ __forceinline__ bool not_finite(unsigned mag) { return mag >= 0x7f800000u; }
__device__ __forceinline__ float max_nan(float a, float b) {             // NaN if one is
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// max over the LANES (a power of two) neighbouring lanes that hold one block
template <int LANES>
__device__ __forceinline__ float lanes_max(float v) {
#pragma unroll
    for (int o = 1; o < LANES; o <<= 1) v = max_nan(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

// Codes of N elements of one block that LANES lanes hold together, four to a word (N = 1: in the low byte); returns s (the
// same in all of the lanes).  All lanes of the warp must call it together (v = 0 where a lane has nothing).
template <int FMT, int LANES, int N>
__device__ __forceinline__ int encode(const float (&v)[N], unsigned (&word)[(N + 3) / 4]) {
    float m = fabsf(v[0]);
#pragma unroll
    for (int i = 1; i < N; ++i) m = max_nan(m, fabsf(v[i]));
    unsigned top = __float_as_uint(lanes_max<LANES>(m));
    const bool odd = not_finite(top);
    if (__any_sync(0xffffffffu, odd)) {                          // the maximum again, over the finite elements (rare)
        m = 0.0f;
#pragma unroll
        for (int i = 0; i < N; ++i) m = fmaxf(m, not_finite(__float_as_uint(v[i]) & 0x7fffffffu) ? 0.0f : fabsf(v[i]));
        top = __float_as_uint(lanes_max<LANES>(m));
    }
    const int s = exponent_of<FMT>(top);
    const float inv = __uint_as_float((unsigned)(127 - s) << 23);
#pragma unroll
    for (int w = 0; w < (N + 3) / 4; ++w) {
        if constexpr (FMT == CNL_CKPT_INT8) {
            // 1.5 * 2^23 + c: the addition rounds to nearest even and leaves c in the low byte
            const float2 c = make_float2(12582912.0f, 12582912.0f), k = make_float2(inv, inv);
            const float2 f = __ffma2_rn(make_float2(v[4 * w], N > 1 ? v[4 * w + (N > 1)] : 0.0f), k, c);
            word[w] = __float_as_uint(f.x);
            if constexpr (N > 1) {
                const float2 g = __ffma2_rn(make_float2(v[4 * w + 2], v[4 * w + 3]), k, c);
                word[w] = __byte_perm(__byte_perm(__float_as_uint(f.x), __float_as_uint(f.y), 0x0040), __byte_perm(__float_as_uint(g.x), __float_as_uint(g.y), 0x0040), 0x5410);
            } else word[w] &= 0xffu;
        } else {
            const float2 k = make_float2(inv, inv), f = __fmul2_rn(make_float2(v[4 * w], N > 1 ? v[4 * w + (N > 1)] : 0.0f), k);
            word[w] = __nv_cvt_float2_to_fp8x2(f, __NV_SATFINITE, __NV_E4M3);
            if constexpr (N > 1) {
                const float2 g = __fmul2_rn(make_float2(v[4 * w + 2], v[4 * w + 3]), k);
                word[w] = __byte_perm(word[w], __nv_cvt_float2_to_fp8x2(g, __NV_SATFINITE, __NV_E4M3), 0x5410);
            } else word[w] &= 0xffu;
        }
    }
    if (odd) {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (not_finite(__float_as_uint(v[i]) & 0x7fffffffu)) {
                const int at = 8 * (i % 4);
                word[i / 4] = (word[i / 4] & ~(0xffu << at)) | (FMT == CNL_CKPT_INT8 ? 0x80u : 0x7fu) << at;
            }
    }
    return s;
}

// The values N codes stand for, in fp32.  word: the codes, four to a word (N a multiple of 4), or one code in the low byte
// (N = 1).  Saturated to fp32's finite range (a code of 64 at s = 122 would be 2^128).
template <int FMT, int N>
__device__ __forceinline__ void decode(const unsigned* word, int s, float (&v)[N]) {
    const float unit = __uint_as_float((unsigned)(s + 127) << 23);
    bool rare = s > 118;                                                  // may leave fp32's range
    if constexpr (FMT == CNL_CKPT_INT8) {
        // a byte c + 128 under the exponent of 2^23 is the float 2^23 + c + 128
#pragma unroll
        for (int i = 0; i < (N + 3) / 4; ++i) {
            const unsigned w = word[i] ^ 0x80808080u;                     // c + 128
            rare |= ((w - 0x01010101u) & ~w & 0x80808080u) != 0 && (N > 1 || (w & 0xffu) == 0);       // some code is -128
#pragma unroll
            for (int j = 0; j < (N < 4 ? N : 4); j += 2) {
                const float2 f = __fadd2_rn(make_float2(__uint_as_float(__byte_perm(w, 0x4b000000u, 0x7440 + j)), __uint_as_float(__byte_perm(w, 0x4b000000u, 0x7441 + j))),
                                            make_float2(-8388736.0f, -8388736.0f));
                const float2 r = __fmul2_rn(f, make_float2(unit, unit));
                v[4 * i + j] = r.x;
                if (4 * i + j + 1 < N) v[4 * i + j + (N > 1)] = r.y;
            }
        }
        if (rare) {
#pragma unroll
            for (int i = 0; i < N; ++i)
                if ((word[i / 4] >> (8 * (i % 4)) & 0xffu) == 0x80u) v[i] = __uint_as_float(0x7fffffffu);
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(word[i / 4] >> (8 * (i % 4)) & 0xffffu), __NV_E4M3);
            const float2 f = __fmul2_rn(__half22float2(__half2(h)), make_float2(unit, unit));
            v[i] = f.x;
            if (i + 1 < N) v[i + (N > 1)] = f.y;
        }
    }
    if (rare) {
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
