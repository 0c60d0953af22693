// Activations kept in 8 bits: store, restore, and activations whose forward pass leaves the codes of its input and whose
// backward pass reads them (format: ckpt8.cuh).
//
// Every kernel is one pass over memory and HBM bound: b + 1 + 1/32 bytes an element for store and restore, 2 b + 1 + 1/32
// for the activations (b = 2 or 4).  A lane holds one 16-byte vector, so a block of 32 elements lies in 4 (16-bit types) or
// 8 (fp32) neighbouring lanes and its maximum costs two or three shuffles; a thread's vectors are all loaded before the first
// is used.  Addresses that are not 16-byte aligned take the same code with one element a lane.
// 126 M elements: fp32 store and restore 100 us (6.3 TB/s, 0.96 of a copy), GELU and SiLU either way 170 to 175 us (1.0 of one);
// 16 bits store 74 (int8) and 82 us (e4m3), restore 66, SiLU 104 and 98, GELU 113 and 125 us (0.76 to 0.98: conversions and the
// error function issue beside the copies).
#include "ckpt8.cuh"

#include <type_traits>

namespace cnl {
namespace ckpt8 {

constexpr int kThreads = 256;
// Vectors a thread has under way.  Store and restore are short and want four (restore bf16 64 us, with two 76 us, for 126M
// elements); the activations need the registers and want two (silu backward 98 us, with four 127 us).
template <int ACT> constexpr int kUnrollOf = ACT ? 2 : 4;

__device__ __forceinline__ float2 pair(float v) { return make_float2(v, v); }
__device__ __forceinline__ float relu(float x) { return max_nan(x, 0.0f); }
__device__ __forceinline__ float below_inf(float x) {                    // +inf as the largest number; NaN and -inf stay
    float r;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(x), "f"(3.402823466e38f));
    return r;
}

// Phi(x) = exp(-x^2/2) t P(t) for x <= 0, t = 1 / (1 + 0.3 |x|), and 1 - that for x > 0.  P was fitted here to the scaled
// complementary error function by least squares with weights moved towards an even relative error over |x| <= 14:
// 8.2e-6 with degree 5 (a 64th of fp16's half step), 1.6e-7 with degree 7.
// Two at a time: packed fp32 arithmetic takes both in one issue slot, and at 5 bytes an element (16-bit types) an SM has some
// 27 slots an element.
template <typename T>
__device__ __forceinline__ float2 cdf_tail(float2 x, float2 magnitude) {                 // Phi(-|x|)
    const float2 k = __fmul2_rn(__fmul2_rn(x, x), pair(-0.7213475204444817f));           // -x^2 / 2 in powers of two
    const float2 d = __ffma2_rn(magnitude, pair(0.3f), pair(1.0f));
    const float2 t = make_float2(rcp_approx(d.x), rcp_approx(d.y));
    float2 p;
    if constexpr (sizeof(T) == 4) {
        p = __ffma2_rn(t, pair(0.03567475825548172f), pair(-0.15720295906066895f));
        p = __ffma2_rn(t, p, pair(0.20635318756103516f));
        p = __ffma2_rn(t, p, pair(-0.053683266043663025f));
        p = __ffma2_rn(t, p, pair(0.12856139242649078f));
        p = __ffma2_rn(t, p, pair(0.0999135747551918f));
        p = __ffma2_rn(t, p, pair(0.1207539439201355f));
        p = __ffma2_rn(t, p, pair(0.11962930113077164f));
    } else {
        p = __ffma2_rn(t, pair(-0.0770978331565857f), pair(0.21603818237781525f));
        p = __ffma2_rn(t, p, pair(-0.0169492457062006f));
        p = __ffma2_rn(t, p, pair(0.14419695734977722f));
        p = __ffma2_rn(t, p, pair(0.11374179273843765f));
        p = __ffma2_rn(t, p, pair(0.12007424235343933f));
    }
    return __fmul2_rn(__fmul2_rn(t, p), make_float2(exp2_approx(k.x), exp2_approx(k.y)));
}

__device__ __forceinline__ float2 logistic(float2 x) {
    const float2 e = __fmul2_rn(x, pair(-1.4426950408889634f));
    const float2 d = __fadd2_rn(make_float2(exp2_approx(e.x), exp2_approx(e.y)), pair(1.0f));
    return make_float2(rcp_approx(d.x), rcp_approx(d.y));
}

template <int ACT, typename T>
__device__ __forceinline__ float2 act(float2 x) {
    if constexpr (ACT == CNL_ACT_GELU) {                                                 // x Phi(x) = max(x, 0) - |x| Phi(-|x|)
        // (a finite factor, so that the tail of +inf, which is 0, leaves +inf as it is; -inf times its Phi, 0, is NaN)
        const float2 m = make_float2(fabsf(below_inf(x.x)), fabsf(below_inf(x.y))), q = cdf_tail<T>(x, m);
        return __ffma2_rn(make_float2(-m.x, -m.y), q, make_float2(relu(x.x), relu(x.y)));
    } else {
        return __fmul2_rn(x, logistic(x));
    }
}

template <int ACT, typename T>
__device__ __forceinline__ float2 act_slope(float2 x) {
    if constexpr (ACT == CNL_ACT_GELU) {                                                 // Phi(x) + x phi(x); Phi(x) = 1/2 + sign(x) (1/2 - Phi(-|x|))
        const float2 m = make_float2(fabsf(x.x), fabsf(x.y)), q = cdf_tail<T>(x, m);
        const float2 h = __fadd2_rn(pair(0.5f), make_float2(-q.x, -q.y));
        const float2 k = __fmul2_rn(__fmul2_rn(x, x), pair(-0.7213475204444817f));
        const float2 e = make_float2(exp2_approx(k.x), exp2_approx(k.y));               // the one in cdf_tail
        return __ffma2_rn(__fmul2_rn(x, pair(0.3989422804014327f)), e, __fadd2_rn(make_float2(copysignf(h.x, x.x), copysignf(h.y, x.y)), pair(0.5f)));
    } else {                                                                             // s + x s (1 - s)
        const float2 g = logistic(x);
        return __ffma2_rn(x, __ffma2_rn(make_float2(-g.x, -g.y), g, g), g);
    }
}

// V consecutive elements from `at` (0 beyond count); V > 1 reads 16 bytes where they all exist.
template <typename T, int V>
__device__ __forceinline__ void read(const T* __restrict__ x, long long at, long long count, float (&v)[V]) {
    if (V > 1 && at + V <= count) {
        if constexpr (V > 1) load_vec<T, V>(x + at, v);
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = at + i < count ? to_f32(x[at + i]) : 0.0f;
    }
}

template <typename T, int V>
__device__ __forceinline__ void write(T* __restrict__ x, long long at, long long count, const float (&v)[V]) {
    if (V > 1 && at + V <= count) {
        if constexpr (V > 1) store_vec<T, V>(x + at, v);
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (at + i < count) x[at + i] = from_f32<T>(v[i]);
    }
}

template <int V>
__device__ __forceinline__ void write_codes(unsigned char* __restrict__ codes, long long at, long long count, const unsigned (&w)[(V + 3) / 4]) {
    if (V > 1 && at + V <= count) {
        if constexpr (V == 8) *reinterpret_cast<uint2*>(codes + at) = make_uint2(w[0], w[(V + 3) / 4 - 1]);
        else *reinterpret_cast<unsigned*>(codes + at) = w[0];
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (at + i < count) codes[at + i] = (unsigned char)(w[i / 4] >> (8 * (i % 4)));
    }
}

template <int V>
__device__ __forceinline__ void read_codes(const unsigned char* __restrict__ codes, long long at, long long count, unsigned (&w)[(V + 3) / 4]) {
    if (V > 1 && at + V <= count) {
        if constexpr (V == 8) {
            const uint2 q = __ldg(reinterpret_cast<const uint2*>(codes + at));
            w[0] = q.x; w[(V + 3) / 4 - 1] = q.y;
        } else w[0] = __ldg(reinterpret_cast<const unsigned*>(codes + at));
    } else {
#pragma unroll
        for (int i = 0; i < (V + 3) / 4; ++i) w[i] = 0;
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (at + i < count) w[i / 4] |= (unsigned)codes[at + i] << (8 * (i % 4));
    }
}

// x -> codes, scales (if not null) and, with ACT, y = act(x)
template <typename T, int V, int FMT, int ACT>
__global__ void __launch_bounds__(kThreads) store_kernel(const T* __restrict__ x, T* __restrict__ y, unsigned char* __restrict__ codes,
                                                         unsigned char* __restrict__ scales, long long count) {
    constexpr int kLanes = kBlock / V, kUnroll = kUnrollOf<ACT>;
    const long long first = ((long long)blockIdx.x * kUnroll * kThreads + threadIdx.x) * V;
    float v[kUnroll][V];
#pragma unroll
    for (int j = 0; j < kUnroll; ++j) read<T, V>(x, first + (long long)j * kThreads * V, count, v[j]);
#pragma unroll
    for (int j = 0; j < kUnroll; ++j) {
        const long long at = first + (long long)j * kThreads * V;
        if (codes) {                                              // the same for the whole grid
            unsigned c[(V + 3) / 4];
            const int s = encode<FMT, kLanes, V>(v[j], c);
            write_codes<V>(codes, at, count, c);
            if (at < count && (threadIdx.x & (kLanes - 1)) == 0) scales[at / kBlock] = scale_byte(s);
        }
        if constexpr (ACT != 0) {
#pragma unroll
            for (int i = 0; i < V; i += 2) {
                const float2 f = act<ACT, T>(make_float2(v[j][i], v[j][i + (V > 1)]));
                v[j][i] = f.x;
                if (V > 1) v[j][i + (V > 1)] = f.y;
            }
            write<T, V>(y, at, count, v[j]);
        }
    }
}

// codes, scales -> x, or with ACT g_x = g_y * act'(x)
template <typename T, int V, int FMT, int ACT>
__global__ void __launch_bounds__(kThreads) restore_kernel(const unsigned char* __restrict__ codes, const unsigned char* __restrict__ scales,
                                                           const T* __restrict__ g, T* __restrict__ out, long long count) {
    constexpr int kUnroll = kUnrollOf<ACT>;
    const long long first = ((long long)blockIdx.x * kUnroll * kThreads + threadIdx.x) * V;
    unsigned w[kUnroll][(V + 3) / 4];
    int s[kUnroll];
    float gv[kUnroll][V];
#pragma unroll
    for (int j = 0; j < kUnroll; ++j) {
        const long long at = first + (long long)j * kThreads * V;
        read_codes<V>(codes, at, count, w[j]);
        s[j] = at < count ? scale_exponent(__ldg(scales + at / kBlock)) : 0;
        if constexpr (ACT != 0) read<T, V>(g, at, count, gv[j]);
    }
    constexpr int kSafe = std::is_same<T, __half>::value ? 7 : 118;                   // no code can leave the type's range up to here
    constexpr float kTop = std::is_same<T, float>::value ? 3.402823466e38f : std::is_same<T, __half>::value ? 65504.0f : 3.38953139e38f;
#pragma unroll
    for (int j = 0; j < kUnroll; ++j) {
        const long long at = first + (long long)j * kThreads * V;
        float v[V];
        decode<FMT, V>(w[j], s[j], v);
        if constexpr (ACT != 0) {
#pragma unroll
            for (int i = 0; i < V; i += 2) {
                const float2 f = __fmul2_rn(make_float2(gv[j][i], gv[j][i + (V > 1)]), act_slope<ACT, T>(make_float2(v[i], v[i + (V > 1)])));
                v[i] = f.x;
                if (V > 1) v[i + (V > 1)] = f.y;
            }
        } else if (s[j] > kSafe) {
#pragma unroll
            for (int i = 0; i < V; ++i)
                if (fabsf(v[i]) > kTop) v[i] = copysignf(kTop, v[i]);
        }
        write<T, V>(out, at, count, v);
    }
}

template <int V, int ACT>
inline int grid_for(long long count, unsigned* grid) {
    const long long per = (long long)kThreads * kUnrollOf<ACT> * V, blocks = (count + per - 1) / per;
    if (blocks > 0x7fffffffLL) return fail(CNL_ERR_BAD_SHAPE, "count %lld is too large", count);
    *grid = (unsigned)blocks;
    return CNL_OK;
}

template <typename T, int FMT, int ACT>
int run_store(const void* x, void* y, unsigned char* codes, unsigned char* scales, long long count, cudaStream_t st) {
    constexpr int V = 16 / (int)sizeof(T);
    unsigned grid = 0;
    // one element a lane where a pointer is not aligned (a view that starts at an odd element)
    if (aligned16(x) && aligned16(y) && aligned16(codes)) {
        CNL_TRY((grid_for<V, ACT>(count, &grid)));
        store_kernel<T, V, FMT, ACT><<<grid, kThreads, 0, st>>>((const T*)x, (T*)y, codes, scales, count);
    } else {
        CNL_TRY((grid_for<1, ACT>(count, &grid)));
        store_kernel<T, 1, FMT, ACT><<<grid, kThreads, 0, st>>>((const T*)x, (T*)y, codes, scales, count);
    }
    return after_launch("ckpt8 store");
}

template <typename T, int FMT, int ACT>
int run_restore(const unsigned char* codes, const unsigned char* scales, const void* g, void* out, long long count, cudaStream_t st) {
    constexpr int V = 16 / (int)sizeof(T);
    unsigned grid = 0;
    if (aligned16(g) && aligned16(out) && aligned16(codes)) {
        CNL_TRY((grid_for<V, ACT>(count, &grid)));
        restore_kernel<T, V, FMT, ACT><<<grid, kThreads, 0, st>>>(codes, scales, (const T*)g, (T*)out, count);
    } else {
        CNL_TRY((grid_for<1, ACT>(count, &grid)));
        restore_kernel<T, 1, FMT, ACT><<<grid, kThreads, 0, st>>>(codes, scales, (const T*)g, (T*)out, count);
    }
    return after_launch("ckpt8 restore");
}

int check(long long count, int dtype, int fmt) {
    if (count < 0) return fail(CNL_ERR_BAD_SHAPE, "count %lld is negative", count);
    CNL_TRY(check_dtype(dtype));
    if (fmt != CNL_CKPT_INT8 && fmt != CNL_CKPT_E4M3) return fail(CNL_ERR_BAD_OPTION, "fmt %d is not CNL_CKPT_INT8 or CNL_CKPT_E4M3", fmt);
    return CNL_OK;
}

int check_act(int act) {
    if (act != CNL_ACT_GELU && act != CNL_ACT_SILU) return fail(CNL_ERR_BAD_OPTION, "act %d is not CNL_ACT_GELU or CNL_ACT_SILU", act);
    return CNL_OK;
}

// F<T, FMT, ACT> for the run-time values
#define CNL_CKPT8_DISPATCH(F, ...)                                                                                      \
    do {                                                                                                                \
        const bool i8 = fmt == CNL_CKPT_INT8;                                                                           \
        if (dtype == CNL_F32) return i8 ? F<float, CNL_CKPT_INT8, ACT>(__VA_ARGS__) : F<float, CNL_CKPT_E4M3, ACT>(__VA_ARGS__);      \
        if (dtype == CNL_F16) return i8 ? F<__half, CNL_CKPT_INT8, ACT>(__VA_ARGS__) : F<__half, CNL_CKPT_E4M3, ACT>(__VA_ARGS__);    \
        return i8 ? F<__nv_bfloat16, CNL_CKPT_INT8, ACT>(__VA_ARGS__) : F<__nv_bfloat16, CNL_CKPT_E4M3, ACT>(__VA_ARGS__);            \
    } while (0)

template <int ACT>
int store_any(const void* x, void* y, unsigned char* codes, unsigned char* scales, long long count, int dtype, int fmt, cudaStream_t st) {
    CNL_CKPT8_DISPATCH(run_store, x, y, codes, scales, count, st);
}
template <int ACT>
int restore_any(const unsigned char* codes, const unsigned char* scales, const void* g, void* out, long long count, int dtype, int fmt, cudaStream_t st) {
    CNL_CKPT8_DISPATCH(run_restore, codes, scales, g, out, count, st);
}

}  // namespace ckpt8
}  // namespace cnl

using namespace cnl;

extern "C" int cnl_ckpt8_store(const void* x, unsigned char* codes, unsigned char* scales, long long count, int dtype, int fmt, void* stream) {
    CNL_TRY(ckpt8::check(count, dtype, fmt));
    if (count == 0) return CNL_OK;
    if (!x || !codes || !scales) return fail(CNL_ERR_NULL, "null pointer argument");
    return ckpt8::store_any<0>(x, nullptr, codes, scales, count, dtype, fmt, static_cast<cudaStream_t>(stream));
}

extern "C" int cnl_ckpt8_restore(const unsigned char* codes, const unsigned char* scales, void* x, long long count, int dtype, int fmt, void* stream) {
    CNL_TRY(ckpt8::check(count, dtype, fmt));
    if (count == 0) return CNL_OK;
    if (!x || !codes || !scales) return fail(CNL_ERR_NULL, "null pointer argument");
    return ckpt8::restore_any<0>(codes, scales, nullptr, x, count, dtype, fmt, static_cast<cudaStream_t>(stream));
}

extern "C" int cnl_act8_forward(const void* x, void* y, unsigned char* codes, unsigned char* scales, long long count, int dtype, int fmt, int act, void* stream) {
    CNL_TRY(ckpt8::check(count, dtype, fmt));
    CNL_TRY(ckpt8::check_act(act));
    if (count == 0) return CNL_OK;
    if (!x || !y || !codes != !scales) return fail(CNL_ERR_NULL, "null pointer argument");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (act == CNL_ACT_GELU) return ckpt8::store_any<CNL_ACT_GELU>(x, y, codes, scales, count, dtype, fmt, st);
    return ckpt8::store_any<CNL_ACT_SILU>(x, y, codes, scales, count, dtype, fmt, st);
}

extern "C" int cnl_act8_backward(const unsigned char* codes, const unsigned char* scales, const void* g_y, void* g_x, long long count, int dtype, int fmt, int act, void* stream) {
    CNL_TRY(ckpt8::check(count, dtype, fmt));
    CNL_TRY(ckpt8::check_act(act));
    if (count == 0) return CNL_OK;
    if (!codes || !scales || !g_y || !g_x) return fail(CNL_ERR_NULL, "null pointer argument");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (act == CNL_ACT_GELU) return ckpt8::restore_any<CNL_ACT_GELU>(codes, scales, g_y, g_x, count, dtype, fmt, st);
    return ckpt8::restore_any<CNL_ACT_SILU>(codes, scales, g_y, g_x, count, dtype, fmt, st);
}
