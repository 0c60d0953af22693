// Norms before and after a block, fused with the block's gate, residual scale and residual sum (sm_100a).
//
// With N(v; w, b) = v^ w + b, v^ = (v - mu) r over the d channels of a row (rms: mu = 0, r = (mean v^2 + eps)^-1/2; layer: the
// centred form):
//     y = x + s act(z) N(u; w2, b2)              after a block with output u, residual stream x, gate z, scale s
//     h = N(y; w1, b1)                           before the next block, of y as computed (not as rounded for storage)
// Backward, from (dy, dh): y is rebuilt from x, u, z with the saved statistics, so the pass reads the same tensors as the
// forward pass and rounds nothing in between:
//     t  = dy + B(dh w1, y^, r_y)                B(g, v^, r) = r (g - [mean g] - v^ mean(g v^))
//     dx = t,   du = B(t s a w2, u^, r_u),   dz = t s n a',   n = u^ w2 + b2, a = act(z)
//     dw1 = sum dh y^, db1 = sum dh;  A = sum t a u^, B = sum t a:  dw2 = s A, db2 = s B, ds = w2 A + b2 B
// so four column sums serve five vectors.  A gate of one row for a group of rows (one image) leaves a out of the sums, which
// are kept per group: dz_g = a' s (w2 A_g + b2 B_g) and A = sum_g a_g A_g.
//
// One pass: a row lies in the registers of tpr threads (8 channels each) from its loads to its stores, the statistics are
// fp32 and two-step (mean, then centred squares).  Column sums stay in a thread's registers over all rows it handles, are
// joined in a fixed order across the block and then, by a second small kernel, over the blocks: same bits every call.
#include <type_traits>

#include "blocknorm.cuh"

namespace cnl {
namespace bnorm {

// ---- eight channels of a row ------------------------------------------------------------------------------------
// VEC: channels 8 t .. 8 t + 7 as 16-byte vectors (d a multiple of 8, aligned rows); otherwise channels t, t + tpr, ...
template <typename T, bool VEC>
__device__ __forceinline__ void get(const T* __restrict__ row, const Args& a, int t, float (&v)[K]) {
    if constexpr (VEC) {
        if (t * K < a.d) {
            load_vec<T, K>(row + t * K, v);
        } else {
#pragma unroll
            for (int k = 0; k < K; ++k) v[k] = 0.0f;
        }
    } else {
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int c = t + k * a.tpr;
            v[k] = c < a.d ? to_f32(row[c]) : 0.0f;
        }
    }
}

template <typename T, bool VEC>
__device__ __forceinline__ void put(T* __restrict__ row, const Args& a, int t, const float (&v)[K]) {
    if constexpr (VEC) {
        if (t * K < a.d) store_vec<T, K>(row + t * K, v);
    } else {
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int c = t + k * a.tpr;
            if (c < a.d) row[c] = from_f32<T>(v[k]);
        }
    }
}

// A parameter vector: of the rows' type or fp32; a null pointer gives `other`.
template <typename T, bool VEC>
__device__ __forceinline__ void param(const void* p, const Args& a, int t, float other, float (&v)[K]) {
    if (!p) {
#pragma unroll
        for (int k = 0; k < K; ++k) v[k] = other;
    } else if (a.w_f32) {
        get<float, VEC>((const float*)p, a, t, v);
    } else {
        get<T, VEC>((const T*)p, a, t, v);
    }
}

template <bool VEC>
__device__ __forceinline__ bool has(const Args& a, int t, int k) { return VEC ? t * K < a.d : t + k * a.tpr < a.d; }

// 8-bit form of a row's channels (a block of 32 is four lanes of a VEC row, or one k of a warp otherwise)
template <bool VEC>
__device__ __forceinline__ void put_codes(unsigned char* __restrict__ codes, unsigned char* __restrict__ scales, const Args& a, int t,
                                          bool live, const float (&v)[K]) {
    if constexpr (VEC) {
        unsigned c[2];
        const int s = a.fmt == CNL_CKPT_INT8 ? ckpt8::encode<CNL_CKPT_INT8, 4, K>(v, c) : ckpt8::encode<CNL_CKPT_E4M3, 4, K>(v, c);
        if (live && t * K < a.d) {
            *reinterpret_cast<uint2*>(codes + t * K) = make_uint2(c[0], c[1]);
            if ((t & 3) == 0) scales[t >> 2] = ckpt8::scale_byte(s);
        }
    } else {
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const float one[1] = {v[k]};
            unsigned c[1];
            const int s = a.fmt == CNL_CKPT_INT8 ? ckpt8::encode<CNL_CKPT_INT8, 32, 1>(one, c) : ckpt8::encode<CNL_CKPT_E4M3, 32, 1>(one, c);
            const int col = t + k * a.tpr;
            if (live && col < a.d) {
                codes[col] = (unsigned char)c[0];
                if ((col & 31) == 0) scales[col >> 5] = ckpt8::scale_byte(s);
            }
        }
    }
}

template <bool VEC>
__device__ __forceinline__ void get_codes(const unsigned char* __restrict__ codes, const unsigned char* __restrict__ scales, const Args& a,
                                          int t, float (&v)[K]) {
    if constexpr (VEC) {
        if (t * K < a.d) {
            const uint2 q = __ldg(reinterpret_cast<const uint2*>(codes + t * K));
            const unsigned w[2] = {q.x, q.y};
            const int s = ckpt8::scale_exponent(__ldg(scales + (t >> 2)));
            if (a.fmt == CNL_CKPT_INT8) ckpt8::decode<CNL_CKPT_INT8, K>(w, s, v);
            else ckpt8::decode<CNL_CKPT_E4M3, K>(w, s, v);
        } else {
#pragma unroll
            for (int k = 0; k < K; ++k) v[k] = 0.0f;
        }
    } else {
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int c = t + k * a.tpr;
            v[k] = 0.0f;
            if (c < a.d) {
                const unsigned w[1] = {codes[c]};
                const int s = ckpt8::scale_exponent(scales[c >> 5]);
                float one[1];
                if (a.fmt == CNL_CKPT_INT8) ckpt8::decode<CNL_CKPT_INT8, 1>(w, s, one);
                else ckpt8::decode<CNL_CKPT_E4M3, 1>(w, s, one);
                v[k] = one[0];
            }
        }
    }
}

// ---- sums over a row --------------------------------------------------------------------------------------------
// WIDE: a row spans several warps, whose sums meet in shared memory (two buffers in turn, so one barrier a sum).
// The barrier is one of its own for every row slot of the block: rows do not wait for one another.
template <bool WIDE, int N>
__device__ __forceinline__ void row_sum(float (&v)[N], int tpr, float* __restrict__ sm, int& turn) {
    if constexpr (!WIDE) {
        for (int o = 1; o < tpr; o <<= 1) {
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
        }
    } else {
        const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, wpr = tpr >> 5;
        const int first = (int)threadIdx.x / tpr * wpr;                    // first warp of this row
        float* buf = sm + turn * (32 * 2);
        turn ^= 1;
#pragma unroll
        for (int i = 0; i < N; ++i) {
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
            if (lane == 0) buf[warp * 2 + i] = v[i];
        }
        asm volatile("bar.sync %0, %1;" ::"r"((int)threadIdx.x / tpr + 1), "r"(tpr) : "memory");
#pragma unroll
        for (int i = 0; i < N; ++i) {
            float p = lane < wpr ? buf[(first + lane) * 2 + i] : 0.0f;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) p += __shfl_xor_sync(0xffffffffu, p, o);
            v[i] = p;
        }
    }
}

// mu and r of a row; v is left centred.  Channels that the thread does not have stay 0.
template <bool VEC, bool WIDE>
__device__ __forceinline__ void center(float (&v)[K], const Args& a, int t, float* sm, int& turn, float& mu, float& r) {
    float s[1];
    mu = 0.0f;
    if (a.layer) {
        s[0] = 0.0f;
#pragma unroll
        for (int k = 0; k < K; ++k) s[0] += v[k];
        row_sum<WIDE, 1>(s, a.tpr, sm, turn);
        mu = s[0] * a.inv_d;
#pragma unroll
        for (int k = 0; k < K; ++k) v[k] = has<VEC>(a, t, k) ? v[k] - mu : 0.0f;
    }
    s[0] = 0.0f;
#pragma unroll
    for (int k = 0; k < K; ++k) s[0] = fmaf(v[k], v[k], s[0]);
    row_sum<WIDE, 1>(s, a.tpr, sm, turn);
    r = rsqrtf(fmaf(s[0], a.inv_d, a.eps));
}

// ---- forward ----------------------------------------------------------------------------------------------------
// Here without vectors: one element a lane and load, so that loads and conversions, not memory, are the bound.  Forward /
// backward: 21996 x 150 fp32 33 / 65 us, 61440 x 501 bf16 218 / 530 us (1.4 and 0.9 TB/s); with vectors, 3840 x 8192 fp32, 172 / 687 us
// (one block of 1024 threads an SM, whose row sums meet at a barrier, is all that the registers of such a row allow).
template <typename T, bool VEC, bool WIDE, int BLOCK>
__global__ void __launch_bounds__(BLOCK, BLOCK <= 256 ? 3 : 1) forward_kernel(const Args a) {
    __shared__ float sm[2 * 32 * 2];
    const int rpb = blockDim.x / a.tpr, slot = threadIdx.x / a.tpr, t = threadIdx.x - slot * a.tpr;
    const long long group = blockIdx.x / a.nb;
    const int j = blockIdx.x - (int)(group * a.nb);
    const long long begin = group * a.per + (long long)j * rpb, end = (group + 1) * a.per, step = (long long)a.nb * rpb;
    const int blocks = (a.d + 31) >> 5;
    int turn = 0;
    for (long long base = begin; base < end; base += step) {
        const long long row = base + slot;
        const bool live = row < end;
        const long long off = (live ? row : base) * a.d;
        float y[K], u[K], z[K];
        get<T, VEC>((const T*)a.x + off, a, t, y);
        if (a.u) get<T, VEC>((const T*)a.u + off, a, t, u);
        if (a.gate_full) get<T, VEC>((const T*)a.gate + off, a, t, z);
        if (a.gate_group) get<T, VEC>((const T*)a.gate + group * a.d, a, t, z);
        float mu_u = 0.0f, r_u = 0.0f, mu_y = 0.0f, r_y = 0.0f;
        if (a.codes) {
            const long long n = a.rows * a.d, nb = a.rows * blocks, so = (live ? row : base) * blocks;
            if (a.w1) put_codes<VEC>(a.codes + off, a.scales + so, a, t, live, y);
            if (a.u) put_codes<VEC>(a.codes + n + off, a.scales + nb + so, a, t, live, u);
            if (a.gate_full) put_codes<VEC>(a.codes + 2 * n + off, a.scales + 2 * nb + so, a, t, live, z);
        }
        if (a.u) {
            center<VEC, WIDE>(u, a, t, sm, turn, mu_u, r_u);
            float w[K], b[K], s[K];
            param<T, VEC>(a.w2, a, t, 0.0f, w);
            param<T, VEC>(a.b2, a, t, 0.0f, b);
            param<T, VEC>(a.scale, a, t, 1.0f, s);
            const bool gated = a.gate_full || a.gate_group;
#pragma unroll
            for (int k = 0; k < K; ++k) {
                float m = s[k];
                if (gated) m *= a.sigmoid ? sigmoid(z[k]) : z[k];
                y[k] = fmaf(m, fmaf(u[k] * r_u, w[k], b[k]), y[k]);
                if (!has<VEC>(a, t, k)) y[k] = 0.0f;
            }
            if (live) put<T, VEC>((T*)a.y + off, a, t, y);
        }
        if (a.w1) {
            center<VEC, WIDE>(y, a, t, sm, turn, mu_y, r_y);
            float w[K], b[K];
            param<T, VEC>(a.w1, a, t, 0.0f, w);
            param<T, VEC>(a.b1, a, t, 0.0f, b);
#pragma unroll
            for (int k = 0; k < K; ++k) y[k] = fmaf(y[k] * r_y, w[k], b[k]);
            if (live) put<T, VEC>((T*)a.h + off, a, t, y);
        }
        if (a.stats && live && t == 0) a.stats[row] = make_float4(mu_u, r_u, mu_y, r_y);
    }
}

// ---- backward ---------------------------------------------------------------------------------------------------
template <typename T, bool VEC, bool WIDE, int BLOCK>
__global__ void __launch_bounds__(BLOCK, BLOCK <= 256 ? 2 : 1) backward_kernel(const Args a) {
    constexpr bool kSharedSums = BLOCK > 256;                              // rows of up to 1024 threads: 64 registers each, sums in shared memory
    extern __shared__ float dyn[];
    __shared__ float sm[2 * 32 * 2];
    const int rpb = blockDim.x / a.tpr, slot = threadIdx.x / a.tpr, t = threadIdx.x - slot * a.tpr;
    const long long group = blockIdx.x / a.nb;
    const int j = blockIdx.x - (int)(group * a.nb);
    const long long begin = group * a.per + (long long)j * rpb, end = (group + 1) * a.per, step = (long long)a.nb * rpb;
    const int blocks = (a.d + 31) >> 5;
    const long long n = a.rows * a.d, nb = a.rows * blocks;
    float acc[kSharedSums ? 1 : kSums][K];
    if constexpr (kSharedSums) {
        for (int i = 0; i < kSums * K; ++i) dyn[i * blockDim.x + threadIdx.x] = 0.0f;
    } else {
#pragma unroll
        for (int i = 0; i < kSums; ++i)
#pragma unroll
            for (int k = 0; k < K; ++k) acc[i][k] = 0.0f;
    }
    auto add = [&](int i, int k, float v) {
        if constexpr (kSharedSums) dyn[(i * K + k) * blockDim.x + threadIdx.x] += v;
        else acc[i][k] += v;
    };
    int turn = 0;
    for (long long base = begin; base < end; base += step) {
        const long long row = base + slot;
        const bool live = row < end;
        const long long at = live ? row : base, off = at * a.d, so = at * blocks;
        const float4 st = __ldg(a.stats + at);
        float g[K], y[K], u[K], z[K], dh[K];
        if (a.fmt) {
            if (a.dh) get_codes<VEC>(a.codes + off, a.scales + so, a, t, y);
            if (a.u) get_codes<VEC>(a.codes + n + off, a.scales + nb + so, a, t, u);
            if (a.gate_full) get_codes<VEC>(a.codes + 2 * n + off, a.scales + 2 * nb + so, a, t, z);
        } else {
            if (a.dh) get<T, VEC>((const T*)a.x + off, a, t, y);
            if (a.u) get<T, VEC>((const T*)a.u + off, a, t, u);
            if (a.gate_full) get<T, VEC>((const T*)a.gate + off, a, t, z);
        }
        if (a.dy) get<T, VEC>((const T*)a.dy + off, a, t, g);
        if (a.dh) get<T, VEC>((const T*)a.dh + off, a, t, dh);
        if (a.gate_group) get<T, VEC>((const T*)a.gate + group * a.d, a, t, z);
        if (!a.dy) {
#pragma unroll
            for (int k = 0; k < K; ++k) g[k] = 0.0f;
        }
        float w[K], b[K], s[K], m[K], slope[K];                            // m = s a, slope = s a' (of a full gate)
        if (a.u) {
            param<T, VEC>(a.w2, a, t, 0.0f, w);
            param<T, VEC>(a.b2, a, t, 0.0f, b);
            param<T, VEC>(a.scale, a, t, 1.0f, s);
#pragma unroll
            for (int k = 0; k < K; ++k) {
                u[k] = (u[k] - st.x) * st.y;                               // u^
                float act = 1.0f, da = 0.0f;
                if (a.gate_full || a.gate_group) {
                    act = a.sigmoid ? sigmoid(z[k]) : z[k];
                    da = a.sigmoid ? act * (1.0f - act) : 1.0f;
                }
                z[k] = act;
                m[k] = s[k] * act;
                slope[k] = s[k] * da;
            }
        }
        if (a.dh) {
            float w1[K], sum[2] = {0.0f, 0.0f};
            param<T, VEC>(a.w1, a, t, 0.0f, w1);
#pragma unroll
            for (int k = 0; k < K; ++k) {
                if (a.u) y[k] = fmaf(m[k], fmaf(u[k], w[k], b[k]), y[k]);
                y[k] = (y[k] - st.z) * st.w;                               // y^
                if (live) { add(2, k, dh[k] * y[k]); add(3, k, dh[k]); }
                dh[k] *= w1[k];
                sum[0] = fmaf(dh[k], y[k], sum[0]);
                sum[1] += dh[k];
            }
            row_sum<WIDE, 2>(sum, a.tpr, sm, turn);
            const float s1 = sum[0] * a.inv_d, s0 = a.layer ? sum[1] * a.inv_d : 0.0f;
#pragma unroll
            for (int k = 0; k < K; ++k) g[k] = fmaf(st.w, dh[k] - s0 - y[k] * s1, g[k]);
        }
        if (live && a.dx) put<T, VEC>((T*)a.dx + off, a, t, g);
        if (a.u) {
            float dn[K], sum[2] = {0.0f, 0.0f};
#pragma unroll
            for (int k = 0; k < K; ++k) {
                const float ta = a.gate_group ? g[k] : g[k] * z[k];
                if (live && has<VEC>(a, t, k)) { add(0, k, ta * u[k]); add(1, k, ta); }
                if (a.gate_full) z[k] = g[k] * slope[k] * fmaf(u[k], w[k], b[k]);
                dn[k] = g[k] * m[k] * w[k];
                sum[0] = fmaf(dn[k], u[k], sum[0]);
                sum[1] += dn[k];
            }
            row_sum<WIDE, 2>(sum, a.tpr, sm, turn);
            const float s1 = sum[0] * a.inv_d, s0 = a.layer ? sum[1] * a.inv_d : 0.0f;
#pragma unroll
            for (int k = 0; k < K; ++k) dn[k] = st.y * (dn[k] - s0 - u[k] * s1);
            if (live && a.du) put<T, VEC>((T*)a.du + off, a, t, dn);
            if (live && a.gate_full && a.dgate) put<T, VEC>((T*)a.dgate + off, a, t, z);
        }
    }
    // sums over the block's rows: lanes of a warp that hold the same channels, then the row slots in order
    float* out = a.partial + (long long)blockIdx.x * kSums * a.d;
    if constexpr (kSharedSums) {                                           // one row a block
        for (int i = 0; i < kSums; ++i)
#pragma unroll
            for (int k = 0; k < K; ++k) {
                const int c = VEC ? t * K + k : t + k * a.tpr;
                if (slot == 0 && c < a.d) out[i * a.d + c] = dyn[(i * K + k) * blockDim.x + threadIdx.x];
            }
    } else {
        const int unit = WIDE ? a.tpr : 32, units = WIDE ? rpb : blockDim.x >> 5;
#pragma unroll
        for (int i = 0; i < kSums; ++i) {
#pragma unroll
            for (int k = 0; k < K; ++k) {
                float v = acc[i][k];
                if constexpr (!WIDE)
                    for (int o = a.tpr; o < 32; o <<= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
                dyn[k * blockDim.x + threadIdx.x] = v;
            }
            __syncthreads();
            if (threadIdx.x < a.tpr) {
#pragma unroll
                for (int k = 0; k < K; ++k) {
                    const int c = VEC ? t * K + k : t + k * a.tpr;
                    float v = 0.0f;
                    for (int q = 0; q < units; ++q) v += dyn[k * blockDim.x + q * unit + threadIdx.x];
                    if (c < a.d) out[i * a.d + c] = v;
                }
            }
            __syncthreads();
        }
    }
}

// ---- column sums over the blocks --------------------------------------------------------------------------------
struct SumArgs {
    const float* partial;                         // [groups * nb][4][d]
    float* per_group;                             // [groups][4][d] when there are several groups
    const void *gate, *scale, *w2, *b2;
    void *dgate, *dscale, *dw2, *db2, *dw1, *db1;
    int d, nb, groups, gate_group, sigmoid, w_f32, need_b;
};

template <typename T>
__device__ __forceinline__ float one_param(const void* p, int w_f32, int c, float other) {
    return !p ? other : w_f32 ? ((const float*)p)[c] : to_f32(((const T*)p)[c]);
}
template <typename T>
__device__ __forceinline__ void put_param(void* p, int w_f32, int c, float v) {
    if (!p) return;
    if (w_f32) ((float*)p)[c] = v;
    else ((T*)p)[c] = from_f32<T>(v);
}

// 32 channels x 32 threads over `count` rows of [4][d] sums; the threads' sums are joined in order, in 64 bits
__device__ __forceinline__ void column_sums(const float* src, long long count, int d, int c, int need_b, double (*sm)[32][33], double (&v)[kSums]) {
    double s[kSums] = {0.0, 0.0, 0.0, 0.0};
    if (c < d) {
        constexpr int kAhead = 4;                                          // rows whose sums are asked for together
        for (long long p0 = threadIdx.y; p0 < count; p0 += 32 * kAhead) {
            float f[kAhead][kSums];
#pragma unroll
            for (int k = 0; k < kAhead; ++k)
#pragma unroll
                for (int i = 0; i < kSums; ++i) {                          // B and db1 are not written where nothing asks for them
                    const long long p = p0 + 32 * k;
                    f[k][i] = p < count && (need_b || !(i & 1)) ? src[(p * kSums + i) * d + c] : 0.0f;
                }
#pragma unroll
            for (int k = 0; k < kAhead; ++k)
#pragma unroll
                for (int i = 0; i < kSums; ++i) s[i] += (double)f[k][i];
        }
    }
#pragma unroll
    for (int i = 0; i < kSums; ++i) sm[i][threadIdx.y][threadIdx.x] = s[i];
    __syncthreads();
    for (int half = 16; half > 0; half >>= 1) {
        if (threadIdx.y < half)
#pragma unroll
            for (int i = 0; i < kSums; ++i) sm[i][threadIdx.y][threadIdx.x] += sm[i][threadIdx.y + half][threadIdx.x];
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < kSums; ++i) v[i] = sm[i][0][threadIdx.x];
}

template <typename T>
__device__ __forceinline__ void finish(const SumArgs& a, int c, float A, float B, float dw1, float db1) {
    const float s = one_param<T>(a.scale, a.w_f32, c, 1.0f), w = one_param<T>(a.w2, a.w_f32, c, 0.0f), b = one_param<T>(a.b2, a.w_f32, c, 0.0f);
    put_param<T>(a.dw2, a.w_f32, c, s * A);
    put_param<T>(a.db2, a.w_f32, c, s * B);
    put_param<T>(a.dscale, a.w_f32, c, fmaf(w, A, b * B));
    put_param<T>(a.dw1, a.w_f32, c, dw1);
    put_param<T>(a.db1, a.w_f32, c, db1);
}

template <typename T>
__global__ void __launch_bounds__(1024) sum_blocks_kernel(const SumArgs a) {
    __shared__ double sm[kSums][32][33];
    const int c = blockIdx.x * 32 + threadIdx.x;
    const long long group = blockIdx.y;
    double v[kSums];
    column_sums(a.partial + group * a.nb * kSums * a.d, a.nb, a.d, c, a.need_b, sm, v);
    if (threadIdx.y != 0 || c >= a.d) return;
    float A = (float)v[0], B = (float)v[1];
    if (a.gate_group) {
        const float z = to_f32(((const T*)a.gate)[group * a.d + c]);
        const float act = a.sigmoid ? sigmoid(z) : z, da = a.sigmoid ? act * (1.0f - act) : 1.0f;
        const float s = one_param<T>(a.scale, a.w_f32, c, 1.0f), w = one_param<T>(a.w2, a.w_f32, c, 0.0f), b = one_param<T>(a.b2, a.w_f32, c, 0.0f);
        if (a.dgate) ((T*)a.dgate)[group * a.d + c] = from_f32<T>(da * s * fmaf(w, A, b * B));
        A *= act;
        B *= act;
    }
    if (a.groups == 1) {
        finish<T>(a, c, A, B, (float)v[2], (float)v[3]);
    } else {
        float* out = a.per_group + group * kSums * a.d + c;
        out[0] = A;
        out[a.d] = B;
        out[2 * a.d] = (float)v[2];
        out[3 * a.d] = (float)v[3];
    }
}

template <typename T>
__global__ void __launch_bounds__(1024) sum_groups_kernel(const SumArgs a) {
    __shared__ double sm[kSums][32][33];
    const int c = blockIdx.x * 32 + threadIdx.x;
    double v[kSums];
    column_sums(a.per_group, a.groups, a.d, c, a.need_b, sm, v);
    if (threadIdx.y == 0 && c < a.d) finish<T>(a, c, (float)v[0], (float)v[1], (float)v[2], (float)v[3]);
}

// ---- launch -----------------------------------------------------------------------------------------------------
// threads of a row: a power of two up to a warp, whole warps above; unaligned rows take whole warps
inline int plan(long long rows, int d, long long groups, bool vec, int blocks_wanted, Plan* p) {
    const int need = (d + K - 1) / K;
    if (need > 32) p->tpr = (need + 31) / 32 * 32;
    else {
        p->tpr = vec ? 4 : 32;
        while (p->tpr < need) p->tpr <<= 1;
    }
    p->block = p->tpr <= 256 ? 256 / p->tpr * p->tpr : p->tpr;
    p->rpb = p->block / p->tpr;
    p->groups = groups;
    const long long per = rows / groups, most = (per + p->rpb - 1) / p->rpb;
    long long nb = blocks_wanted / groups;
    nb = nb < 1 ? 1 : nb;
    p->nb = (int)(nb < most ? nb : most < 1 ? 1 : most);
    if (groups * p->nb > 0x7fffffffLL) return fail(CNL_ERR_BAD_SHAPE, "%lld groups are too many", groups);
    return CNL_OK;
}

inline int check(long long rows, int d, long long groups, int dtype, int wdtype, int fmt) {
    if (rows < 0 || d < 1 || d > kMaxD) return fail(CNL_ERR_BAD_SHAPE, "rows %lld, d %d: rows must not be negative and d within 1..%d", rows, d, kMaxD);
    if (groups < 1 || rows % groups) return fail(CNL_ERR_BAD_SHAPE, "%lld groups do not divide %lld rows", groups, rows);
    CNL_TRY(check_dtype(dtype));
    CNL_TRY(check_dtype(wdtype));
    if (wdtype != dtype && wdtype != CNL_F32) return fail(CNL_ERR_BAD_OPTION, "parameters must be of the rows' type or fp32");
    if (fmt != CNL_CKPT_NONE && fmt != CNL_CKPT_INT8 && fmt != CNL_CKPT_E4M3) return fail(CNL_ERR_BAD_OPTION, "fmt %d is not a checkpoint format", fmt);
    return CNL_OK;
}

inline bool aligned_all(const void* const* p, int n) {
    for (int i = 0; i < n; ++i)
        if (!aligned16(p[i])) return false;
    return true;
}

// Rows without vectors, or over kVecMaxD channels.
template <typename T, bool VEC>
int launch_forward(const Args& a, const Plan& p, cudaStream_t st) {
    const unsigned grid = (unsigned)(p.groups * p.nb);
    if constexpr (VEC) forward_kernel<T, true, true, 1024><<<grid, p.block, 0, st>>>(a);
    else if (p.tpr <= 32) forward_kernel<T, false, false, 256><<<grid, p.block, 0, st>>>(a);
    else if (p.tpr <= 256) forward_kernel<T, false, true, 256><<<grid, p.block, 0, st>>>(a);
    else forward_kernel<T, false, true, 1024><<<grid, p.block, 0, st>>>(a);
    return after_launch("blocknorm forward");
}

template <typename T, bool VEC>
int launch_backward(const Args& a, const Plan& p, cudaStream_t st) {
    const unsigned grid = (unsigned)(p.groups * p.nb);
    const int join = K * p.block * (int)sizeof(float);                   // the block's join of one of the four sums
    const int bytes = p.tpr <= 256 ? join : kSums * join;
    void (*kernel)(const Args);
    if constexpr (VEC) kernel = backward_kernel<T, true, true, 1024>;
    else kernel = p.tpr <= 32 ? backward_kernel<T, false, false, 256> : p.tpr <= 256 ? backward_kernel<T, false, true, 256> : backward_kernel<T, false, true, 1024>;
    CNL_TRY(ensure_dynamic_smem(kernel, bytes));
    kernel<<<grid, p.block, bytes, st>>>(a);
    return after_launch("blocknorm backward");
}

template <typename T>
int sums(const SumArgs& s, cudaStream_t st) {
    const unsigned cols = (unsigned)((s.d + 31) / 32);
    for (int g0 = 0; g0 < s.groups; g0 += 65535) {                     // the y extent of a grid
        SumArgs part = s;
        const int n = s.groups - g0 < 65535 ? s.groups - g0 : 65535;
        const long long skip = (long long)g0 * s.d;
        part.partial += skip * s.nb * kSums;
        if (s.per_group) part.per_group += skip * kSums;
        if (s.gate_group) {
            part.gate = (const T*)s.gate + skip;
            if (s.dgate) part.dgate = (T*)s.dgate + skip;
        }
        sum_blocks_kernel<T><<<dim3(cols, (unsigned)n), dim3(32, 32), 0, st>>>(part);
        CNL_TRY(after_launch("blocknorm column sums"));
    }
    if (s.groups > 1) {
        sum_groups_kernel<T><<<cols, dim3(32, 32), 0, st>>>(s);
        CNL_TRY(after_launch("blocknorm group sums"));
    }
    return CNL_OK;
}

// blocks of the backward grid: two of 256 threads or one of up to 1024 an SM
inline int backward_blocks(int d, int* out) {
    int sms = 0;
    CNL_TRY(sm_count(&sms));
    *out = d > 256 * K ? sms : 2 * sms;
    return CNL_OK;
}

}  // namespace bnorm
}  // namespace cnl

using namespace cnl;
using namespace cnl::bnorm;

extern "C" long long cnl_blocknorm_scratch_bytes(long long rows, int d, long long groups) {
    int want = 0;
    if (rows < 0 || d < 1 || groups < 1 || backward_blocks(d, &want) != CNL_OK) return 0;
    Plan p;
    long long most = 0;
    for (int vec = 0; vec < 2; ++vec) {
        if (plan(rows, d, groups, vec, want, &p) != CNL_OK) return 0;
        most = p.nb > most ? p.nb : most;
    }
    return (groups * most + (groups > 1 ? groups : 0)) * kSums * d * (long long)sizeof(float);
}

extern "C" int cnl_blocknorm_forward(const void* x, const void* u, const void* gate, const void* scale, const void* w_post, const void* b_post,
                                     const void* w_pre, const void* b_pre, void* y, void* h, float* stats, unsigned char* codes,
                                     unsigned char* scales, long long rows, int d, long long groups, int gate_mode, int sigmoid_gate, int layer,
                                     float eps, int dtype, int wdtype, int fmt, void* stream) {
    CNL_TRY(check(rows, d, groups, dtype, wdtype, fmt));
    if (rows == 0) return CNL_OK;
    if (!x || (u && (!w_post || !y)) || (w_pre && !h) || (!u && !w_pre) || (fmt && (!codes || !scales)) || (gate_mode && (!u || !gate)))
        return fail(CNL_ERR_NULL, "null pointer argument");
    if (gate_mode < 0 || gate_mode > 2) return fail(CNL_ERR_BAD_OPTION, "gate_mode %d is not 0, 1 or 2", gate_mode);
    Args a = {};
    a.x = x; a.u = u; a.gate = gate; a.scale = scale; a.w2 = w_post; a.b2 = b_post; a.w1 = w_pre; a.b1 = b_pre;
    a.y = y; a.h = h; a.stats = reinterpret_cast<float4*>(stats);
    a.codes = fmt ? codes : nullptr; a.scales = scales;
    const void* all[] = {x, u, gate, scale, w_post, b_post, w_pre, b_pre, y, h, stats, codes};
    const bool vec = d % K == 0 && aligned_all(all, 12);
    if (!aligned16(stats)) return fail(CNL_ERR_BAD_SHAPE, "stats must be 16-byte aligned");
    int sms = 0;
    CNL_TRY(sm_count(&sms));
    Plan p;
    CNL_TRY(plan(rows, d, gate_mode == 2 ? groups : 1, vec, d > 256 * K ? sms : vec && (b_post || b_pre) ? 2 * sms : 3 * sms, &p));      // as many blocks as are resident
    a.rows = rows; a.per = rows / p.groups; a.d = d; a.tpr = p.tpr; a.nb = p.nb; a.eps = eps; a.inv_d = 1.0f / (float)d;
    a.layer = layer; a.gate_full = gate_mode == 1; a.gate_group = gate_mode == 2; a.sigmoid = sigmoid_gate;
    a.w_f32 = wdtype == CNL_F32; a.fmt = fmt;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (vec && d <= kVecMaxD) return run_forward_vec(a, p, dtype, st);
    if (dtype == CNL_F32) return vec ? launch_forward<float, true>(a, p, st) : launch_forward<float, false>(a, p, st);
    if (dtype == CNL_F16) return vec ? launch_forward<__half, true>(a, p, st) : launch_forward<__half, false>(a, p, st);
    return vec ? launch_forward<__nv_bfloat16, true>(a, p, st) : launch_forward<__nv_bfloat16, false>(a, p, st);
}

extern "C" int cnl_blocknorm_backward(const void* x, const void* u, const void* gate, const unsigned char* codes, const unsigned char* scales,
                                      const float* stats, const void* scale, const void* w_post, const void* b_post, const void* w_pre,
                                      const void* b_pre, const void* g_y, const void* g_h, void* g_x, void* g_u, void* g_gate, void* g_scale,
                                      void* g_w_post, void* g_b_post, void* g_w_pre, void* g_b_pre, void* scratch, long long rows, int d,
                                      long long groups, int gate_mode, int sigmoid_gate, int layer, int dtype, int wdtype, int fmt, void* stream) {
    CNL_TRY(check(rows, d, groups, dtype, wdtype, fmt));
    if (gate_mode < 0 || gate_mode > 2) return fail(CNL_ERR_BAD_OPTION, "gate_mode %d is not 0, 1 or 2", gate_mode);
    if (groups > 0x7fffffffLL) return fail(CNL_ERR_BAD_SHAPE, "%lld groups are too many", groups);
    const bool post = w_post != nullptr;
    if (!scratch || (!post && !w_pre) || (gate_mode == 2 && !gate) || (g_h && !w_pre)) return fail(CNL_ERR_NULL, "null pointer argument");
    if (rows > 0) {
        if (!stats || (fmt && (!codes || !scales)) || (!fmt && post && !u) || (!fmt && g_h && !x) || (!fmt && gate_mode == 1 && !gate))
            return fail(CNL_ERR_NULL, "null pointer argument");
    }
    Args a = {};
    // with codes the tensors themselves are not read; `u` then only says that there is a block output
    a.x = x; a.u = post ? (fmt ? (const void*)codes : u) : nullptr; a.gate = gate;
    a.scale = scale; a.w2 = w_post; a.b2 = b_post; a.w1 = w_pre; a.b1 = b_pre;
    a.stats = reinterpret_cast<float4*>(const_cast<float*>(stats));
    a.codes = const_cast<unsigned char*>(codes); a.scales = const_cast<unsigned char*>(scales);
    a.dy = g_y; a.dh = g_h; a.dx = g_x; a.du = g_u; a.dgate = gate_mode == 1 ? g_gate : nullptr;
    a.partial = static_cast<float*>(scratch);
    const void* all[] = {x, u, gate, scale, w_post, b_post, w_pre, b_pre, g_y, g_h, g_x, g_u, gate_mode == 1 ? g_gate : nullptr, codes};
    const bool vec = d % K == 0 && aligned_all(all, 14);
    if (!aligned16(stats)) return fail(CNL_ERR_BAD_SHAPE, "stats must be 16-byte aligned");
    int want = 0;
    CNL_TRY(backward_blocks(d, &want));
    Plan p;
    CNL_TRY(plan(rows, d, gate_mode == 2 ? groups : 1, vec, want, &p));
    a.rows = rows; a.per = rows / p.groups; a.d = d; a.tpr = p.tpr; a.nb = p.nb; a.inv_d = 1.0f / (float)d;
    a.layer = layer; a.gate_full = gate_mode == 1; a.gate_group = gate_mode == 2; a.sigmoid = sigmoid_gate;
    a.w_f32 = wdtype == CNL_F32; a.fmt = fmt;
    a.need_b = b_post || b_pre || g_b_post || g_b_pre;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (rows > 0) {
        if (vec && d <= kVecMaxD) CNL_TRY(run_backward_vec(a, p, dtype, st));
        else if (dtype == CNL_F32) CNL_TRY((vec ? launch_backward<float, true>(a, p, st) : launch_backward<float, false>(a, p, st)));
        else if (dtype == CNL_F16) CNL_TRY((vec ? launch_backward<__half, true>(a, p, st) : launch_backward<__half, false>(a, p, st)));
        else CNL_TRY((vec ? launch_backward<__nv_bfloat16, true>(a, p, st) : launch_backward<__nv_bfloat16, false>(a, p, st)));
    }
    SumArgs s = {};
    s.partial = a.partial; s.per_group = a.partial + (long long)p.groups * p.nb * kSums * d;
    s.gate = gate; s.scale = scale; s.w2 = w_post; s.b2 = b_post;
    s.dgate = gate_mode == 2 ? g_gate : nullptr; s.dscale = g_scale; s.dw2 = g_w_post; s.db2 = g_b_post; s.dw1 = g_w_pre; s.db1 = g_b_pre;
    s.d = d; s.nb = rows > 0 ? p.nb : 0; s.groups = (int)p.groups; s.gate_group = gate_mode == 2; s.sigmoid = sigmoid_gate; s.w_f32 = a.w_f32; s.need_b = a.need_b;
    if (dtype == CNL_F32) return sums<float>(s, st);
    if (dtype == CNL_F16) return sums<__half>(s, st);
    return sums<__nv_bfloat16>(s, st);
}
