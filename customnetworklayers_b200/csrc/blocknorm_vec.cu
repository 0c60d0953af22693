// Block norms on rows that are 16-byte vectors: d a multiple of 8, at most 4096 (formulas: blocknorm.cu).
//
// HBM bound: 10 bytes an element forward and 16 backward with a full gate in 16 bits, which at 6.5 TB/s leaves an SM some 55
// and 90 issue slots (of 128 lanes) an element and clock; so what the kernels are built for is few instructions.  A thread
// keeps 8 channels in pairs (packed fp32 arithmetic takes two a slot), the parameters of its channels in registers, folded
// (s w and s b, since s, w, b only appear so), and rows arrive by cp.async in shared-memory slots that belong to one thread
// each: it waits for its own copies, needs no barrier, and STAGES - 1 rows are under way while one is worked on.
// 61440 x 512 bf16 with a full gate: rms forward 60 us (5.2 TB/s, 0.8 of a copy), layer norm with biases 84 us (two blocks an SM
// instead of three; three with spills 90); backward 110 us without biases (4.6 TB/s), with them 160 and 167 us (3.0 TB/s); with
// 8-bit checkpoints and biases 117 and 187 us.  Wide or narrow rows run alike (with biases, 32: 64 and 153, 4096: 74 and 196 us for as many elements).
// fp32 with a full gate, rms: 152 and 261 us (4.1 and 3.9 TB/s; two rows under way instead of three), 30720 x 1024 150 and 265 us.  A norm
// alone: bf16 34 and 71 us, fp32 66 and 112 us.  Instructions issue on half of the cycles at 16
// warps an SM; mean and squares in one way through the row instead of two left all of these times as they are.
#include "blocknorm.cuh"

namespace cnl {
namespace bnorm {

constexpr int kStages16 = 3, kStages32 = 2;              // rows under way in shared memory, and the one in hand

__device__ __forceinline__ float2 f2(float v) { return make_float2(v, v); }

// ---- slots --------------------------------------------------------------------------------------------------------
template <typename T, int TENSORS, int BLOCK>
struct Slots {
    static constexpr int kStages = sizeof(T) == 4 ? kStages32 : kStages16;
    static constexpr int kParts = (int)sizeof(T) / 2;    // 16-byte parts of a thread's 8 channels
    static constexpr int kTensor = kParts * BLOCK * 16, kStage = TENSORS * kTensor, kBytes = kStages * kStage;
    unsigned at;                                         // this thread's first slot, as a shared-memory address

    __device__ __forceinline__ void ask(unsigned stage, int tensor, const T* p) const {
#pragma unroll
        for (int i = 0; i < kParts; ++i)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(at + stage + tensor * kTensor + i * BLOCK * 16), "l"(reinterpret_cast<const char*>(p) + 16 * i) : "memory");
    }
    __device__ __forceinline__ void ask_codes(unsigned stage, int tensor, const unsigned char* p) const {
        asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(at + stage + tensor * kTensor), "l"(p) : "memory");
    }
    __device__ __forceinline__ static void close() { asm volatile("cp.async.commit_group;" ::: "memory"); }
    __device__ __forceinline__ static void wait() { asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory"); }

    __device__ __forceinline__ void take(unsigned stage, int tensor, float2 (&v)[4]) const {
#pragma unroll
        for (int i = 0; i < kParts; ++i) {
            unsigned w[4];
            asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(at + stage + tensor * kTensor + i * BLOCK * 16) : "memory");
            if constexpr (kParts == 2) {
                v[2 * i] = make_float2(__uint_as_float(w[0]), __uint_as_float(w[1]));
                v[2 * i + 1] = make_float2(__uint_as_float(w[2]), __uint_as_float(w[3]));
            } else {
#pragma unroll
                for (int k = 0; k < 4; ++k) v[k] = unpack2(w[k], T());
            }
        }
    }
    __device__ __forceinline__ void take_codes(unsigned stage, int tensor, int s, int fmt, float2 (&v)[4]) const {
        unsigned w[2];
        asm volatile("ld.shared.v2.b32 {%0,%1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(at + stage + tensor * kTensor) : "memory");
        float f[8];
        if (fmt == CNL_CKPT_INT8) ckpt8::decode<CNL_CKPT_INT8, 8>(w, s, f);
        else ckpt8::decode<CNL_CKPT_E4M3, 8>(w, s, f);
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = make_float2(f[2 * k], f[2 * k + 1]);
    }
};

template <typename T>
__device__ __forceinline__ void put(T* p, const float2 (&v)[4]) {
    if constexpr (sizeof(T) == 4) {
        reinterpret_cast<float4*>(p)[0] = make_float4(v[0].x, v[0].y, v[1].x, v[1].y);
        reinterpret_cast<float4*>(p)[1] = make_float4(v[2].x, v[2].y, v[3].x, v[3].y);
    } else {
        *reinterpret_cast<uint4*>(p) = make_uint4(pack2<T>(v[0].x, v[0].y), pack2<T>(v[1].x, v[1].y), pack2<T>(v[2].x, v[2].y), pack2<T>(v[3].x, v[3].y));
    }
}

// 8 channels of a vector in the rows' type or (wide) fp32; `other` for a null pointer
template <typename T>
__device__ __forceinline__ void vector8(const void* p, int wide, int c, float other, float2 (&v)[4]) {
    float f[8];
    if (!p) {
#pragma unroll
        for (int k = 0; k < 8; ++k) f[k] = other;
    } else if (wide) {
        load_vec<float, 8>((const float*)p + c, f);
    } else {
        load_vec<T, 8>((const T*)p + c, f);
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = make_float2(f[2 * k], f[2 * k + 1]);
}

__device__ __forceinline__ void put_codes(unsigned char* codes, unsigned char* scale, int fmt, bool on, bool first, const float2 (&v)[4]) {
    const float f[8] = {v[0].x, v[0].y, v[1].x, v[1].y, v[2].x, v[2].y, v[3].x, v[3].y};
    unsigned c[2];
    const int s = fmt == CNL_CKPT_INT8 ? ckpt8::encode<CNL_CKPT_INT8, 4, 8>(f, c) : ckpt8::encode<CNL_CKPT_E4M3, 4, 8>(f, c);
    if (on) {
        *reinterpret_cast<uint2*>(codes) = make_uint2(c[0], c[1]);
        if (first) *scale = ckpt8::scale_byte(s);
    }
}

// ---- sums over a row ----------------------------------------------------------------------------------------------
// Up to a warp: butterflies.  Several warps: their sums meet in shared memory, two buffers in turn, at a barrier of the row's own.
struct Row {
    int tpr, wpr, slot;              // threads and warps of a row; the row slot
    float* buffer;                   // [2][warps][2]
    int turn;
};

template <bool WIDE, int N>
__device__ __forceinline__ void row_sum(float (&v)[N], Row& r) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1)
        if (WIDE || o < r.tpr) {
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
        }
    if constexpr (WIDE) {
        const int lane = threadIdx.x & 31;
        float* buf = r.buffer + r.turn;
        r.turn ^= 64;
        if (lane == 0) {
#pragma unroll
            for (int i = 0; i < N; ++i) buf[(threadIdx.x >> 5) * 2 + i] = v[i];
        }
        asm volatile("bar.sync %0, %1;" ::"r"(r.slot + 1), "r"(r.tpr) : "memory");
        const int at = (r.slot * r.wpr + (lane & 15)) * 2;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            float p = (lane & 15) < r.wpr ? buf[at + i] : 0.0f;
#pragma unroll
            for (int o = 1; o < 16; o <<= 1) p += __shfl_xor_sync(0xffffffffu, p, o);
            v[i] = p;
        }
    }
}

// mu and r; v becomes v^
template <bool WIDE, bool LAYER>
__device__ __forceinline__ void normalise(float2 (&v)[4], bool on, const Args& a, Row& row, float& mu, float& r) {
    float s[1];
    mu = 0.0f;
    if constexpr (LAYER) {
        const float2 t = __fadd2_rn(__fadd2_rn(v[0], v[1]), __fadd2_rn(v[2], v[3]));
        s[0] = t.x + t.y;
        row_sum<WIDE, 1>(s, row);
        mu = s[0] * a.inv_d;
        const float2 m = f2(on ? -mu : 0.0f);                              // nothing stays nothing
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = __fadd2_rn(v[k], m);
    }
    float2 q = __fmul2_rn(v[0], v[0]);
#pragma unroll
    for (int k = 1; k < 4; ++k) q = __ffma2_rn(v[k], v[k], q);
    s[0] = q.x + q.y;
    row_sum<WIDE, 1>(s, row);
    r = rsqrtf(fmaf(s[0], a.inv_d, a.eps));
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = __fmul2_rn(v[k], f2(r));
}

__device__ __forceinline__ float2 gate2(float2 z, int sig) {
    if (!sig) return z;
    const float2 e = __fmul2_rn(z, f2(-1.4426950408889634f));
    const float2 p = __fadd2_rn(make_float2(exp2_approx(e.x), exp2_approx(e.y)), f2(1.0f));
    return make_float2(rcp_approx(p.x), rcp_approx(p.y));
}

// ---- forward --------------------------------------------------------------------------------------------------------
// BIAS: a bias takes part.  Without one the registers allow three blocks of 256 an SM.
template <typename T, bool WIDE, bool LAYER, bool BIAS, int BLOCK>
__global__ void __launch_bounds__(BLOCK, BLOCK == 512 ? 1 : BIAS ? 2 : 3) forward_vec(const Args a) {
    using S = Slots<T, 3, BLOCK>;
    extern __shared__ __align__(16) unsigned char dynamic[];
    __shared__ float meet[128];
    const int rpb = blockDim.x / a.tpr, slot = threadIdx.x / a.tpr, t = threadIdx.x - slot * a.tpr, c = t * 8;
    Row row = {a.tpr, a.tpr >> 5, slot, meet, 0};
    const S slots = {(unsigned)__cvta_generic_to_shared(dynamic) + threadIdx.x * 16};
    const long long group = blockIdx.x / a.nb;
    const int first = blockIdx.x - (int)(group * a.nb);
    const bool in = c < a.d;
    // rows are counted from this thread's first one
    const long long begin = group * a.per + (long long)first * rpb + slot, step = (long long)a.nb * rpb, left = (group + 1) * a.per - begin;
    const int count = (int)((left + slot + step - 1) / step);              // of the block's first slot: every slot goes round as often
    const int mine = left > 0 ? (int)((left + step - 1) / step) : 0;
    const long long stride = step * a.d;
    const bool has_u = a.u != nullptr, has_h = a.w1 != nullptr;
    long long at = begin * a.d + c, next = at;
    int asked = 0;
    unsigned into = 0, from = 0;
    auto ask = [&]() {
        if (in && asked < mine) {
            slots.ask(into, 0, (const T*)a.x + next);
            if (has_u) slots.ask(into, 1, (const T*)a.u + next);
            if (a.gate_full) slots.ask(into, 2, (const T*)a.gate + next);
        }
        S::close();
        next += stride;
        ++asked;
        into = into == (S::kStages - 1) * S::kStage ? 0 : into + S::kStage;
    };
#pragma unroll
    for (int i = 0; i < S::kStages - 1; ++i) ask();

    float2 sw[4], sb[4], w1[4], b1[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) sw[k] = sb[k] = w1[k] = b1[k] = f2(0.0f);
    if (in) {
        if (has_u) {
            float2 s[4];
            vector8<T>(a.scale, a.w_f32, c, 1.0f, s);
            vector8<T>(a.w2, a.w_f32, c, 0.0f, sw);
            if constexpr (BIAS) vector8<T>(a.b2, a.w_f32, c, 0.0f, sb);
#pragma unroll
            for (int k = 0; k < 4; ++k) { sw[k] = __fmul2_rn(sw[k], s[k]); sb[k] = __fmul2_rn(sb[k], s[k]); }
            if (a.gate_group) {                                            // one gate for all rows of this block: part of s
                float f[8];
                load_vec<T, 8>((const T*)a.gate + group * a.d + c, f);
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const float2 g = gate2(make_float2(f[2 * k], f[2 * k + 1]), a.sigmoid);
                    sw[k] = __fmul2_rn(sw[k], g);
                    sb[k] = __fmul2_rn(sb[k], g);
                }
            }
        }
        if (has_h) {
            vector8<T>(a.w1, a.w_f32, c, 0.0f, w1);
            if constexpr (BIAS) vector8<T>(a.b1, a.w_f32, c, 0.0f, b1);
        }
    }
    const int blocks = (a.d + 31) >> 5;
    for (int it = 0; it < count; ++it) {
        const bool on = in && it < mine;
        float2 z[4], x[4], u[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) z[k] = x[k] = u[k] = f2(0.0f);
        S::wait();
        if (on) {
            slots.take(from, 0, x);
            if (has_u) slots.take(from, 1, u);
            if (a.gate_full) slots.take(from, 2, z);
        }
        from = from == (S::kStages - 1) * S::kStage ? 0 : from + S::kStage;
        ask();
        float mu_u = 0.0f, r_u = 0.0f, mu_y = 0.0f, r_y = 0.0f;
        if (a.codes) {
            const long long n = a.rows * a.d, nb = a.rows * blocks, so = (begin + it * step) * blocks + (t >> 2);
            if (has_h) put_codes(a.codes + at, a.scales + so, a.fmt, on, (t & 3) == 0, x);
            if (has_u) put_codes(a.codes + n + at, a.scales + nb + so, a.fmt, on, (t & 3) == 0, u);
            if (a.gate_full) put_codes(a.codes + 2 * n + at, a.scales + 2 * nb + so, a.fmt, on, (t & 3) == 0, z);
        }
        if (has_u) {
            normalise<WIDE, LAYER>(u, in, a, row, mu_u, r_u);
            if (a.gate_full) {
#pragma unroll
                for (int k = 0; k < 4; ++k) x[k] = __ffma2_rn(gate2(z[k], a.sigmoid), BIAS ? __ffma2_rn(u[k], sw[k], sb[k]) : __fmul2_rn(u[k], sw[k]), x[k]);
            } else {
#pragma unroll
                for (int k = 0; k < 4; ++k) x[k] = BIAS ? __fadd2_rn(__ffma2_rn(u[k], sw[k], sb[k]), x[k]) : __ffma2_rn(u[k], sw[k], x[k]);
            }
            if (on) put<T>((T*)a.y + at, x);
        }
        if (has_h) {
            normalise<WIDE, LAYER>(x, in, a, row, mu_y, r_y);
#pragma unroll
            for (int k = 0; k < 4; ++k) x[k] = BIAS ? __ffma2_rn(x[k], w1[k], b1[k]) : __fmul2_rn(x[k], w1[k]);
            if (on) put<T>((T*)a.h + at, x);
        }
        if (a.stats && on && t == 0) a.stats[begin + it * step] = make_float4(mu_u, r_u, mu_y, r_y);
        at += stride;
    }
}

// ---- backward -------------------------------------------------------------------------------------------------------
// BIAS: a bias takes part or its gradient is asked for, so the sums of t a and of dh are kept too (without: 110 us where the
// rms norm of 61440 x 512 bf16 takes 160).
template <typename T, bool WIDE, bool LAYER, bool BIAS, int BLOCK>
__global__ void __launch_bounds__(BLOCK, 512 / BLOCK) backward_vec(const Args a) {
    using S = Slots<T, 5, BLOCK>;
    extern __shared__ __align__(16) unsigned char dynamic[];
    __shared__ float meet[128];
    const int rpb = blockDim.x / a.tpr, slot = threadIdx.x / a.tpr, t = threadIdx.x - slot * a.tpr, c = t * 8;
    Row row = {a.tpr, a.tpr >> 5, slot, meet, 0};
    const S slots = {(unsigned)__cvta_generic_to_shared(dynamic) + threadIdx.x * 16};
    const long long group = blockIdx.x / a.nb;
    const int first = blockIdx.x - (int)(group * a.nb);
    const bool in = c < a.d;
    const long long begin = group * a.per + (long long)first * rpb + slot, step = (long long)a.nb * rpb, left = (group + 1) * a.per - begin;
    const int count = (int)((left + slot + step - 1) / step);
    const int mine = left > 0 ? (int)((left + step - 1) / step) : 0;
    const long long stride = step * a.d;
    const bool has_u = a.u != nullptr, has_h = a.dh != nullptr, has_y = a.dy != nullptr;
    const int blocks = (a.d + 31) >> 5;
    const long long n = a.rows * a.d, nb = a.rows * blocks;
    long long at = begin * a.d + c, next = at;
    int asked = 0;
    unsigned into = 0, from = 0;
    float4 st_next = {};
    unsigned sc_x = 0, sc_u = 0, sc_z = 0;                                 // not joined before use: that would wait for them
    auto ask = [&]() {
        if (in && asked < mine) {
            if (has_y) slots.ask(into, 0, (const T*)a.dy + next);
            if (has_h) slots.ask(into, 1, (const T*)a.dh + next);
            if (a.fmt) {
                if (has_h) slots.ask_codes(into, 2, a.codes + next);
                if (has_u) slots.ask_codes(into, 3, a.codes + n + next);
                if (a.gate_full) slots.ask_codes(into, 4, a.codes + 2 * n + next);
            } else {
                if (has_h) slots.ask(into, 2, (const T*)a.x + next);
                if (has_u) slots.ask(into, 3, (const T*)a.u + next);
                if (a.gate_full) slots.ask(into, 4, (const T*)a.gate + next);
            }
        }
        S::close();
        next += stride;
        ++asked;
        into = into == (S::kStages - 1) * S::kStage ? 0 : into + S::kStage;
    };
    // statistics and scale bytes of a row: registers, one row ahead
    auto small = [&](int it) {
        if (in && it < mine) {
            const long long r = begin + it * step;
            st_next = __ldg(a.stats + r);
            if (a.fmt) {
                const unsigned char* sc = a.scales + r * blocks + (t >> 2);
                if (has_h) sc_x = __ldg(sc);
                if (has_u) sc_u = __ldg(sc + nb);
                if (a.gate_full) sc_z = __ldg(sc + 2 * nb);
            }
        }
    };
    small(0);
#pragma unroll
    for (int i = 0; i < S::kStages - 1; ++i) ask();

    float2 sw[4], sb[4], w1[4], gg[4];                                     // gg: the group's gate
#pragma unroll
    for (int k = 0; k < 4; ++k) { sw[k] = sb[k] = w1[k] = f2(0.0f); gg[k] = f2(1.0f); }
    if (in) {
        if (has_u) {
            float2 s[4];
            vector8<T>(a.scale, a.w_f32, c, 1.0f, s);
            vector8<T>(a.w2, a.w_f32, c, 0.0f, sw);
            if (BIAS) vector8<T>(a.b2, a.w_f32, c, 0.0f, sb);
#pragma unroll
            for (int k = 0; k < 4; ++k) { sw[k] = __fmul2_rn(sw[k], s[k]); sb[k] = __fmul2_rn(sb[k], s[k]); }
            if (a.gate_group) {
                float f[8];
                load_vec<T, 8>((const T*)a.gate + group * a.d + c, f);
#pragma unroll
                for (int k = 0; k < 4; ++k) gg[k] = gate2(make_float2(f[2 * k], f[2 * k + 1]), a.sigmoid);
            }
        }
        if (has_h) vector8<T>(a.w1, a.w_f32, c, 0.0f, w1);
    }
    if (a.gate_group) {                                                    // part of s, but not of the sums
#pragma unroll
        for (int k = 0; k < 4; ++k) { sw[k] = __fmul2_rn(sw[k], gg[k]); sb[k] = __fmul2_rn(sb[k], gg[k]); }
    }
    float2 accA[4], accB[BIAS ? 4 : 1], acc1[4], acc2[BIAS ? 4 : 1];
#pragma unroll
    for (int k = 0; k < 4; ++k) accA[k] = acc1[k] = f2(0.0f);
    if constexpr (BIAS) {
#pragma unroll
        for (int k = 0; k < 4; ++k) accB[k] = acc2[k] = f2(0.0f);
    }
    for (int it = 0; it < count; ++it) {
        const bool on = in && it < mine;
        const float4 st = st_next;
        const int e_x = (int)sc_x - 127, e_u = (int)sc_u - 127, e_z = (int)sc_z - 127;
        float2 g[4], dh[4], y[4], u[4], z[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) g[k] = dh[k] = y[k] = u[k] = z[k] = f2(0.0f);      // a slot without a row adds nothing
        S::wait();
        if (on) {
            if (has_h) slots.take(from, 1, dh);
            if (a.fmt) {
                if (has_h) slots.take_codes(from, 2, e_x, a.fmt, y);
                if (has_u) slots.take_codes(from, 3, e_u, a.fmt, u);
                if (a.gate_full) slots.take_codes(from, 4, e_z, a.fmt, z);
            } else {
                if (has_h) slots.take(from, 2, y);
                if (has_u) slots.take(from, 3, u);
                if (a.gate_full) slots.take(from, 4, z);
            }
        }
        const unsigned here = from;                                        // dy stays in its slot until it is needed
        from = from == (S::kStages - 1) * S::kStage ? 0 : from + S::kStage;
        ask();
        small(it + 1);
        float2 nn[4];                                                      // s n
        if (has_u) {
            const float2 r = f2(st.y), m = f2(-st.x * st.y);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                u[k] = LAYER ? __ffma2_rn(u[k], r, m) : __fmul2_rn(u[k], r);
                nn[k] = BIAS ? __ffma2_rn(u[k], sw[k], sb[k]) : __fmul2_rn(u[k], sw[k]);
                if (a.gate_full) z[k] = gate2(z[k], a.sigmoid);
            }
        }
        if (has_h) {
            const float2 r = f2(st.w), m = f2(-st.z * st.w);
            float2 s1 = f2(0.0f), s0 = f2(0.0f);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                if (has_u) y[k] = a.gate_full ? __ffma2_rn(z[k], nn[k], y[k]) : __fadd2_rn(nn[k], y[k]);
                y[k] = LAYER ? __ffma2_rn(y[k], r, m) : __fmul2_rn(y[k], r);
                acc1[k] = __ffma2_rn(dh[k], y[k], acc1[k]);
                if constexpr (BIAS) acc2[k] = __fadd2_rn(dh[k], acc2[k]);
                dh[k] = __fmul2_rn(dh[k], w1[k]);
                s1 = __ffma2_rn(dh[k], y[k], s1);
                if constexpr (LAYER) s0 = __fadd2_rn(dh[k], s0);
            }
            float sum[LAYER ? 2 : 1];
            sum[0] = s1.x + s1.y;
            if constexpr (LAYER) sum[1] = s0.x + s0.y;
            row_sum<WIDE, LAYER ? 2 : 1>(sum, row);
            const float2 m1 = f2(-sum[0] * a.inv_d);
            if (on && has_y) slots.take(here, 0, g);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                float2 v = __ffma2_rn(y[k], m1, dh[k]);
                if constexpr (LAYER) v = __fadd2_rn(v, f2(-sum[1] * a.inv_d));
                g[k] = __ffma2_rn(v, r, g[k]);
            }
        } else if (on && has_y) slots.take(here, 0, g);
        if (on && a.dx) put<T>((T*)a.dx + at, g);
        if (has_u) {
            float2 s1 = f2(0.0f), s0 = f2(0.0f), dn[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                float2 ta = g[k];
                if (a.gate_full) {
                    ta = __fmul2_rn(ta, z[k]);
                    // dz = t (s n) a', a' = a - a^2
                    const float2 slope = a.sigmoid ? __ffma2_rn(make_float2(-z[k].x, -z[k].y), z[k], z[k]) : f2(1.0f);
                    nn[k] = __fmul2_rn(__fmul2_rn(g[k], nn[k]), slope);
                }
                accA[k] = __ffma2_rn(ta, u[k], accA[k]);
                if constexpr (BIAS) accB[k] = __fadd2_rn(ta, accB[k]);
                dn[k] = __fmul2_rn(ta, sw[k]);
                s1 = __ffma2_rn(dn[k], u[k], s1);
                if constexpr (LAYER) s0 = __fadd2_rn(dn[k], s0);
            }
            float sum[LAYER ? 2 : 1];
            sum[0] = s1.x + s1.y;
            if constexpr (LAYER) sum[1] = s0.x + s0.y;
            row_sum<WIDE, LAYER ? 2 : 1>(sum, row);
            const float2 m1 = f2(-sum[0] * a.inv_d), r = f2(st.y);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                float2 v = __ffma2_rn(u[k], m1, dn[k]);
                if constexpr (LAYER) v = __fadd2_rn(v, f2(-sum[1] * a.inv_d));
                dn[k] = __fmul2_rn(v, r);
            }
            if (on) {
                if (a.du) put<T>((T*)a.du + at, dn);
                if (a.gate_full && a.dgate) put<T>((T*)a.dgate + at, nn);
            }
        }
        at += stride;
    }
    // sums over the block's rows: lanes of a warp that hold the same channels, then the row slots in order
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();
    float2* room = reinterpret_cast<float2*>(dynamic);                     // [4][BLOCK]
    float* out = a.partial + (long long)blockIdx.x * kSums * a.d;
    const int unit = WIDE ? a.tpr : 32, units = WIDE ? rpb : BLOCK >> 5;
    auto join = [&](int which, float2 (&acc)[4]) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if constexpr (!WIDE) {
#pragma unroll
                for (int o = 16; o > 0; o >>= 1)
                    if (o >= a.tpr) {
                        acc[k].x += __shfl_xor_sync(0xffffffffu, acc[k].x, o);
                        acc[k].y += __shfl_xor_sync(0xffffffffu, acc[k].y, o);
                    }
            }
            room[k * BLOCK + threadIdx.x] = acc[k];
        }
        __syncthreads();
        if (slot == 0 && in) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                float2 v = f2(0.0f);
                for (int q = 0; q < units; ++q) v = __fadd2_rn(v, room[k * BLOCK + q * unit + t]);
                *reinterpret_cast<float2*>(out + which * a.d + c + 2 * k) = v;
            }
        }
        __syncthreads();
    };
    join(0, accA);
    join(2, acc1);
    if constexpr (BIAS) {
        join(1, accB);
        join(3, acc2);
    }
}

template <typename T, bool WIDE, int BLOCK>
int forward_as(const Args& a, const Plan& p, cudaStream_t st) {
    const bool bias = a.b2 || a.b1;
    auto* kernel = bias ? (a.layer ? forward_vec<T, WIDE, true, true, BLOCK> : forward_vec<T, WIDE, false, true, BLOCK>)
                        : (a.layer ? forward_vec<T, WIDE, true, false, BLOCK> : forward_vec<T, WIDE, false, false, BLOCK>);
    constexpr int bytes = Slots<T, 3, BLOCK>::kBytes;
    CNL_TRY(ensure_dynamic_smem(kernel, bytes));
    kernel<<<(unsigned)(p.groups * p.nb), p.block, bytes, st>>>(a);
    return after_launch("blocknorm forward");
}

template <typename T, bool WIDE, int BLOCK>
int backward_as(const Args& a, const Plan& p, cudaStream_t st) {
    auto* kernel = a.need_b ? (a.layer ? backward_vec<T, WIDE, true, true, BLOCK> : backward_vec<T, WIDE, false, true, BLOCK>)
                            : (a.layer ? backward_vec<T, WIDE, true, false, BLOCK> : backward_vec<T, WIDE, false, false, BLOCK>);
    constexpr int bytes = Slots<T, 5, BLOCK>::kBytes > BLOCK * 32 ? Slots<T, 5, BLOCK>::kBytes : BLOCK * 32;
    CNL_TRY(ensure_dynamic_smem(kernel, bytes));
    kernel<<<(unsigned)(p.groups * p.nb), p.block, bytes, st>>>(a);
    return after_launch("blocknorm backward");
}

int run_forward_vec(const Args& a, const Plan& p, int dtype, cudaStream_t st) {
#define CNL_SHAPE(T) (p.tpr <= 32 ? forward_as<T, false, 256>(a, p, st) : p.tpr <= 256 ? forward_as<T, true, 256>(a, p, st) : forward_as<T, true, 512>(a, p, st))
    return dtype == CNL_F32 ? CNL_SHAPE(float) : dtype == CNL_F16 ? CNL_SHAPE(__half) : CNL_SHAPE(__nv_bfloat16);
#undef CNL_SHAPE
}

int run_backward_vec(const Args& a, const Plan& p, int dtype, cudaStream_t st) {
#define CNL_SHAPE(T) (p.tpr <= 32 ? backward_as<T, false, 256>(a, p, st) : p.tpr <= 256 ? backward_as<T, true, 256>(a, p, st) : backward_as<T, true, 512>(a, p, st))
    return dtype == CNL_F32 ? CNL_SHAPE(float) : dtype == CNL_F16 ? CNL_SHAPE(__half) : CNL_SHAPE(__nv_bfloat16);
#undef CNL_SHAPE
}

}  // namespace bnorm
}  // namespace cnl
