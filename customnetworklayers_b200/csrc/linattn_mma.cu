// Linear attention sweep for fp16 and bf16 on the tensor cores (formulas: linattn.cuh).
//
// A block walks one segment of one head in chunks of 64 positions, one warp for every 16 columns of the output.  A warp keeps
// its 16 columns of W, transposed, as fp32 accumulators: W^T [16 x da] is what the product (weighted c)^T b adds to, and the
// same registers, rounded to the type and paired, are the second operand of a W -- W never goes through shared memory.  Per
// chunk: P = a b^T (ten 16 x 16 blocks at or under the diagonal, shared out over the warps), out = l^{i+off} (a W) + P c,
// W = l^m W + (weighted c)^T b.  The next chunk's rows arrive by cp.async meanwhile.
//
// Roundings to the type: P's weights and W where they meet the outputs, once each, as the outputs themselves.  The weighted
// c of the state is split into SPLIT parts of the type (bf16: two carry 16 bits, three all 24; fp16: the second part times
// 2^11, summed apart, so that it does not fall under fp16's range) so that what is carried, and the state a caller gets back,
// is a 32-bit sum; a chunk is summed apart and added to W by one rounded multiply-add, because the tensor cores truncate
// their sums.  fp16's range: W is brought to at most 2^8 by a power of two for its product (the sum over a head can leave
// the range that the inputs are in), P carries the whole scale of its outputs.
#include <type_traits>

#include "linattn.cuh"

namespace cnl {
namespace lin {

constexpr int kChunk = 64;
constexpr int kPad = 8;                      // elements behind a row in shared memory: rows 16 bytes apart modulo 128

__device__ __forceinline__ void ldsm(unsigned (&r)[4], const void* p) {
    const unsigned at = (unsigned)__cvta_generic_to_shared(p);
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void ldsm_t(unsigned (&r)[4], const void* p) {
    const unsigned at = (unsigned)__cvta_generic_to_shared(p);
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void mma(float (&c)[4], const unsigned (&a)[4], unsigned b0, unsigned b1, __nv_bfloat16) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma(float (&c)[4], const unsigned (&a)[4], unsigned b0, unsigned b1, __half) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <int DA, int DC, bool OUT>
struct Layout {                              // shared memory, in elements of the type
    static constexpr int ra = DA + kPad, rc = DC + kPad, rp = kChunk + kPad;
    static constexpr int a = 0, b = OUT ? kChunk * ra : 0, c = b + kChunk * ra, stage = c + kChunk * rc;
    static constexpr int p = 2 * stage, o = p + (OUT ? kChunk * rp : 0);
    static constexpr bool own_o = OUT && DC > DA;              // otherwise outputs pass through the rows of a just read
    static constexpr int end = o + (own_o ? kChunk * rc : 0);
    static constexpr int bytes = end * 2 + (kChunk + 1) * 4;
};

template <typename T, int DA, int DC, bool OUT, int SPLIT>
__global__ void __launch_bounds__(2 * DC, DC == 128 ? 2 : DC == 64 ? 4 : 8) mma_kernel(const Sweep s, const int vec) {
    using L = Layout<DA, DC, OUT>;
    constexpr int kThreads = 2 * DC, kWarps = DC / 16, KT = DA / 16;
    constexpr bool kHalf = std::is_same<T, __half>::value;
    constexpr float kNext = kHalf ? 2048.0f : 1.0f;            // a part's size against the one before
    extern __shared__ __align__(16) unsigned char raw[];
    T* sm = reinterpret_cast<T*>(raw);
    float* pw = reinterpret_cast<float*>(raw + (L::end * 2 + 3) / 4 * 4);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, q2 = (lane & 3) * 2;
    const int seg = blockIdx.x % s.segments, bh = blockIdx.x / s.segments, head = bh % s.h, bat = bh / s.h;
    const float ld = clamp_log(s.log_decay[head]);
    const int n = s.lengths ? min(max(s.lengths[bat], 0), s.t) : s.t;
    const long long first = (long long)seg * s.seg;
    const int lo = (int)(first < n ? first : n), hi = (int)(first + s.seg < n ? first + s.seg : n);
    const int da = s.da, dc = s.dc;
    const long long size = (long long)da * dc;

    for (int i = tid; i <= kChunk; i += kThreads) pw[i] = power(ld, i);
    if (da < DA || dc < DC) {                                  // what lies behind the head sizes stays 0
        for (int i = tid; i < L::p / 8; i += kThreads) reinterpret_cast<uint4*>(sm)[i] = make_uint4(0, 0, 0, 0);
        __syncthreads();
    }

    auto fetch_rows = [&](const Rows& r, T* dst, int d, int stride, int c0) {
        const T* src = (const T*)r.p + bat * r.sb + head * r.sh;
        const int m = hi - c0;
        if (vec) {
            const int per = d >> 3;
            for (int e = tid; e < kChunk * per; e += kThreads) {
                const int j = e / per, x = (e - j * per) * 8;
                const bool live = j < m;
                const long long tok = live ? (s.reversed ? n - 1 - (c0 + j) : c0 + j) : 0;
                const unsigned to = (unsigned)__cvta_generic_to_shared(dst + j * stride + x);
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(src + tok * r.st + x), "r"(live ? 16 : 0) : "memory");
            }
        } else {
            for (int e = tid; e < kChunk * d; e += kThreads) {
                const int j = e / d, x = e - j * d;
                const long long tok = s.reversed ? n - 1 - (c0 + j) : c0 + j;
                dst[j * stride + x] = j < m ? src[tok * r.st + x] : from_f32<T>(0.0f);
            }
        }
    };
    auto fetch = [&](int c0, int stage) {
        T* base = sm + stage * L::stage;
        if constexpr (OUT) fetch_rows(s.a, base + L::a, da, L::ra, c0);
        fetch_rows(s.b, base + L::b, da, L::ra, c0);
        fetch_rows(s.c, base + L::c, dc, L::rc, c0);
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    if (lo < hi) fetch(lo, 0);

    // W^T: tile x holds rows (columns of c) 16 warp + g, + 8 and columns (of a) 8 x + q2, + 1
    float w[DA / 8][4];
    const int row0 = warp * 16 + g;
    const float* w0 = s.start ? s.start + ((long long)bh * s.segments + seg) * size : nullptr;
#pragma unroll
    for (int x = 0; x < DA / 8; ++x)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int i = 8 * x + q2 + (e & 1), j = row0 + (e >> 1) * 8;
            w[x][e] = w0 && i < da && j < dc ? (s.transposed ? w0[(long long)j * da + i] : w0[(long long)i * dc + j]) : 0.0f;
        }

    int stage = 0;
    for (int c0 = lo; c0 < hi; c0 += kChunk, stage ^= 1) {
        const int m = min(kChunk, hi - c0);
        asm volatile("cp.async.wait_all;" ::: "memory");
        __syncthreads();
        if (c0 + kChunk < hi) fetch(c0 + kChunk, stage ^ 1);
        T* A = sm + stage * L::stage + L::a;
        const T* B = sm + stage * L::stage + L::b;
        const T* C = sm + stage * L::stage + L::c;
        if constexpr (OUT) {
            T* P = sm + L::p;
            const float both = s.in_scale * s.out_scale;
            // P: blocks (i, j) of 16 x 16, j <= i, numbered row by row
            for (int id = warp; id < 10; id += kWarps) {
                const int bi = id >= 6 ? 3 : id >= 3 ? 2 : id >= 1 ? 1 : 0, bj = id - bi * (bi + 1) / 2;
                float acc[2][4] = {};
#pragma unroll
                for (int k = 0; k < KT; ++k) {
                    unsigned a[4], b[4];
                    ldsm(a, A + (bi * 16 + (lane & 15)) * L::ra + k * 16 + (lane >> 4) * 8);
                    ldsm(b, B + (bj * 16 + (lane & 7) + (lane >> 4) * 8) * L::ra + k * 16 + ((lane >> 3) & 1) * 8);
                    mma(acc[0], a, b[0], b[1], T());
                    mma(acc[1], a, b[2], b[3], T());
                }
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        const int i = bi * 16 + g + h * 8, j = bj * 16 + x * 8 + q2;
                        const float v0 = j <= i ? acc[x][2 * h] * (both * pw[max(i - j, 0)]) : 0.0f;
                        const float v1 = j + 1 <= i ? acc[x][2 * h + 1] * (both * pw[max(i - j - 1, 0)]) : 0.0f;
                        *reinterpret_cast<unsigned*>(P + i * L::rp + j) = pack2<T>(v0, v1);
                    }
            }
            float o[4][2][4];
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[i][0][e] = o[i][1][e] = 0.0f;
            float down = 1.0f, up = s.out_scale;
            if constexpr (kHalf) {
                float top = 0.0f;
#pragma unroll
                for (int x = 0; x < DA / 8; ++x)
#pragma unroll
                    for (int e = 0; e < 4; ++e) top = fmaxf(top, fabsf(w[x][e]));
#pragma unroll
                for (int k = 16; k > 0; k >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, k));
                const int ex = min(max((int)(__float_as_uint(top) >> 23) - 127, -100), 100);
                down = __uint_as_float((unsigned)(127 + 7 - ex) << 23);
                up *= __uint_as_float((unsigned)(127 - 7 + ex) << 23);
            }
#pragma unroll
            for (int k = 0; k < KT; ++k) {
                const unsigned b00 = pack2<T>(down * w[2 * k][0], down * w[2 * k][1]), b01 = pack2<T>(down * w[2 * k + 1][0], down * w[2 * k + 1][1]);
                const unsigned b10 = pack2<T>(down * w[2 * k][2], down * w[2 * k][3]), b11 = pack2<T>(down * w[2 * k + 1][2], down * w[2 * k + 1][3]);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    unsigned a[4];
                    ldsm(a, A + (i * 16 + (lane & 15)) * L::ra + k * 16 + (lane >> 4) * 8);
                    mma(o[i][0], a, b00, b01, T());
                    mma(o[i][1], a, b10, b11, T());
                }
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float f0 = up * pw[min(i * 16 + g + s.off, kChunk)], f1 = up * pw[min(i * 16 + g + 8 + s.off, kChunk)];
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    o[i][x][0] *= f0; o[i][x][1] *= f0; o[i][x][2] *= f1; o[i][x][3] *= f1;
                }
            }
            __syncthreads();
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                unsigned b[4];
                ldsm_t(b, C + (k * 16 + (lane & 15)) * L::rc + warp * 16 + (lane >> 4) * 8);
#pragma unroll
                for (int i = k; i < 4; ++i) {
                    unsigned a[4];
                    ldsm(a, P + (i * 16 + (lane & 15)) * L::rp + k * 16 + (lane >> 4) * 8);
                    mma(o[i][0], a, b[0], b[1], T());
                    mma(o[i][1], a, b[2], b[3], T());
                }
            }
            // through shared memory, so that a warp stores whole 32-byte pieces of its rows
            T* O = L::own_o ? sm + L::o : A;
            constexpr int ro = L::own_o ? L::rc : L::ra;
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int x = 0; x < 2; ++x)
#pragma unroll
                    for (int h = 0; h < 2; ++h)
                        *reinterpret_cast<unsigned*>(O + (i * 16 + h * 8 + g) * ro + warp * 16 + x * 8 + q2) =
                            pack2<T>(o[i][x][2 * h], o[i][x][2 * h + 1]);
            __syncwarp();
            T* out = (T*)s.out + ((long long)bat * s.t * s.h + head) * dc;
#pragma unroll
            for (int e = lane; e < kChunk * 2; e += 32) {
                const int i = e >> 1, x = warp * 16 + (e & 1) * 8;
                if (i < m && x < dc) {
                    const long long tok = s.reversed ? n - 1 - (c0 + i) : c0 + i;
                    T* to = out + tok * s.h * dc + x;
                    if (vec) *reinterpret_cast<uint4*>(to) = *reinterpret_cast<const uint4*>(O + i * ro + x);
                    else
                        for (int k = 0; k < 8 && x + k < dc; ++k) to[k] = O[i * ro + x + k];
                }
                if (!L::own_o && x + 8 > da)                     // back to the zeros that stand behind a head smaller than DA
                    for (int k = max(da - x, 0); k < 8; ++k) O[i * ro + x + k] = from_f32<T>(0.0f);
            }
        }
        // W^T = l^m W^T + in_scale sum_j (l^{m-off-j} c_j) b_j^T, 32 positions at a time
        float keep = pw[m];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            unsigned part[2][SPLIT][4];
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const int j0 = half * 32 + k * 16;
                unsigned a[4];
                ldsm_t(a, C + (j0 + (lane & 7) + (lane >> 4) * 8) * L::rc + warp * 16 + ((lane >> 3) & 1) * 8);
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int j = j0 + q2 + (r >> 1) * 8;
                    const float2 v = unpack2(a[r], T());
                    float x = v.x * pw[max(m - s.off - j, 0)], y = v.y * pw[max(m - s.off - j - 1, 0)];
#pragma unroll
                    for (int p = 0; p < SPLIT; ++p) {
                        part[k][p][r] = pack2<T>(x, y);
                        const float2 f = unpack2(part[k][p][r], T());
                        x = (x - f.x) * kNext;
                        y = (y - f.y) * kNext;
                    }
                }
            }
#pragma unroll
            for (int x = 0; x < DA / 16; ++x) {
                float t[2][4] = {}, small[2][4] = {};
#pragma unroll
                for (int p = SPLIT - 1; p >= 0; --p)
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        unsigned b[4];
                        ldsm_t(b, B + (half * 32 + k * 16 + (lane & 15)) * L::ra + x * 16 + (lane >> 4) * 8);
                        mma(kHalf && p > 0 ? small[0] : t[0], part[k][p], b[0], b[1], T());
                        mma(kHalf && p > 0 ? small[1] : t[1], part[k][p], b[2], b[3], T());
                    }
#pragma unroll
                for (int e = 0; e < 4; ++e)
#pragma unroll
                    for (int y = 0; y < 2; ++y) {
                        const float sum = kHalf ? fmaf(small[y][e], 1.0f / kNext, t[y][e]) : t[y][e];
                        w[2 * x + y][e] = fmaf(s.in_scale, sum, keep * w[2 * x + y][e]);
                    }
            }
            keep = 1.0f;
        }
    }
    if (s.end) {
        float* w1 = s.end + ((long long)bh * s.segments + seg) * size;
#pragma unroll
        for (int x = 0; x < DA / 8; ++x)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int i = 8 * x + q2 + (e & 1), j = row0 + (e >> 1) * 8;
                if (i < da && j < dc) w1[(long long)i * dc + j] = w[x][e];
            }
    }
    if constexpr (OUT) {                                         // rows behind the sequence's end
        const long long zlo = first > n ? first : n, zhi = first + s.seg < s.t ? first + s.seg : s.t;
        for (long long e = zlo * dc + tid; e < zhi * dc; e += kThreads) {
            const long long tok = e / dc;
            ((T*)s.out)[(((long long)bat * s.t + tok) * s.h + head) * dc + (e - tok * dc)] = from_f32<T>(0.0f);
        }
    }
}

template <typename T, int DA, int DC, bool OUT, int SPLIT>
int launch(const Sweep& s, int vec, cudaStream_t st) {
    constexpr int bytes = Layout<DA, DC, OUT>::bytes;
    CNL_TRY(ensure_dynamic_smem(mma_kernel<T, DA, DC, OUT, SPLIT>, bytes));
    mma_kernel<T, DA, DC, OUT, SPLIT><<<(unsigned)((long long)s.batch * s.h * s.segments), 2 * DC, bytes, st>>>(s, vec);
    return after_launch("linear attention sweep");
}

template <typename T, int DA, int DC>
int pick(const Sweep& s, int vec, cudaStream_t st) {
    // a state that leaves the kernel is kept to 32 bits (fp16 has 22 in two parts); one that only feeds rounded outputs to 16
    constexpr int kExact = std::is_same<T, __half>::value ? 2 : 3;
    if (!s.out) return launch<T, DA, DC, false, kExact>(s, vec, st);
    if (s.end) return launch<T, DA, DC, true, kExact>(s, vec, st);
    return launch<T, DA, DC, true, 2>(s, vec, st);
}

inline bool rows_aligned(const Rows& r, int d) { return !r.p || (aligned16(r.p) && d % 8 == 0 && r.sb % 8 == 0 && r.st % 8 == 0 && r.sh % 8 == 0); }

template <typename T>
int run(const Sweep& s, cudaStream_t st) {
    const int vec = rows_aligned(s.a, s.da) && rows_aligned(s.b, s.da) && rows_aligned(s.c, s.dc) && aligned16(s.out);
    // head sizes are filled up to 32, 64 or 128; 64 with 128 has its own form, other mixed sizes take the larger for both
    const int a = s.da <= 32 ? 32 : s.da <= 64 ? 64 : 128, c = s.dc <= 32 ? 32 : s.dc <= 64 ? 64 : 128;
    if (a <= 32 && c <= 32) return pick<T, 32, 32>(s, vec, st);
    if (a <= 64 && c <= 64) return pick<T, 64, 64>(s, vec, st);
    if (a <= 64) return pick<T, 64, 128>(s, vec, st);
    if (c <= 64) return pick<T, 128, 64>(s, vec, st);
    return pick<T, 128, 128>(s, vec, st);
}

int run_sweep_mma(const Sweep& s, int dtype, cudaStream_t st) {
    return dtype == CNL_F16 ? run<__half>(s, st) : run<__nv_bfloat16>(s, st);
}

}  // namespace lin
}  // namespace cnl
