// Linear attention sweep for fp16 and bf16 on the tensor cores (formulas: linattn.cuh).
//
// A block walks one segment of one head in chunks of 64 positions, one warp for every 16 columns of the output.  A warp keeps
// its 16 columns of W, transposed, as fp32 accumulators: W^T [16 x da] is what the product (weighted c)^T b adds to, and the
// same registers, rounded to the type and paired, are the second operand of a W -- W never goes through shared memory.  Per
// chunk: P = a b^T (ten 16 x 16 blocks at or under the diagonal, shared out over the warps), out = l^{i+off} (a W) + P c,
// W = l^m W + (weighted c)^T b.  The next chunk's rows arrive by cp.async meanwhile.
//
// Roundings to the type: P and, where it meets the outputs, W go in two parts each, so that a result carries its own rounding
// and little else (each rounded once, a result would be off by 1.4 times what its own rounding costs).  The weighted
// c of the state is split into parts of the type (one part would be off by 1.6e-3): fp16 into two, 22 bits, the second times
// 2^11 and summed apart, so that it does not fall under fp16's range; bf16 into two (16 bits, 7e-7 rms) where W only feeds
// rounded outputs, and into all three where a caller gets the state (EXACT).  A chunk is summed apart and added to W by one
// rounded multiply-add, because the tensor cores truncate their sums.  fp16's range: W is brought to at most 2^15 by a power
// of two for its product (the sum over a head can leave the range that the inputs are in, and a column that is small beside
// its neighbours keeps 2^-40 of their largest).  P, a product of two rows that may each be near either end, stays fp32 in
// shared memory and meets c as two parts in tf32, which has fp32's range and holds fp16's values of c as they are.
//
// fp16, forward / backward: 8 x 7680 tokens x 8 heads of 128 609 / 1541 us, of 64 222 / 566 us, 4 x 7680 x 8 of 32 65 / 148 us (with P
// as two parts in fp16, which loses weights above 65504, and W as one, 478 / 1148, 179 / 437 and 56 / 130 us); bound
// by the legacy tensor path and the fragments' way through shared memory.  The tcgen05 sweep takes 208 / 497 and 140 / 308 us for
// the same in bf16; fp16 stays here, where the state's second part can be summed apart.
#include <type_traits>

#include "linattn.cuh"

namespace cnl {
namespace lin {

constexpr int kChunk = 64;
constexpr int kPad = 8;                      // elements behind a row in shared memory: rows 16 bytes apart modulo 128

__device__ __forceinline__ void ldsm(unsigned (&r)[4], const void* p) {
    const unsigned at = (unsigned)__cvta_generic_to_shared(p);
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at));
}
__device__ __forceinline__ void ldsm_t(unsigned (&r)[4], const void* p) {
    const unsigned at = (unsigned)__cvta_generic_to_shared(p);
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at));
}
__device__ __forceinline__ void mma(float (&c)[4], const unsigned (&a)[4], unsigned b0, unsigned b1, __nv_bfloat16) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma(float (&c)[4], const unsigned (&a)[4], unsigned b0, unsigned b1, __half) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Eight rows summed: tf32, whose 11 significant bits are fp16's
__device__ __forceinline__ void mma_tf32(float (&c)[4], const unsigned (&a)[4], float2 b) {
    asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(__float_as_uint(b.x)), "r"(__float_as_uint(b.y)));
}
__device__ __forceinline__ unsigned to_tf32(float v) {
    unsigned r;
    asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(r) : "f"(v));
    return r;
}

template <int DA, int DC, bool OUT>
struct Layout {                              // shared memory, in elements of the type
    static constexpr int ra = DA + kPad, rc = DC + kPad, rp = kChunk + kPad;
    static constexpr int a = 0, b = OUT ? kChunk * ra : 0, c = b + kChunk * ra, stage = c + kChunk * rc;
    static constexpr int p = 2 * stage, p2 = kChunk * rp, o = p + (OUT ? 2 * p2 : 0);      // P's two parts, or P in fp32
    static constexpr bool own_o = OUT && DC > DA;              // otherwise outputs pass through the rows of a just read
    static constexpr int end = o + (own_o ? kChunk * rc : 0);
    static constexpr int bytes = (end * 2 + 15) / 16 * 16 + (3 * kChunk + 24) * 4;      // and the three tables of powers
};

template <typename T, int DA, int DC, bool OUT, bool EXACT>
__global__ void __launch_bounds__(2 * DC, DC == 128 ? 2 : DC == 64 ? 4 : 8) mma_kernel(const Sweep s, const int vec) {
    using L = Layout<DA, DC, OUT>;
    constexpr int kThreads = 2 * DC, kWarps = DC / 16, KT = DA / 16;
    constexpr bool kHalf = std::is_same<T, __half>::value;
    constexpr int kSplit = EXACT && !kHalf ? 3 : 2;
    constexpr float kNext = kHalf ? 2048.0f : 1.0f;            // a part's size against the one before
    extern __shared__ __align__(16) unsigned char raw[];
    T* sm = reinterpret_cast<T*>(raw);
    float* pw = reinterpret_cast<float*>(raw + (L::end * 2 + 15) / 16 * 16);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, q2 = (lane & 3) * 2;
    const int seg = blockIdx.x % s.segments, bh = blockIdx.x / s.segments, head = bh % s.h, bat = bh / s.h;
    const float ld = clamp_log(s.log_decay[head]);
    const int n = s.lengths ? min(max(s.lengths[bat], 0), s.t) : s.t;
    const long long first = (long long)seg * s.seg;
    const int lo = (int)(first < n ? first : n), hi = (int)(first + s.seg < n ? first + s.seg : n);
    const int da = s.da, dc = s.dc;
    const long long size = (long long)da * dc;

    float* wt = pw + kChunk + 4;                               // what a position of the chunk weighs in the state
    float* pz = wt + kChunk + 16;                              // what one position weighs for another d later; 0 for d < 0
    auto weight = [&](int j, int m) { return j < m ? power(ld, m - s.off - j) * (kHalf ? 1.0f : s.in_scale) : 0.0f; };
    for (int i = tid; i <= kChunk; i += kThreads) pw[i] = power(ld, i);
    for (int i = tid; i < kChunk; i += kThreads) wt[i] = weight(i, kChunk);
    for (int i = tid; i < kChunk + 16; i += kThreads) pz[i - 16] = i < 16 ? 0.0f : power(ld, i - 16) * (s.in_scale * s.out_scale);
    if (da < DA || dc < DC) {                                  // what lies behind the head sizes stays 0
        for (int i = tid; i < L::p / 8; i += kThreads) reinterpret_cast<uint4*>(sm)[i] = make_uint4(0, 0, 0, 0);
        __syncthreads();
    }

    // rows of one operand; FULL: the head fills its columns, so a thread's pieces lie a fixed number of rows apart
    auto fetch_rows = [&](const Rows& r, T* dst, int d, auto full, int stride, int c0) {
        constexpr int kFull = decltype(full)::value;
        const int m = hi - c0;
        const long long by = s.reversed ? -r.st : r.st;
        const T* row = (const T*)r.p + bat * r.sb + head * r.sh + (s.reversed ? n - 1 - c0 : c0) * r.st;
        auto piece = [&](unsigned to, const T* from, bool live) {
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(live ? from : row), "r"(live ? 16 : 0) : "memory");
        };
        if (vec && d == kFull) {
            constexpr int per = kFull / 8, rows = kThreads / per;
            const int j = tid / per, x = tid % per * 8;
            unsigned to = (unsigned)__cvta_generic_to_shared(dst + j * stride + x);
            const T* from = row + j * by + x;
            if (m >= kChunk) {
#pragma unroll
                for (int i = 0; i < kChunk / rows; ++i) {
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + i * rows * stride * (int)sizeof(T)), "l"(from) : "memory");
                    from += rows * by;
                }
            } else {
#pragma unroll 1
                for (int i = 0; i < kChunk / rows; ++i) {
                    piece(to + i * rows * stride * (int)sizeof(T), from, j + i * rows < m);
                    from += rows * by;
                }
            }
        } else if (vec) {
            const int per = d >> 3;
#pragma unroll 1
            for (int e = tid; e < kChunk * per; e += kThreads) {
                const int j = e / per, x = (e - j * per) * 8;
                piece((unsigned)__cvta_generic_to_shared(dst + j * stride + x), row + j * by + x, j < m);
            }
        } else {
#pragma unroll 1
            for (int e = tid; e < kChunk * d; e += kThreads) {
                const int j = e / d, x = e - j * d;
                dst[j * stride + x] = j < m ? row[j * by + x] : from_f32<T>(0.0f);
            }
        }
    };
    auto fetch = [&](int c0, int stage) {
        T* base = sm + stage * L::stage;
        if constexpr (OUT) fetch_rows(s.a, base + L::a, da, std::integral_constant<int, DA>(), L::ra, c0);
        fetch_rows(s.b, base + L::b, da, std::integral_constant<int, DA>(), L::ra, c0);
        fetch_rows(s.c, base + L::c, dc, std::integral_constant<int, DC>(), L::rc, c0);
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    if (lo < hi) fetch(lo, 0);

    // W^T: tile x holds rows (columns of c) 16 warp + g, + 8 and columns (of a) 8 x + q2, + 1
    float2 w[DA / 8][2];                                       // [tile][row g or g + 8], two neighbouring columns
    const int row0 = warp * 16 + g;
    const float* w0 = s.start ? s.start + ((long long)bh * s.segments + seg) * size : nullptr;
#pragma unroll
    for (int x = 0; x < DA / 8; ++x)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int i = 8 * x + q2, j = row0 + h * 8;
            float v[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) v[e] = w0 && i + e < da && j < dc ? (s.transposed ? w0[(long long)j * da + i + e] : w0[(long long)(i + e) * dc + j]) : 0.0f;
            w[x][h] = make_float2(v[0], v[1]);
        }

    int stage = 0;
    for (int c0 = lo; c0 < hi; c0 += kChunk, stage ^= 1) {
        const int m = min(kChunk, hi - c0);
        asm volatile("cp.async.wait_all;" ::: "memory");
        __syncthreads();
        if (c0 + kChunk < hi) fetch(c0 + kChunk, stage ^ 1);
        if (m < kChunk) {                                      // the last chunk: its weights end at m (uniform for the block)
            if (tid < kChunk) wt[tid] = weight(tid, m);
            __syncthreads();
        }
        T* A = sm + stage * L::stage + L::a;
        const T* B = sm + stage * L::stage + L::b;
        const T* C = sm + stage * L::stage + L::c;
        if constexpr (OUT) {
            T* P = sm + L::p;
            // P: blocks (i, j) of 16 x 16, j <= i, numbered row by row
#pragma unroll 1
            for (int id = warp; id < 10; id += kWarps) {
                const int bi = id >= 6 ? 3 : id >= 3 ? 2 : id >= 1 ? 1 : 0, bj = id - bi * (bi + 1) / 2;
                const T* pa = A + (bi * 16 + (lane & 15)) * L::ra + (lane >> 4) * 8;
                const T* pb = B + (bj * 16 + (lane & 7) + (lane >> 4) * 8) * L::ra + ((lane >> 3) & 1) * 8;
                float acc[2][4] = {};
#pragma unroll
                for (int k = 0; k < KT; ++k) {
                    unsigned a[4], b[4];
                    ldsm(a, pa + k * 16);
                    ldsm(b, pb + k * 16);
                    mma(acc[0], a, b[0], b[1], T());
                    mma(acc[1], a, b[2], b[3], T());
                }
                const float* z = pz + (bi - bj) * 16 + g - q2;               // position i after position j: 8 h - 8 x - e more
                const int at = (bi * 16 + g) * L::rp + bj * 16 + q2;
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int x = 0; x < 2; ++x)
                    {
                        const float2 v = make_float2(acc[x][2 * h] * z[8 * h - 8 * x], acc[x][2 * h + 1] * z[8 * h - 8 * x - 1]);
                        const int to = at + h * 8 * L::rp + x * 8;
                        if constexpr (kHalf) {
                            *reinterpret_cast<float2*>(reinterpret_cast<float*>(P) + to) = v;
                        } else {
                            const unsigned top = pack2<T>(v.x, v.y);
                            const float2 f = unpack2(top, T());
                            *reinterpret_cast<unsigned*>(P + to) = top;
                            *reinterpret_cast<unsigned*>(P + L::p2 + to) = pack2<T>(v.x - f.x, v.y - f.y);
                        }
                    }
            }
            __syncthreads();
            float down = 1.0f, up = s.out_scale;
            if constexpr (kHalf) {
                float top = 0.0f;
#pragma unroll
                for (int x = 0; x < DA / 8; ++x)
#pragma unroll
                    for (int h = 0; h < 2; ++h) top = fmaxf(top, fmaxf(fabsf(w[x][h].x), fabsf(w[x][h].y)));
#pragma unroll
                for (int k = 16; k > 0; k >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, k));
                const int ex = min(max((int)(__float_as_uint(top) >> 23) - 127, -100), 100);
                down = __uint_as_float((unsigned)(127 + 14 - ex) << 23);
                up *= __uint_as_float((unsigned)(127 - 14 + ex) << 23);
            }
            auto round = [&](float2 v, unsigned& small) {            // W in two parts
                if constexpr (kHalf) v = __fmul2_rn(v, make_float2(down, down));
                const unsigned top = pack2<T>(v.x, v.y);
                const float2 f = unpack2(top, T());
                small = pack2<T>(v.x - f.x, v.y - f.y);
                return top;
            };
            // outputs pass through shared memory, so that a warp stores whole 32-byte pieces of its rows
            T* O = L::own_o ? sm + L::o : A;
            constexpr int ro = L::own_o ? L::rc : L::ra;
            // 32 positions at a time: with all 64 the sums and W do not fit the registers of two blocks an SM
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                float o[2][2][4];
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[i][0][e] = o[i][1][e] = 0.0f;
#pragma unroll
                for (int k = 0; k < KT; ++k) {
                    unsigned s00, s01, s10, s11;
                    const unsigned b00 = round(w[2 * k][0], s00), b01 = round(w[2 * k + 1][0], s01), b10 = round(w[2 * k][1], s10), b11 = round(w[2 * k + 1][1], s11);
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        unsigned a[4];
                        ldsm(a, A + (half * 32 + i * 16 + (lane & 15)) * L::ra + k * 16 + (lane >> 4) * 8);
                        mma(o[i][0], a, s00, s01, T());
                        mma(o[i][1], a, s10, s11, T());
                        mma(o[i][0], a, b00, b01, T());
                        mma(o[i][1], a, b10, b11, T());
                    }
                }
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float f0 = up * pw[half * 32 + i * 16 + g + s.off], f1 = up * pw[half * 32 + i * 16 + g + 8 + s.off];
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        o[i][x][0] *= f0; o[i][x][1] *= f0; o[i][x][2] *= f1; o[i][x][3] *= f1;
                    }
                }
#pragma unroll
                for (int k = 0; k < 2 * half + 2; ++k) {
                    unsigned b[4];
                    ldsm_t(b, C + (k * 16 + (lane & 15)) * L::rc + warp * 16 + (lane >> 4) * 8);
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        if (k > half * 2 + i) continue;
                        unsigned a[4];
                        if constexpr (kHalf) {
                            // columns 2 t and 2 t + 1 of 8 stand where the product sums over t and t + 4: c's pairs are there already
                            const float* from = reinterpret_cast<const float*>(P) + (half * 32 + i * 16 + g) * L::rp + k * 16 + q2;
#pragma unroll
                            for (int e = 0; e < 2; ++e) {
                                const float2 p0 = *reinterpret_cast<const float2*>(from + e * 8), p1 = *reinterpret_cast<const float2*>(from + e * 8 + 8 * L::rp);
                                const float v[4] = {p0.x, p1.x, p0.y, p1.y};
                                unsigned small[4];
#pragma unroll
                                for (int x = 0; x < 4; ++x) {
                                    a[x] = to_tf32(v[x]);
                                    small[x] = to_tf32(v[x] - __uint_as_float(a[x]));
                                }
                                const float2 b0 = unpack2(b[e], T()), b1 = unpack2(b[2 + e], T());
                                mma_tf32(o[i][0], small, b0);
                                mma_tf32(o[i][1], small, b1);
                                mma_tf32(o[i][0], a, b0);
                                mma_tf32(o[i][1], a, b1);
                            }
                            continue;
                        }
                        ldsm(a, P + (half * 32 + i * 16 + (lane & 15)) * L::rp + k * 16 + (lane >> 4) * 8);
                        mma(o[i][0], a, b[0], b[1], T());
                        mma(o[i][1], a, b[2], b[3], T());
                        ldsm(a, P + L::p2 + (half * 32 + i * 16 + (lane & 15)) * L::rp + k * 16 + (lane >> 4) * 8);
                        mma(o[i][0], a, b[0], b[1], T());
                        mma(o[i][1], a, b[2], b[3], T());
                    }
                }
                if (!L::own_o) __syncthreads();                  // all warps have read these rows of A
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int x = 0; x < 2; ++x)
#pragma unroll
                        for (int h = 0; h < 2; ++h)
                            *reinterpret_cast<unsigned*>(O + (half * 32 + i * 16 + h * 8 + g) * ro + warp * 16 + x * 8 + q2) = pack2<T>(o[i][x][2 * h], o[i][x][2 * h + 1]);
            }
            __syncwarp();
            const int x = warp * 16 + (lane & 1) * 8, i0 = lane >> 1;
            const long long by = (s.reversed ? -1LL : 1LL) * s.h * dc;
            T* to = (T*)s.out + ((long long)bat * s.t * s.h + head) * dc + (s.reversed ? n - 1 - c0 : c0) * ((long long)s.h * dc) + i0 * by + x;
            if (vec) {
                if (x < dc) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        if (i0 + 16 * i < m) *reinterpret_cast<uint4*>(to) = *reinterpret_cast<const uint4*>(O + (i0 + 16 * i) * ro + x);
                        to += 16 * by;
                    }
                }
            } else {
#pragma unroll 1
                for (int i = i0; i < m; i += 16, to += 16 * by)
                    for (int k = 0; k < 8 && x + k < dc; ++k) to[k] = O[i * ro + x + k];
            }
            if (!L::own_o && x + 8 > da)                         // back to the zeros that stand behind a head smaller than DA
#pragma unroll 1
                for (int i = i0; i < kChunk; i += 16)
                    for (int k = max(da - x, 0); k < 8; ++k) O[i * ro + x + k] = from_f32<T>(0.0f);
        }
        // W^T = l^m W^T + in_scale sum_j (l^{m-off-j} c_j) b_j^T, 32 positions at a time
        const float2 keep = make_float2(pw[m], pw[m]), sc = make_float2(s.in_scale, s.in_scale);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            unsigned part[2][kSplit][4];
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const int j0 = half * 32 + k * 16;
                unsigned a[4];
                ldsm_t(a, C + (j0 + (lane & 7) + (lane >> 4) * 8) * L::rc + warp * 16 + ((lane >> 3) & 1) * 8);
                const float2 f0 = *reinterpret_cast<const float2*>(wt + j0 + q2), f1 = *reinterpret_cast<const float2*>(wt + j0 + q2 + 8);
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    float2 v = __fmul2_rn(unpack2(a[r], T()), r < 2 ? f0 : f1);
#pragma unroll
                    for (int p = 0; p < kSplit; ++p) {
                        part[k][p][r] = pack2<T>(v.x, v.y);
                        if (p + 1 < kSplit) {
                            const float2 f = unpack2(part[k][p][r], T());
                            v = __fadd2_rn(v, make_float2(-f.x, -f.y));
                            if constexpr (kHalf) v = __fmul2_rn(v, make_float2(kNext, kNext));
                        }
                    }
                }
            }
#pragma unroll
            for (int x = 0; x < DA / 16; ++x) {
                float t[2][4] = {}, small[2][4] = {};
                unsigned b[2][4];
#pragma unroll
                for (int k = 0; k < 2; ++k) ldsm_t(b[k], B + (half * 32 + k * 16 + (lane & 15)) * L::ra + x * 16 + (lane >> 4) * 8);
#pragma unroll
                for (int p = kSplit - 1; p >= 0; --p)
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        mma(kHalf && p > 0 ? small[0] : t[0], part[k][p], b[k][0], b[k][1], T());
                        mma(kHalf && p > 0 ? small[1] : t[1], part[k][p], b[k][2], b[k][3], T());
                    }
#pragma unroll
                for (int y = 0; y < 2; ++y)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        float2 sum = make_float2(t[y][2 * h], t[y][2 * h + 1]);
                        float2& to = w[2 * x + y][h];
                        if constexpr (kHalf) {
                            sum = __ffma2_rn(make_float2(small[y][2 * h], small[y][2 * h + 1]), make_float2(1.0f / kNext, 1.0f / kNext), sum);
                            to = __ffma2_rn(sc, sum, half ? to : __fmul2_rn(keep, to));
                        } else {                               // in_scale is in the weights
                            to = half ? __fadd2_rn(to, sum) : __ffma2_rn(keep, to, sum);
                        }
                    }
            }
        }
    }
    if (s.end) {
        float* w1 = s.end + ((long long)bh * s.segments + seg) * size;
#pragma unroll
        for (int x = 0; x < DA / 8; ++x)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int i = 8 * x + q2 + (e & 1), j = row0 + (e >> 1) * 8;
                if (i < da && j < dc) w1[(long long)i * dc + j] = e & 1 ? w[x][e >> 1].y : w[x][e >> 1].x;
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

template <typename T, int DA, int DC, bool OUT, bool EXACT>
int launch(const Sweep& s, int vec, cudaStream_t st) {
    constexpr int bytes = Layout<DA, DC, OUT>::bytes;
    CNL_TRY(ensure_dynamic_smem(mma_kernel<T, DA, DC, OUT, EXACT>, bytes));
    mma_kernel<T, DA, DC, OUT, EXACT><<<(unsigned)((long long)s.batch * s.h * s.segments), 2 * DC, bytes, st>>>(s, vec);
    return after_launch("linear attention sweep");
}

template <typename T, int DA, int DC>
int pick(const Sweep& s, int vec, cudaStream_t st) {
    constexpr bool kParts = std::is_same<T, __nv_bfloat16>::value;           // fp16 has one form
    if (s.exact && kParts) return s.out ? launch<T, DA, DC, true, kParts>(s, vec, st) : launch<T, DA, DC, false, kParts>(s, vec, st);
    return s.out ? launch<T, DA, DC, true, false>(s, vec, st) : launch<T, DA, DC, false, false>(s, vec, st);
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
