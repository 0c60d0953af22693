// Linear attention sweep in fp32 (formulas: linattn.cuh).
//
// A block of 256 threads walks one segment of one head in chunks of 64 positions.  Every product is plain multiply-adds on
// register tiles: a thread of the 16 x 16 grid holds rows ty, ty + 16, ... and D / 16 columns of the chunk's products, and a
// D / 16 x D / 16 tile of W in registers from chunk to chunk (a copy of W in shared memory is what a W reads).  Bound by the
// fp32 pipe: 2 D^2 + 1.25 * 64 D multiply-adds a position; the tiles keep shared-memory reads at 0.2 to 0.6 of what a
// multiply-add's issue slot leaves (rows are D + 4 floats apart, so that a warp's reads meet no bank twice).
// 2 x 7680 tokens x 8 heads of 128: 556 us forward (states and outputs), 1310 us backward; heads of 64 224 and 519 us.  Products
// that read both operands from shared memory a multiply-add at a time took 1516 us forward.
#include "linattn.cuh"

namespace cnl {
namespace lin {
namespace {

constexpr int kRows = 64, kThreads = 256;

template <int D>
struct Room {                                    // shared memory, in floats
    static constexpr int rd = D + 4, rp = kRows + 4;
    static constexpr int a = 0, b = a + kRows * rd, c = b + kRows * rd, w = c + kRows * rd, p = w + D * rd, pw = p + kRows * rp;
    static constexpr int end = pw + kRows + 4, bytes = end * 4;
};

template <int D>
__global__ void __launch_bounds__(kThreads, D == 128 ? 1 : D == 64 ? 2 : 4) sweep_f32(const Sweep s, const int vec) {
    using R = Room<D>;
    constexpr int G = D >= 64 ? D / 64 : 1, V = D >= 64 ? 4 : 2, TW = D / 16;        // column groups of a thread, their width; rows of its tile of W
    extern __shared__ float4 smem4[];
    float* sm = reinterpret_cast<float*>(smem4);
    const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
    const int seg = blockIdx.x % s.segments, bh = blockIdx.x / s.segments, head = bh % s.h, bat = bh / s.h;
    const float ld = clamp_log(s.log_decay[head]);
    const int n = s.lengths ? min(max(s.lengths[bat], 0), s.t) : s.t;
    const long long first = (long long)seg * s.seg;
    const int lo = (int)(first < n ? first : n), hi = (int)(first + s.seg < n ? first + s.seg : n);
    const int da = s.da, dc = s.dc;
    const long long size = (long long)da * dc;
    const bool out = s.out != nullptr;

    auto col = [&](int g) { return g * 64 + tx * V; };          // first column of group g
    auto wrow = [&](int r) { return (r / V) * 64 + ty * V + r % V; };      // row r of the tile of W (the same pattern)
    for (int i = tid; i <= kRows; i += kThreads) sm[R::pw + i] = power(ld, i);

    const float* w0 = s.start ? s.start + ((long long)bh * s.segments + seg) * size : nullptr;
    float w[TW][G][V];
#pragma unroll
    for (int r = 0; r < TW; ++r)
#pragma unroll
        for (int g = 0; g < G; ++g)
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const int i = wrow(r), j = col(g) + v;
                w[r][g][v] = w0 && i < da && j < dc ? (s.transposed ? w0[(long long)j * da + i] : w0[(long long)i * dc + j]) : 0.0f;
            }
    auto put = [](float* p, const float (&v)[V]) {
        if constexpr (V == 4) *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
        else *reinterpret_cast<float2*>(p) = make_float2(v[0], v[1]);
    };
    auto get = [](const float* p, float (&v)[V]) {
        if constexpr (V == 4) {
            const float4 f = *reinterpret_cast<const float4*>(p);
            v[0] = f.x; v[1] = f.y; v[2] = f.z; v[3] = f.w;
        } else {
            const float2 f = *reinterpret_cast<const float2*>(p);
            v[0] = f.x; v[1] = f.y;
        }
    };
    auto fetch = [&](const Rows& r, float* dst, int d, int c0, int m) {
        const long long by = s.reversed ? -r.st : r.st;
        const float* row = (const float*)r.p + bat * r.sb + head * r.sh + (s.reversed ? n - 1 - c0 : c0) * r.st;
        if (vec) {
#pragma unroll 4
            for (int e = tid; e < kRows * D / 4; e += kThreads) {
                const int j = e / (D / 4), x = e % (D / 4) * 4;
                *reinterpret_cast<float4*>(dst + j * R::rd + x) = j < m && x < d ? __ldg(reinterpret_cast<const float4*>(row + j * by + x)) : make_float4(0, 0, 0, 0);
            }
        } else {
            for (int e = tid; e < kRows * D; e += kThreads) {
                const int j = e / D, x = e % D;
                dst[j * R::rd + x] = j < m && x < d ? __ldg(row + j * by + x) : 0.0f;
            }
        }
    };

    for (int c0 = lo; c0 < hi; c0 += kRows) {
        const int m = min(kRows, hi - c0);
        __syncthreads();
        if (out) {
            fetch(s.a, sm + R::a, da, c0, m);
#pragma unroll
            for (int r = 0; r < TW; ++r)
#pragma unroll
                for (int g = 0; g < G; ++g) put(sm + R::w + wrow(r) * R::rd + col(g), w[r][g]);
        }
        fetch(s.b, sm + R::b, da, c0, m);
        fetch(s.c, sm + R::c, dc, c0, m);
        __syncthreads();
        if (out) {
            // P: rows ty + 16 i, columns tx + 16 j, blocks on and under the diagonal
            {
                float p[4][4] = {};
#pragma unroll 2
                for (int x = 0; x < D; x += 4) {
                    float4 a[4], b[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        a[i] = *reinterpret_cast<const float4*>(sm + R::a + (ty + 16 * i) * R::rd + x);
                        b[i] = *reinterpret_cast<const float4*>(sm + R::b + (tx + 16 * i) * R::rd + x);
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i)
#pragma unroll
                        for (int j = 0; j <= i; ++j) {
                            p[i][j] = fmaf(a[i].x, b[j].x, p[i][j]); p[i][j] = fmaf(a[i].y, b[j].y, p[i][j]);
                            p[i][j] = fmaf(a[i].z, b[j].z, p[i][j]); p[i][j] = fmaf(a[i].w, b[j].w, p[i][j]);
                        }
                }
                const float both = s.in_scale * s.out_scale;
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int j = 0; j <= i; ++j) {
                        const int d = ty + 16 * i - tx - 16 * j;
                        sm[R::p + (ty + 16 * i) * R::rp + tx + 16 * j] = d >= 0 ? p[i][j] * (both * sm[R::pw + max(d, 0)]) : 0.0f;
                    }
            }
            // l^{i + off} a W
            float o[4][G][V] = {};
#pragma unroll 2
            for (int x = 0; x < D; x += 4) {
                float4 a[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) a[i] = *reinterpret_cast<const float4*>(sm + R::a + (ty + 16 * i) * R::rd + x);
#pragma unroll
                for (int y = 0; y < 4; ++y)
#pragma unroll
                    for (int g = 0; g < G; ++g) {
                        float q[V];
                        get(sm + R::w + (x + y) * R::rd + col(g), q);
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const float f = y == 0 ? a[i].x : y == 1 ? a[i].y : y == 2 ? a[i].z : a[i].w;
#pragma unroll
                            for (int v = 0; v < V; ++v) o[i][g][v] = fmaf(f, q[v], o[i][g][v]);
                        }
                    }
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float f = s.out_scale * power(ld, ty + 16 * i + s.off);
#pragma unroll
                for (int g = 0; g < G; ++g)
#pragma unroll
                    for (int v = 0; v < V; ++v) o[i][g][v] *= f;
            }
            __syncthreads();
            // + P c
#pragma unroll
            for (int jb = 0; jb < 4; ++jb)
#pragma unroll 2
                for (int x = 0; x < 16; x += 4) {
                    float4 p[4];
#pragma unroll
                    for (int i = jb; i < 4; ++i) p[i] = *reinterpret_cast<const float4*>(sm + R::p + (ty + 16 * i) * R::rp + jb * 16 + x);
#pragma unroll
                    for (int y = 0; y < 4; ++y)
#pragma unroll
                        for (int g = 0; g < G; ++g) {
                            float q[V];
                            get(sm + R::c + (jb * 16 + x + y) * R::rd + col(g), q);
#pragma unroll
                            for (int i = jb; i < 4; ++i) {
                                const float f = y == 0 ? p[i].x : y == 1 ? p[i].y : y == 2 ? p[i].z : p[i].w;
#pragma unroll
                                for (int v = 0; v < V; ++v) o[i][g][v] = fmaf(f, q[v], o[i][g][v]);
                            }
                        }
                }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int r = ty + 16 * i;
                if (r < m) {
                    const long long tok = s.reversed ? n - 1 - (c0 + r) : c0 + r;
                    float* to = (float*)s.out + (((long long)bat * s.t + tok) * s.h + head) * dc;
#pragma unroll
                    for (int g = 0; g < G; ++g) {
                        if (V == 4 && vec) {
                            if (col(g) < dc) put(to + col(g), o[i][g]);
                        } else {
#pragma unroll
                            for (int v = 0; v < V; ++v)
                                if (col(g) + v < dc) to[col(g) + v] = o[i][g][v];
                        }
                    }
                }
            }
        }
        // W <- l^m W + in_scale sum_j l^{m - off - j} b_j c_j^T
        const float keep = sm[R::pw + m];
#pragma unroll
        for (int r = 0; r < TW; ++r)
#pragma unroll
            for (int g = 0; g < G; ++g)
#pragma unroll
                for (int v = 0; v < V; ++v) w[r][g][v] *= keep;
#pragma unroll 2
        for (int j = 0; j < m; ++j) {
            const float f = s.in_scale * sm[R::pw + max(m - s.off - j, 0)];
            float b[TW], c[G][V];
#pragma unroll
            for (int r = 0; r < TW; r += V) {
                float q[V];
                get(sm + R::b + j * R::rd + wrow(r), q);
#pragma unroll
                for (int v = 0; v < V; ++v) b[r + v] = f * q[v];
            }
#pragma unroll
            for (int g = 0; g < G; ++g) get(sm + R::c + j * R::rd + col(g), c[g]);
#pragma unroll
            for (int r = 0; r < TW; ++r)
#pragma unroll
                for (int g = 0; g < G; ++g)
#pragma unroll
                    for (int v = 0; v < V; ++v) w[r][g][v] = fmaf(b[r], c[g][v], w[r][g][v]);
        }
    }
    if (s.end) {
        float* w1 = s.end + ((long long)bh * s.segments + seg) * size;
#pragma unroll
        for (int r = 0; r < TW; ++r)
#pragma unroll
            for (int g = 0; g < G; ++g)
#pragma unroll
                for (int v = 0; v < V; ++v)
                    if (wrow(r) < da && col(g) + v < dc) w1[(long long)wrow(r) * dc + col(g) + v] = w[r][g][v];
    }
    if (out) {                                                   // rows behind the sequence's end
        const long long zlo = first > n ? first : n, zhi = first + s.seg < s.t ? first + s.seg : s.t;
        for (long long e = zlo * dc + tid; e < zhi * dc; e += kThreads) {
            const long long tok = e / dc;
            ((float*)s.out)[(((long long)bat * s.t + tok) * s.h + head) * dc + (e - tok * dc)] = 0.0f;
        }
    }
}

template <int D>
int launch(const Sweep& s, int vec, cudaStream_t st) {
    CNL_TRY(ensure_dynamic_smem(sweep_f32<D>, Room<D>::bytes));
    sweep_f32<D><<<(unsigned)((long long)s.batch * s.h * s.segments), kThreads, Room<D>::bytes, st>>>(s, vec);
    return after_launch("linear attention sweep");
}

}  // namespace

int run_sweep_f32(const Sweep& s, cudaStream_t st) {
    auto ok = [](const Rows& r) { return !r.p || (aligned16(r.p) && r.sb % 4 == 0 && r.st % 4 == 0 && r.sh % 4 == 0); };
    const int vec = s.da % 4 == 0 && s.dc % 4 == 0 && ok(s.a) && ok(s.b) && ok(s.c) && aligned16(s.out);
    const int d = s.da > s.dc ? s.da : s.dc;
    return d <= 32 ? launch<32>(s, vec, st) : d <= 64 ? launch<64>(s, vec, st) : launch<128>(s, vec, st);
}

}  // namespace lin
}  // namespace cnl
