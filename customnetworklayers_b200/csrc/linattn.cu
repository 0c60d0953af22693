// Linear attention with a decay for each head: drivers, the scan over segments and the single-token step (formulas:
// linattn.cuh; sweeps: linattn_f32.cu, linattn_mma.cu, linattn_tc.cu).
#include "linattn.cuh"

namespace cnl {
namespace lin {

constexpr int kMaxD = 128;

int run_sweep(const Sweep& s, int dtype, cudaStream_t st) {
    if (dtype == CNL_F32) return run_sweep_f32(s, st);
    return tc_serves(s, dtype) ? run_sweep_tc(s, st) : run_sweep_mma(s, dtype, st);
}

// ---- scan over the segments -------------------------------------------------------------------------------------
// local[seg] (W of every segment from 0) becomes W at the segment's start; `last` receives W at the sequence's end.
// Four entries a thread where the sizes allow it, eight segments asked for together.  Latency of the few segments; 64 heads of
// 128 x 128 in 9 segments 14 us, of 38 MB read and written.
template <int V>
__global__ void __launch_bounds__(128) scan_kernel(float* __restrict__ local, const float* __restrict__ init, float* __restrict__ last,
                                                   const float* __restrict__ log_decay, const int* __restrict__ lengths, int t, int h,
                                                   int size, int segments, int seg) {
    const int parts = (size + 128 * V - 1) / (128 * V);
    const long long bh = blockIdx.x / parts;
    const int e = ((int)(blockIdx.x - bh * parts) * 128 + threadIdx.x) * V;
    if (e >= size) return;
    const float ld = clamp_log(log_decay[bh % h]);
    const int n = lengths ? min(max(lengths[bh / h], 0), t) : t;
    float* p = local + bh * segments * size + e;
    const float whole = power(ld, seg);
    auto get = [](const float* q, float (&v)[V]) {
        if constexpr (V == 4) {
            const float4 f = *reinterpret_cast<const float4*>(q);
            v[0] = f.x; v[1] = f.y; v[2] = f.z; v[3] = f.w;
        } else v[0] = *q;
    };
    auto put = [](float* q, const float (&v)[V]) {
        if constexpr (V == 4) *reinterpret_cast<float4*>(q) = make_float4(v[0], v[1], v[2], v[3]);
        else *q = v[0];
    };
    float w[V] = {};
    if (init) get(init + bh * size + e, w);
    constexpr int kAhead = 8;
    for (int s0 = 0; s0 < segments; s0 += kAhead) {
        float v[kAhead][V];
#pragma unroll
        for (int i = 0; i < kAhead; ++i)
            if (s0 + i < segments) get(p + (long long)(s0 + i) * size, v[i]);
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            if (s0 + i >= segments) break;
            put(p + (long long)(s0 + i) * size, w);
            const long long left = n - (long long)(s0 + i) * seg;
            const float keep = left >= seg ? whole : power(ld, (int)(left < 0 ? 0 : left));
#pragma unroll
            for (int x = 0; x < V; ++x) w[x] = fmaf(keep, w[x], v[i][x]);
        }
    }
    if (last) put(last + bh * size + e, w);
}

int run_scan(float* local, const float* init, float* last, const float* log_decay, const int* lengths, int b, int t, int h, int size,
             int segments, int seg, cudaStream_t st) {
    const bool four = size % 4 == 0 && aligned16(local) && aligned16(init) && aligned16(last);
    const int per = four ? 512 : 128;
    const unsigned grid = (unsigned)((long long)((size + per - 1) / per) * b * h);
    if (four) scan_kernel<4><<<grid, 128, 0, st>>>(local, init, last, log_decay, lengths, t, h, size, segments, seg);
    else scan_kernel<1><<<grid, 128, 0, st>>>(local, init, last, log_decay, lengths, t, h, size, segments, seg);
    return after_launch("linear attention scan");
}

// ---- one token --------------------------------------------------------------------------------------------------
// S <- l S + k v^T in place, o = scale q^T S.  One block a head; reads and writes the state once: HBM bound, 8 dk dv bytes.
// 128 x 16 heads of 128 x 128 47 us (268 MB, 5.8 TB/s); with eight rows of the loop merely unrolled, 51 us.  Small calls are one
// launch's latency: 16 heads 10 us.
template <typename T, int V>
__global__ void __launch_bounds__(256, 4) step_kernel(const T* __restrict__ q, const T* __restrict__ k, const T* __restrict__ v,
                                                   const float* __restrict__ log_decay, float* __restrict__ state, T* __restrict__ out,
                                                   int h, int dk, int dv, int cols, float scale, long long qb, long long qh, long long kb,
                                                   long long kh, long long vb, long long vh) {
    __shared__ float sq[kMaxD], sk[kMaxD], red[256 * V];
    const long long bh = blockIdx.x;
    const int head = (int)(bh % h);
    const long long bat = bh / h;
    for (int i = threadIdx.x; i < dk; i += 256) {
        sq[i] = to_f32(q[bat * qb + head * qh + i]);
        sk[i] = to_f32(k[bat * kb + head * kh + i]);
    }
    const int tx = threadIdx.x % cols, ty = threadIdx.x / cols, rows = 256 / cols, x = tx * V;
    const bool live = x < dv;
    const float l = expf(clamp_log(log_decay[head]));
    float vv[V], acc[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        vv[i] = live ? to_f32(v[bat * vb + head * vh + x + i]) : 0.0f;
        acc[i] = 0.0f;
    }
    __syncthreads();
    float* s = state + bh * dk * dv + x;
    if (live) {
        constexpr int kAhead = 8;                                // rows of the state asked for together
        for (int y0 = ty; y0 < dk; y0 += kAhead * rows) {
            float w[kAhead][V];
#pragma unroll
            for (int k = 0; k < kAhead; ++k) {
                const int y = y0 + k * rows;
                if (y < dk) {
                    if constexpr (V == 4) {
                        const float4 f = *reinterpret_cast<const float4*>(s + (long long)y * dv);
                        w[k][0] = f.x; w[k][1] = f.y; w[k][2] = f.z; w[k][3] = f.w;
                    } else w[k][0] = s[(long long)y * dv];
                }
            }
#pragma unroll
            for (int k = 0; k < kAhead; ++k) {
                const int y = y0 + k * rows;
                if (y >= dk) break;
                const float kk = sk[y], qq = sq[y];
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    w[k][i] = fmaf(l, w[k][i], kk * vv[i]);
                    acc[i] = fmaf(qq, w[k][i], acc[i]);
                }
                if constexpr (V == 4) *reinterpret_cast<float4*>(s + (long long)y * dv) = make_float4(w[k][0], w[k][1], w[k][2], w[k][3]);
                else s[(long long)y * dv] = w[k][0];
            }
        }
    }
#pragma unroll
    for (int i = 0; i < V; ++i) red[i * 256 + threadIdx.x] = acc[i];
    __syncthreads();
    if (ty == 0 && live) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            float o = 0.0f;
            for (int r = 0; r < rows; ++r) o += red[i * 256 + r * cols + tx];
            out[bh * dv + x + i] = from_f32<T>(scale * o);
        }
    }
}

template <typename T>
int launch_step(const void* q, const void* k, const void* v, const long long* st6, const float* log_decay, float* state, void* out, int b,
                int h, int dk, int dv, float scale, cudaStream_t st) {
    const bool vec = dv % 4 == 0 && aligned16(state);
    const int need = vec ? dv / 4 : dv;
    int cols = 1;
    while (cols < need) cols <<= 1;
    const unsigned grid = (unsigned)((long long)b * h);
    if (vec)
        step_kernel<T, 4><<<grid, 256, 0, st>>>((const T*)q, (const T*)k, (const T*)v, log_decay, state, (T*)out, h, dk, dv, cols, scale, st6[0], st6[1], st6[2], st6[3], st6[4], st6[5]);
    else
        step_kernel<T, 1><<<grid, 256, 0, st>>>((const T*)q, (const T*)k, (const T*)v, log_decay, state, (T*)out, h, dk, dv, cols, scale, st6[0], st6[1], st6[2], st6[3], st6[4], st6[5]);
    return after_launch("linear attention step");
}

int check(int b, int t, int h, int dk, int dv, int dtype) {
    if (b < 0 || t < 0 || h < 1 || dk < 1 || dv < 1 || dk > kMaxD || dv > kMaxD)
        return fail(CNL_ERR_BAD_SHAPE, "b %d, t %d, h %d, dk %d, dv %d: head sizes must be within 1..%d", b, t, h, dk, dv, kMaxD);
    if ((long long)b * h > (1 << 24)) return fail(CNL_ERR_BAD_SHAPE, "b * h = %lld is above 2^24", (long long)b * h);
    return check_dtype(dtype);
}

// Segments of a sequence.  All blocks take about the same time, so a launch lasts as many rounds as it has blocks for one
// place: the segment count with the fewest rounds times positions wins, a segment counting `kExtra` positions more for its
// state's way through memory.
int segment_plan(int b, int t, int h, int dk, int dv, int dtype, int* segments, int* seg) {
    constexpr int kExtra = 128;
    int sms = 0;
    CNL_TRY(sm_count(&sms));
    const int d = dk > dv ? dk : dv;
    const bool tc = tc_sizes(t, dk, dv, dtype);
    const long long heads = ((long long)b * h > 0 ? (long long)b * h : 1);
    // blocks that an SM holds of the kernel that serves these sizes
    const int each = dtype == CNL_F32 ? (d > 64 ? 1 : d > 32 ? 2 : 4) : tc ? 1 : d > 64 ? 2 : d > 32 ? 4 : 8;
    const long long places = (long long)sms * each, most = (t + 127) / 128;
    long long best = 0;
    *segments = 1;
    *seg = (int)(((long long)t + 127) / 128 * 128);
    if (*seg < 128) *seg = 128;
    for (long long want = 1; want <= most && (want - 1) * heads < 4 * places; ++want) {
        const long long len = ((t + want - 1) / want + 127) / 128 * 128, have = (t + len - 1) / len;
        const long long cost = (heads * have + places - 1) / places * (len + kExtra);
        if (best == 0 || cost < best) {
            best = cost;
            *segments = (int)have;
            *seg = (int)len;
        }
    }
    return CNL_OK;
}

}  // namespace lin
}  // namespace cnl

using namespace cnl;
using namespace cnl::lin;

extern "C" int cnl_linattn_segments(int b, int t, int h, int dk, int dv, int dtype) {
    int segments = 0, seg = 0;
    if (lin::check(b, t, h, dk, dv, dtype) != CNL_OK || segment_plan(b, t, h, dk, dv, dtype, &segments, &seg) != CNL_OK) return -1;
    return segments;
}

extern "C" int cnl_linattn_forward(const void* q, const void* k, const void* v, const long long* strides_host, const float* log_decay,
                                   const int* lengths, const float* state, void* out, float* state_out, float* starts, int b, int t, int h,
                                   int dk, int dv, float scale, int dtype, void* stream) {
    CNL_TRY(lin::check(b, t, h, dk, dv, dtype));
    if (b == 0) return CNL_OK;
    if ((t > 0 && (!q || !k || !v || !out)) || !strides_host || !log_decay) return fail(CNL_ERR_NULL, "null pointer argument");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    int segments = 0, seg = 0;
    CNL_TRY(segment_plan(b, t, h, dk, dv, dtype, &segments, &seg));
    if (segments > 1 && !starts) return fail(CNL_ERR_NULL, "%d segments need the starts buffer", segments);
    const long long* s = strides_host;
    const Rows Q = {q, s[0], s[1], s[2]}, Kk = {k, s[3], s[4], s[5]}, V = {v, s[6], s[7], s[8]};
    Sweep w = {};
    w.log_decay = log_decay; w.lengths = lengths; w.batch = b; w.t = t; w.h = h; w.segments = segments; w.seg = seg;
    w.b = Kk; w.c = V; w.da = dk; w.dc = dv; w.off = 1; w.in_scale = 1.0f; w.out_scale = scale; w.exact = state_out != nullptr;
    if (segments > 1) {
        w.end = starts;
        CNL_TRY(run_sweep(w, dtype, st));
        CNL_TRY(run_scan(starts, state, state_out, log_decay, lengths, b, t, h, dk * dv, segments, seg, st));
        w.start = starts; w.end = nullptr; w.exact = 0;
    } else {
        w.start = state; w.end = state_out;
    }
    w.a = Q; w.out = out;
    return run_sweep(w, dtype, st);
}

extern "C" int cnl_linattn_backward(const void* q, const void* k, const void* v, const void* g_out, const long long* strides_host,
                                    const float* log_decay, const int* lengths, const float* state, const float* starts,
                                    const float* g_state_out, void* g_q, void* g_k, void* g_v, float* g_state, float* scratch, int b, int t,
                                    int h, int dk, int dv, float scale, int dtype, void* stream) {
    CNL_TRY(lin::check(b, t, h, dk, dv, dtype));
    if (b == 0) return CNL_OK;
    if ((t > 0 && (!q || !k || !v || !g_out || !g_q || !g_k || !g_v)) || !strides_host || !log_decay) return fail(CNL_ERR_NULL, "null pointer argument");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    int segments = 0, seg = 0;
    CNL_TRY(segment_plan(b, t, h, dk, dv, dtype, &segments, &seg));
    if (segments > 1 && (!starts || !scratch)) return fail(CNL_ERR_NULL, "%d segments need starts and scratch", segments);
    const long long* s = strides_host;
    const Rows Q = {q, s[0], s[1], s[2]}, Kk = {k, s[3], s[4], s[5]}, V = {v, s[6], s[7], s[8]}, G = {g_out, s[9], s[10], s[11]};
    Sweep w = {};
    w.log_decay = log_decay; w.lengths = lengths; w.batch = b; w.t = t; w.h = h; w.segments = segments; w.seg = seg;
    // dq
    w.a = G; w.b = V; w.c = Kk; w.da = dv; w.dc = dk; w.off = 1; w.in_scale = 1.0f; w.out_scale = scale;
    w.start = segments > 1 ? starts : state; w.transposed = 1; w.out = g_q;
    CNL_TRY(run_sweep(w, dtype, st));
    // the reversed sweeps: W = sum of scale l^.. q do^T
    w.off = 0; w.reversed = 1; w.in_scale = scale; w.out_scale = 1.0f;
    w.b = Q; w.c = G; w.da = dk; w.dc = dv; w.transposed = 0; w.start = nullptr; w.out = nullptr; w.exact = g_state != nullptr;
    if (segments > 1) {
        w.end = scratch;
        CNL_TRY(run_sweep(w, dtype, st));
        CNL_TRY(run_scan(scratch, g_state_out, g_state, log_decay, lengths, b, t, h, dk * dv, segments, seg, st));
        w.start = scratch; w.end = nullptr; w.exact = 0;
    } else {
        w.start = g_state_out; w.end = g_state;
    }
    w.a = Kk; w.out = g_v;
    CNL_TRY(run_sweep(w, dtype, st));
    w.end = nullptr; w.exact = 0;
    w.a = V; w.b = G; w.c = Q; w.da = dv; w.dc = dk; w.transposed = 1; w.out = g_k;
    return run_sweep(w, dtype, st);
}

extern "C" int cnl_linattn_step(const void* q, const void* k, const void* v, const long long* strides_host, const float* log_decay, float* state,
                                void* out, int b, int h, int dk, int dv, float scale, int dtype, void* stream) {
    CNL_TRY(lin::check(b, 1, h, dk, dv, dtype));
    if (b == 0) return CNL_OK;
    if (!q || !k || !v || !strides_host || !log_decay || !state || !out) return fail(CNL_ERR_NULL, "null pointer argument");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (dtype == CNL_F32) return launch_step<float>(q, k, v, strides_host, log_decay, state, out, b, h, dk, dv, scale, st);
    if (dtype == CNL_F16) return launch_step<__half>(q, k, v, strides_host, log_decay, state, out, b, h, dk, dv, scale, st);
    return launch_step<__nv_bfloat16>(q, k, v, strides_host, log_decay, state, out, b, h, dk, dv, scale, st);
}
