// One sweep of linear attention with a decay for each head: shared by the kernels and the drivers.
//
// Sweep over positions i = 0 .. n-1 of one head (l = exp(log_decay)):
//     out_i = out_scale ( in_scale sum_{j <= i} l^{i-j} (a_i . b_j) c_j  +  l^{i + off} a_i^T W_0 )
//     W_n   = l^n W_0 + in_scale sum_j l^{n - off - j} b_j c_j^T                          [da x dc]
// The four products of a training step are sweeps of this one form:
//     o : a = q,  b = k,  c = v,  forward,  off 1, W_0 = S_0,    W_n = S_T
//     dq: a = do, b = v,  c = k,  forward,  off 1, W_0 = S_0^T
//     dk: a = v,  b = do, c = q,  reversed, off 0, W_0 = dS_T^T
//     dv: a = k,  b = q,  c = do, reversed, off 0, W_0 = dS_T,   W_n = dS_0
// (reversed: position i is token n-1-i.)  A chunk of C positions keeps its own part in a C x C product and passes the rest
// through W, so the work is 2 C + 2 d multiply-adds an element instead of T.
#pragma once
#include "dtypes.cuh"

namespace cnl {
namespace lin {

struct Rows {                        // one operand [b][t][h][d], d contiguous
    const void* p;
    long long sb, st, sh;            // strides in elements
};

struct Sweep {
    Rows a, b, c;
    void* out;                       // [b][t][h][dc]; null: only W
    const float* log_decay;          // [h]
    const int* lengths;              // [b] or null
    const float* start;              // W at the start of every segment [b][h][segments][...] (one segment: W_0); null: 0
    float* end;                      // W at the end of every segment, from `start`; may be null
    int batch, t, h, da, dc;
    int segments, seg;               // segments of a sequence, positions of a segment
    int reversed, off;
    int transposed;                  // `start` is stored [dc][da]
    float in_scale, out_scale;
    int exact;                       // W at the end is a result, not only what later outputs are rounded from
};

__device__ __forceinline__ float clamp_log(float a) { return a < -1e30f ? -1e30f : a; }   // l = 0 keeps l^0 = 1; NaN stays

// l^n; n >= 0.  The product is rounded to 2^-24 of itself, so where l^n matters (a n > -20) it is off by 1e-6 at most
__device__ __forceinline__ float power(float a, int n) { return expf(a * (float)n); }

int run_sweep(const Sweep& s, int dtype, cudaStream_t st);          // dispatches to the kernel that serves the type and sizes
int run_sweep_f32(const Sweep& s, cudaStream_t st);
int run_sweep_mma(const Sweep& s, int dtype, cudaStream_t st);      // fp16, bf16: mma.sync
bool tc_sizes(int t, int da, int dc, int dtype);                    // sizes that the tcgen05 sweep serves
bool tc_serves(const Sweep& s, int dtype);                          // ... and rows that TMA can take
int run_sweep_tc(const Sweep& s, cudaStream_t st);                  // ... on the fifth-generation tensor cores

}  // namespace lin
}  // namespace cnl
