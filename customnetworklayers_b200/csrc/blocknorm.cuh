// Shared by the two translation units of the block norms: arguments, the plan of a launch, small helpers.
#pragma once
#include "ckpt8.cuh"

namespace cnl {
namespace bnorm {

constexpr int K = 8;                 // channels a thread holds
constexpr int kMaxD = 8192;
constexpr int kSums = 4;             // A, B, dw1, db1

struct Args {
    const void *x, *u, *gate;                     // [rows][d]; gate [rows][d], [groups][d] or null
    const void *scale, *w2, *b2, *w1, *b1;        // [d] each, scale / b2 / b1 may be null; w1 null: no h
    void *y, *h;
    float4* stats;                                // per row: mu_u, r_u, mu_y, r_y
    unsigned char *codes, *scales;                // 8-bit forms of x, u and a full gate, [3][rows][d] and [3][rows][blocks]
    const void *dy, *dh;
    void *dx, *du, *dgate;
    float* partial;                               // [groups * nb][4][d]
    long long rows, per;                          // rows in all, rows of a group
    int d, tpr, nb;                               // channels, threads of a row, blocks of a group
    float eps, inv_d;
    int layer, gate_full, gate_group, sigmoid, w_f32, fmt;
    int need_b;                                   // the sums B and db1 are asked for, or a bias enters n
};

// Threads of a row, rows of a block, blocks of a group.
struct Plan {
    int tpr, block, rpb, nb;
    long long groups;
};

__device__ __forceinline__ float sigmoid(float z) { return rcp_approx(1.0f + exp2_approx(-1.4426950408889634f * z)); }

// The vector kernels (blocknorm_vec.cu): d a multiple of 8 and at most kVecMaxD, 16-byte aligned rows.
constexpr int kVecMaxD = 4096;
int run_forward_vec(const Args& a, const Plan& p, int dtype, cudaStream_t st);
int run_backward_vec(const Args& a, const Plan& p, int dtype, cudaStream_t st);

}  // namespace bnorm
}  // namespace cnl
