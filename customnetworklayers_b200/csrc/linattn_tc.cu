// Linear attention sweep for bf16 on the fifth-generation tensor cores (formulas: linattn.cuh).
//
// A block of 18 warps walks one segment of one head in chunks of 128 tokens.  One warp brings a, b, c rows by TMA (128-byte
// swizzle), one thread issues the products, sixteen warps do what lies between.  Per chunk, accumulators in tensor memory:
//     P = a b^T                 [128 tokens x 128 tokens]   -> weighted, masked, rounded, put back in tensor memory
//     X = a W                   [128 tokens x dc]           W as the sweep has it before the chunk
//     O = P c                   [128 tokens x dc]
//     T = (weighted c)^T b      [dc x da]                   what the chunk adds to W^T
// and in registers W^T <- l^m W^T + T (fp32), out = l^{pos + off} X + O.  Nothing of the recurrence passes through the tensor
// cores: T needs only the chunk's own rows, so it is summed while the outputs are finished.  Reversed sweeps take the tokens
// of a chunk in their order in memory and turn the mask and the weights around instead.
//
// Operands: a and b for P, P, and W lie with the summed dimension contiguous; c, its parts, and b for T with it strided
// (their rows are tokens), which the descriptors say.  Roundings as in the mma.sync kernel, so that a result carries its own
// rounding and little else: P and W are two bf16 parts each (16 bits; P's lie side by side in P's columns of tensor memory, W's
// smaller one waits in the parts' room until X has read it), the weighted c two or, where the state is a result, three.  With up to 64 columns of
// c (DC = 64) two parts fill the 128 rows of T, so W is kept in two addends, which X meets side by side; three parts are
// (c0 | c1 / 2) and (c1 / 2 | c2).  With 128 columns the parts add up in T.  P and W rounded once would take 10 to 13 % less time
// (1 x 122880 x 8 x 64 forward 194 instead of 216 us, 8 x 7680 x 8 x 128 backward 451 instead of 497 us) at 1.4 times the error: 2.35e-3 rms of
// the outputs against 1.66e-3, which the outputs' own rounding is.
//
// Measured, bf16 (one sweep with its outputs; beside it a call's states take 61 and 64 us, a scan 12 to 20): 1 x 122880 tokens x 8
// heads of 64 148 us, 8 x 7680 x 8 x 128 134 us (rows of 503 MB in and out: 3.4 and 3.8 TB/s).  Tensor pipes are active on 28 to
// 39 % of cycles, instructions issue on 35 to 43 %: what bounds a chunk is the chain weights -> P -> outputs with 16 warps to hide
// it, and the operands' way through shared memory; a second block would not fit either memory.
//
// Every wait is bounded: a block that gives up marks the status word, fills what it owes with NaN, and returns after its
// copies and products have ended.
#include <cuda.h>

#include <atomic>

#include "linattn.cuh"

namespace cnl {
namespace lin {

__device__ int g_gave_up = 0;

constexpr int kTok = 128;                       // tokens of a chunk
constexpr int kBlk = kTok * 128;                // bytes of 128 rows of 64 elements
constexpr int kWorkers = 16;                    // warps between the products
constexpr int kTcThreads = (kWorkers + 2) * 32;
constexpr int kSpins = 1 << 22;

// ---- the machine's words ------------------------------------------------------------------------------------------
__device__ __forceinline__ unsigned smem_at(const void* p) { return (unsigned)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void bar_init(unsigned bar, int count) { asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory"); }
__device__ __forceinline__ void bar_arrive(unsigned bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory"); }
__device__ __forceinline__ void bar_expect(unsigned bar, int bytes) { asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory"); }
__device__ __forceinline__ bool bar_try(unsigned bar, unsigned parity) {
    unsigned ok;
    asm volatile("{\n.reg .pred p;\nmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\nselp.u32 %0, 1, 0, p;\n}" : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    return ok != 0;
}
// true when the phase has ended; false when it did not within the limit or another warp has given up
__device__ __forceinline__ bool bar_wait(unsigned bar, unsigned parity, volatile int* dead) {
    for (int i = 0; i < kSpins; ++i) {
        if (bar_try(bar, parity)) return true;
        if ((i & 255) == 255 && *dead) return false;
    }
    *dead = 1;
    return false;
}
__device__ __forceinline__ void tma_load(unsigned to, const CUtensorMap* map, int x, int h, int t, int b, unsigned bar) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(to), "l"(map), "r"(x), "r"(h), "r"(t), "r"(b), "r"(bar) : "memory");
}
__device__ __forceinline__ void tma_ahead(const CUtensorMap* map, int x, int h, int t, int b) {      // into L2
    asm volatile("cp.async.bulk.prefetch.tensor.4d.L2.global.tile [%0, {%1, %2, %3, %4}];" ::"l"(map), "r"(x), "r"(h), "r"(t), "r"(b) : "memory");
}
// 16 bytes of shared memory by address: a generic pointer, which alignment by hand leaves, would cost the slower path
__device__ __forceinline__ uint4 smem_get(unsigned at) {
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ void smem_put(unsigned at, uint4 v) { asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(at), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory"); }
__device__ __forceinline__ void smem_put(unsigned at, float v) { asm volatile("st.shared.f32 [%0], %1;" ::"r"(at), "f"(v) : "memory"); }
__device__ __forceinline__ float smem_get1(unsigned at) {
    float v;
    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ void tma_store(const CUtensorMap* map, unsigned from, int x, int h, int t, int b) {
    asm volatile("cp.async.bulk.tensor.4d.global.shared::cta.tile.bulk_group [%0, {%1, %2, %3, %4}], [%5];" ::"l"(map), "r"(x), "r"(h), "r"(t), "r"(b), "r"(from) : "memory");
}
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void tc_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_commit(unsigned bar) { asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory"); }
__device__ __forceinline__ void tc_mma(unsigned d, unsigned long long a, unsigned long long b, unsigned what, bool add) {
    asm volatile("{\n.reg .pred p;\nsetp.ne.u32 p, %4, 0;\ntcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d), "l"(a), "l"(b), "r"(what), "r"((unsigned)add) : "memory");
}
// the same with the rows' operand in tensor memory: 128 lanes, two summed elements a column
__device__ __forceinline__ void tc_mma_t(unsigned d, unsigned a, unsigned long long b, unsigned what, bool add) {
    asm volatile("{\n.reg .pred p;\nsetp.ne.u32 p, %4, 0;\ntcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}" ::"r"(d), "r"(a), "l"(b), "r"(what), "r"((unsigned)add) : "memory");
}
// 32 lanes of the warp's quarter, 16 or 32 columns
__device__ __forceinline__ void tc_load(unsigned at, unsigned (&r)[16]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                 : "r"(at));
}
__device__ __forceinline__ void tc_load(unsigned at, unsigned (&r)[32]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
                 : "r"(at));
}
__device__ __forceinline__ void tc_store(unsigned at, const unsigned (&r)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(at) : "memory");
}
__device__ __forceinline__ void tc_wait_store() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tc_wait_load() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

// Descriptor of an operand in shared memory, 128-byte swizzle, groups of 8 rows 1024 bytes apart.  Its upper word is the same
// for all; the lower one is the address, and with the summed dimension strided the distance of 64-element columns.  Products
// differ by a constant in it: built anew for every product, and by one lane on its own, the descriptors cost 150 to 200 clocks
// a product, where the product itself takes 43 + n / 2 (10 + n / 2 with the rows' operand in tensor memory), measured.
__device__ __forceinline__ unsigned rows_word(unsigned at) { return (at & 0x3ffffu) >> 4 | 1u << 16; }
__device__ __forceinline__ unsigned columns_word(unsigned at, int blk = kBlk) { return (at & 0x3ffffu) >> 4 | (unsigned)(blk >> 4) << 16; }
__device__ __forceinline__ unsigned long long operand(unsigned word, int further) {
    return (unsigned long long)(1024u >> 4 | 1u << 14 | 2u << 29) << 32 | (word + (unsigned)(further >> 4));
}
__device__ __forceinline__ bool elected() {                     // one lane of the warp
    unsigned one;
    asm volatile("{\n.reg .pred q;\nelect.sync _|q, 0xffffffff;\nselp.u32 %0, 1, 0, q;\n}" : "=r"(one));
    return one != 0;
}
// Instruction word: fp32 sums of bf16 products, 128 rows, n columns; strided a / b
__host__ __device__ constexpr unsigned product(int n, int strided_a, int strided_b) {
    return 1u << 4 | 1u << 7 | 1u << 10 | (unsigned)strided_a << 15 | (unsigned)strided_b << 16 | (unsigned)(n >> 3) << 17 | 8u << 24;
}

// W^T <- keep W^T + T of tensor memory
template <int HC>
__device__ __forceinline__ void add_chunk(float2 (&w)[HC / 2], unsigned from, float keep) {
    unsigned r[HC];
    tc_load(from, r);
    tc_wait_load();
#pragma unroll
    for (int x = 0; x < HC / 2; ++x) w[x] = __ffma2_rn(make_float2(keep, keep), w[x], make_float2(__uint_as_float(r[2 * x]), __uint_as_float(r[2 * x + 1])));
}
// Eight elements of c, weighted, in parts of 8 bits each
template <int PARTS, bool kStack>
__device__ __forceinline__ void split(uint4 v, float weight, uint4 (&out)[PARTS]) {
    const unsigned in[4] = {v.x, v.y, v.z, v.w};
    unsigned part[PARTS][4];
    const float2 f = make_float2(weight, weight);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        float2 y = __fmul2_rn(unpack2(in[e], __nv_bfloat16()), f);
#pragma unroll
        for (int p = 0; p < PARTS; ++p) {
            part[p][e] = pack2<__nv_bfloat16>(y.x, y.y);
            if (p + 1 < PARTS) {
                const float2 z = unpack2(part[p][e], __nv_bfloat16());
                y = __fadd2_rn(y, make_float2(-z.x, -z.y));
                if (kStack && PARTS == 3 && p == 1) part[p][e] = pack2<__nv_bfloat16>(0.5f * z.x, 0.5f * z.y);       // it is there twice
            }
        }
    }
#pragma unroll
    for (int p = 0; p < PARTS; ++p) out[p] = make_uint4(part[p][0], part[p][1], part[p][2], part[p][3]);
}

template <int DA, int DC, int PARTS>
struct Map {                                    // shared memory in bytes from a 1024-byte boundary
    static constexpr int one = DA / 64 * kBlk, one_c = DC / 64 * kBlk;     // a's or b's rows; c's, or one part of them
    // rooms: two of each as far as they go.  a is free first, then c; b is held longest
    static constexpr int two_a = DA == 128 ? 1 : 2, two_b = 2, two_c = DA == 128 && DC == 128 ? 1 : 2;
    // output rows on their way: rooms of their own, or (128 columns) c's, which O and the parts were the last to read
    static constexpr bool through_c = DC == 128;
    static constexpr int two_r = through_c ? two_c : DA == 128 && PARTS == 3 ? 1 : 2;
    static constexpr int a = 0, b = a + two_a * one, c = b + two_b * one, w = c + two_c * one_c;
    static constexpr int parts = w + one, rows = parts + PARTS * one_c;
    static constexpr int bars = rows + (through_c ? 0 : two_r * kBlk);
    static constexpr int bytes = bars + 272 + 1024;              // and the way to the boundary
};

// ---- the sweep -----------------------------------------------------------------------------------------------------
template <int DA, int DC, int PARTS>
__global__ void __launch_bounds__(kTcThreads, 1) tc_kernel(const Sweep s, const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                                                           const __grid_constant__ CUtensorMap map_c, const __grid_constant__ CUtensorMap map_o) {
    using M = Map<DA, DC, PARTS>;
    constexpr bool kStack = DC == 64;
    extern __shared__ unsigned char raw[];
    __shared__ float whole[32], edge[64];                        // powers of the decay for P: for whole tiles, for diagonal ones
    __shared__ int dead_word;
    __shared__ unsigned tmem_word;
    const unsigned base = (smem_at(raw) + 1023u) & ~1023u, bars = base + M::bars;
    volatile int* dead = &dead_word;
    // barriers, two of each: chunk i uses number i mod 2, whose phase is then i / 2
    enum { FULL_A, FULL_B, FULL_C, DONE_P, DONE_X, DONE_T, DONE_O, HAS_C, HAS_P, HAS_W, HAS_O, HAS_R, CLEARED, SENT, KINDS };
    auto read_p = [&](int quarter) { return bars + (unsigned)(KINDS * 2 + quarter) * 8; };      // P's fp32 columns of these lanes have been read
    auto bar = [&](int kind, int i) { return bars + (unsigned)(kind * 2 + (i & 1)) * 8; };
    auto phase = [](int i) { return (unsigned)(i >> 1) & 1u; };
    auto at_a = [](int i) { return M::a + i % M::two_a * M::one; };
    auto at_b = [](int i) { return M::b + i % M::two_b * M::one; };
    auto at_c = [](int i) { return M::c + i % M::two_c * M::one_c; };
    auto at_r = [](int i) { return M::through_c ? M::c + i % M::two_c * M::one_c : M::rows + i % (M::two_r > 1 ? 2 : 1) * kBlk; };

    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int seg = blockIdx.x % s.segments, bh = blockIdx.x / s.segments, head = bh % s.h, bat = bh / s.h;
    const int n = s.lengths ? min(max(s.lengths[bat], 0), s.t) : s.t;
    const long long first = (long long)seg * s.seg;
    const int lo = (int)(first < n ? first : n), hi = (int)(first + s.seg < n ? first + s.seg : n);
    const int chunks = (hi - lo + kTok - 1) / kTok;
    const int da = s.da, dc = s.dc;
    const long long size = (long long)da * dc;
    // first token of chunk i; positions lo + 128 i ... of the sweep
    auto token0 = [&](int i) { return s.reversed ? n - (lo + i * kTok) - kTok : lo + i * kTok; };

    if (tid == 0) {
        *dead = 0;
        for (int i = 0; i < 2; ++i) {
            for (int k = FULL_A; k <= DONE_O; ++k) bar_init(bar(k, i), 1);
            for (int k = HAS_C; k <= CLEARED; ++k) bar_init(bar(k, i), kWorkers);
            bar_init(bar(SENT, i), 1);
        }
        for (int k = 0; k < 4; ++k) bar_init(read_p(k), kWorkers / 4);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kWorkers + 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_at(&tmem_word)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        tc_before();
    }
    __syncthreads();
    tc_after();
    const unsigned tmem = tmem_word, tP = tmem, tX = tmem + 128, tO = tmem + 256, tT = tmem + 256 + DC;

    if (warp == kWorkers) {
        // ---- rows arrive
        if (lane == 0) {
            int i = 0;
            auto send = [&](int j) {                             // the output rows of chunk j
                if (!bar_wait(bar(HAS_R, j), phase(j), dead)) return false;
                if (token0(j) >= 0) {                            // (a store must not start before the tensor: those rows go without it)
                    for (int x = 0; x < DC / 64; ++x)
                        if (x * 64 < dc) tma_store(&map_o, base + at_r(j) + x * kBlk, x * 64, head, token0(j), bat);
                    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
                    asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
                }
                bar_arrive(bar(SENT, j));
                return true;
            };
            for (; i < chunks; ++i) {
                const int t0 = token0(i);
                auto take = [&](int full, int done, int room, const CUtensorMap* map, const Rows& r, int to, int bytes) {
                    if (i >= room && !bar_wait(bar(done, i - room), phase(i - room), dead)) return false;
                    if (i >= room && full == FULL_C && !bar_wait(bar(HAS_C, i - room), phase(i - room), dead)) return false;
                    bar_expect(bar(full, i), bytes);
                    for (int x = 0; x < bytes / kBlk; ++x) tma_load(base + to + x * kBlk, map, x * 64, r.sh ? head : 0, t0, r.sb ? bat : 0, bar(full, i));
                    return true;
                };
                // room comes free: b after T, a after X, c after O and its parts (and the output rows that pass through it)
                if (!take(FULL_B, DONE_T, M::two_b, &map_b, s.b, at_b(i), M::one)) break;
                if (M::through_c && M::two_c == 1 && i > 0)      // its room comes free late: at least from L2 then
                    for (int x = 0; x < DC / 64; ++x) tma_ahead(&map_c, x * 64, s.c.sh ? head : 0, t0, s.c.sb ? bat : 0);
                if (!M::through_c && i >= M::two_r && !send(i - M::two_r)) break;
                if (!take(FULL_A, DONE_X, M::two_a, &map_a, s.a, at_a(i), M::one)) break;
                if (M::through_c && i >= M::two_r && !send(i - M::two_r)) break;
                if (!take(FULL_C, DONE_O, M::two_c, &map_c, s.c, at_c(i), M::one_c)) break;
            }
            for (int j = max(0, chunks - M::two_r); j < chunks && !*dead; ++j)
                if (!send(j)) break;
            asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
            if (*dead) {                                         // what was asked for has to land before the block leaves
                for (int j = max(0, i - 2); j <= min(i, chunks - 1); ++j)
                    for (int k = FULL_A; k <= FULL_C; ++k)
                        for (int spin = 0; spin < 4096 && !bar_try(bar(k, j), phase(j)); ++spin) {}
            }
        }
        __syncwarp();
    } else if (warp == kWorkers + 1) {
        // ---- products.  The warp runs as one, so that what the products are given is uniform; one lane issues them
        const bool one = elected();
        const unsigned W = rows_word(base + M::w), Wlow = rows_word(base + M::parts), Q = columns_word(base + M::parts);
        for (int i = 0; i < chunks; ++i) {
            const unsigned ph = phase(i);
            const bool cut = hi - lo - i * kTok < kTok && !s.reversed;       // rows behind the end are cleared first
            const unsigned A = rows_word(base + at_a(i)), B = rows_word(base + at_b(i)), Bt = columns_word(base + at_b(i)), C = columns_word(base + at_c(i));
            if (!bar_wait(bar(FULL_A, i), ph, dead) || !bar_wait(bar(FULL_B, i), ph, dead)) break;
            if (cut && !bar_wait(bar(CLEARED, i), 0, dead)) break;          // once in a sweep
            if (i > 0 && !bar_wait(bar(DONE_O, i - 1), phase(i - 1), dead)) break;       // O has read the P before
            tc_after();
            if (one) {
#pragma unroll
                for (int k = 0; k < DA / 16; ++k) tc_mma(tP, operand(A, (k / 4) * kBlk + (k % 4) * 32), operand(B, (k / 4) * kBlk + (k % 4) * 32), product(128, 0, 0), k > 0);
                tc_commit(bar(DONE_P, i));
            }
            __syncwarp();
            if (!bar_wait(bar(HAS_W, i), ph, dead)) break;
            if (i > 0 && !bar_wait(bar(HAS_O, i - 1), phase(i - 1), dead)) break;
            tc_after();
            if (one) {
#pragma unroll
                for (int k = 0; k < DA / 16; ++k) tc_mma(tX, operand(A, (k / 4) * kBlk + (k % 4) * 32), operand(W, (k / 4) * kBlk + (k % 4) * 32), product(128, 0, 0), k > 0);
#pragma unroll
                for (int k = 0; k < DA / 16; ++k) tc_mma(tX, operand(A, (k / 4) * kBlk + (k % 4) * 32), operand(Wlow, (k / 4) * kBlk + (k % 4) * 32), product(DC, 0, 0), true);
                tc_commit(bar(DONE_X, i));
            }
            __syncwarp();
            if (!bar_wait(bar(HAS_P, i), ph, dead) || !bar_wait(bar(FULL_C, i), ph, dead)) break;
            tc_after();
            if (one) {
#pragma unroll
                for (int k = 0; k < 16; ++k) tc_mma_t(tO, tP + (k ^ 8) * 8, operand(C, (k & 7) * 2048), product(DC, 0, 1), k > 0);      // small parts first
                tc_commit(bar(DONE_O, i));
            }
            __syncwarp();
            if (!bar_wait(bar(HAS_C, i), ph, dead)) break;
            tc_after();
            if (one) {
                // small parts first
                constexpr int kSets = kStack ? PARTS - 1 : PARTS;
#pragma unroll
                for (int p = kSets - 1; p >= 0; --p)
#pragma unroll
                    for (int k = 0; k < 8; ++k) tc_mma(tT, operand(Q, p * M::one_c + k * 2048), operand(Bt, k * 2048), product(DA, 1, 1), p < kSets - 1 || k > 0);
                tc_commit(bar(DONE_T, i));
            }
            __syncwarp();
        }
        if (*dead) {                                             // products under way end before the tensor memory goes
            if (one) tc_commit(bar(DONE_P, 0));
            for (int spin = 0; spin < 4096; ++spin)
                if (bar_try(bar(DONE_P, 0), 0) && bar_try(bar(DONE_P, 0), 1)) break;
        }
        __syncwarp();
    } else {
        // ---- between the products: warp w holds lanes 32 (w mod 4) .. of tensor memory and a quarter of the columns
        constexpr int HC = DA / 4;                               // columns of T that a thread holds
        constexpr int kAll = kWorkers * 32;
        const int q = warp & 3, cq = warp >> 2, row = q * 32 + lane;
        const unsigned lanes = (unsigned)(q * 32) << 16;
        const float ld = clamp_log(s.log_decay[head]), both = s.in_scale * s.out_scale;
        const float keep_full = power(ld, kTok);
        const int pos = s.reversed ? kTok - 1 - row : row;
        const float far = s.out_scale * power(ld, pos + s.off);
        // P: a tile of 32 x 32 that lies off the diagonal weighs u (this thread's) times a row of 32; one on it l^(lane - x)
        const int behind = s.reversed ? 32 * cq - row : row - 32 * cq - 31;
        const float u = behind > 0 ? both * power(ld, behind) : both;
        if (tid < 96) {
            if (tid < 32) whole[tid] = power(ld, s.reversed ? tid : 31 - tid);
            else edge[tid - 32] = tid < 64 ? 0.0f : power(ld, tid - 64);      // edge[32 + d] = l^d, 0 for d < 0
        }
        // weights of the token rows of this thread's pieces: rows tid / 8 and 64 more
        const int prow = tid >> 3;
        float wt[2];
        auto weigh = [&](int m) {
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const int r = prow + 64 * k, j = s.reversed ? kTok - 1 - r : r;
                wt[k] = j < m ? power(ld, m - s.off - j) * s.in_scale : 0.0f;
            }
        };
        weigh(kTok);
        // W^T: a row for a column of c (kStack: rows 0..63 first addend, 64..127 second)
        const int wrow = kStack ? row & 63 : row, wcol = cq * HC;
        float2 w[HC / 2];
        {
            const float* w0 = s.start ? s.start + ((long long)bh * s.segments + seg) * size : nullptr;
            const bool has = w0 && wrow < dc && (!kStack || row < 64);
            // (a transposed state by vectors, as its rows lie apart: 8 x 7680 x 8 x 128, 4 floats at a time 12 us less than 1 at a time)
            if (s.transposed && ((unsigned long long)w0 & 15) == 0) {
#pragma unroll
                for (int x = 0; x < HC; x += 4) {
                    const float4 f = has && wcol + x < da ? *reinterpret_cast<const float4*>(w0 + (long long)wrow * da + wcol + x) : make_float4(0, 0, 0, 0);
                    w[x / 2] = make_float2(f.x, f.y);
                    w[x / 2 + 1] = make_float2(f.z, f.w);
                }
            } else {
#pragma unroll
                for (int x = 0; x < HC; ++x) {
                    const int i = wcol + x;
                    const float v = has && i < da ? (s.transposed ? w0[(long long)wrow * da + i] : w0[(long long)i * dc + wrow]) : 0.0f;
                    if (x & 1) w[x / 2].y = v;
                    else w[x / 2].x = v;
                }
            }
        }
        auto four = [](const float2* v) {                        // eight numbers as a 16-byte piece
            return make_uint4(pack2<__nv_bfloat16>(v[0].x, v[0].y), pack2<__nv_bfloat16>(v[1].x, v[1].y), pack2<__nv_bfloat16>(v[2].x, v[2].y), pack2<__nv_bfloat16>(v[3].x, v[3].y));
        };
        auto rest = [&](const float2* v, uint4 top) {            // what those leave of them
            const unsigned t[4] = {top.x, top.y, top.z, top.w};
            float2 r[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float2 f = unpack2(t[e], __nv_bfloat16());
                r[e] = __fadd2_rn(v[e], make_float2(-f.x, -f.y));
            }
            return four(r);
        };
        auto tell = [&](int kind, int i) {
            tc_before();
            __syncwarp();
            if (lane == 0) bar_arrive(bar(kind, i));
        };
        auto put_w = [&](int i) {                                // W as the operand of chunk i
            const unsigned to = base + M::w + (DA == 128 ? (cq >> 1) * kBlk : 0) + row * 128;
            const int piece = DA == 128 ? (cq & 1) * 4 : cq * 2;
#pragma unroll
            for (int x = 0; x < HC / 8; ++x) {
                const unsigned at = to + (((piece + x) ^ (row & 7)) << 4);
                const uint4 top = four(w + 4 * x);
                smem_put(at, top);
                if (!kStack || row < 64) smem_put(at + (M::parts - M::w), rest(w + 4 * x, top));
            }
            fence_async();
            tell(HAS_W, i);
        };
        constexpr int OC = DC / 4;                               // columns of X and O that a thread holds
        const long long by = (long long)s.h * dc;
        const int ocol = cq * OC;
        asm volatile("bar.sync 1, %0;" ::"n"(kAll) : "memory");  // the tables
        __nv_bfloat16* first_out = (__nv_bfloat16*)s.out + ((long long)bat * s.t * s.h + head) * dc + ocol;
        if (chunks > 0) put_w(0);

        for (int i = 0; i < chunks; ++i) {
            const unsigned ph = phase(i);
            const int left = hi - lo - i * kTok, m = left < kTok ? left : kTok;
            if (m < kTok && !s.reversed) {                       // rows behind the end become nothing, whatever they hold
                if (!bar_wait(bar(FULL_B, i), ph, dead) || !bar_wait(bar(FULL_C, i), ph, dead) || !bar_wait(bar(FULL_A, i), ph, dead)) break;
                for (int e = tid; e < (M::one > M::one_c ? M::one : M::one_c) / 16; e += kAll)
                    if ((e >> 3 & 127) >= m) {
                        const uint4 none = make_uint4(0, 0, 0, 0);
                        if (e < M::one / 16) smem_put(base + at_b(i) + e * 16, none);
                        if (e < M::one / 16) smem_put(base + at_a(i) + e * 16, none);
                        if (e < M::one_c / 16) smem_put(base + at_c(i) + e * 16, none);
                    }
                fence_async();
                tell(CLEARED, i);
            }
            // P: weights and mask; back into tensor memory, two columns in one, once the four warps of these lanes have read it
            if (!bar_wait(bar(DONE_P, i), ph, dead)) break;
            tc_after();
            unsigned r[32], to[16], low[16];
            auto parts = [&](int x, float2 y) {
                to[x] = pack2<__nv_bfloat16>(y.x, y.y);
                const float2 f = unpack2(to[x], __nv_bfloat16());
                y = __fadd2_rn(y, make_float2(-f.x, -f.y));
                low[x] = pack2<__nv_bfloat16>(y.x, y.y);
            };
            if (s.reversed ? cq < q : cq > q) {              // above the diagonal
#pragma unroll
                for (int x = 0; x < 16; ++x) to[x] = low[x] = 0;
            } else {
                tc_load(tP + lanes + cq * 32, r);
                tc_wait_load();
                if (cq == q) {
                    const float* e = edge + 32 + (s.reversed ? -lane : lane);
#pragma unroll
                    for (int x = 0; x < 16; ++x) {
                        const float2 f = s.reversed ? make_float2(e[2 * x], e[2 * x + 1]) : make_float2(e[-2 * x], e[-2 * x - 1]);
                        const float2 y = __fmul2_rn(__fmul2_rn(make_float2(__uint_as_float(r[2 * x]), __uint_as_float(r[2 * x + 1])), make_float2(both, both)), f);
                        parts(x, y);
                    }
                } else {
#pragma unroll
                    for (int x = 0; x < 16; ++x) {
                        const float2 f = *reinterpret_cast<const float2*>(whole + 2 * x);
                        const float2 y = __fmul2_rn(__fmul2_rn(make_float2(__uint_as_float(r[2 * x]), __uint_as_float(r[2 * x + 1])), make_float2(u, u)), f);
                        parts(x, y);
                    }
                }
            }
            tc_before();
            __syncwarp();
            if (lane == 0) bar_arrive(read_p(q));
            if (!bar_wait(read_p(q), (unsigned)i & 1u, dead)) break;
            tc_after();
            tc_store(tP + lanes + cq * 16, to);
            tc_store(tP + lanes + 64 + cq * 16, low);
            tc_wait_store();
            tell(HAS_P, i);
            // the weighted c in parts
            if (!bar_wait(bar(FULL_C, i), ph, dead) || !bar_wait(bar(DONE_X, i), ph, dead)) break;      // (X reads W's smaller part in their room)
            if (m < kTok) weigh(m);
#pragma unroll
            for (int x = 0; x < DC / 64; ++x)
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const int off = x * kBlk + (tid + kAll * k) * 16;
                    const uint4 v = smem_get(base + at_c(i) + off);
                    uint4 part[PARTS];
                    split<PARTS, kStack>(v, wt[k], part);
#pragma unroll
                    for (int p = 0; p < PARTS; ++p) smem_put(base + M::parts + p * M::one_c + off, part[p]);
                }
            fence_async();
            tell(HAS_C, i);
            // out = l^{pos + off} X + O
            if (!bar_wait(bar(DONE_O, i), ph, dead)) break;
            tc_after();
            const bool live = pos < m, turned = token0(i) < 0;           // a TMA store must not start before the tensor
            if (M::through_c ? !bar_wait(bar(HAS_C, i), ph, dead)        // every warp has read c
                             : i >= M::two_r && !bar_wait(bar(SENT, i - M::two_r), phase(i - M::two_r), dead)) break;
#pragma unroll
            for (int y = 0; y < OC / 16; ++y) {
                unsigned r0[16], r1[16], r2[16];
                tc_load(tX + lanes + ocol + y * 16, r0);
                if constexpr (kStack) tc_load(tX + lanes + 64 + ocol, r1);
                tc_load(tO + lanes + ocol + y * 16, r2);
                tc_wait_load();
                if (y == OC / 16 - 1) tell(HAS_O, i);
                float2 v[8];
#pragma unroll
                for (int x = 0; x < 8; ++x) {
                    float2 z = make_float2(__uint_as_float(r0[2 * x]), __uint_as_float(r0[2 * x + 1]));
                    if constexpr (kStack) z = __fadd2_rn(z, make_float2(__uint_as_float(r1[2 * x]), __uint_as_float(r1[2 * x + 1])));
                    v[x] = __ffma2_rn(make_float2(far, far), z, make_float2(__uint_as_float(r2[2 * x]), __uint_as_float(r2[2 * x + 1])));
                }
                const uint4 lo8 = four(v), hi8 = four(v + 4);
                const int piece = (ocol + y * 16) / 8;       // rows leave by TMA (those behind the end as the zeros they are)
                if (!turned) {
                    const unsigned to = base + at_r(i) + (piece >> 3) * kBlk + row * 128;
                    smem_put(to + (((piece & 7) ^ (row & 7)) << 4), live ? lo8 : make_uint4(0, 0, 0, 0));
                    smem_put(to + (((piece + 1 & 7) ^ (row & 7)) << 4), live ? hi8 : make_uint4(0, 0, 0, 0));
                } else if (live) {
                    __nv_bfloat16* to = first_out + (token0(i) + row) * by + y * 16;
                    if (ocol + y * 16 < dc) *reinterpret_cast<uint4*>(to) = lo8;
                    if (ocol + y * 16 + 8 < dc) *reinterpret_cast<uint4*>(to + 8) = hi8;
                }
            }
            fence_async();
            tell(HAS_R, i);
            // W^T <- l^m W^T + T
            if (!bar_wait(bar(DONE_T, i), ph, dead)) break;
            tc_after();
            add_chunk<HC>(w, tT + lanes + wcol, m < kTok ? power(ld, m) : keep_full);
            if (i + 1 < chunks) put_w(i + 1);                    // X has read the last one: waited for above
        }
        if (s.end) {
            float* w1 = s.end + ((long long)bh * s.segments + seg) * size;
            if constexpr (kStack) {
                asm volatile("bar.sync 1, %0;" ::"n"(kAll) : "memory");
                const unsigned meet = base + M::parts + (row & 63) * 4;        // the two addends meet in the parts' room
                if (row >= 64)
#pragma unroll
                    for (int x = 0; x < HC / 2; ++x) {
                        smem_put(meet + (wcol + 2 * x) * 256, w[x].x);
                        smem_put(meet + (wcol + 2 * x + 1) * 256, w[x].y);
                    }
                asm volatile("bar.sync 1, %0;" ::"n"(kAll) : "memory");
                if (row < 64)
#pragma unroll
                    for (int x = 0; x < HC / 2; ++x) {
                        w[x].x += smem_get1(meet + (wcol + 2 * x) * 256);
                        w[x].y += smem_get1(meet + (wcol + 2 * x + 1) * 256);
                    }
            }
            const bool lost = *dead != 0;
            if (wrow < dc && (!kStack || row < 64))
#pragma unroll
                for (int x = 0; x < HC; ++x)
                    if (wcol + x < da) w1[(long long)(wcol + x) * dc + wrow] = lost ? __uint_as_float(0x7fffffffu) : x & 1 ? w[x / 2].y : w[x / 2].x;
        }
    }
    tc_before();
    __syncthreads();
    tc_after();
    if (warp == kWorkers + 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    const bool lost = *dead != 0;
    if (lost && tid == 0) g_gave_up = 1;
    const long long zlo = lost ? lo : (first > n ? first : n), zhi = first + s.seg < s.t ? first + s.seg : s.t;
    for (long long e = zlo * dc + tid; e < zhi * dc; e += kTcThreads) {
        const long long i = e / dc, tok = i < n && s.reversed ? n - 1 - i : i;
        ((__nv_bfloat16*)s.out)[(((long long)bat * s.t + tok) * s.h + head) * dc + (e - i * dc)] = from_f32<__nv_bfloat16>(i < n ? __uint_as_float(0x7fffffffu) : 0.0f);
    }
}

// A thread's share of W^T as a sweep begins and ends: a row of it (a column of c) and HC of its columns.  kStack: rows 64..127 are
// a second addend, which starts at 0 and meets the first in `room` (256 da bytes of shared memory, free by then).
// (no sweep that makes a state begins from a transposed one)
template <int HC, bool kStack>
__device__ __forceinline__ void take_start(const Sweep& s, int row, int wcol, float2 (&w)[HC / 2]) {
    const int wrow = kStack ? row & 63 : row;
    const float* w0 = s.start ? s.start + (long long)blockIdx.x * s.da * s.dc : nullptr;      // a block has one segment
    const bool has = w0 && wrow < s.dc && (!kStack || row < 64);
#pragma unroll
    for (int x = 0; x < HC; ++x) {
        const int i = wcol + x;
        const float v = has && i < s.da ? w0[(long long)i * s.dc + wrow] : 0.0f;
        if (x & 1) w[x / 2].y = v;
        else w[x / 2].x = v;
    }
}
template <int HC, bool kStack>
__device__ __forceinline__ void give_end(const Sweep& s, int row, int wcol, float2 (&w)[HC / 2], unsigned room, const volatile int* dead) {
    if constexpr (kStack) {
        asm volatile("bar.sync 1, %0;" ::"n"(kWorkers * 32) : "memory");
        const unsigned meet = room + (row & 63) * 4;
        if (row >= 64)
#pragma unroll
            for (int x = 0; x < HC / 2; ++x) {
                smem_put(meet + (wcol + 2 * x) * 256, w[x].x);
                smem_put(meet + (wcol + 2 * x + 1) * 256, w[x].y);
            }
        asm volatile("bar.sync 1, %0;" ::"n"(kWorkers * 32) : "memory");
        if (row < 64)
#pragma unroll
            for (int x = 0; x < HC / 2; ++x) {
                w[x].x += smem_get1(meet + (wcol + 2 * x) * 256);
                w[x].y += smem_get1(meet + (wcol + 2 * x + 1) * 256);
            }
    }
    const bool lost = *dead != 0;
    float* w1 = s.end + (long long)blockIdx.x * s.da * s.dc;
    const int wrow = kStack ? row & 63 : row;
    if (wrow < s.dc && (!kStack || row < 64))
#pragma unroll
        for (int x = 0; x < HC; ++x)
            if (wcol + x < s.da) w1[(long long)(wcol + x) * s.dc + wrow] = lost ? __uint_as_float(0x7fffffffu) : x & 1 ? w[x / 2].y : w[x / 2].x;
}
// ---- the state alone ------------------------------------------------------------------------------------------------
// W^T <- l^m W^T + T without the outputs: what a cut sequence needs first.  Chunks follow one another in two to four rooms; the
// first part of the weighted c takes c's own place.  T has two places in tensor memory, so that the workers add chunk i - 1 to
// W while the products of chunk i run: nothing waits but for rows to come.  Three parts of 128 columns leave room for two
// chunks only with 64 tokens in each; elsewhere 64 would cost (three parts of 64 columns, 1 x 122880 x 8 heads: 72 us).
//     k, v 252 MB, three parts: 1 x 122880 x 8 x 64 61 us (4.1 TB/s), 8 x 7680 x 8 x 128 64 us; 82 and 75 us as a sweep of the
//     kernel above, which takes T, W and the parts one after another.  Bound by shared memory: rows in, parts out and the
//     products' operands are some 1500 of a chunk's 2200 clocks; two groups of workers in turn, which hide each other's waits,
//     took the same 61 us.
template <int DA, int DC, int PARTS>
struct StateMap {
    static constexpr int tok = DA == 128 && DC == 128 && PARTS == 3 ? 64 : kTok, blk = tok * 128;
    static constexpr int one = DA / 64 * blk, one_c = DC / 64 * blk, parts = one + one_c, room = parts + (PARTS - 1) * one_c;
    static constexpr int most = 14 * kBlk / room, rooms = most < 4 ? most : 4, bars = rooms * room;
    static constexpr int bytes = bars + 128 + 1024;                        // and the way to the boundary
    static_assert(rooms >= 2, "T of a chunk is read while the next one is summed");
};

template <int DA, int DC, int PARTS>
__global__ void __launch_bounds__(kTcThreads, 1) state_kernel(const Sweep s, const __grid_constant__ CUtensorMap map_b, const __grid_constant__ CUtensorMap map_c) {
    using M = StateMap<DA, DC, PARTS>;
    constexpr bool kStack = DC == 64;
    constexpr int R = M::rooms, kTok = M::tok, kBlk = M::blk;
    extern __shared__ unsigned char raw[];
    __shared__ int dead_word;
    __shared__ unsigned tmem_word;
    const unsigned base = (smem_at(raw) + 1023u) & ~1023u, bars = base + M::bars;
    volatile int* dead = &dead_word;
    enum { FULL, HAS_C, DONE_T, KINDS };
    const unsigned ended = bars + KINDS * R * 8;
    auto bar = [&](int kind, int i) { return bars + (unsigned)(kind * R + i % R) * 8; };         // chunk i uses number i mod R
    auto phase = [](int i) { return (unsigned)(i / R) & 1u; };
    auto at = [](int i) { return i % R * M::room; };

    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int seg = blockIdx.x % s.segments, bh = blockIdx.x / s.segments, head = bh % s.h, bat = bh / s.h;
    const int n = s.lengths ? min(max(s.lengths[bat], 0), s.t) : s.t;
    const long long first = (long long)seg * s.seg;
    const int lo = (int)(first < n ? first : n), hi = (int)(first + s.seg < n ? first + s.seg : n);
    const int chunks = (hi - lo + kTok - 1) / kTok;
    if (tid == 0) {
        *dead = 0;
        for (int i = 0; i < R; ++i) {
            bar_init(bar(FULL, i), 1);
            bar_init(bar(HAS_C, i), kWorkers);
            bar_init(bar(DONE_T, i), 1);
        }
        bar_init(ended, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kWorkers + 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_at(&tmem_word)), "n"(2 * DA) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        tc_before();
    }
    __syncthreads();
    tc_after();
    const unsigned tmem = tmem_word;

    if (warp == kWorkers) {
        if (lane == 0) {
            int i = 0;
            for (; i < chunks; ++i) {
                if (i >= R && !bar_wait(bar(DONE_T, i - R), phase(i - R), dead)) break;
                const int t0 = s.reversed ? n - (lo + i * kTok) - kTok : lo + i * kTok;
                bar_expect(bar(FULL, i), M::one + M::one_c);
                for (int x = 0; x < DC / 64; ++x) tma_load(base + at(i) + M::one + x * kBlk, &map_c, x * 64, s.c.sh ? head : 0, t0, s.c.sb ? bat : 0, bar(FULL, i));
                for (int x = 0; x < DA / 64; ++x) tma_load(base + at(i) + x * kBlk, &map_b, x * 64, s.b.sh ? head : 0, t0, s.b.sb ? bat : 0, bar(FULL, i));
            }
            if (*dead)                                           // what was asked for has to land before the block leaves
                for (int j = max(0, i - R); j < i; ++j)
                    for (int spin = 0; spin < 4096 && !bar_try(bar(FULL, j), phase(j)); ++spin) {}
        }
        __syncwarp();
    } else if (warp == kWorkers + 1) {
        const bool one = elected();
        for (int i = 0; i < chunks; ++i) {
            // (the workers have read T of chunk i - 2 before they say that c of chunk i is there)
            if (!bar_wait(bar(FULL, i), phase(i), dead) || !bar_wait(bar(HAS_C, i), phase(i), dead)) break;
            tc_after();
            const unsigned B = columns_word(base + at(i), kBlk), C = columns_word(base + at(i) + M::one, kBlk);
            if (one) {
                constexpr int kSets = kStack ? PARTS - 1 : PARTS;
#pragma unroll
                for (int p = kSets - 1; p >= 0; --p)             // small parts first
#pragma unroll
                    for (int k = 0; k < kTok / 16; ++k)
                        tc_mma(tmem + (i & 1) * DA, operand(C, p * M::one_c + k * 2048), operand(B, k * 2048), product(DA, 1, 1), p < kSets - 1 || k > 0);
                tc_commit(bar(DONE_T, i));
            }
            __syncwarp();
        }
        if (*dead) {                                             // products under way end before the tensor memory goes
            if (one) tc_commit(ended);
            for (int spin = 0; spin < 4096 && !bar_try(ended, 0); ++spin) {}
        }
        __syncwarp();
    } else {
        constexpr int HC = DA / 4, kAll = kWorkers * 32;
        const int q = warp & 3, cq = warp >> 2, row = q * 32 + lane, wcol = cq * HC;
        const unsigned from = tmem + ((unsigned)(q * 32) << 16) + wcol;
        const float ld = clamp_log(s.log_decay[head]), keep_full = power(ld, kTok);
        const int prow = tid >> 3;                               // token rows of this thread's pieces: tid / 8 and, of 128, 64 more
        float wt[kTok / 64];
        bool live[kTok / 64];
        auto weigh = [&](int m) {
#pragma unroll
            for (int k = 0; k < kTok / 64; ++k) {
                const int r = prow + 64 * k, j = s.reversed ? kTok - 1 - r : r;
                live[k] = j < m;
                wt[k] = live[k] ? power(ld, m - s.off - j) * s.in_scale : 0.0f;
            }
        };
        weigh(kTok);
        float2 w[HC / 2];
        take_start<HC, kStack>(s, row, wcol, w);
        int i = 0;
        for (; i < chunks; ++i) {
            const int left = hi - lo - i * kTok, m = left < kTok ? left : kTok;
            if (!bar_wait(bar(FULL, i), phase(i), dead)) break;
            if (m < kTok) {                                      // rows behind the end become nothing, whatever they hold
                weigh(m);
                for (int e = tid; e < M::one / 16; e += kAll)
                    if (s.reversed ? (e >> 3 & kTok - 1) < kTok - m : (e >> 3 & kTok - 1) >= m) smem_put(base + at(i) + e * 16, make_uint4(0, 0, 0, 0));
            }
#pragma unroll
            for (int x = 0; x < DC / 64; ++x)
#pragma unroll
                for (int k = 0; k < kTok / 64; ++k) {
                    const int off = x * kBlk + (tid + kAll * k) * 16;
                    const uint4 v = smem_get(base + at(i) + M::one + off);
                    uint4 part[PARTS];
                    split<PARTS, kStack>(live[k] ? v : make_uint4(0, 0, 0, 0), wt[k], part);
                    smem_put(base + at(i) + M::one + off, part[0]);
#pragma unroll
                    for (int p = 1; p < PARTS; ++p) smem_put(base + at(i) + M::parts + (p - 1) * M::one_c + off, part[p]);
                }
            fence_async();
            tc_before();
            __syncwarp();
            if (lane == 0) bar_arrive(bar(HAS_C, i));
            if (i > 0) {
                if (!bar_wait(bar(DONE_T, i - 1), phase(i - 1), dead)) break;
                tc_after();
                add_chunk<HC>(w, from + (i - 1 & 1) * DA, keep_full);
            }
        }
        if (i == chunks && chunks > 0 && bar_wait(bar(DONE_T, chunks - 1), phase(chunks - 1), dead)) {
            const int m = hi - lo - (chunks - 1) * kTok;
            tc_after();
            add_chunk<HC>(w, from + (chunks - 1 & 1) * DA, m < kTok ? power(ld, m) : keep_full);
        }
        give_end<HC, kStack>(s, row, wcol, w, base, dead);
    }
    tc_before();
    __syncthreads();
    tc_after();
    if (warp == kWorkers + 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(2 * DA) : "memory");
    if (*dead && tid == 0) g_gave_up = 1;
}

// ---- launch --------------------------------------------------------------------------------------------------------
using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*, const cuuint32_t*,
                            CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

int encoder(Encode* out) {
    static std::atomic<Encode> known{nullptr};
    Encode fn = known.load();
    if (!fn) {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult found;
        CNL_TRY(check_cuda(cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &found), "cudaGetDriverEntryPoint"));
        if (!p || found != cudaDriverEntryPointSuccess) return fail(CNL_ERR_CUDA, "the driver has no cuTensorMapEncodeTiled");
        known.store(fn = reinterpret_cast<Encode>(p));
    }
    *out = fn;
    return CNL_OK;
}

// [b][t][h][d] in boxes of 64 elements x 128 (or 64) tokens of one head; what lies outside reads as 0.  A head or batch stride of 0
// (rows shared by all heads or sequences) is a dimension of one element, whose coordinate stays 0.
int encode(CUtensorMap* map, const Rows& r, int b, int t, int h, int d, int tok = kTok) {
    Encode fn = nullptr;
    CNL_TRY(encoder(&fn));
    if (r.sh == 0) h = 1;
    if (r.sb == 0) b = 1;
    const long long some = 16;                                   // the stride of a dimension of one element is not used
    const cuuint64_t sizes[4] = {(cuuint64_t)d, (cuuint64_t)h, (cuuint64_t)t, (cuuint64_t)b};
    const cuuint64_t strides[3] = {(cuuint64_t)(h > 1 ? 2 * r.sh : some), (cuuint64_t)(t > 1 ? 2 * r.st : some), (cuuint64_t)(b > 1 ? 2 * r.sb : some)};
    const cuuint32_t box[4] = {64, 1, (cuuint32_t)tok, 1}, ones[4] = {1, 1, 1, 1};
    const CUresult e = fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(r.p), sizes, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
                          CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (e != CUDA_SUCCESS) return fail(CNL_ERR_CUDA, "cuTensorMapEncodeTiled: error %d", (int)e);
    return CNL_OK;
}

template <int DA, int DC, int PARTS>
int launch_tc(const Sweep& s, cudaStream_t st) {
    CUtensorMap a, b, c, o;
    CNL_TRY(encode(&a, s.a, s.batch, s.t, s.h, s.da));
    CNL_TRY(encode(&o, Rows{s.out, (long long)s.t * s.h * s.dc, (long long)s.h * s.dc, s.dc}, s.batch, s.t, s.h, s.dc));
    CNL_TRY(encode(&b, s.b, s.batch, s.t, s.h, s.da));
    CNL_TRY(encode(&c, s.c, s.batch, s.t, s.h, s.dc));
    constexpr int bytes = Map<DA, DC, PARTS>::bytes;
    static_assert(bytes <= 232448, "more shared memory than a block may have");
    CNL_TRY(ensure_dynamic_smem(tc_kernel<DA, DC, PARTS>, bytes));
    tc_kernel<DA, DC, PARTS><<<(unsigned)((long long)s.batch * s.h * s.segments), kTcThreads, bytes, st>>>(s, a, b, c, o);
    return after_launch("linear attention sweep");
}

template <int DA, int DC, int PARTS>
int launch_state(const Sweep& s, cudaStream_t st) {
    CUtensorMap b, c;
    CNL_TRY(encode(&b, s.b, s.batch, s.t, s.h, s.da, StateMap<DA, DC, PARTS>::tok));
    CNL_TRY(encode(&c, s.c, s.batch, s.t, s.h, s.dc, StateMap<DA, DC, PARTS>::tok));
    constexpr int bytes = StateMap<DA, DC, PARTS>::bytes;
    static_assert(bytes <= 232448, "more shared memory than a block may have");
    CNL_TRY(ensure_dynamic_smem(state_kernel<DA, DC, PARTS>, bytes));
    state_kernel<DA, DC, PARTS><<<(unsigned)((long long)s.batch * s.h * s.segments), kTcThreads, bytes, st>>>(s, b, c);
    return after_launch("linear attention states");
}

template <int DA, int DC>
int run_tc(Sweep s, cudaStream_t st) {
    const bool exact = s.end && s.exact;
    if constexpr (DC == 64) {
        if (s.out) return exact ? launch_tc<DA, DC, 3>(s, st) : launch_tc<DA, DC, 2>(s, st);
    }
    if (s.out && exact) {                                        // no room for three parts beside the outputs: the state on its own
        Sweep only = s;
        only.out = nullptr;
        CNL_TRY((launch_state<DA, DC, 3>(only, st)));
        s.end = nullptr;
    }
    if (s.out) return launch_tc<DA, DC, 2>(s, st);
    return exact ? launch_state<DA, DC, 3>(s, st) : launch_state<DA, DC, 2>(s, st);
}

// Measured against the mma.sync sweep (forward / backward, us): 64 x 128 tokens x 8 heads of 128 69 / 159 against 76 / 259, of 64
// 34 / 89 against 29 / 77; 1 x 128 of 64 12 / 29 against 14 / 36; 16 x 1024 of 64 33 / 85 against 67 / 144; 8 x 7680 of 128
// 204 / 458 against 544 / 1304.  Heads of 32 would fill half of its tiles; shorter sequences less than one chunk.
bool tc_sizes(int t, int da, int dc, int dtype) { return dtype == CNL_BF16 && t >= kTok && da > 32 && dc > 32 && da % 8 == 0 && dc % 8 == 0; }

bool tc_serves(const Sweep& s, int dtype) {
    auto fits = [&](const Rows& r) {
        auto ok = [](long long n, long long stride) { return n <= 1 || (stride >= 0 && stride % 8 == 0 && stride < (1LL << 38)); };
        return !r.p || (aligned16(r.p) && ok(s.h, r.sh) && ok(s.t, r.st) && r.st > 0 && ok(s.batch, r.sb));
    };
    return tc_sizes(s.t, s.da, s.dc, dtype) && fits(s.a) && fits(s.b) && fits(s.c) && aligned16(s.out);
}

int run_sweep_tc(const Sweep& s, cudaStream_t st) {
    if (s.da <= 64) return s.dc <= 64 ? run_tc<64, 64>(s, st) : run_tc<64, 128>(s, st);
    return s.dc <= 64 ? run_tc<128, 64>(s, st) : run_tc<128, 128>(s, st);
}

}  // namespace lin
}  // namespace cnl

extern "C" int cnl_linattn_status(void) {
    // the copy alone would wait for the default stream and not for those that are independent of it
    int v = 0;
    if (cudaDeviceSynchronize() != cudaSuccess || cudaMemcpyFromSymbol(&v, cnl::lin::g_gave_up, sizeof(int)) != cudaSuccess) { cudaGetLastError(); return -1; }
    return v;
}
