// Softmax cross entropy of a linear layer's logits, and its gradient, without the logits in memory (HipGPT multiplies by its output
// projection, stores [N][V] logits and their gradient, and multiplies twice more: src/gpt_model.cpp, softmax_loss_kernel
// src/hip_kernels.cpp:606-657).
//
//   z[n][v] = x[n] . w[v]        lse[n] = log sum_v exp z[n][v]        loss[n] = lse[n] - z[n][t_n]
//   dz[n][v] = g_n (exp(z[n][v] - lse[n]) - [v = t_n])        dx = dz W        dW = dz^T x
//
// Three forms of one product kernel (loss_gemm_kernel), which differ in what they do with an accumulator tile:
//   kLse   (forward)   a row's maximum and sum of exponentials over 128 columns, kept for loss_join_kernel; the target's logit
//   kDz    (backward)  forms the logits of a piece of the vocabulary again and stores their gradient as 16-bit numbers: the piece's
//                      gradient stays within L2 (kPieceBytes) until the next form has read it twice
//   kOut   (backward)  dx (summed over the pieces in fp32) and the piece's rows of dW, in one launch
// The backward pass costs 6 N E V operations instead of 4, and no [N][V] array exists in either.
//
// Rows whose target lies outside the vocabulary are left out at the start: loss_pack_x_kernel moves the others together, so they cost
// nothing and what they hold (NaN from padding) meets no product.
//
// Products: tcgen05.mma.cta_group::2, 256 x 256 tiles of two blocks, 64 deep stages by TMA in a ring, two accumulators in TMEM: the products of a
// tile run while eight warps take the tile before it out.  Any operand may be contiguous along the reduction or across it (a descriptor
// bit), so neither x, W nor dz is ever transposed.  bf16: operands as they are, dz rounded to bf16.  fp32: each operand as two fp16 numbers
// hi + lo of the value times a power of two (one per matrix; 2^-22 of the value), three products a pair: lo hi + hi lo + hi hi.  The tensor
// core's fp32 sums are cut off, not rounded, so fp32 sums leave TMEM every kPromote stages and go on in registers.
#include "elem_types.cuh"
#include "stream_workspace.hpp"
#include "tma_host.cuh"

#include <cuda_fp16.h>
#include <math.h>

#include <algorithm>

namespace hipgpt {
namespace {

constexpr int kHalfM = 128, kTileM = 2 * kHalfM, kTileN = 256, kDeep = 64;
constexpr int kOperand = kHalfM * kDeep * 2;            // bytes of one block's share of an operand of a stage: 128 rows or columns
constexpr int kEpiWarps = 8, kThreads = 32 * (kEpiWarps + 2);
constexpr int kTmemColumns = 512;
constexpr int kPromote = 2;
constexpr size_t kPieceBytes = 64u << 20;
template <int NP> constexpr int kStageBytes = 2 * NP * kOperand;
template <int NP> constexpr int kRing = NP == 1 ? 6 : 3;
constexpr size_t kGemmSmem = 6 * 2 * kOperand + 1024;

enum Form { kLse, kDz, kOut };

__device__ int g_loss_status = 0;

// Sizes of one product D = A B (A: M x K, B: K x N), its place in the operands and what becomes of the result.
struct Problem {
    int m_tiles, n_tiles, stages;            // of 256, 256 and 64
    int a_across, b_across;                  // operand contiguous across the reduction (along M or N) instead of along it
    int a_k0, a_m0, b_k0, b_n0;              // where the product begins in the operands
    int m_by_count, k_by_count;              // M, or K, is the number of rows that take part
    // kOut
    void *out;                               // element (row, column) at row * ld + column
    long long ld;
    int rows, cols;
    int by_map;                              // row i of the product is row row_map[i] of the output
    int accumulate, first, last;             // pieces of the sum over the vocabulary: `sum` (fp32) holds what the earlier ones gave
    float *sum;
    int scale_of;                            // kOut: 0 of x's gradient, 1 of W's
};

struct LossArgs {
    CUtensorMap a[2], b[2];
    Problem p[2];
    int problems;
    const int *count;                        // rows that take part
    const int *row_map, *targets;            // of the rows that take part
    const float *lse, *g;
    const unsigned *amax;                    // fp32: bits of the largest |x|, |w|, |g|
    float2 *part;                            // kLse: [half tile of the vocabulary][row] maximum and sum
    float *z_target;
    uint16_t *dz;                            // kDz: [piece of the operand][rows][ld]
    size_t dz_ld, dz_plane;
    size_t rows_alloc;
    int v0, V;                               // kLse, kDz: first column of the call, and of all
    int expire;
};

// fp32 operands: x = (hi + lo) / scale.  The gradient of the logits is |dz| <= 2 |g|: 2^14 / (power of two above the largest |g|) leaves room
__device__ __forceinline__ float operand_scale(const unsigned *amax, int which) { return pow2_scale(__uint_as_float(amax[which])); }
__device__ __forceinline__ float grad_scale(const unsigned *amax) { return operand_scale(amax, 2) * 0.5f; }

__device__ __forceinline__ void split_half(float x, __half &hi, __half &lo)
{
    hi = __float2half_rn(x);
    lo = __float2half_rn(x - __half2float(hi));
}

// ---- rows that take part, moved together ------------------------------------------------------------------------------

__global__ void __launch_bounds__(256)
loss_amax_kernel(const float *__restrict__ x, const float *__restrict__ w, const float *__restrict__ g, const int *__restrict__ targets, int N, int E, int V, unsigned *amax)
{
    dependency_wait();
    dependents_may_start();
    const int which = blockIdx.y;
    float m = 0.0f;
    auto take = [&](float v) { v = fabsf(v); m = v <= 3.0e38f ? fmaxf(m, v) : m; };      // (not of infinities and NaN: they stay what they are)
    const long long step = (long long)gridDim.x * 256, at = (long long)blockIdx.x * 256 + threadIdx.x;
    if (which == 1) {
        const long long total = (long long)V * E;
        if ((reinterpret_cast<uintptr_t>(w) & 15) == 0) {
            for (long long i = at; i < total / 4; i += step) {
                const float4 v = __ldg(reinterpret_cast<const float4 *>(w) + i);
                take(v.x); take(v.y); take(v.z); take(v.w);
            }
            for (long long i = total / 4 * 4 + at; i < total; i += step) take(w[i]);
        } else {
            for (long long i = at; i < total; i += step) take(w[i]);
        }
    } else {
        const int lane = threadIdx.x & 31;
        for (long long n = at >> 5; n < N; n += step >> 5) {
            const int t = targets[n];
            if (t < 0 || t >= V) continue;
            if (which == 2) {
                if (lane == 0) take(g[n]);
            } else {
                for (int e = lane; e < E; e += 32) take(x[(size_t)n * E + e]);
            }
        }
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if ((threadIdx.x & 31) == 0 && m > 0.0f) atomicMax(&amax[which], __float_as_uint(m));
}

// One row of `cols` values -> a row of `ld` 16-bit ones (zeros behind the last) in each plane, by one warp
template <typename T>
__device__ __forceinline__ void pack_row(const T *src, uint16_t *dst, size_t plane, int cols, int ld, float scale, int lane, bool vec)
{
    if constexpr (sizeof(T) == 2) {
        if (vec) {
            for (int c = lane * 8; c < ld; c += 256) *reinterpret_cast<uint4 *>(dst + c) = *reinterpret_cast<const uint4 *>(src + c);
        } else {
            for (int c = lane; c < ld; c += 32) dst[c] = c < cols ? reinterpret_cast<const uint16_t *>(src)[c] : (uint16_t)0;
        }
    } else {
        for (int c = lane * 4; c < ld; c += 128) {
            float v[4];
            if (vec) {
                load_values<float, 4>(src + c, v);
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) v[j] = c + j < cols ? src[c + j] : 0.0f;
            }
            union { __half h[4]; uint2 u; } hi, lo;
#pragma unroll
            for (int j = 0; j < 4; ++j) split_half(v[j] * scale, hi.h[j], lo.h[j]);
            *reinterpret_cast<uint2 *>(dst + c) = hi.u;
            *reinterpret_cast<uint2 *>(dst + plane + c) = lo.u;
        }
    }
}

struct PackX {
    const int *targets;
    const float *lse, *g;                    // backward
    int N, E, V, ld, per_block;
    uint16_t *xp;
    size_t plane;
    int *count, *row_map, *c_targets;
    float *c_lse, *c_g;
    const unsigned *amax;
    float *zero_loss, *zero_lse;             // forward: what rows that take no part get
    uint8_t *zero_grad;                      // backward: their rows of the gradient
};

template <typename T>
__global__ void __launch_bounds__(256)
loss_pack_x_kernel(const T *__restrict__ x, PackX p, int vec)
{
    dependency_wait();
    dependents_may_start();
    __shared__ int warp_sum[8];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int from = blockIdx.x * p.per_block, to = min(p.N, from + p.per_block);
    auto inside = [&](int t) { return t >= 0 && t < p.V; };
    int before = 0;
    for (int i = tid; i < from; i += 256) before += inside(__ldg(p.targets + i));
#pragma unroll
    for (int o = 16; o; o >>= 1) before += __shfl_xor_sync(0xffffffffu, before, o);
    if (lane == 0) warp_sum[warp] = before;
    __syncthreads();
    int base = 0;
#pragma unroll
    for (int w = 0; w < 8; ++w) base += warp_sum[w];
    const float scale = sizeof(T) == 4 ? operand_scale(p.amax, 0) : 1.0f, gscale = sizeof(T) == 4 && p.g ? grad_scale(p.amax) : 1.0f;
    for (int r0 = from; r0 < to; r0 += 32) {
        const int t = r0 + lane < to ? __ldg(p.targets + r0 + lane) : -1;
        const unsigned mask = __ballot_sync(0xffffffffu, inside(t));
        for (int j = warp; j < 32 && r0 + j < to; j += 8) {
            const int n = r0 + j;
            if (mask >> j & 1) {
                const int i = base + __popc(mask & ((1u << j) - 1));
                if (lane == j) {
                    p.row_map[i] = n;
                    p.c_targets[i] = t;
                    if (p.g) { p.c_g[i] = p.g[n] * gscale; p.c_lse[i] = p.lse[n]; }
                }
                pack_row<T>(x + (size_t)n * p.E, p.xp + (size_t)i * p.ld, p.plane, p.E, p.ld, scale, lane, vec != 0);
            } else {
                if (p.zero_loss && lane == 0) p.zero_loss[n] = p.zero_lse[n] = 0.0f;
                if (p.zero_grad) {
                    T *row = reinterpret_cast<T *>(p.zero_grad) + (size_t)n * p.E;
                    for (int e = lane; e < p.E; e += 32) row[e] = from_float<T>(0.0f);
                }
            }
        }
        base += __popc(mask);
    }
    if (to == p.N && from < p.N) {           // the last block that has rows: their number, and zeros up to a whole stage of the products that sum over them
        if (tid == 0) *p.count = base;
        const int end = (base + kDeep - 1) / kDeep * kDeep;
        for (int i = base + warp; i < end; i += 8)
            for (int c = lane * 4; c < p.ld; c += 128)
                for (int pl = 0; pl < (sizeof(T) == 4 ? 2 : 1); ++pl) *reinterpret_cast<uint2 *>(p.xp + pl * p.plane + (size_t)i * p.ld + c) = make_uint2(0u, 0u);
    }
}

// W [rows][cols] -> 16-bit rows of ld
template <typename T>
__global__ void __launch_bounds__(256)
loss_pack_w_kernel(const T *__restrict__ w, uint16_t *wp, size_t plane, int rows, int cols, int ld, const unsigned *amax, int vec)
{
    dependency_wait();
    dependents_may_start();
    const float scale = sizeof(T) == 4 ? operand_scale(amax, 1) : 1.0f;
    for (int r = blockIdx.x * 8 + (threadIdx.x >> 5); r < rows; r += gridDim.x * 8)
        pack_row<T>(w + (size_t)r * cols, wp + (size_t)r * ld, plane, cols, ld, scale, threadIdx.x & 31, vec != 0);
}

// ---- the products -----------------------------------------------------------------------------------------------------

__device__ __forceinline__ void tma_load_pair(void *dst, const CUtensorMap *map, int c0, int c1, int c2, uint32_t bar)
{
    // completes on a barrier of the pair's first block, whichever block asks
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3, %4}], [%5];"
                 ::"r"(smem_u32(dst)), "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(bar) : "memory");
}
__device__ __forceinline__ void mma_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate)
{
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
// arrives at the barrier of both blocks once the products before it have completed
__device__ __forceinline__ void commit_pair(uint64_t *bar)
{
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(smem_u32(bar)), "h"((uint16_t)3) : "memory");
}

__device__ __noinline__ bool loss_wait_slow(uint64_t *bar, uint32_t parity, int site, volatile int *abort_flag, uint32_t peer_flag, int expire)
{
    if (!expires_now(expire, site) && mbar_wait(bar, parity)) return true;
    *abort_flag = 1;
    asm volatile("st.volatile.shared::cluster.u32 [%0], %1;" ::"r"(peer_flag), "r"(1) : "memory");      // the other block's rows of the tile are not stored either
    atomicCAS(&g_loss_status, 0, site);
    linger();
    return false;
}

template <typename T>
__device__ __forceinline__ void put_columns(T *dst, const float (&v)[32], int cols, bool accumulate, bool vec)
{
    if (vec && cols >= 32) {
        constexpr int W = kPer16<T>;
#pragma unroll
        for (int j = 0; j < 32; j += W) {
            float x[W];
#pragma unroll
            for (int k = 0; k < W; ++k) x[k] = v[j + k];
            if (accumulate) {
                float old[W];
                load_values<T, W>(dst + j, old);
#pragma unroll
                for (int k = 0; k < W; ++k) x[k] += old[k];
            }
            store_values<T, W>(dst + j, x);
        }
    } else {
#pragma unroll
        for (int j = 0; j < 32; ++j)
            if (j < cols) dst[j] = from_float<T>(accumulate ? to_float(dst[j]) + v[j] : v[j]);
    }
}

// T: the storage type of kOut's results; NP: planes of an operand (1: bf16, 2: fp16 hi and lo).  site codes in the status word: 1 stage landed, 2 stage free,
// 3 accumulator complete, 4 accumulator drained
template <Form FORM, typename T>
__global__ void __launch_bounds__(kThreads, 1)
loss_gemm_kernel(const __grid_constant__ LossArgs args)
{
    constexpr int NP = sizeof(T) == 4 ? 2 : 1;
    constexpr int RING = kRing<NP>, STAGE = kStageBytes<NP>;
    extern __shared__ __align__(1024) uint8_t loss_smem[];
    uint8_t *ring = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(loss_smem) + 1023) & ~(uintptr_t)1023);      // [stage][A's planes | B's planes]
    __shared__ uint64_t full[RING], empty[RING], acc_full[2], acc_empty[2];
    __shared__ uint32_t tmem_slot;
    __shared__ volatile int abort_flag;
    const int lane = threadIdx.x & 31;
    const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0);
    int rank;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));

    if (threadIdx.x == 0) {
        abort_flag = 0;
        for (int i = 0; i < RING; ++i) { mbar_init(&full[i], 1); mbar_init(&empty[i], 1); }
        for (int i = 0; i < 2; ++i) { mbar_init(&acc_full[i], 1); mbar_init(&acc_empty[i], 2 * kEpiWarps); }
    }
    if (warp == kEpiWarps) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(kTmemColumns) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    dependents_may_start();
    tc_fence_before();
    __syncthreads();
    cluster_sync();
    tc_fence_after();
    const uint32_t tmem = tmem_slot, peer_flag = peer_addr(smem_u32(const_cast<const int *>(&abort_flag)), rank ^ 1);
    dependency_wait();

    bool seen = true;                         // what this thread waited for last has come
    auto wait = [&](uint64_t *bar, uint32_t parity, int site) {
        const int gone = abort_flag;
        const bool done = mbar_test(bar, parity);
        seen = !gone;
        if (!gone && !done) seen = loss_wait_slow(bar, parity, site, &abort_flag, peer_flag, args.expire);
    };

    // the tiles of a call: those of the first problem, then those of the second; m runs fastest, so pairs that run side by side share B's columns
    const int count = *args.count;
    struct Tile { int which, m, n, stages; };
    const int pairs = (int)gridDim.x / 2, first_tile = (int)blockIdx.x / 2;
    int m_tiles[2] = {0, 0}, tiles[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < 2; ++i)
        if (i < args.problems) {
            m_tiles[i] = args.p[i].m_by_count ? (count + kTileM - 1) / kTileM : args.p[i].m_tiles;
            tiles[i] = m_tiles[i] * args.p[i].n_tiles;
        }
    const int all_tiles = tiles[0] + tiles[1];
    auto tile_of = [&](int t) {
        const int which = t >= tiles[0], u = which ? t - tiles[0] : t, mt = which ? m_tiles[1] : m_tiles[0];
        const Problem &p = args.p[which];
        return Tile{which, u % mt, u / mt, p.k_by_count ? (count + kDeep - 1) / kDeep : p.stages};
    };

    if (warp == kEpiWarps) {
        // ---- producer: this block's halves of both operands ----
        uint32_t full_of_first[RING];
#pragma unroll
        for (int s = 0; s < RING; ++s) full_of_first[s] = peer_addr(smem_u32(&full[s]), 0);
        int s = 0, round = 0;
        for (int t = first_tile; t < all_tiles; t += pairs) {
            const Tile w = tile_of(t);
            const Problem &p = args.p[w.which];
            const CUtensorMap *ma = &args.a[w.which], *mb = &args.b[w.which];
            const int m0 = p.a_m0 + w.m * kTileM + rank * kHalfM, n0 = p.b_n0 + w.n * kTileN + rank * kHalfM;
            for (int k = 0; k < w.stages; ++k) {
                if (round) wait(&empty[s], (uint32_t)((round - 1) & 1), 2);
                if (lane == 0 && seen) {
                    if (rank == 0) mbar_arrive_expect_tx(&full[s], 2 * STAGE);
                    uint32_t bar = full_of_first[0];
#pragma unroll
                    for (int i = 1; i < RING; ++i) bar = i == s ? full_of_first[i] : bar;
                    uint8_t *at = ring + s * STAGE;
#pragma unroll
                    for (int pl = 0; pl < NP; ++pl) {
                        uint8_t *a = at + pl * kOperand, *b = at + (NP + pl) * kOperand;
                        const int ka = p.a_k0 + k * kDeep, kb = p.b_k0 + k * kDeep;
                        if (p.a_across) {
                            tma_load_pair(a, ma, m0, ka, pl, bar);
                            tma_load_pair(a + kOperand / 2, ma, m0 + 64, ka, pl, bar);
                        } else {
                            tma_load_pair(a, ma, ka, m0, pl, bar);
                        }
                        if (p.b_across) {
                            tma_load_pair(b, mb, n0, kb, pl, bar);
                            tma_load_pair(b + kOperand / 2, mb, n0 + 64, kb, pl, bar);
                        } else {
                            tma_load_pair(b, mb, kb, n0, pl, bar);
                        }
                    }
                }
                __syncwarp();
                if (++s == RING) { s = 0; ++round; }
            }
        }
        if (abort_flag) linger();
    } else if (warp == kEpiWarps + 1) {
        // ---- products, issued by the pair's first block for both ----
        if (rank == 0) {
            int s = 0, round = 0, unit = 0;
            for (int t = first_tile; t < all_tiles; t += pairs) {
                const Tile w = tile_of(t);
                const Problem &p = args.p[w.which];
                // operand along the reduction: rows of 128 bytes in groups of 8 (1024 bytes), 16 deep = 32 bytes; across it: blocks of 64 x 64 deep (8192 bytes),
                // 8 deep = 1024 bytes.  Swizzled by 128 bytes either way.
                const uint32_t idesc = (1u << 4) | (NP == 1 ? (1u << 7) | (1u << 10) : 0u) | ((uint32_t)p.a_across << 15) | ((uint32_t)p.b_across << 16) | ((uint32_t)(kTileN >> 3) << 17) |
                                       ((uint32_t)(kTileM >> 4) << 24);
                const uint32_t a_lbo = p.a_across ? kOperand / 2 : 16, b_lbo = p.b_across ? kOperand / 2 : 16;
                const uint64_t a_step = p.a_across ? 128 : 2, b_step = p.b_across ? 128 : 2;
                const int unit_stages = NP == 1 ? w.stages : kPromote;
                for (int k0 = 0; k0 < w.stages; k0 += unit_stages, ++unit) {
                    const uint32_t acc = tmem + (uint32_t)((unit & 1) * kTileN);
                    if (unit >= 2) wait(&acc_empty[unit & 1], (uint32_t)((unit / 2 - 1) & 1), 4);
                    tc_fence_after();
                    const int k1 = min(w.stages, k0 + unit_stages);
                    for (int k = k0; k < k1; ++k) {
                        wait(&full[s], (uint32_t)(round & 1), 1);
                        tc_fence_after();
                        const uint32_t at = smem_u32(ring + s * STAGE);
                        const uint64_t a = make_desc(at, a_lbo, 1024, 2), b = make_desc(at + NP * kOperand, b_lbo, 1024, 2);
                        constexpr uint64_t lo = kOperand >> 4;
#pragma unroll
                        for (int j = 0; j < kDeep / 16; ++j) {
                            if constexpr (NP == 2) {
                                if (elect_one()) mma_pair(acc, a + lo + j * a_step, b + j * b_step, idesc, (k > k0 || j) ? 1u : 0u);
                                if (elect_one()) mma_pair(acc, a + j * a_step, b + lo + j * b_step, idesc, 1u);
                                if (elect_one()) mma_pair(acc, a + j * a_step, b + j * b_step, idesc, 1u);
                            } else {
                                if (elect_one()) mma_pair(acc, a + j * a_step, b + j * b_step, idesc, (k > k0 || j) ? 1u : 0u);
                            }
                        }
                        if (elect_one()) commit_pair(&empty[s]);
                        if (++s == RING) { s = 0; ++round; }
                    }
                    if (elect_one()) commit_pair(&acc_full[unit & 1]);
                }
            }
            __syncwarp();
            if (abort_flag) linger();
        }
    } else {
        // ---- what becomes of an accumulator: thread = row = TMEM lane; two warps share a row's columns ----
        const int quarter = warp & 3, half = warp >> 2;
        const uint32_t lane_base = tmem + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(half * 128);
        const uint32_t drained[2] = {peer_addr(smem_u32(&acc_empty[0]), 0), peer_addr(smem_u32(&acc_empty[1]), 0)};
        const float x_inv = NP == 2 ? pow2_inverse(operand_scale(args.amax, 0)) : 1.0f, w_inv = NP == 2 ? pow2_inverse(operand_scale(args.amax, 1)) : 1.0f;
        const float z_scale = x_inv * w_inv;
        int unit = 0;
        for (int t = first_tile; t < all_tiles; t += pairs) {
            const Tile w = tile_of(t);
            const Problem &p = args.p[w.which];
            const int row = w.m * kTileM + rank * kHalfM + quarter * 32 + lane;
            const int col0 = w.n * kTileN + half * 128;
            auto release = [&](int buf) {
                tc_fence_before();
                __syncwarp();
                if (lane == 0) asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(buf ? drained[1] : drained[0]) : "memory");
            };

            // per row
            const bool here = row < count;
            int target = -1;
            float lse = 0.0f, g = 0.0f;
            if constexpr (FORM != kOut) {
                if (here) target = __ldg(args.targets + row) - args.v0;
                if constexpr (FORM == kDz) if (here) { lse = __ldg(args.lse + row); g = __ldg(args.g + row); }
            }
            float run_max = -INFINITY, run_sum = 0.0f;
            size_t out_row = 0;
            float out_scale = 1.0f;
            bool out_here = false, out_vec = false;
            if constexpr (FORM == kOut) {
                out_here = row < (p.m_by_count ? count : p.rows);
                if (out_here) out_row = (size_t)(p.by_map ? __ldg(args.row_map + row) : row) * p.ld;
                if constexpr (NP == 2) out_scale = pow2_inverse(grad_scale(args.amax)) * (p.scale_of ? x_inv : w_inv);
                out_vec = p.ld % kPer16<T> == 0 && (reinterpret_cast<uintptr_t>(p.out) & 15) == 0;
            }

            // 32 columns from col0 + 32 c on
            auto columns = [&](int c, float (&v)[32]) {
                const int col = col0 + 32 * c;
                if constexpr (FORM == kLse) {
                    const int left = args.V - args.v0 - col;
                    if (left <= 0) return;
                    if (left < 32) {
#pragma unroll
                        for (int j = 0; j < 32; ++j) if (j >= left) v[j] = -INFINITY;
                    }
                    if (target >= col && target < col + 32 && !abort_flag) {
#pragma unroll
                        for (int j = 0; j < 32; ++j) if (target - col == j) args.z_target[row] = v[j] * z_scale;
                    }
                    float m = run_max;
#pragma unroll
                    for (int j = 0; j < 32; j += 2) m = max3(m, v[j] * z_scale, v[j + 1] * z_scale);
                    const float ref = m == -INFINITY ? 0.0f : m;
                    float s0 = run_sum * ex2_approx((run_max - ref) * kLog2e), s1 = 0.0f;
#pragma unroll
                    for (int j = 0; j < 32; j += 2) {
                        const float2 d = fmul2(ffma2(make_float2(v[j], v[j + 1]), make_float2(z_scale, z_scale), make_float2(-ref, -ref)), make_float2(kLog2e, kLog2e));
                        s0 += ex2_approx(d.x);
                        s1 += ex2_approx(d.y);
                    }
                    run_max = m;
                    run_sum = s0 + s1;
                } else if constexpr (FORM == kDz) {
                    const int left = args.V - args.v0 - col;
#pragma unroll
                    for (int j = 0; j < 32; j += 2) {
                        const float2 d = fmul2(ffma2(make_float2(v[j], v[j + 1]), make_float2(z_scale, z_scale), make_float2(-lse, -lse)), make_float2(kLog2e, kLog2e));
                        v[j] = ex2_approx(d.x);
                        v[j + 1] = ex2_approx(d.y);
                    }
                    if (target >= col && target < col + 32) {
#pragma unroll
                        for (int j = 0; j < 32; ++j) v[j] = target - col == j ? v[j] - 1.0f : v[j];
                    }
#pragma unroll
                    for (int j = 0; j < 32; ++j) v[j] = here && j < left ? v[j] * g : 0.0f;
                    if (abort_flag) return;
                    float *dst = reinterpret_cast<float *>(args.dz + (size_t)row * args.dz_ld + col);
                    float o[16];
                    if constexpr (NP == 1) {
#pragma unroll
                        for (int j = 0; j < 16; ++j) o[j] = __uint_as_float(pack_bf16(v[2 * j], v[2 * j + 1]));
                    } else {
#pragma unroll
                        for (int j = 0; j < 16; ++j) {
                            const __half2 h = __floats2half2_rn(v[2 * j], v[2 * j + 1]);
                            o[j] = __uint_as_float(*reinterpret_cast<const uint32_t *>(&h));
                            v[2 * j] -= __low2float(h);
                            v[2 * j + 1] -= __high2float(h);
                        }
                    }
                    store_sector(dst, o[0], o[1], o[2], o[3], o[4], o[5], o[6], o[7]);
                    store_sector(dst + 8, o[8], o[9], o[10], o[11], o[12], o[13], o[14], o[15]);
                    if constexpr (NP == 2) {
                        dst += args.dz_plane / 2;
#pragma unroll
                        for (int j = 0; j < 16; ++j) {
                            const __half2 h = __floats2half2_rn(v[2 * j], v[2 * j + 1]);
                            o[j] = __uint_as_float(*reinterpret_cast<const uint32_t *>(&h));
                        }
                        store_sector(dst, o[0], o[1], o[2], o[3], o[4], o[5], o[6], o[7]);
                        store_sector(dst + 8, o[8], o[9], o[10], o[11], o[12], o[13], o[14], o[15]);
                    }
                } else {
                    const int left = p.cols - col;
                    if (!out_here || left <= 0 || abort_flag) return;
                    if (p.sum && !(p.first && p.last)) {
                        float *sum = p.sum + (size_t)row * p.cols + col;
                        const bool vec = p.cols % 4 == 0;
                        if (!p.first) {              // (past L1: another SM may have written it, in the launch before)
#pragma unroll
                            for (int j = 0; j < 32; ++j) if (j < left) v[j] += __ldcg(sum + j);
                        }
                        if (!p.last) {
                            put_columns<float>(sum, v, left, false, vec);
                            return;
                        }
                    }
                    if constexpr (NP == 2) {
#pragma unroll
                        for (int j = 0; j < 32; ++j) v[j] *= out_scale;
                    }
                    put_columns<T>(static_cast<T *>(p.out) + out_row + col, v, left, p.accumulate != 0, out_vec);
                }
            };

            if constexpr (NP == 2) {
                float acc[4][32];
#pragma unroll
                for (int c = 0; c < 4; ++c)
#pragma unroll
                    for (int j = 0; j < 32; ++j) acc[c][j] = 0.0f;
                for (int k0 = 0; k0 < w.stages; k0 += kPromote, ++unit) {
                    wait(&acc_full[unit & 1], (uint32_t)((unit / 2) & 1), 3);
                    tc_fence_after();
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
#pragma unroll
                        for (int h = 0; h < 32; h += 16) {
                            float v[16];
                            tmem_ld16(lane_base + (uint32_t)((unit & 1) * kTileN + 32 * c + h), v);
                            tmem_wait_ld();
#pragma unroll
                            for (int j = 0; j < 16; ++j) acc[c][h + j] += v[j];
                        }
                    }
                    release(unit & 1);
                }
#pragma unroll
                for (int c = 0; c < 4; ++c) columns(c, acc[c]);
            } else {
                if (w.stages) {
                    wait(&acc_full[unit & 1], (uint32_t)((unit / 2) & 1), 3);
                    tc_fence_after();
                }
#pragma unroll 1
                for (int c = 0; c < 4; ++c) {
                    float v[32];
                    if (w.stages) {
                        tmem_ld32(lane_base + (uint32_t)((unit & 1) * kTileN + 32 * c), v);
                        tmem_wait_ld();
                        if (c == 3) release(unit & 1);
                    } else {
#pragma unroll
                        for (int j = 0; j < 32; ++j) v[j] = 0.0f;
                    }
                    columns(c, v);
                }
                if (w.stages) ++unit;
            }
            if constexpr (FORM == kLse)
                if (here && !abort_flag) args.part[(size_t)(2 * w.n + half) * args.rows_alloc + row] = make_float2(run_max, run_sum);
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    cluster_sync();                           // no block of the pair is still to be signalled, and no accumulator to be read
    if (warp == kEpiWarps) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemColumns) : "memory");
}

// Forward: a block joins the parts of 32 rows, each of its warps every eighth part in order, then the eight in order
__global__ void __launch_bounds__(256)
loss_join_kernel(const float2 *__restrict__ part, int parts, size_t rows_alloc, const float *__restrict__ z_target, const int *__restrict__ row_map, const int *__restrict__ count,
                 float *loss, float *lse)
{
    dependency_wait();
    dependents_may_start();
    __shared__ float2 sh[8][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, n = *count;
    for (int r0 = blockIdx.x * 32; r0 < n; r0 += gridDim.x * 32) {
        const int row = r0 + lane;
        float m = -INFINITY, s = 0.0f;
        auto join = [&](float2 x) {
            const float mn = fmaxf(m, x.x), ref = mn == -INFINITY ? 0.0f : mn;
            s = s * ex2_approx((m - ref) * kLog2e) + x.y * ex2_approx((x.x - ref) * kLog2e);
            m = mn;
        };
        if (row < n) {
#pragma unroll 8
            for (int i = warp; i < parts; i += 8) join(__ldg(part + (size_t)i * rows_alloc + row));
        }
        sh[warp][lane] = make_float2(m, s);
        __syncthreads();
        if (warp == 0 && row < n) {
            m = -INFINITY;
            s = 0.0f;
#pragma unroll
            for (int w = 0; w < 8; ++w) join(sh[w][lane]);
            const float l = m + logf(s);
            const int at = row_map[row];
            lse[at] = l;
            loss[at] = l - z_target[row];
        }
        __syncthreads();
    }
}

// ---- host -------------------------------------------------------------------------------------------------------------

StreamWorkspace g_loss_ws;

size_t padded(size_t bytes) { return (bytes + 1023) & ~(size_t)1023; }
long long round_up(long long a, long long b) { return (a + b - 1) / b * b; }

// {inner, outer, plane} of 16-bit values; box: 64 inner values (128 bytes, swizzled) of `box_outer` outer ones
int operand_map(CUtensorMap *m, const void *base, bool half, long long inner, long long outer, long long ld, size_t plane, int planes, int box_outer)
{
    EncodeTiledFn enc = tma_encode_fn();
    if (!enc) return fail(HIPGPT_ERR_CUDA, "cuTensorMapEncodeTiled is not available from this driver");
    const cuuint64_t dims[3] = {(cuuint64_t)inner, (cuuint64_t)outer, (cuuint64_t)planes};
    const cuuint64_t strides[2] = {(cuuint64_t)ld * 2, (cuuint64_t)plane * 2};
    const cuuint32_t box[3] = {64, (cuuint32_t)box_outer, 1}, estr[3] = {1, 1, 1};
    const CUresult r = enc(m, half ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void *>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                           CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(HIPGPT_ERR_CUDA, "cuTensorMapEncodeTiled failed with code %d", (int)r);
    return HIPGPT_OK;
}

template <Form FORM, typename T>
int launch_loss_gemm(LossArgs &a, long long most_tiles, int dev, cudaStream_t st)
{
    static std::atomic<unsigned long long> done{0};
    cudaError_t e = once_per_device(done, dev, [] { return cudaFuncSetAttribute(loss_gemm_kernel<FORM, T>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kGemmSmem); });
    int sms = 0;
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    if (e != cudaSuccess) return fail(HIPGPT_ERR_CUDA, "loss_gemm_kernel: %s", cudaGetErrorString(e));
    if (most_tiles > 1LL << 30) return fail(HIPGPT_ERR_UNSUPPORTED, "%lld tiles are beyond one call", most_tiles);
    const long long pairs = std::min<long long>(most_tiles, sms / 2);
    e = launch_overlapped_clusters(loss_gemm_kernel<FORM, T>, 2, dim3((unsigned)(2 * pairs)), dim3(kThreads), kGemmSmem, st, a);
    return e == cudaSuccess ? check_launch("loss_gemm_kernel") : fail(HIPGPT_ERR_CUDA, "loss_gemm_kernel: %s", cudaGetErrorString(e));
}

// What both directions share: the rows that take part, the weights as the tensor core takes them, and the workspace.
struct Plan {
    int N, E, V, layout, dev;
    long long x_ld, w_rows, w_cols, w_ld, rows_alloc;
    bool pack_w;
    size_t x_plane, w_plane;
    // places in the workspace
    size_t x_at, w_at, ints_at, floats_at, amax_at, end;
};

template <typename T>
int plan_call(Plan &p, const void *w, int N, int E, int V, int layout)
{
    constexpr int NP = sizeof(T) == 4 ? 2 : 1;
    p.N = N; p.E = E; p.V = V; p.layout = layout;
    const cudaError_t e = cudaGetDevice(&p.dev);
    if (e != cudaSuccess) return fail(HIPGPT_ERR_CUDA, "cudaGetDevice: %s", cudaGetErrorString(e));
    p.x_ld = round_up(E, 8);
    p.rows_alloc = round_up(N, kTileM);
    p.w_rows = layout == HIPGPT_WEIGHTS_VE ? V : E;
    p.w_cols = layout == HIPGPT_WEIGHTS_VE ? E : V;
    // 16-bit weights are read where they lie if TMA can (rows of whole 16-byte words); others are copied once per call
    p.pack_w = NP == 2 || p.w_cols % 8 != 0 || (reinterpret_cast<uintptr_t>(w) & 15) != 0;
    p.w_ld = round_up(p.w_cols, 8);
    p.x_plane = (size_t)p.rows_alloc * p.x_ld;
    p.w_plane = (size_t)p.w_rows * p.w_ld;
    size_t at = 0;
    auto take = [&](size_t bytes) { const size_t r = at; at += padded(bytes); return r; };
    p.x_at = take(NP * p.x_plane * 2);
    p.w_at = take(p.pack_w ? NP * p.w_plane * 2 : 0);
    p.ints_at = take((1 + 2 * (size_t)p.rows_alloc) * sizeof(int));
    p.floats_at = take(2 * (size_t)p.rows_alloc * sizeof(float));
    p.amax_at = take(16);
    p.end = at;
    return HIPGPT_OK;
}

// Fills what the plan has in the workspace, and of `a` what every form reads
template <typename T>
int pack_call(const Plan &p, uint8_t *ws, LossArgs &a, const T *x, const T *w, const int *targets, const float *lse, const float *g, float *zero_loss, float *zero_lse, void *zero_grad,
              cudaStream_t st, const void **w_base)
{
    unsigned *amax = reinterpret_cast<unsigned *>(ws + p.amax_at);
    int *ints = reinterpret_cast<int *>(ws + p.ints_at);
    float *floats = reinterpret_cast<float *>(ws + p.floats_at);
    cudaError_t e;
    if constexpr (sizeof(T) == 4) {
        e = cudaMemsetAsync(amax, 0, 16, st);
        if (e != cudaSuccess) return fail(HIPGPT_ERR_CUDA, "cudaMemsetAsync: %s", cudaGetErrorString(e));
        const long long blocks = std::min<long long>(592, std::max<long long>(((long long)p.V * p.E + 4095) / 4096, ((long long)p.N + 7) / 8));
        e = launch_overlapped(loss_amax_kernel, dim3((unsigned)blocks, g ? 3 : 2), dim3(256), 0, st, (const float *)x, (const float *)w, g, targets, p.N, p.E, p.V, amax);
        if (e != cudaSuccess) return fail(HIPGPT_ERR_CUDA, "loss_amax_kernel: %s", cudaGetErrorString(e));
    }
    if (p.pack_w) {
        const bool vec = p.w_cols % kPer16<T> == 0 && p.w_cols == p.w_ld && (reinterpret_cast<uintptr_t>(w) & 15) == 0;
        const long long blocks = std::min<long long>((p.w_rows + 7) / 8, 148 * 16);
        e = launch_overlapped(loss_pack_w_kernel<T>, dim3((unsigned)blocks), dim3(256), 0, st, w, reinterpret_cast<uint16_t *>(ws + p.w_at), p.w_plane, (int)p.w_rows, (int)p.w_cols, (int)p.w_ld,
                              (const unsigned *)amax, (int)vec);
        if (e != cudaSuccess) return fail(HIPGPT_ERR_CUDA, "loss_pack_w_kernel: %s", cudaGetErrorString(e));
    }
    *w_base = p.pack_w ? static_cast<const void *>(ws + p.w_at) : w;
    PackX px = {};
    px.targets = targets; px.lse = lse; px.g = g;
    px.N = p.N; px.E = p.E; px.V = p.V; px.ld = (int)p.x_ld;
    px.per_block = (int)std::max<long long>(32, round_up((p.N + 295) / 296, 32));
    px.xp = reinterpret_cast<uint16_t *>(ws + p.x_at);
    px.plane = p.x_plane;
    px.count = ints; px.row_map = ints + 1; px.c_targets = ints + 1 + p.rows_alloc;
    px.c_lse = floats; px.c_g = floats + p.rows_alloc;
    px.amax = amax;
    px.zero_loss = zero_loss; px.zero_lse = zero_lse; px.zero_grad = static_cast<uint8_t *>(zero_grad);
    const bool xvec = p.E % kPer16<T> == 0 && p.E == p.x_ld && (reinterpret_cast<uintptr_t>(x) & 15) == 0;
    e = launch_overlapped(loss_pack_x_kernel<T>, dim3((unsigned)((p.N + px.per_block - 1) / px.per_block)), dim3(256), 0, st, x, px, (int)xvec);
    if (e != cudaSuccess) return fail(HIPGPT_ERR_CUDA, "loss_pack_x_kernel: %s", cudaGetErrorString(e));
    a.count = px.count; a.row_map = px.row_map; a.targets = px.c_targets;
    a.lse = px.c_lse; a.g = px.c_g; a.amax = amax;
    a.rows_alloc = (size_t)p.rows_alloc;
    a.V = p.V;
    return HIPGPT_OK;
}

// Maps of the operands of one problem: `across`: contiguous across the reduction, boxes of 64 x 64; along it: boxes of 64 x 128 rows
template <typename T>
int x_map(CUtensorMap *m, const Plan &p, const uint8_t *ws, bool across)
{
    return operand_map(m, ws + p.x_at, sizeof(T) == 4, p.E, p.rows_alloc, p.x_ld, p.x_plane, sizeof(T) == 4 ? 2 : 1, across ? kDeep : kHalfM);
}
template <typename T>
int w_map(CUtensorMap *m, const Plan &p, const void *w, bool across)
{
    return operand_map(m, w, sizeof(T) == 4, p.w_cols, p.w_rows, p.w_ld, p.w_plane, sizeof(T) == 4 ? 2 : 1, across ? kDeep : kHalfM);
}

template <typename T>
int forward(const void *xv, const void *wv, const int *targets, float *loss, float *lse, int N, int E, int V, int layout, cudaStream_t st)
{
    const T *x = static_cast<const T *>(xv), *w = static_cast<const T *>(wv);
    Plan p;
    int rc = plan_call<T>(p, w, N, E, V, layout);
    if (rc != HIPGPT_OK) return rc;
    const int n_tiles = (int)((V + kTileN - 1) / kTileN), parts = (int)((V + 127) / 128);
    const size_t part_at = p.end, zt_at = part_at + padded((size_t)2 * n_tiles * p.rows_alloc * sizeof(float2));
    StreamWorkspace::Lease lease;
    rc = g_loss_ws.enter(st, zt_at + padded((size_t)p.rows_alloc * sizeof(float)), &lease);
    if (rc != HIPGPT_OK) return rc;
    uint8_t *ws = lease.get();
    LossArgs a = {};
    const void *wb = nullptr;
    rc = pack_call<T>(p, ws, a, x, w, targets, nullptr, nullptr, loss, lse, nullptr, st, &wb);
    const bool ev = layout == HIPGPT_WEIGHTS_EV;
    if (rc == HIPGPT_OK) rc = x_map<T>(&a.a[0], p, ws, false);
    if (rc == HIPGPT_OK) rc = w_map<T>(&a.b[0], p, wb, ev);
    if (rc != HIPGPT_OK) return rc;
    a.problems = 1;
    a.p[0].n_tiles = n_tiles;
    a.p[0].stages = (E + kDeep - 1) / kDeep;
    a.p[0].b_across = ev;
    a.p[0].m_by_count = 1;
    a.part = reinterpret_cast<float2 *>(ws + part_at);
    a.z_target = reinterpret_cast<float *>(ws + zt_at);
    a.expire = take_expiry(700);
    rc = launch_loss_gemm<kLse, T>(a, (p.rows_alloc / kTileM) * n_tiles, p.dev, st);
    if (rc != HIPGPT_OK) return rc;
    const cudaError_t e = launch_overlapped(loss_join_kernel, dim3((unsigned)std::min<long long>((N + 31) / 32, 148 * 8)), dim3(256), 0, st, (const float2 *)a.part, parts, a.rows_alloc,
                                            (const float *)a.z_target, a.row_map, a.count, loss, lse);
    return e == cudaSuccess ? check_launch("loss_join_kernel") : fail(HIPGPT_ERR_CUDA, "loss_join_kernel: %s", cudaGetErrorString(e));
}

template <typename T>
int backward(const void *xv, const void *wv, const int *targets, const float *lse, const float *grad_loss, void *grad_x, void *grad_w, int accumulate_w, int N, int E, int V, int layout,
             cudaStream_t st)
{
    constexpr int NP = sizeof(T) == 4 ? 2 : 1;
    const T *x = static_cast<const T *>(xv), *w = static_cast<const T *>(wv);
    Plan p;
    int rc = plan_call<T>(p, w, N, E, V, layout);
    if (rc != HIPGPT_OK) return rc;
    // pieces of the vocabulary of like size
    const long long most = std::max<long long>(1024, (long long)(kPieceBytes / ((size_t)p.rows_alloc * 2 * NP)) / kTileN * kTileN);
    const int pieces = (int)((V + most - 1) / most);
    const long long width = round_up((V + pieces - 1) / pieces, kTileN);
    const size_t dz_plane = (size_t)p.rows_alloc * width;
    const size_t dz_at = p.end, sum_at = dz_at + padded(NP * dz_plane * 2);
    const bool sums = grad_x && pieces > 1;
    StreamWorkspace::Lease lease;
    rc = g_loss_ws.enter(st, sum_at + (sums ? padded((size_t)p.rows_alloc * E * sizeof(float)) : 0), &lease);
    if (rc != HIPGPT_OK) return rc;
    uint8_t *ws = lease.get();
    LossArgs a = {};
    const void *wb = nullptr;
    rc = pack_call<T>(p, ws, a, x, w, targets, lse, grad_loss, nullptr, nullptr, grad_x, st, &wb);
    if (rc != HIPGPT_OK) return rc;
    const bool ev = layout == HIPGPT_WEIGHTS_EV;
    const int e_tiles = (E + kTileN - 1) / kTileN, m_tiles = (int)(p.rows_alloc / kTileM);
    const int expire = take_expiry(700);
    a.dz = reinterpret_cast<uint16_t *>(ws + dz_at);
    a.dz_ld = (size_t)width;
    a.dz_plane = dz_plane;
    LossArgs o = a;
    rc = x_map<T>(&a.a[0], p, ws, false);
    if (rc == HIPGPT_OK) rc = w_map<T>(&a.b[0], p, wb, ev);
    a.problems = 1;
    a.p[0].stages = (E + kDeep - 1) / kDeep;
    a.p[0].b_across = ev;
    a.p[0].m_by_count = 1;
    a.expire = o.expire = expire;
    // dx[n][e] = sum_v dz[n][v] w[v][e]; dW[v][e] = sum_n dz[n][v] x[n][e], or dW[e][v]
    auto dz_map = [&](CUtensorMap *m, bool across) { return operand_map(m, a.dz, NP == 2, width, p.rows_alloc, width, dz_plane, NP, across ? kDeep : kHalfM); };
    const int ix = 0, iw = grad_x ? 1 : 0;
    o.problems = (grad_x ? 1 : 0) + (grad_w ? 1 : 0);
    if (grad_x) {
        if (rc == HIPGPT_OK) rc = dz_map(&o.a[ix], false);
        if (rc == HIPGPT_OK) rc = w_map<T>(&o.b[ix], p, wb, !ev);
        Problem &q = o.p[ix];
        q.n_tiles = e_tiles;
        q.b_across = !ev;
        q.m_by_count = 1;
        q.out = grad_x;
        q.ld = q.cols = E;
        q.by_map = 1;
        q.sum = sums ? reinterpret_cast<float *>(ws + sum_at) : nullptr;
        q.scale_of = 0;
    }
    if (grad_w) {
        Problem &q = o.p[iw];
        if (rc == HIPGPT_OK) rc = ev ? x_map<T>(&o.a[iw], p, ws, true) : dz_map(&o.a[iw], true);
        if (rc == HIPGPT_OK) rc = ev ? dz_map(&o.b[iw], true) : x_map<T>(&o.b[iw], p, ws, true);
        q.a_across = q.b_across = 1;
        q.k_by_count = 1;
        q.accumulate = accumulate_w;
        q.first = q.last = 1;
        q.scale_of = 1;
        q.ld = ev ? V : E;
    }
    if (rc != HIPGPT_OK) return rc;
    for (int i = 0; i < pieces; ++i) {
        const long long v0 = i * width, here = std::min<long long>(width, V - v0);
        if (here <= 0) break;
        const int v_tiles = (int)((here + kTileN - 1) / kTileN);
        a.v0 = (int)v0;
        a.p[0].n_tiles = v_tiles;
        a.p[0].b_n0 = (int)v0;
        rc = launch_loss_gemm<kDz, T>(a, (long long)m_tiles * v_tiles, p.dev, st);
        if (rc != HIPGPT_OK) return rc;
        long long tiles = 0;
        if (grad_x) {
            Problem &q = o.p[ix];
            q.stages = (int)((here + kDeep - 1) / kDeep);
            q.b_k0 = (int)v0;
            q.first = i == 0;
            q.last = v0 + width >= V;
            tiles += (long long)m_tiles * e_tiles;
        }
        if (grad_w) {
            Problem &q = o.p[iw];
            q.m_tiles = ev ? e_tiles : v_tiles;
            q.n_tiles = ev ? v_tiles : e_tiles;
            q.rows = ev ? E : (int)here;
            q.cols = ev ? (int)here : E;
            q.out = static_cast<T *>(grad_w) + (ev ? v0 : v0 * E);
            tiles += (long long)q.m_tiles * q.n_tiles;
        }
        rc = launch_loss_gemm<kOut, T>(o, tiles, p.dev, st);
        if (rc != HIPGPT_OK) return rc;
    }
    return HIPGPT_OK;
}

int check_loss_args(int N, int E, int V, int layout, int type)
{
    if (type != HIPGPT_TYPE_F32 && type != HIPGPT_TYPE_BF16) return fail(HIPGPT_ERR_BAD_ARG, "unknown type %d", type);
    if (layout != HIPGPT_WEIGHTS_VE && layout != HIPGPT_WEIGHTS_EV) return fail(HIPGPT_ERR_BAD_ARG, "unknown layout of the weights %d", layout);
    if (N < 0 || E <= 0 || V <= 0) return fail(HIPGPT_ERR_BAD_ARG, "bad size: N=%d E=%d V=%d", N, E, V);
    if (N > 1 << 26 || E > 1 << 20 || V > 1 << 28) return fail(HIPGPT_ERR_UNSUPPORTED, "N=%d E=%d V=%d is beyond one call", N, E, V);
    return HIPGPT_OK;
}

}  // namespace

void loss_release_scratch() { g_loss_ws.release(); }

int loss_status_fetch(int *status)
{
    int v = 0;
    const cudaError_t e = cudaMemcpyFromSymbol(&v, g_loss_status, sizeof(v));
    if (e != cudaSuccess) return fail(HIPGPT_ERR_CUDA, "cudaMemcpyFromSymbol: %s", cudaGetErrorString(e));
    if (v) { const int zero = 0; cudaMemcpyToSymbol(g_loss_status, &zero, sizeof(zero)); }
    *status = v;
    return HIPGPT_OK;
}

}  // namespace hipgpt

using namespace hipgpt;

extern "C" {

int hipgpt_linear_cross_entropy(const void *d_x, const void *d_w, const int *d_targets, float *d_loss, float *d_lse, int N, int E, int V, int layout, int type, void *stream)
{
    const int rc = check_loss_args(N, E, V, layout, type);
    if (rc != HIPGPT_OK) return rc;
    if (N == 0) return HIPGPT_OK;
    if (!d_x || !d_w || !d_targets || !d_loss || !d_lse) return fail(HIPGPT_ERR_NULL, "x, w, targets, loss and lse must not be NULL");
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    return type == HIPGPT_TYPE_F32 ? forward<float>(d_x, d_w, d_targets, d_loss, d_lse, N, E, V, layout, st)
                                   : forward<__nv_bfloat16>(d_x, d_w, d_targets, d_loss, d_lse, N, E, V, layout, st);
}

int hipgpt_linear_cross_entropy_backward(const void *d_x, const void *d_w, const int *d_targets, const float *d_lse, const float *d_grad_loss, void *d_grad_x, void *d_grad_w,
                                         int accumulate_w, int N, int E, int V, int layout, int type, void *stream)
{
    const int rc = check_loss_args(N, E, V, layout, type);
    if (rc != HIPGPT_OK) return rc;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (N == 0) {
        if (!d_grad_w || accumulate_w) return HIPGPT_OK;
        const cudaError_t e = cudaMemsetAsync(d_grad_w, 0, (size_t)V * E * (type == HIPGPT_TYPE_F32 ? 4 : 2), st);
        return e == cudaSuccess ? HIPGPT_OK : fail(HIPGPT_ERR_CUDA, "cudaMemsetAsync: %s", cudaGetErrorString(e));
    }
    if (!d_grad_x && !d_grad_w) return HIPGPT_OK;
    if (!d_x || !d_w || !d_targets || !d_lse || !d_grad_loss) return fail(HIPGPT_ERR_NULL, "x, w, targets, lse and grad_loss must not be NULL");
    return type == HIPGPT_TYPE_F32
               ? backward<float>(d_x, d_w, d_targets, d_lse, d_grad_loss, d_grad_x, d_grad_w, accumulate_w, N, E, V, layout, st)
               : backward<__nv_bfloat16>(d_x, d_w, d_targets, d_lse, d_grad_loss, d_grad_x, d_grad_w, accumulate_w, N, E, V, layout, st);
}

}  // extern "C"
