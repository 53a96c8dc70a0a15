// Softmax cross entropy of a linear layer's logits, and its gradient, without stored logits (HipGPT multiplies by its output
// projection, stores [N][V] logits and their gradient, and multiplies twice more: src/gpt_model.cpp, softmax_loss_kernel
// src/hip_kernels.cpp:606-657).
//
//   z[n][v] = x[n] . w[v]        lse[n] = log sum_v exp z[n][v]        loss[n] = lse[n] - z[n][t_n]
//   dz[n][v] = g_n (exp(z[n][v] - lse[n]) - [v = t_n])        dx = dz W        dW = dz^T x
//
// Two forms of one product kernel (loss_gemm_kernel), which differ in what they do with an accumulator tile:
//   kForward    a row's maximum and sum of exponentials over 256 columns, kept for loss_join_kernel; the target's logit
//   kBackward   the vocabulary in pieces.  Of one piece the logits are formed again and their gradient stored as 16-bit numbers (kDz); the
//               same launch forms, from the gradient of the piece before, that piece's share of dx (kDx, summed over the pieces in fp32) and its rows of
//               dW (kDw).  Two pieces' gradients exist at a time (kPieceBytes each at most, or 1024 columns); where one piece takes the whole vocabulary, so much is stored of the
//               gradient of the logits as a whole.
// The backward pass costs 6 N E V operations instead of 4; the forward stores nothing of size [N][V].
//
// The two large sums of a launch have few tiles and long reductions (default model, one piece: 32 tiles of 79 stages and 20 of 128), so the tiles that
// do not come out even are not dealt out whole: their stages in a row are cut into a length for each pair of blocks (plan_launch).  A tile that falls to several pairs
// is left by each as a sum in fp32; the one that comes last adds them up, in the order of their stages.  Nothing waits for another pair, and the order of a sum depends on the
// sizes alone.
//
// Rows whose target lies outside the vocabulary are left out at the start: loss_pack_kernel moves the others together, so they cost
// nothing and what they hold (NaN from padding) meets no product.
//
// Products: tcgen05.mma.cta_group::2, 256 x 256 tiles of two blocks, 64 deep stages by TMA in a ring, two accumulators in TMEM: the products of a
// tile run while sixteen warps take the tile before it out.  Any operand may be contiguous along the reduction or across it (a descriptor
// bit), so neither x, W nor dz is ever transposed.  bf16: operands as they are, dz / (largest |g|) rounded to bf16.  fp32: each operand as two fp16 numbers
// hi + lo of the value times a power of two (2^-22 of the value; row_scales), three products a pair: lo hi + hi lo + hi hi.  The tensor
// core's fp32 sums are cut off, not rounded, so sums leave TMEM every kSumStages stages.
//
// Bound, on one B200 (profiles/loss_gemm_kernel.md).  Loss: the tensor pipe and the power it draws: 8192 x 1024 x 65536 bf16 673 us in a short run (1634 TFLOP/s), 775 where the power cap sets the clock (1.37 GHz); a stage takes
// 521 cycles, 512 of them products.  8192 x 256 x 5000 fp32 (three products) 64 us, 48 of them products at 0.73 of the pipe (9 rounds of tiles where 8.65 are needed, the last one's way out).
// Gradient, bf16, large: 2370 in the best short run, 2500 - 2850 in longer ones; its sums keep the pipe 0.88 busy with operands at 57 of the 64 bytes a cycle that an SM takes from L2, the launches that also store dz 0.72.
// Gradient, fp32, 8192 x 256 x 5000: 194, 70 + 100 in its two launches of products.  There the operands take 22 and 31 bytes a cycle: the first waits for dz's way out (one place of 2 KB a warp; 0.46 of the pipe), the second reads
// dz out of HBM twice (168 MB in one piece: 0.3 GB) and joins shares (0.69).  64 x 256 x 5000: 21 us, a chain of four launches.
#include "elem_types.cuh"
#include "stream_workspace.hpp"
#include "tma_host.cuh"

#include <cuda_fp16.h>
#include <float.h>
#include <math.h>

#include <algorithm>
#include <type_traits>

namespace hipgpt {
namespace {

constexpr int kHalfM = 128, kTileM = 2 * kHalfM, kTileN = 256, kDeep = 64;
constexpr int kOperand = kHalfM * kDeep * 2;            // bytes of one block's share of an operand of a stage: 128 rows or columns
constexpr int kEpiWarps = 16, kThreads = 32 * (kEpiWarps + 2);      // four warps share a row's columns
constexpr int kWarpChunks = kTileN / 4 / 32;              // 32-column chunks of a warp
constexpr int kTmemColumns = 512;
// Stages that TMEM sums by itself, and what the sums lose: default model's gradient 281 us and 2.2e-7 (of the largest value) with one, 229 and 4.6e-7 with two, 209 and 1.1e-6 with four
// (8192 x 256 x 5000, before the accumulators were given back earlier)
constexpr int kPromote = 2;
// bf16: a sum that stays in TMEM is cut off by up to 2^-23 of itself for each 16 terms, always towards zero (262144 terms of one sign in one sum: 1.6e-3 short, 65536: 3e-4).  The loss adds its logits up in registers
// every 16 stages (64 instructions: within 2^-17).  The backward, whose results are rounded to bf16, stores a tile's sum every 128 (512: within 2^-14, a 64th of a rounding) and adds it to the next one's: accumulators
// kept in registers there cost every tile (8192 x 256 x 5000 93 -> 106 us, by what else then leaves the registers).
constexpr int kLossStages = 16, kGradStages = 128;
// What a piece's gradient of the logits takes at most.  Longer pieces mean fewer launches and joins, and lie in HBM instead of L2 (which 64 MB would leave room for): 8192 x 1024 x 65536 bf16 in pieces of 64 MB 3190 us, 128 MB 2850, 192 MB
// 2800, 256 MB 2750; 8192 x 256 x 5000 fp32 226 us in two pieces (128 MB), 201 in one
constexpr size_t kPieceBytes = 192u << 20;
template <int NP> constexpr int kStageBytes = 2 * NP * kOperand;
// What a tile of kDz costs a pair beside its stages, in quarter stages (8 and 24 measure alike)
template <int NP> constexpr int kDzExtra = 8;
template <int NP> constexpr int kRing = NP == 1 ? 6 : 3;
constexpr int kRingBytes = 6 * 2 * kOperand;
enum Form { kForward, kBackward };
constexpr int kOutBytes = 32 * 64;                      // a warp's 32 rows of 64 bytes on their way out
template <Form FORM> constexpr size_t kGemmSmem = kRingBytes + (FORM == kBackward ? kEpiWarps * kOutBytes : 0) + 1024;
template <Form FORM, int NP> constexpr int kSumStages = NP == 2 ? kPromote : FORM == kForward ? kLossStages : kGradStages;
enum Kind { kDx, kDw, kDz };                            // problems of kBackward; kForward's one problem lies at kDz's place

__device__ int g_loss_status = 0;

// Sizes of one product D = A B (A: M x K, B: K x N), its place in the operands and what becomes of the result.
struct Problem {
    int n_tiles, stages;                     // kDz: columns of 256, depth of 64; n_tiles 0: not asked for
    int a_across, b_across;                  // operand contiguous across the reduction (along M or N) instead of along it
    int b_k0, b_n0;                          // where the product begins in B
    // kDx, kDw: element (row, column) of the result at row * ld + column
    void *out;
    long long ld;
    int rows, cols;
    int accumulate;
};

struct LossArgs {
    CUtensorMap a[3], b[3], dz_out, xq;      // xq: takes the place of x in dW where scales[3] says so (fp32)
    Problem p[3];
    const int *count;                        // rows that take part
    int *failed;                             // a wait of this call has run out: its later launches do nothing
    const int *row_map, *targets;            // of the rows that take part
    const float *lse, *g;
    const float *x_inv, *row_unit;           // fp32: what takes a row's scale out of its logits, and out of its row of dx
    const float *scales;                     // fp32: what takes W's scale out; two whose product takes the scales of dz and x out of dW; 1: dW takes xq.  bf16: [2] the largest |g|
    float2 *part;                            // kForward: [tile of the vocabulary][row] maximum and sum
    float *z_target;
    float4 *shares, *sum;                    // kBackward: tiles left by several pairs, [2 a pair], and (bf16) long ones so far, [1 a pair]; dx so far, [tile].  Of a tile: [column / 4][row]
    int *arrived;                            // [tile][block of the pair][warp]: pairs that have left their share of a tile
    const struct Cut *cut;                   // the launch's
    int first, last;                         // the launch's share of dx is that of the first, the last piece
    size_t rows_alloc;
    int v0, V;                               // first column of the piece whose logits are formed, and of all
    int x_is_a;                              // dW's first operand is x
    int expire;
};

// bf16: the gradient of the logits is rounded in units of the largest |g|.  With one g for all rows (a mean) the target's element then is p - 1, all but exact where p is small;
// rounded as it is, -g would be off by the same half step of bf16 in every row, and that element is most of the row's gradient.
//
// fp32: an operand is hi + lo, two fp16 numbers of the value times a power of two that brings the largest of its row (x) or of the matrix (W) into [2^14, 2^15); nothing is kept below 2^-39 of that one.
// The gradient of the logits, of at most a few times |g| (p may pass 1 a little where lse is the caller's), is scaled row by row to [2^13, 2^14) at |g|, so a row that weighs little keeps its bits; what takes
// that out multiplies its row of dx.  In dW, a sum over the rows, |g| max|x| of all rows lie under one scale.  A row h binades below the largest of these leaves up to 8 of them to its dz, of which its
// row of dx can spare that many (2^-30 of g is left, and the errors of 65536 columns add up to 2^-24).  Only where a row lies deeper does dW take a second copy of x, whose rows are smaller by the rest.
constexpr int kMostShift = 8;
// floor(log2 a) of a finite a > 0, at least -112
__device__ __forceinline__ int exponent_of(float a) { return max((int)(__float_as_uint(a) >> 23) - 127, -112); }
// 2^e; zero below the normal numbers
__device__ __forceinline__ float pow2(int e) { return e < -126 ? 0.0f : __uint_as_float((uint32_t)(127 + min(e, 127)) << 23); }

struct RowScales {
    float x, x_inv;                          // of a row of x in the logits, and its inverse
    float x_dw;                              // ... in dW
    float dz, dz_inv;                        // of the row's gradient of the logits
};
// m: the row's largest finite |x|; most: the largest exponent_of(|g|) + exponent_of(m) of all rows
__device__ __forceinline__ RowScales row_scales(float m, float g, int most)
{
    const float ga = fabsf(g);
    const bool weighs = ga > 0.0f && ga <= FLT_MAX;
    const int ex = m > 0.0f ? exponent_of(m) : 14, eg = weighs ? exponent_of(ga) : 0;
    const int below = weighs && m > 0.0f ? most - ex - eg : 0, shift = min(below, kMostShift);
    return {pow2(14 - ex), pow2(ex - 14), pow2(14 - ex - (below - shift)), pow2(13 - eg - shift), pow2(eg + shift - 13)};
}

__device__ __forceinline__ void split_half(float x, __half &hi, __half &lo)
{
    hi = __float2half_rn(x);
    lo = __float2half_rn(x - __half2float(hi));
}

// ---- what the backward's launches do -----------------------------------------------------------------------------------

// How the tiles of kDx and kDw fall to the pairs.  In a row (kDx's first; the tiles that share rows or columns of dz next to one another, so that pairs that run
// side by side read the same stages of it), as many whole rounds as leave every pair something over are dealt out tile by tile; the stages of the rest are cut into a length for
// each pair such that all pairs have the same to do, the whole tiles of kDz counted in.  Places are in quarter stages: a narrow
// tile's stages count three (they fetch three quarters, and that is what bounds them).
constexpr int kPackThreads = 256;            // of a block of the kernels before the products
struct Place { int tile, k; };               // tile: kDx's, then kDw's
constexpr int kMostPairs = 128;
// A tile counts so many stages more: what becomes of its accumulator is not hidden by the products of a short one (24 stages of 24 + 8: 12 us)
constexpr int kTileExtra = 8;
struct Cut {
    int m_tiles[2], n_tiles[2], stages[2], tiles[2], narrow[2], n_fast[2];
    int dealt;                               // tiles that are dealt out whole
    Place begin[kMostPairs + 1];             // each pair's length of the rest
};

// Tile u of problem i: its row and column of tiles, and what a stage of it counts
struct TileOf { int m, n, unit; };
__device__ __forceinline__ TileOf tile_of(const Cut &c, int i, int u)
{
    const int nt = c.n_tiles[i], mt = c.m_tiles[i];
    const int m = c.n_fast[i] ? u / nt : u % mt, n = c.n_fast[i] ? u % nt : u / mt;
    return {m, n, c.narrow[i] && n == nt - 1 ? 3 : 4};
}
// Quarter stages of kDx, of both
struct Lengths { long long first, all; };
__device__ __forceinline__ Lengths lengths_of(const Cut &c)
{
    long long total[2];
    for (int i = 0; i < 2; ++i) total[i] = (long long)c.m_tiles[i] * (c.stages[i] + kTileExtra) * max(0, 4 * c.n_tiles[i] - c.narrow[i]);
    return {total[0], total[0] + total[1]};
}
// Quarter stages before tile t
__device__ __forceinline__ long long place_before(const Cut &c, const Lengths &len, int t)
{
    const int i = t >= c.tiles[0], u = t - (i ? c.tiles[0] : 0);
    if (u >= c.tiles[i]) return len.all;
    const TileOf x = tile_of(c, i, u);
    const long long stages = c.stages[i] + kTileExtra;
    const long long here = c.n_fast[i] ? stages * ((long long)x.m * (4 * c.n_tiles[i] - c.narrow[i]) + 4 * x.n) : stages * (4LL * x.n * c.m_tiles[i] + (long long)x.m * x.unit);
    return (i ? len.first : 0) + here;
}
__device__ __forceinline__ Place place_of(const Cut &c, const Lengths &len, long long at)
{
    if (at >= len.all) return {c.tiles[0] + c.tiles[1], 0};
    const int i = at >= len.first;
    if (i) at -= len.first;
    const long long stages = c.stages[i] + kTileExtra;
    int u, unit;
    if (c.n_fast[i]) {
        const long long row = stages * (4 * c.n_tiles[i] - c.narrow[i]);
        const long long m = at / row;
        at -= m * row;
        const int n = (int)min(at / (4 * stages), (long long)c.n_tiles[i] - 1);
        at -= n * 4 * stages;
        unit = c.narrow[i] && n == c.n_tiles[i] - 1 ? 3 : 4;
        u = (int)m * c.n_tiles[i] + n;
    } else {
        const long long column = 4 * stages * c.m_tiles[i];
        const int n = (int)min(at / column, (long long)c.n_tiles[i] - 1);
        at -= n * column;
        unit = c.narrow[i] && n == c.n_tiles[i] - 1 ? 3 : 4;
        const int m = (int)(at / (unit * stages));
        at -= m * unit * stages;
        u = n * c.m_tiles[i] + m;
    }
    const int k = (int)(at / unit), tile = (i ? c.tiles[0] : 0) + u;
    return k < c.stages[i] ? Place{tile, k} : Place{tile + 1, 0};             // (a tile's last stages are what it costs otherwise)
}
__device__ __forceinline__ bool before(const Place &a, const Place &b) { return a.tile < b.tile || (a.tile == b.tile && a.k < b.k); }

// What a call's launches are cut from
struct PlanArgs {
    int pieces, width, V, E, pairs, dz_stages, dz_extra;
    int ev, with_x, with_w;
    const int *targets;
    const float *g;                          // bf16: where the largest finite |g| goes, of rows that take part; 1 if there is none
    int N;
    float *most;
};

// By a block of kPackThreads for each launch of the backward, among the first kernel's.  Tiles of kDz are dealt out one by one from pair 0 on.
__device__ __forceinline__ void plan_launch(const PlanArgs &a, int launch, Cut *cuts)
{
    __shared__ Cut c;
    __shared__ Lengths len;
    __shared__ long long scan[kPackThreads / 32];
    __shared__ int warp_count[kPackThreads / 32];
    __shared__ float warp_most[kPackThreads / 32];
    const int q = threadIdx.x, lane = q & 31, warp = q >> 5, pairs = a.pairs;
    int count = 0;
    float most = 0.0f;
    const bool find_most = a.most && launch == 0;
#pragma unroll 8
    for (int n = q; n < a.N; n += kPackThreads) {
        const int t = __ldg(a.targets + n);
        const bool inside = t >= 0 && t < a.V;
        count += inside;
        if (find_most && inside) {
            const float g = fabsf(__ldg(a.g + n));
            if (g <= 3.0e38f) most = fmaxf(most, g);
        }
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        count += __shfl_xor_sync(0xffffffffu, count, o);
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
    }
    if (lane == 0) { warp_count[warp] = count; warp_most[warp] = most; }
    __syncthreads();
    count = 0;
#pragma unroll
    for (int w = 0; w < kPackThreads / 32; ++w) { count += warp_count[w]; most = fmaxf(most, warp_most[w]); }
    if (find_most && q == 0) *a.most = most > 0.0f ? most : 1.0f;
    const int count_tiles = max(1, (count + kTileM - 1) / kTileM), count_stages = max(1, (count + kDeep - 1) / kDeep), e_tiles = (a.E + kTileN - 1) / kTileN;
    auto columns = [&](int piece) { return piece < 0 || piece >= a.pieces ? 0 : (int)min((long long)a.width, a.V - (long long)piece * a.width); };
    auto narrow = [](int n) { return n && (n - 1) % kTileN < kTileN / 2 ? 1 : 0; };
    const int old = columns(launch - 1), v_tiles = (old + kTileN - 1) / kTileN;
    if (q == 0) {
        c.m_tiles[0] = count_tiles;
        c.n_tiles[0] = a.with_x && old ? e_tiles : 0;
        c.stages[0] = (old + kDeep - 1) / kDeep;
        c.narrow[0] = narrow(a.E);
        c.n_fast[0] = 1;
        c.m_tiles[1] = a.ev ? e_tiles : v_tiles;
        c.n_tiles[1] = a.with_w && old ? (a.ev ? v_tiles : e_tiles) : 0;
        c.stages[1] = count_stages;
        c.narrow[1] = narrow(a.ev ? old : a.E);
        c.n_fast[1] = !a.ev;
        for (int i = 0; i < 2; ++i) c.tiles[i] = c.m_tiles[i] * c.n_tiles[i];
        len = lengths_of(c);
    }
    __syncthreads();
    const int tiles = c.tiles[0] + c.tiles[1], dz_tiles = count_tiles * ((columns(launch) + kTileN - 1) / kTileN);
    const long long dz_cost = 4 * a.dz_stages + a.dz_extra, both = len.all + dz_cost * dz_tiles;
    for (int rounds = tiles / pairs;; --rounds) {
        const int dealt = max(0, rounds) * pairs;
        const long long rest = len.all - place_before(c, len, dealt);
        long long load = 0;
        if (q < pairs) {
            for (int t = q; t < dealt; t += pairs) {
                const int i = t >= c.tiles[0];
                load += (long long)tile_of(c, i, t - (i ? c.tiles[0] : 0)).unit * (c.stages[i] + kTileExtra);
            }
            load += dz_cost * (dz_tiles / pairs + (q < dz_tiles % pairs));
        }
        long long incl = load;
#pragma unroll
        for (int o = 1; o < 32; o *= 2) {
            const long long up = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += up;
        }
        if (lane == 31) scan[warp] = incl;
        __syncthreads();
        for (int w = 0; w < warp; ++w) incl += scan[w];
        // what is left for the pairs before this one when each has an equal part of everything; a length of at least eight stages each (four: 90 x 256 x 6163 fp32 58 us instead
        // of 55, 300 x 256 x 5000 56 instead of 54, longer ones alike)
        const long long begin = both * q / pairs - (incl - load), mine = both * (q + 1) / pairs - incl - begin;
        const bool fits = __syncthreads_and(q >= pairs || mine >= 32) != 0;
        if (!fits && rounds > 0) continue;
        if (q == 0) c.dealt = dealt;
        if (q <= pairs) {
            long long at;
            if (fits) {
                at = (len.all - rest) + (q < pairs ? begin : rest);
            } else {                         // too little for equal parts beside kDz's tiles: equal lengths of eight stages or more, for as many pairs as that gives
                const int active = (int)max(1LL, min((long long)pairs, len.all / 32));
                at = q >= active ? len.all : len.all * q / active;
            }
            c.begin[q] = place_of(c, len, at);
        }
        break;
    }
    __syncthreads();
    for (int i = q; i < (int)(sizeof(Cut) / sizeof(int)); i += kPackThreads) reinterpret_cast<int *>(cuts + launch)[i] = reinterpret_cast<const int *>(&c)[i];
}

// ---- rows that take part, moved together ------------------------------------------------------------------------------

constexpr int kAmaxBlocks = 4 * 148;

// partial[1][block] = the largest finite |w| that the block has seen; row_max[n] = that of row n of x, of the rows that take part.  Backward: partial[0][block] = the largest exponent_of(|g_n|) +
// exponent_of(row_max[n]) of the rows that have both, partial[2][block] = minus the smallest.
__global__ void __launch_bounds__(kPackThreads)
loss_amax_kernel(const float *__restrict__ x, const float *__restrict__ w, const float *__restrict__ g, const int *__restrict__ targets, int N, int E, int V, float *partial, float *row_max, int blocks,
                 PlanArgs plan, int launches, Cut *cuts)
{
    dependency_wait();
    dependents_may_start();
    if ((int)blockIdx.x < launches) { plan_launch(plan, blockIdx.x, cuts); return; }
    __shared__ float warp_max[2][8];
    const int which = ((int)blockIdx.x - launches) / blocks, block = ((int)blockIdx.x - launches) % blocks, lane = threadIdx.x & 31;
    float m = 0.0f, minus_least = -INFINITY;
    auto take = [&](float v) { v = fabsf(v); m = v <= FLT_MAX ? fmaxf(m, v) : m; };      // (not of infinities and NaN: they stay what they are)
    auto take4 = [&](const float4 &v) { take(v.x); take(v.y); take(v.z); take(v.w); };
    auto over_warp = [](float v) {
#pragma unroll
        for (int o = 16; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
        return v;
    };
    const long long step = (long long)blocks * 256, at = (long long)block * 256 + threadIdx.x;
    if (which == 1) {
        const long long total = (long long)V * E, words = (reinterpret_cast<uintptr_t>(w) & 15) == 0 ? total / 4 : 0;
        const float4 *w4 = reinterpret_cast<const float4 *>(w);
        long long i = at;
        for (; i + 3 * step < words; i += 4 * step) {
            const float4 a = __ldg(w4 + i), b = __ldg(w4 + i + step), c = __ldg(w4 + i + 2 * step), d = __ldg(w4 + i + 3 * step);
            take4(a); take4(b); take4(c); take4(d);
        }
        for (; i < words; i += step) take4(__ldg(w4 + i));
        for (i = words * 4 + at; i < total; i += step) take(__ldg(w + i));
    } else {
        const bool vec = E % 4 == 0 && (reinterpret_cast<uintptr_t>(x) & 15) == 0;
        const long long warps = step >> 5;
        float most = -INFINITY;
        for (long long n0 = at >> 5; n0 < N; n0 += 32 * warps) {             // a warp's next 32 rows: their targets at once
            const long long mine = n0 + lane * warps;
            const int t = mine < N ? __ldg(targets + mine) : -1;
            const float weight = g && t >= 0 && t < V ? fabsf(__ldg(g + mine)) : 0.0f;
            unsigned inside = __ballot_sync(0xffffffffu, t >= 0 && t < V);
            for (; inside; inside &= inside - 1) {
                const int from = __ffs(inside) - 1;
                const long long n = n0 + from * warps;
                const float *row = x + (size_t)n * E;
                m = 0.0f;
                if (vec) {
#pragma unroll 4
                    for (int e = lane * 4; e < E; e += 128) take4(__ldg(reinterpret_cast<const float4 *>(row + e)));
                } else {
#pragma unroll 4
                    for (int e = lane; e < E; e += 32) take(__ldg(row + e));
                }
                m = over_warp(m);
                if (lane == 0) row_max[n] = m;
                const float ga = __shfl_sync(0xffffffffu, weight, from);
                if (m > 0.0f && ga > 0.0f && ga <= FLT_MAX) {
                    const float e = (float)(exponent_of(m) + exponent_of(ga));
                    most = fmaxf(most, e);
                    minus_least = fmaxf(minus_least, -e);
                }
            }
        }
        m = most;
    }
    m = over_warp(m);
    if (lane == 0) {                         // (the least is the same in all lanes)
        warp_max[0][threadIdx.x >> 5] = m;
        warp_max[1][threadIdx.x >> 5] = minus_least;
    }
    __syncthreads();
    if (threadIdx.x < 2 - which) {
        m = -INFINITY;
#pragma unroll
        for (int i = 0; i < 8; ++i) m = fmaxf(m, warp_max[threadIdx.x][i]);
        partial[(which + 2 * threadIdx.x) * kAmaxBlocks + block] = m;
    }
}

// The largest of each of loss_amax_kernel's rows (backward: all three, forward: the second); every thread of 256 gets them
__device__ __forceinline__ void block_max(const float *partial, bool backward, int count, float (&sh)[3][8], float (&most)[3])
{
#pragma unroll
    for (int r = 0; r < 3; ++r) most[r] = -INFINITY;
    for (int i = threadIdx.x; i < count; i += 256)
#pragma unroll
        for (int r = 0; r < 3; ++r) if (backward || r == 1) most[r] = fmaxf(most[r], partial[r * kAmaxBlocks + i]);
#pragma unroll
    for (int r = 0; r < 3; ++r) {
#pragma unroll
        for (int o = 16; o; o >>= 1) most[r] = fmaxf(most[r], __shfl_xor_sync(0xffffffffu, most[r], o));
        if ((threadIdx.x & 31) == 0) sh[r][threadIdx.x >> 5] = most[r];
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < 3; ++r)
#pragma unroll
        for (int i = 0; i < 8; ++i) most[r] = fmaxf(most[r], sh[r][i]);
}

// The values of a row of `cols` from `begin` to `end` -> 16-bit ones in each plane, by one warp.  (What lies between `cols` and the next row is never read.)
template <typename T>
__device__ __forceinline__ void pack_row(const T *src, uint16_t *dst, size_t plane, int begin, int end, int cols, float scale, int lane, bool vec)
{
    end = min(end, cols);
    if constexpr (sizeof(T) == 2) {
        if (vec) {
#pragma unroll 4
            for (int c = begin + lane * 8; c < end; c += 256) *reinterpret_cast<uint4 *>(dst + c) = __ldg(reinterpret_cast<const uint4 *>(src + c));
        } else {
#pragma unroll 4
            for (int c = begin + lane; c < end; c += 32) dst[c] = reinterpret_cast<const uint16_t *>(src)[c];
        }
    } else {
#pragma unroll 4
        for (int c = begin + lane * 4; c < end; c += 128) {
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

struct Pack {
    const float *partial, *row_max;          // fp32: loss_amax_kernel's
    int amax_blocks;
    float *scales;
    // the rows of x
    const int *targets;
    const float *lse, *g;                    // backward
    int N, E, V, ld, per_block, x_blocks, x_vec;
    uint16_t *xp, *xq;                       // xq: the rows as dW takes them (fp32), or NULL
    size_t plane;
    int *count, *failed, *row_map, *c_targets;
    float *c_lse, *c_g, *c_x_inv, *c_unit;
    float *zero_loss, *zero_lse;             // forward: what rows that take no part get
    uint8_t *zero_grad;                      // backward: their rows of the gradient
    int *zero_ints;
    int zeros;
    // the weights, in pieces of kPackCols columns of a row
    uint16_t *wp;
    size_t w_plane;
    int w_rows, w_cols, w_ld, w_col_pieces, w_vec;
    int targets_vec;
};
constexpr int kPackCols = 1024;

template <typename T>
__global__ void __launch_bounds__(kPackThreads)
loss_pack_kernel(const T *__restrict__ x, const T *__restrict__ w, Pack p, PlanArgs plan, int launches, Cut *cuts)
{
    dependency_wait();
    dependents_may_start();
    if constexpr (sizeof(T) == 2)            // (fp32: among loss_amax_kernel's blocks)
        if ((int)blockIdx.x < launches) { plan_launch(plan, blockIdx.x, cuts); return; }
    const int block = sizeof(T) == 2 ? (int)blockIdx.x - launches : (int)blockIdx.x;
    __shared__ int warp_sum[8];
    __shared__ float warp_max[3][8];
    int w_exp = 14, most = 27;                // (scales of 1)
    bool deep = false;                       // a row lies more than kMostShift below the largest
    if constexpr (sizeof(T) == 4) {
        float largest[3];
        block_max(p.partial, p.g != nullptr, p.amax_blocks, warp_max, largest);
        if (largest[1] > 0.0f) w_exp = exponent_of(largest[1]);
        if (largest[0] > -INFINITY) most = (int)largest[0];
        deep = largest[0] + largest[2] > (float)kMostShift;
    }
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (block >= p.x_blocks) {               // eight pieces of rows of the weights a block
        const float scale = pow2(14 - w_exp);
        const long long job = (long long)(block - p.x_blocks) * 8 + warp;
        const int r = (int)(job / p.w_col_pieces), c = (int)(job % p.w_col_pieces) * kPackCols;
        if (r < p.w_rows) pack_row<T>(w + (size_t)r * p.w_cols, p.wp + (size_t)r * p.w_ld, p.w_plane, c, min(p.w_ld, c + kPackCols), p.w_cols, scale, lane, p.w_vec != 0);
        return;
    }
    if (sizeof(T) == 4 && block == 0 && tid == 0) {
        p.scales[0] = pow2(w_exp - 14);
        const int e = most - 27;              // (one power of two could pass the range of fp32)
        p.scales[1] = pow2(e / 2);
        p.scales[2] = pow2(e - e / 2);
        p.scales[3] = deep ? 1.0f : 0.0f;
    }
    if (block == 0 && tid == 0) *p.failed = 0;
    for (int i = block * 256 + tid; i < p.zeros; i += p.x_blocks * 256) p.zero_ints[i] = 0;
    const int from = block * p.per_block, to = min(p.N, from + p.per_block);
    auto inside = [&](int t) { return t >= 0 && t < p.V; };
    int before = 0, done = 0;
    if (p.targets_vec) {
        done = from / 4 * 4;
#pragma unroll 8
        for (int i = tid; i < done / 4; i += 256) {
            const int4 t = __ldg(reinterpret_cast<const int4 *>(p.targets) + i);
            before += inside(t.x) + inside(t.y) + inside(t.z) + inside(t.w);
        }
    }
#pragma unroll 8
    for (int i = done + tid; i < from; i += 256) before += inside(__ldg(p.targets + i));
#pragma unroll
    for (int o = 16; o; o >>= 1) before += __shfl_xor_sync(0xffffffffu, before, o);
    if (lane == 0) warp_sum[warp] = before;
    __syncthreads();
    int base = 0;
#pragma unroll
    for (int w8 = 0; w8 < 8; ++w8) base += warp_sum[w8];
    for (int r0 = from; r0 < to; r0 += 32) {
        // each lane looks at one row; what belongs to it is stored by the first warp
        const bool there = r0 + lane < to;
        const int t = there ? __ldg(p.targets + r0 + lane) : -1;
        const float g = p.g && there ? __ldg(p.g + r0 + lane) : 0.0f;
        const unsigned mask = __ballot_sync(0xffffffffu, inside(t));
        RowScales scale = {1.0f, 1.0f, 1.0f, 1.0f, 1.0f};
        if (sizeof(T) == 4 && there) scale = row_scales(p.row_max[r0 + lane], g, most);       // (of a row that takes no part: not used)
        if (warp == 0 && inside(t)) {
            const int i = base + __popc(mask & ((1u << lane) - 1));
            p.row_map[i] = r0 + lane;
            p.c_targets[i] = t;
            if (sizeof(T) == 4) p.c_x_inv[i] = scale.x_inv;
            if (p.g) {
                p.c_g[i] = g * scale.dz;
                p.c_lse[i] = p.lse[r0 + lane];
                if (sizeof(T) == 4) p.c_unit[i] = scale.dz_inv;
            }
        }
        float x_scale[4], x_dw_scale[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            x_scale[k] = __shfl_sync(0xffffffffu, scale.x, warp + 8 * k);
            x_dw_scale[k] = __shfl_sync(0xffffffffu, scale.x_dw, warp + 8 * k);
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int j = warp + 8 * k, n = r0 + j;
            if (n >= to) break;
            if (mask >> j & 1) {
                const size_t at = (size_t)(base + __popc(mask & ((1u << j) - 1))) * p.ld;
                pack_row<T>(x + (size_t)n * p.E, p.xp + at, p.plane, 0, p.ld, p.E, x_scale[k], lane, p.x_vec != 0);
                if (sizeof(T) == 4 && deep && p.xq) pack_row<T>(x + (size_t)n * p.E, p.xq + at, p.plane, 0, p.ld, p.E, x_dw_scale[k], lane, p.x_vec != 0);
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
    if (to == p.N && from < p.N) {           // the last block that has rows: their number, and zeros up to a whole stage (one at least) of the products that sum over them
        if (tid == 0) *p.count = base;
        const int end = max(kDeep, (base + kDeep - 1) / kDeep * kDeep);
        uint16_t *rows = p.xq && deep ? p.xq : p.xp;
        for (int i = base + warp; i < end; i += 8)
            for (int c = lane * 4; c < p.ld; c += 128)
                for (int pl = 0; pl < (sizeof(T) == 4 ? 2 : 1); ++pl) *reinterpret_cast<uint2 *>(rows + pl * p.plane + (size_t)i * p.ld + c) = make_uint2(0u, 0u);
    }
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

__device__ __noinline__ bool loss_wait_slow(uint64_t *bar, uint32_t parity, int site, volatile int *abort_flag, uint32_t peer_flag, int *failed, int expire)
{
    if (!expires_now(expire, site) && mbar_wait(bar, parity)) return true;
    *abort_flag = 1;
    asm volatile("st.volatile.shared::cluster.u32 [%0], %1;" ::"r"(peer_flag), "r"(1) : "memory");      // the other block's rows of the tile are not stored either
    atomicCAS(&g_loss_status, 0, site);
    atomicExch(failed, 1);
    linger();
    return false;
}

// What a pair does, one after the other: its tiles of kDx and kDw, its length of the rest of them, its tiles of kDz
struct Work {
    int kind, m, n, k0, k1, stages, tile;    // tile: of kDx and kDw, as in Place
    bool narrow;
};
struct Walk {
    int dealt;
    Place at, end;
    int dz, dz_tiles, dz_m_tiles;
};

// What exponentials are taken relative to: the maximum, or the next finite number.  (So beside a logit of +infinity the others count for nothing and the sum is infinite, and infinity - infinity is met nowhere.)
__device__ __forceinline__ float reference(float m) { return fminf(fmaxf(m, -FLT_MAX), FLT_MAX); }

// Two parts of a row: (maximum, sum of exponentials relative to its reference)
__device__ __forceinline__ float2 join_parts(float2 a, float2 b)
{
    const float m = fmaxf(a.x, b.x), ref = reference(m);
    return make_float2(m, a.y * ex2_approx((a.x - ref) * kLog2e) + b.y * ex2_approx((b.x - ref) * kLog2e));
}

// 32 columns of a thread's row, four of them at `to`, the next kTileM further on
__device__ __forceinline__ void put_tile(float4 *to, const float (&v)[32])
{
#pragma unroll
    for (int j = 0; j < 8; ++j) __stcg(to + j * kTileM, make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]));
}
__device__ __forceinline__ void add_tile(const float4 *from, float (&v)[32])
{
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float4 o = __ldcg(from + j * kTileM);
        v[4 * j] += o.x; v[4 * j + 1] += o.y; v[4 * j + 2] += o.z; v[4 * j + 3] += o.w;
    }
}
// A sum of TMEM's, added to what a thread has stored at `so_far` if `more`, and stored there.  (Not inline: few calls come here, and those that do not keep their registers.)
__device__ __noinline__ void put_by(uint32_t tmem, float4 *so_far, int chunks, bool more)
{
#pragma unroll 1
    for (int c = 0; c < chunks; ++c) {
        float v[32];
        tmem_ld32(tmem + (uint32_t)(32 * c), v);
        tmem_wait_ld();
        if (more) add_tile(so_far + c * 8 * kTileM, v);
        put_tile(so_far + c * 8 * kTileM, v);
    }
}

// T: the storage type; operands have one plane (bf16) or two (fp32 as fp16 hi and lo).  site codes in the status word: 1 stage landed, 2 stage free,
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
    __shared__ float scales_s[4];             // LossArgs::scales
    __shared__ float2 part_s[FORM == kForward ? 2 : 1][4][kHalfM];
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
        if (!gone && !done) seen = loss_wait_slow(bar, parity, site, &abort_flag, peer_flag, args.failed, args.expire);
    };

    // No row may take part: one tile of rows of zeros, and one stage, are then worked on (so gradients of zero are written)
    if (threadIdx.x < 4 && (NP == 2 || FORM == kBackward)) scales_s[threadIdx.x] = args.scales[threadIdx.x];
    const bool failed = *args.failed != 0;
    const int count = *args.count, pairs = (int)gridDim.x / 2, pair = (int)blockIdx.x / 2;
    const int count_tiles = max(1, (count + kTileM - 1) / kTileM), count_stages = max(1, (count + kDeep - 1) / kDeep);
    __shared__ Cut cut;
    if constexpr (FORM == kBackward)
        for (int i = threadIdx.x; i < (int)(sizeof(Cut) / sizeof(int)); i += kThreads) reinterpret_cast<int *>(&cut)[i] = reinterpret_cast<const int *>(args.cut)[i];
    __syncthreads();
    Walk first = {0, {0, 0}, {0, 0}, pair, failed ? 0 : count_tiles * args.p[kDz].n_tiles, count_tiles};
    if constexpr (FORM == kBackward) {
        first.dealt = failed ? cut.dealt : min(pair, cut.dealt);
        first.at = cut.begin[pair];
        first.end = failed ? first.at : cut.begin[pair + 1];
    }
    auto next = [&](Walk &w, Work &x) {
        if constexpr (FORM == kBackward) {
            const bool deal = w.dealt < cut.dealt;
            if (deal || before(w.at, w.end)) {
                const int t = deal ? w.dealt : w.at.tile, i = t >= cut.tiles[0];
                const TileOf place = tile_of(cut, i, t - (i ? cut.tiles[0] : 0));
                x = {i, place.m, place.n, deal ? 0 : w.at.k, deal || t != w.end.tile ? cut.stages[i] : w.end.k, cut.stages[i], t, place.unit == 3};
                if (deal) w.dealt += pairs; else w.at = {t + 1, 0};
                return true;
            }
        }
        if (w.dz >= w.dz_tiles) return false;
        const int stages = args.p[kDz].stages;
        x = {kDz, w.dz % w.dz_m_tiles, w.dz / w.dz_m_tiles, 0, stages, stages, 0, false};      // m runs fastest, so pairs that run side by side share B's columns
        w.dz += pairs;
        return true;
    };
    // f(kind) with the kind as a constant: what is read of the problem then lies at a fixed place among the kernel's arguments.  (With the place in a variable a stage took
    // 950 cycles instead of 740 for the logits, 800 instead of 620 for the sums: copies and products were issued late.)
    auto by_kind = [](int kind, auto f) {
        if (FORM == kForward || kind == kDz) f(std::integral_constant<int, kDz>());
        else if (kind == kDx) f(std::integral_constant<int, kDx>());
        else f(std::integral_constant<int, kDw>());
    };

    Work x;
    Walk walk = first;
    if (warp == kEpiWarps) {
        // ---- producer: this block's halves of both operands ----
        const uint32_t full_of_first = peer_addr(smem_u32(&full[0]), 0);
        int s = 0, round = 0;
        while (next(walk, x)) {
            by_kind(x.kind, [&](auto kind) {
                constexpr int KIND = decltype(kind)::value;
                const Problem &p = args.p[KIND];
                const CUtensorMap *ma = &args.a[KIND], *mb = &args.b[KIND];
                if (NP == 2 && KIND == kDw && scales_s[3] != 0.0f) (args.x_is_a ? ma : mb) = &args.xq;
                const int m0 = x.m * kTileM + rank * kHalfM, n0 = p.b_n0 + x.n * kTileN + rank * (x.narrow ? kHalfM / 2 : kHalfM);
                const int end = KIND == kDz ? p.stages : x.k1;
                for (int k = KIND == kDz ? 0 : x.k0; k < end; ++k) {
                    if (round) wait(&empty[s], (uint32_t)((round - 1) & 1), 2);
                    if (elect_one() && seen) {
                        if (rank == 0) mbar_arrive_expect_tx(&full[s], (uint32_t)(x.narrow ? 2 * STAGE - NP * kOperand : 2 * STAGE));
                        const uint32_t bar = full_of_first + (uint32_t)(s * sizeof(uint64_t));
                        uint8_t *at = ring + s * STAGE;
#pragma unroll
                        for (int pl = 0; pl < NP; ++pl) {
                            uint8_t *a = at + pl * kOperand, *b = at + (NP + pl) * kOperand;
                            const int ka = k * kDeep, kb = p.b_k0 + k * kDeep;
                            if (p.a_across) {
                                tma_load_pair(a, ma, m0, ka, pl, bar);
                                tma_load_pair(a + kOperand / 2, ma, m0 + 64, ka, pl, bar);
                            } else {
                                tma_load_pair(a, ma, ka, m0, pl, bar);
                            }
                            // (64 columns at a time either way: a narrow tile has no more)
                            tma_load_pair(b, mb, p.b_across ? n0 : kb, p.b_across ? kb : n0, pl, bar);
                            if (!x.narrow) tma_load_pair(b + kOperand / 2, mb, p.b_across ? n0 + 64 : kb, p.b_across ? kb : n0 + 64, pl, bar);
                        }
                    }
                    __syncwarp();
                    if (++s == RING) { s = 0; ++round; }
                }
            });
        }
        if (abort_flag) linger();
    } else if (warp == kEpiWarps + 1) {
        // ---- products, issued by the pair's first block for both ----
        if (rank == 0) {
            int s = 0, round = 0, unit = 0;
            while (next(walk, x)) {
                by_kind(x.kind, [&](auto kind) {
                constexpr int KIND = decltype(kind)::value;
                const Problem &p = args.p[KIND];
                // operand along the reduction: rows of 128 bytes in groups of 8 (1024 bytes), 16 deep = 32 bytes; across it: blocks of 64 x 64 deep (8192 bytes),
                // 8 deep = 1024 bytes.  Swizzled by 128 bytes either way.
                const uint32_t idesc = (1u << 4) | (NP == 1 ? (1u << 7) | (1u << 10) : 0u) | ((uint32_t)p.a_across << 15) | ((uint32_t)p.b_across << 16) |
                                       ((uint32_t)((x.narrow ? kTileN / 2 : kTileN) >> 3) << 17) | ((uint32_t)(kTileM >> 4) << 24);
                const uint32_t a_lbo = p.a_across ? kOperand / 2 : 16, b_lbo = p.b_across ? kOperand / 2 : 16;
                const uint64_t a_step = p.a_across ? 128 : 2, b_step = p.b_across ? 128 : 2;
                constexpr int unit_stages = kSumStages<FORM, NP>;
                const int begin = KIND == kDz ? 0 : x.k0, end = KIND == kDz ? p.stages : x.k1;
                for (int k0 = begin; k0 < end; k0 += unit_stages, ++unit) {
                    const uint32_t acc = tmem + (uint32_t)((unit & 1) * kTileN);
                    if (unit >= 2) wait(&acc_empty[unit & 1], (uint32_t)((unit / 2 - 1) & 1), 4);
                    tc_fence_after();
                    const int k1 = min(end, k0 + unit_stages);
                    for (int k = k0; k < k1; ++k) {
                        wait(&full[s], (uint32_t)(round & 1), 1);
                        tc_fence_after();
                        const uint32_t at = smem_u32(ring + s * STAGE);
                        const uint64_t a = make_desc(at, a_lbo, 1024, 2), b = make_desc(at + NP * kOperand, b_lbo, 1024, 2);
                        [[maybe_unused]] constexpr uint64_t lo = kOperand >> 4;
                        if constexpr (NP == 2) {     // the small products before the large ones: less of them is cut off
#pragma unroll
                            for (int j = 0; j < kDeep / 16; ++j) {
                                if (elect_one()) mma_pair(acc, a + lo + j * a_step, b + j * b_step, idesc, (k > k0 || j) ? 1u : 0u);
                                if (elect_one()) mma_pair(acc, a + j * a_step, b + lo + j * b_step, idesc, 1u);
                            }
                        }
#pragma unroll
                        for (int j = 0; j < kDeep / 16; ++j)
                            if (elect_one()) mma_pair(acc, a + j * a_step, b + j * b_step, idesc, (NP == 2 || k > k0 || j) ? 1u : 0u);
                        if (elect_one()) commit_pair(&empty[s]);
                        if (++s == RING) { s = 0; ++round; }
                    }
                    if (elect_one()) commit_pair(&acc_full[unit & 1]);
                }
                });
            }
            __syncwarp();
            if (abort_flag) linger();
        }
    } else {
        // ---- what becomes of an accumulator: thread = row = TMEM lane; four warps share a row's columns ----
        const int quarter = warp & 3, fourth = warp >> 2, row_in_tile = rank * kHalfM + quarter * 32 + lane;
        const uint32_t lane_base = tmem + ((uint32_t)(quarter * 32) << 16);
        const uint32_t drained = peer_addr(smem_u32(&acc_empty[0]), 0);
        uint8_t *out_s = ring + kRingBytes + warp * kOutBytes;           // (kBackward)
        int unit = 0, part_at = 0;
        while (next(walk, x)) {
            const Problem &p = args.p[x.kind];
            const int row = x.m * kTileM + row_in_tile;
            const int chunks = x.narrow ? kWarpChunks / 2 : kWarpChunks, mine0 = fourth * 32 * chunks, col0 = x.n * kTileN + mine0;      // its 32-column chunks
            // The reads of TMEM have completed and nothing in memory goes with it, so the arrival need not wait for the stores that are on their way
            auto release = [&](int buf) {
                tc_fence_before();
                __syncwarp();
                if (lane == 0) asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(drained + (uint32_t)(buf * sizeof(uint64_t))) : "memory");
            };
            const bool whole = x.kind == kDz || (x.k0 == 0 && x.k1 == x.stages);

            // per row: whether it is there, and its target (of the logits), or its row of the result
            const bool here = row < (FORM == kForward || x.kind != kDw ? count : p.rows);
            int of_row = -1;
            float lse = 0.0f, g = 0.0f, z_scale = 1.0f, run_max = -INFINITY, run_sum = 0.0f;
            if (here) {
                if (FORM == kForward || x.kind == kDz) {
                    of_row = __ldg(args.targets + row) - args.v0;
                    if constexpr (NP == 2) z_scale = __ldg(args.x_inv + row);          // (W's joins it behind the waits, so that they begin before this has come)
                } else {
                    of_row = x.kind == kDx ? __ldg(args.row_map + row) : row;
                    if (NP == 2 && x.kind == kDx) g = __ldg(args.row_unit + row);
                }
                if (FORM == kBackward && x.kind == kDz) { lse = __ldg(args.lse + row); g = NP == 2 ? __ldg(args.g + row) : __fdiv_rn(__ldg(args.g + row), scales_s[2]); }
            }
            const int left_all = (FORM == kForward || x.kind == kDz ? args.V - args.v0 : p.cols) - col0;           // columns from col0 on

            // where 32 columns of this thread's row begin in a tile of `shares` or `sum`
            auto tile_at = [&](int tile, int c) { return ((size_t)tile * (kTileN / 4) + (size_t)((mine0 + 32 * c) / 4)) * kTileM + row_in_tile; };

            // the sum of a long tile's stages so far, behind the pairs' shares
            auto so_far = [&](int c) { return args.shares + tile_at(2 * pairs + pair, c); };

            // kForward: 32 columns from col0 + 32 c on
            auto log_sum = [&](int c, float (&v)[32]) {
                const int col = col0 + 32 * c, left = left_all - 32 * c;
                if (left <= 0) return;
                if (left < 32) {
#pragma unroll
                    for (int j = 0; j < 32; ++j) if (j >= left) v[j] = -INFINITY;
                }
                if (of_row >= col && of_row < col + 32 && !abort_flag) {
#pragma unroll
                    for (int j = 0; j < 32; ++j) if (of_row - col == j) args.z_target[row] = v[j] * z_scale;
                }
                float m = run_max;
#pragma unroll
                for (int j = 0; j < 32; j += 2) m = max3(m, v[j] * z_scale, v[j + 1] * z_scale);
                const float ref = reference(m);
                float s0 = run_sum * ex2_approx((run_max - ref) * kLog2e), s1 = 0.0f;
#pragma unroll
                for (int j = 0; j < 32; j += 2) {
                    const float2 d = fmul2(ffma2(make_float2(v[j], v[j + 1]), make_float2(z_scale, z_scale), make_float2(-ref, -ref)), make_float2(kLog2e, kLog2e));
                    s0 += ex2_approx(d.x);
                    s1 += ex2_approx(d.y);
                }
                run_max = m;
                run_sum = s0 + s1;
            };
            // A thread's 64 bytes of its row into the warp's place in shared memory, swizzled so that a store instruction meets every bank once
            auto stage_at = [&](int r, int j) { return reinterpret_cast<uint4 *>(out_s + r * 64 + ((j ^ (r >> 1 & 3)) << 4)); };
            auto stage = [&](const uint32_t (&o)[16]) {
#pragma unroll
                for (int j = 0; j < 4; ++j) *stage_at(lane, j) = make_uint4(o[4 * j], o[4 * j + 1], o[4 * j + 2], o[4 * j + 3]);
            };
            auto out_free = [&] {                 // what lay there is out
                if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
                __syncwarp();
            };
            // kDz: 32 columns of a plane by a bulk copy out of there
            auto put_dz = [&](int c, int plane, const uint32_t (&o)[16]) {
                out_free();
                stage(o);
                proxy_fence();
                __syncwarp();
                if (lane == 0 && !abort_flag) {
                    asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%1, %2, %3}], [%4];"
                                 ::"l"(reinterpret_cast<uint64_t>(&args.dz_out)), "r"(col0 + 32 * c), "r"(x.m * kTileM + rank * kHalfM + quarter * 32), "r"(plane), "r"(smem_u32(out_s)) : "memory");
                    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
                }
            };
            auto logit_gradient = [&](int c, float (&v)[32]) {
                const int col = col0 + 32 * c, left = here ? left_all - 32 * c : 0;
#pragma unroll
                for (int j = 0; j < 32; j += 2) {
                    const float2 d = fmul2(ffma2(make_float2(v[j], v[j + 1]), make_float2(z_scale, z_scale), make_float2(-lse, -lse)), make_float2(kLog2e, kLog2e));
                    v[j] = ex2_approx(d.x);
                    v[j + 1] = ex2_approx(d.y);
                }
                if (of_row >= col && of_row < col + 32) {
#pragma unroll
                    for (int j = 0; j < 32; ++j) v[j] -= of_row - col == j ? 1.0f : 0.0f;
                }
#pragma unroll
                for (int j = 0; j < 32; j += 2) {
                    const float2 d = fmul2(make_float2(v[j], v[j + 1]), make_float2(g, g));
                    v[j] = d.x;
                    v[j + 1] = d.y;
                }
                if (left < 32) {
#pragma unroll
                    for (int j = 0; j < 32; ++j) v[j] = j < left ? v[j] : 0.0f;
                }
                uint32_t o[16];
                if constexpr (NP == 1) {
#pragma unroll
                    for (int j = 0; j < 16; ++j) o[j] = pack_bf16(v[2 * j], v[2 * j + 1]);
                    put_dz(c, 0, o);
                } else {
#pragma unroll
                    for (int plane = 0; plane < 2; ++plane) {
#pragma unroll
                        for (int j = 0; j < 16; ++j) {
                            const __half2 h = __floats2half2_rn(v[2 * j], v[2 * j + 1]);
                            o[j] = *reinterpret_cast<const uint32_t *>(&h);
                            v[2 * j] -= __low2float(h);
                            v[2 * j + 1] -= __high2float(h);
                        }
                        put_dz(c, plane, o);
                    }
                }
            };
            // kDx, kDw: 32 columns of a tile that is complete
            auto finish = [&](int c, float (&v)[32]) {
                const int left = left_all - 32 * c;
                if (left <= 0 || __any_sync(0xffffffffu, abort_flag)) return;
                if (x.kind == kDx && !args.last) {
                    put_tile(args.sum + tile_at(x.tile, c), v);
                    return;
                }
                // fp32: two powers of two whose product may pass the range of fp32; the smaller one first, so that no result is lost on the way that is not too large itself
                const float a = NP == 1 ? scales_s[2] : scales_s[x.kind == kDx ? 0 : 1], b = NP == 1 ? 1.0f : x.kind == kDx ? g : scales_s[2], s0 = fminf(a, b), s1 = fmaxf(a, b);
#pragma unroll
                for (int j = 0; j < 32; ++j) v[j] = NP == 1 ? v[j] * a : v[j] * s0 * s1;
                const unsigned rows_here = __ballot_sync(0xffffffffu, here);
                const bool out_vec = p.ld % kPer16<T> == 0 && (reinterpret_cast<uintptr_t>(p.out) & 15) == 0;
                if (p.accumulate || !out_vec || left < 32) {
                    // added to what is there, rows of any alignment, or the last columns: 16 fp32 values of each row at a time, half a warp a row, a value a lane
#pragma unroll
                    for (int h = 0; h < 32; h += 16) {
                        uint32_t o[16];
#pragma unroll
                        for (int j = 0; j < 16; ++j) o[j] = __float_as_uint(v[h + j]);
                        out_free();
                        stage(o);
                        __syncwarp();
                        const int col = lane & 15;
#pragma unroll 4
                        for (int i = 0; i < 16; ++i) {
                            const int r = 2 * i + (lane >> 4);
                            T *to = static_cast<T *>(p.out) + __shfl_sync(0xffffffffu, of_row, r) * p.ld + col0 + 32 * c + h + col;
                            if ((rows_here >> r & 1) && h + col < left) {
                                const float y = reinterpret_cast<const float *>(stage_at(r, col >> 2))[col & 3];
                                *to = from_float<T>(p.accumulate ? to_float(*to) + y : y);
                            }
                        }
                    }
                    return;
                }
                // 64 bytes of each row at a time, four lanes a row: whole sectors, where a thread's own row by itself would be stored 16 bytes here and 16 there
                constexpr int kPer64 = 64 / (int)sizeof(T);
#pragma unroll
                for (int h = 0; h < 32; h += kPer64) {
                    uint32_t o[16];
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        if constexpr (NP == 1) o[j] = pack_bf16(v[2 * j], v[2 * j + 1]);
                        else o[j] = __float_as_uint(v[h + j]);
                    }
                    out_free();
                    stage(o);
                    __syncwarp();
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int r = 8 * i + (lane >> 2);
                        const long long at = __shfl_sync(0xffffffffu, of_row, r) * p.ld;
                        const uint4 u = *stage_at(r, lane & 3);
                        if (rows_here >> r & 1) *reinterpret_cast<uint4 *>(static_cast<T *>(p.out) + at + col0 + 32 * c + h + (lane & 3) * kPer16<T>) = u;
                    }
                }
            };
            // ... and of one that is not: into this pair's share
            auto leave = [&](int c, const float (&v)[32]) {
                put_tile(args.shares + tile_at(2 * pair + (x.k0 == 0), c), v);
            };

            // A tile that falls to several pairs (they follow one another, each with a part of its stages): the first of them is usually the last to come to it,
            // finds the others' shares there and adds them to what it has in hand.  Whichever comes last adds them in the same order.
            int p0 = pair, p1 = pair, sources = 0;
            bool complete = whole;
            int *arrived = nullptr;
            if (FORM == kBackward && x.kind != kDz) {
                if (!whole) {
                    const Place tile_begin = {x.tile, 0}, tile_end = {x.tile, x.stages};
                    while (p0 > 0 && before(tile_begin, cut.begin[p0])) --p0;
                    while (before(cut.begin[p1 + 1], tile_end)) ++p1;
                    arrived = args.arrived + ((size_t)x.tile * 2 + rank) * kEpiWarps + warp;
                }
                sources = (p1 - p0) + (x.kind == kDx && !args.first);
            }
            // source i of what is added to this pair's own part: the pairs behind the first, then dx so far
            auto source = [&](int i, int c) { return i < p1 - p0 ? args.shares + tile_at(2 * (p0 + 1 + i), c) : args.sum + tile_at(x.tile, c); };

            auto add_sources = [&](int c, float (&v)[32]) {
#pragma unroll 1
                for (int i = 0; i < sources; ++i) add_tile(source(i, c), v);
            };

            // whether the others' shares of a tile that this pair is the first of are there
            auto others_there = [&] {
                int there = 0;
                if (lane == 0) there = *reinterpret_cast<volatile int *>(arrived);
                there = __shfl_sync(0xffffffffu, there, 0);
                __threadfence();
                if (there == p1 - p0 && lane == 0) *arrived = 0;         // for the next launch
                return there == p1 - p0;
            };
            auto take = [&](int c, float (&v)[32]) {
                if constexpr (FORM == kForward) {
                    log_sum(c, v);
                } else if (x.kind == kDz) {
                    logit_gradient(c, v);
                } else if (complete) {
                    add_sources(c, v);
                    finish(c, v);
                } else {
                    leave(c, v);
                }
            };
            constexpr int unit_stages = kSumStages<FORM, NP>;
            auto await_sum = [&] {
                wait(&acc_full[unit & 1], (uint32_t)((unit / 2) & 1), 3);
                tc_fence_after();
            };
            if (NP == 2 || (FORM == kForward && x.k1 - x.k0 > unit_stages)) {
                // TMEM's sums are added up in registers
                float acc[kWarpChunks][32];
#pragma unroll
                for (int c = 0; c < kWarpChunks; ++c)
#pragma unroll
                    for (int j = 0; j < 32; ++j) acc[c][j] = 0.0f;
                for (int k0 = x.k0; k0 < x.k1; k0 += unit_stages, ++unit) {
                    await_sum();
#pragma unroll
                    for (int c = 0; c < kWarpChunks; ++c) {
                        if (c >= chunks) continue;
#pragma unroll
                        for (int h = 0; h < 32; h += 16) {
                            float v[16];
                            tmem_ld16(lane_base + (uint32_t)((unit & 1) * kTileN + mine0 + 32 * c + h), v);
                            tmem_wait_ld();
#pragma unroll
                            for (int j = 0; j < 16; ++j) acc[c][h + j] += v[j];
                        }
                    }
                    release(unit & 1);
                }
                if (FORM == kBackward && !whole && pair == p0) complete = others_there();
                if constexpr (NP == 2) z_scale = fminf(z_scale * scales_s[0], FLT_MAX);           // (an infinite one would make NaN of a logit of zero)
#pragma unroll
                for (int c = 0; c < kWarpChunks; ++c)
                    if (FORM == kForward || c < chunks) take(c, acc[c]);
            } else {
                for (int k0 = x.k0; FORM == kBackward && k0 + unit_stages < x.k1; k0 += unit_stages, ++unit) {
                    await_sum();
                    put_by(lane_base + (uint32_t)((unit & 1) * kTileN + mine0), so_far(0), chunks, k0 > x.k0);
                    release(unit & 1);
                }
                await_sum();
                if (FORM == kBackward && !whole && pair == p0) complete = others_there();
#pragma unroll 1
                for (int c = 0; c < chunks; ++c) {
                    float v[32];
                    tmem_ld32(lane_base + (uint32_t)((unit & 1) * kTileN + mine0 + 32 * c), v);
                    tmem_wait_ld();
                    if (c == chunks - 1) release(unit & 1);
                    if (FORM == kBackward && x.k1 - x.k0 > unit_stages) add_tile(so_far(c), v);
                    take(c, v);
                }
                ++unit;
            }
            if constexpr (FORM == kForward) {
                // the four warps that share these rows meet; one joins what they have (two buffers: a warp is at most a tile ahead)
                float2 (&mine)[4][kHalfM] = part_s[part_at];
                part_at ^= 1;
                mine[fourth][quarter * 32 + lane] = make_float2(run_max, run_sum);
                asm volatile("bar.sync %0, 128;" ::"r"(1 + quarter) : "memory");
                if (fourth == 0 && here && !abort_flag) {
                    float2 all = mine[0][quarter * 32 + lane];
#pragma unroll
                    for (int i = 1; i < 4; ++i) all = join_parts(all, mine[i][quarter * 32 + lane]);
                    args.part[(size_t)x.n * args.rows_alloc + row] = all;
                }
            } else if (!complete) {
                __threadfence();
                __syncwarp();
                int seen_before = 0;
                if (lane == 0 && !abort_flag) seen_before = atomicAdd(arrived, 1);
                seen_before = __shfl_sync(0xffffffffu, seen_before, 0);
                __threadfence();
                if (seen_before == p1 - p0) {        // the last of them: all shares are there
                    if (lane == 0) *arrived = 0;
#pragma unroll 1
                    for (int c = 0; c < chunks; ++c) {
                        float v[32];
                        const float4 *own = args.shares + tile_at(2 * p0 + 1, c);
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            const float4 o = __ldcg(own + j * kTileM);
                            v[4 * j] = o.x; v[4 * j + 1] = o.y; v[4 * j + 2] = o.z; v[4 * j + 3] = o.w;
                        }
                        add_sources(c, v);
                        finish(c, v);
                    }
                }
            }
        }
        if (FORM == kBackward && lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
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
                 const int *__restrict__ failed, float *loss, float *lse)
{
    dependency_wait();
    dependents_may_start();
    __shared__ float2 sh[8][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, n = *failed ? 0 : *count;
    for (int r0 = blockIdx.x * 32; r0 < n; r0 += gridDim.x * 32) {
        const int row = r0 + lane;
        float2 all = make_float2(-INFINITY, 0.0f);
        if (row < n) {
#pragma unroll 8
            for (int i = warp; i < parts; i += 8) all = join_parts(all, __ldg(part + (size_t)i * rows_alloc + row));
        }
        sh[warp][lane] = all;
        __syncthreads();
        if (warp == 0 && row < n) {
#pragma unroll
            for (int w = 1; w < 8; ++w) all = join_parts(all, sh[w][lane]);
            const float l = all.x + logf(all.y);
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

// {inner, outer, plane} of 16-bit values; box: 64 inner values (128 bytes; 32: 64 bytes) of `box_outer` outer ones, swizzled by its width
int operand_map(CUtensorMap *m, const void *base, bool half, long long inner, long long outer, long long ld, size_t plane, int planes, int box_outer, int box_inner = 64)
{
    EncodeTiledFn enc = tma_encode_fn();
    if (!enc) return fail(HIPGPT_ERR_CUDA, "cuTensorMapEncodeTiled is not available from this driver");
    const cuuint64_t dims[3] = {(cuuint64_t)inner, (cuuint64_t)outer, (cuuint64_t)planes};
    const cuuint64_t strides[2] = {(cuuint64_t)ld * 2, (cuuint64_t)plane * 2};
    const cuuint32_t box[3] = {(cuuint32_t)box_inner, (cuuint32_t)box_outer, 1}, estr[3] = {1, 1, 1};
    const CUresult r = enc(m, half ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void *>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                           box_inner == 64 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(HIPGPT_ERR_CUDA, "cuTensorMapEncodeTiled failed with code %d", (int)r);
    return HIPGPT_OK;
}

// The grid of a call: a pair of blocks for each two SMs, or for each tile where there are fewer
int loss_pairs(int dev, long long most, int *pairs)
{
    int sms = 0;
    const cudaError_t e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    if (e != cudaSuccess) return fail(HIPGPT_ERR_CUDA, "loss_gemm_kernel: %s", cudaGetErrorString(e));
    *pairs = (int)std::max<long long>(1, std::min<long long>(most, std::min(sms / 2, kMostPairs - 1)));
    return HIPGPT_OK;
}

template <Form FORM, typename T>
int launch_loss_gemm(LossArgs &a, int pairs, int dev, cudaStream_t st)
{
    static std::atomic<unsigned long long> done{0};
    cudaError_t e = once_per_device(done, dev, [] { return cudaFuncSetAttribute(loss_gemm_kernel<FORM, T>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kGemmSmem<FORM>); });
    if (e == cudaSuccess) e = launch_overlapped_clusters(loss_gemm_kernel<FORM, T>, 2, dim3((unsigned)(2 * pairs)), dim3(kThreads), kGemmSmem<FORM>, st, a);
    return e == cudaSuccess ? check_launch("loss_gemm_kernel") : fail(HIPGPT_ERR_CUDA, "loss_gemm_kernel: %s", cudaGetErrorString(e));
}

// What both directions share: the rows that take part, the weights as the tensor core takes them, and the workspace.
struct Plan {
    int N, E, V, layout, dev;
    long long x_ld, w_rows, w_cols, w_ld, rows_alloc;
    bool pack_w;
    size_t x_plane, w_plane;
    // places in the workspace
    size_t x_at, xq_at, w_at, ints_at, floats_at, amax_at, end;
    bool with_xq;                                    // room for a second copy of the rows
};

template <typename T>
int plan_call(Plan &p, const void *w, int N, int E, int V, int layout, bool with_w_grad)
{
    constexpr int NP = sizeof(T) == 4 ? 2 : 1;
    p.N = N; p.E = E; p.V = V; p.layout = layout;
    const cudaError_t e = cudaGetDevice(&p.dev);
    if (e != cudaSuccess) return fail(HIPGPT_ERR_CUDA, "cudaGetDevice: %s", cudaGetErrorString(e));
    p.x_ld = round_up(E, 64);                        // (whole lines)
    p.rows_alloc = round_up(N, kTileM);
    p.w_rows = layout == HIPGPT_WEIGHTS_VE ? V : E;
    p.w_cols = layout == HIPGPT_WEIGHTS_VE ? E : V;
    // 16-bit weights are read where they lie if TMA can (rows of whole 16-byte words).  Others are copied once per call.  (Where rows do not begin on lines the products
    // read two lines for each, but a copy gains nothing by that: forward, E = 776 and 1544, V = 20011: 1024 rows 40.5 -> 36.3 and 69 -> 56 us without it, 8192 rows 185 -> 186 and 343 -> 336;
    // gradient, 776 and 1544: 1024 rows 134 -> 129 and 209 -> 198, 4096 and 8192 rows the same.)
    p.pack_w = NP == 2 || p.w_cols % 8 != 0 || (reinterpret_cast<uintptr_t>(w) & 15) != 0;
    p.w_ld = p.pack_w ? round_up(p.w_cols, 64) : p.w_cols;
    p.x_plane = (size_t)p.rows_alloc * p.x_ld;
    p.w_plane = (size_t)p.w_rows * p.w_ld;
    size_t at = 0;
    auto take = [&](size_t bytes) { const size_t r = at; at += padded(bytes); return r; };
    p.with_xq = with_w_grad && NP == 2;
    p.x_at = take(NP * p.x_plane * 2);
    p.xq_at = take(p.with_xq ? NP * p.x_plane * 2 : 0);
    p.w_at = take(p.pack_w ? NP * p.w_plane * 2 : 0);
    p.ints_at = take((2 + 2 * (size_t)p.rows_alloc) * sizeof(int));
    p.floats_at = take((NP == 2 ? 5 : 2) * (size_t)p.rows_alloc * sizeof(float));
    p.amax_at = take((4 + 3 * kAmaxBlocks) * sizeof(float));
    p.end = at;
    return HIPGPT_OK;
}

// Fills what the plan has in the workspace, and of `a` what every form reads
template <typename T>
int pack_call(const Plan &p, uint8_t *ws, LossArgs &a, const T *x, const T *w, const int *targets, const float *lse, const float *g, float *zero_loss, float *zero_lse, void *zero_grad,
              int *zero_ints, int zeros, const PlanArgs &plan, int launches, Cut *cuts, cudaStream_t st, const void **w_base)
{
    int *ints = reinterpret_cast<int *>(ws + p.ints_at);
    float *floats = reinterpret_cast<float *>(ws + p.floats_at), *scales = reinterpret_cast<float *>(ws + p.amax_at), *partial = scales + 4, *row_max = floats + 4 * p.rows_alloc;
    Pack k = {};
    cudaError_t e;
    if constexpr (sizeof(T) == 4) {
        k.amax_blocks = (int)std::min<long long>(kAmaxBlocks, std::max<long long>(((long long)p.V * p.E + 4095) / 4096, ((long long)p.N + 7) / 8));
        e = launch_overlapped(loss_amax_kernel, dim3((unsigned)(launches + 2 * k.amax_blocks)), dim3(kPackThreads), 0, st, (const float *)x, (const float *)w, g, targets, p.N, p.E, p.V, partial, row_max,
                              k.amax_blocks, plan, launches, cuts);
        launches = 0;
        if (e != cudaSuccess) return fail(HIPGPT_ERR_CUDA, "loss_amax_kernel: %s", cudaGetErrorString(e));
    }
    k.partial = partial;
    k.row_max = row_max;
    k.scales = scales;
    k.targets = targets; k.lse = lse; k.g = g;
    k.N = p.N; k.E = p.E; k.V = p.V; k.ld = (int)p.x_ld;
    k.targets_vec = (reinterpret_cast<uintptr_t>(targets) & 15) == 0;
    k.per_block = (int)(p.N <= 2048 ? 8 : p.N <= 16384 ? 32 : round_up((p.N + 511) / 512, 32));      // (a block counts the targets before its rows; of 8192, 8 and 32 are alike)
    k.x_blocks = (p.N + k.per_block - 1) / k.per_block;
    k.x_vec = p.E % kPer16<T> == 0 && (reinterpret_cast<uintptr_t>(x) & 15) == 0;
    k.xp = reinterpret_cast<uint16_t *>(ws + p.x_at);
    k.xq = p.with_xq ? reinterpret_cast<uint16_t *>(ws + p.xq_at) : nullptr;
    k.plane = p.x_plane;
    k.count = ints; k.failed = ints + 1; k.row_map = ints + 2; k.c_targets = ints + 2 + p.rows_alloc;
    k.c_lse = floats; k.c_g = floats + p.rows_alloc; k.c_x_inv = floats + 2 * p.rows_alloc; k.c_unit = floats + 3 * p.rows_alloc;       // (the last two in fp32 only)
    k.zero_loss = zero_loss; k.zero_lse = zero_lse; k.zero_grad = static_cast<uint8_t *>(zero_grad);
    k.zero_ints = zero_ints; k.zeros = zeros;
    long long w_blocks = 0;
    if (p.pack_w) {
        k.wp = reinterpret_cast<uint16_t *>(ws + p.w_at);
        k.w_plane = p.w_plane;
        k.w_rows = (int)p.w_rows; k.w_cols = (int)p.w_cols; k.w_ld = (int)p.w_ld;
        k.w_col_pieces = (int)((p.w_ld + kPackCols - 1) / kPackCols);
        k.w_vec = p.w_cols % kPer16<T> == 0 && (reinterpret_cast<uintptr_t>(w) & 15) == 0;
        w_blocks = (p.w_rows * k.w_col_pieces + 7) / 8;
    }
    *w_base = p.pack_w ? static_cast<const void *>(ws + p.w_at) : w;
    if (launches + k.x_blocks + w_blocks > 2147483647LL) return fail(HIPGPT_ERR_UNSUPPORTED, "weights of %lld rows of %lld values are beyond one call", p.w_rows, p.w_cols);
    e = launch_overlapped(loss_pack_kernel<T>, dim3((unsigned)(launches + k.x_blocks + w_blocks)), dim3(kPackThreads), 0, st, x, w, k, plan, launches, cuts);
    if (e != cudaSuccess) return fail(HIPGPT_ERR_CUDA, "loss_pack_kernel: %s", cudaGetErrorString(e));
    a.count = k.count; a.failed = k.failed; a.row_map = k.row_map; a.targets = k.c_targets;
    a.lse = k.c_lse; a.g = k.c_g; a.x_inv = k.c_x_inv; a.row_unit = k.c_unit; a.scales = scales;
    a.rows_alloc = (size_t)p.rows_alloc;
    a.V = p.V;
    return check_launch("loss_pack_kernel");
}

// Maps of the operands of one problem, in boxes of 64 x 64; A contiguous along the reduction: of 64 x 128 rows
template <typename T>
int x_map(CUtensorMap *m, const Plan &p, const uint8_t *ws, int box, bool second = false)
{
    return operand_map(m, ws + (second ? p.xq_at : p.x_at), sizeof(T) == 4, p.E, p.rows_alloc, p.x_ld, p.x_plane, sizeof(T) == 4 ? 2 : 1, box);
}
template <typename T>
int w_map(CUtensorMap *m, const Plan &p, const void *w)
{
    return operand_map(m, w, sizeof(T) == 4, p.w_cols, p.w_rows, p.w_ld, p.w_plane, sizeof(T) == 4 ? 2 : 1, 64);
}

template <typename T>
int forward(const void *xv, const void *wv, const int *targets, float *loss, float *lse, int N, int E, int V, int layout, cudaStream_t st)
{
    const T *x = static_cast<const T *>(xv), *w = static_cast<const T *>(wv);
    Plan p;
    int rc = plan_call<T>(p, w, N, E, V, layout, false);
    if (rc != HIPGPT_OK) return rc;
    const int n_tiles = (int)((V + kTileN - 1) / kTileN), m_tiles = (int)(p.rows_alloc / kTileM);
    if ((long long)m_tiles * n_tiles > 1LL << 30) return fail(HIPGPT_ERR_UNSUPPORTED, "N=%d V=%d is beyond one call", N, V);
    const size_t part_at = p.end, zt_at = part_at + padded((size_t)n_tiles * p.rows_alloc * sizeof(float2));
    StreamWorkspace::Lease lease;
    rc = g_loss_ws.enter(st, zt_at + padded((size_t)p.rows_alloc * sizeof(float)), &lease);
    if (rc != HIPGPT_OK) return rc;
    uint8_t *ws = lease.get();
    LossArgs a = {};
    const void *wb = nullptr;
    const bool ev = layout == HIPGPT_WEIGHTS_EV;
    int pairs = 1;
    rc = loss_pairs(p.dev, (long long)m_tiles * n_tiles, &pairs);
    if (rc == HIPGPT_OK) rc = pack_call<T>(p, ws, a, x, w, targets, nullptr, nullptr, loss, lse, nullptr, nullptr, 0, PlanArgs(), 0, nullptr, st, &wb);
    if (rc == HIPGPT_OK) rc = x_map<T>(&a.a[kDz], p, ws, kHalfM);
    if (rc == HIPGPT_OK) rc = w_map<T>(&a.b[kDz], p, wb);
    if (rc != HIPGPT_OK) return rc;
    Problem &q = a.p[kDz];
    q.n_tiles = n_tiles;
    q.stages = (E + kDeep - 1) / kDeep;
    q.b_across = ev;
    a.part = reinterpret_cast<float2 *>(ws + part_at);
    a.z_target = reinterpret_cast<float *>(ws + zt_at);
    a.expire = take_expiry(700);
    rc = launch_loss_gemm<kForward, T>(a, pairs, p.dev, st);
    if (rc != HIPGPT_OK) return rc;
    const cudaError_t e = launch_overlapped(loss_join_kernel, dim3((unsigned)std::min<long long>((N + 31) / 32, 148 * 8)), dim3(256), 0, st, (const float2 *)a.part, n_tiles, a.rows_alloc,
                                            (const float *)a.z_target, a.row_map, a.count, (const int *)a.failed, loss, lse);
    return e == cudaSuccess ? check_launch("loss_join_kernel") : fail(HIPGPT_ERR_CUDA, "loss_join_kernel: %s", cudaGetErrorString(e));
}

template <typename T>
int backward(const void *xv, const void *wv, const int *targets, const float *lse, const float *grad_loss, void *grad_x, void *grad_w, int accumulate_w, int N, int E, int V, int layout,
             cudaStream_t st)
{
    constexpr int NP = sizeof(T) == 4 ? 2 : 1;
    const T *x = static_cast<const T *>(xv), *w = static_cast<const T *>(wv);
    Plan p;
    int rc = plan_call<T>(p, w, N, E, V, layout, grad_w != nullptr);
    if (rc != HIPGPT_OK) return rc;
    // pieces of the vocabulary of like size
    const long long most = std::max<long long>(1024, (long long)(kPieceBytes / ((size_t)p.rows_alloc * 2 * NP)) / kTileN * kTileN);
    const long long width = round_up((V + (V + most - 1) / most - 1) / ((V + most - 1) / most), kTileN);
    const int pieces = (int)((V + width - 1) / width);
    const bool ev = layout == HIPGPT_WEIGHTS_EV;
    const int e_tiles = (E + kTileN - 1) / kTileN, m_tiles = (int)(p.rows_alloc / kTileM), piece_tiles = (int)(width / kTileN);
    const long long dx_tiles = grad_x ? (long long)m_tiles * e_tiles : 0, dw_tiles = grad_w ? (long long)piece_tiles * e_tiles : 0;
    if (dx_tiles + dw_tiles > 1 << 25 || (long long)m_tiles * piece_tiles > 1 << 30) return fail(HIPGPT_ERR_UNSUPPORTED, "N=%d E=%d V=%d is beyond one call", N, E, V);
    int pairs = 1;
    rc = loss_pairs(p.dev, 1 << 30, &pairs);
    if (rc != HIPGPT_OK) return rc;

    const size_t tile_bytes = (size_t)kTileM * kTileN * sizeof(float), dz_plane = (size_t)p.rows_alloc * width, dz_bytes = padded(NP * dz_plane * 2);
    const size_t dz_at = p.end, shares_at = dz_at + (pieces > 1 ? 2 : 1) * dz_bytes, sum_at = shares_at + (NP == 1 ? 3 : 2) * pairs * tile_bytes, arrived_at = sum_at + (pieces > 1 ? dx_tiles * tile_bytes : 0);
    const int arrived = (int)(dx_tiles + dw_tiles) * 2 * kEpiWarps;
    const size_t cuts_at = arrived_at + padded((size_t)arrived * sizeof(int));
    StreamWorkspace::Lease lease;
    rc = g_loss_ws.enter(st, cuts_at + padded((size_t)(pieces + 1) * sizeof(Cut)), &lease);
    if (rc != HIPGPT_OK) return rc;
    uint8_t *ws = lease.get();
    LossArgs a = {};
    const void *wb = nullptr;
    a.arrived = reinterpret_cast<int *>(ws + arrived_at);
    Cut *cuts = reinterpret_cast<Cut *>(ws + cuts_at);
    const PlanArgs plan = {pieces, (int)width, V, E, pairs, (E + kDeep - 1) / kDeep, kDzExtra<NP>, ev, grad_x != nullptr, grad_w != nullptr, targets, grad_loss, N,
                           NP == 1 ? reinterpret_cast<float *>(ws + p.amax_at) + 2 : nullptr};
    rc = pack_call<T>(p, ws, a, x, w, targets, lse, grad_loss, nullptr, nullptr, grad_x, a.arrived, arrived, plan, pieces + 1, cuts, st, &wb);
    if (rc != HIPGPT_OK) return rc;
    a.shares = reinterpret_cast<float4 *>(ws + shares_at);
    a.sum = reinterpret_cast<float4 *>(ws + sum_at);
    a.expire = take_expiry(700);
    // z[n][v]; dx[n][e] = sum_v dz[n][v] w[v][e]; dW[v][e] = sum_n dz[n][v] x[n][e], or dW[e][v]
    auto dz_map = [&](CUtensorMap *m, int piece, int box, int inner = 64) {
        return operand_map(m, ws + dz_at + (piece & 1) * dz_bytes, NP == 2, width, p.rows_alloc, width, dz_plane, NP, box, inner);
    };
    rc = x_map<T>(&a.a[kDz], p, ws, kHalfM);
    if (rc == HIPGPT_OK) rc = w_map<T>(&a.b[kDz], p, wb);
    if (rc == HIPGPT_OK) rc = w_map<T>(&a.b[kDx], p, wb);
    if (rc == HIPGPT_OK) rc = x_map<T>(ev ? &a.a[kDw] : &a.b[kDw], p, ws, 64);
    if (rc == HIPGPT_OK && p.with_xq) rc = x_map<T>(&a.xq, p, ws, 64, true);
    a.x_is_a = ev;
    if (rc != HIPGPT_OK) return rc;
    a.p[kDz].stages = (E + kDeep - 1) / kDeep;
    a.p[kDz].b_across = ev;
    a.p[kDx].b_across = !ev;
    a.p[kDx].out = grad_x;
    a.p[kDx].ld = a.p[kDx].cols = E;
    a.p[kDw].a_across = a.p[kDw].b_across = 1;
    a.p[kDw].accumulate = accumulate_w;
    a.p[kDw].ld = ev ? V : E;
    for (int i = 0; i <= pieces; ++i) {              // the logits' gradient of piece i, the products with that of piece i - 1
        Problem &z = a.p[kDz], &dx = a.p[kDx], &dw = a.p[kDw];
        const long long v0 = i * width, here = std::min<long long>(width, V - v0);
        a.cut = cuts + i;
        z.n_tiles = i < pieces ? (int)((here + kTileN - 1) / kTileN) : 0;
        if (z.n_tiles) {
            a.v0 = z.b_n0 = (int)v0;
            rc = dz_map(&a.dz_out, i, 32, 32);
        }
        if (i > 0) {
            const long long o0 = v0 - width, old = std::min<long long>(width, V - o0);
            a.first = i == 1;
            a.last = i == pieces;
            if (grad_x) {
                dx.b_k0 = (int)o0;
                if (rc == HIPGPT_OK) rc = dz_map(&a.a[kDx], i - 1, kHalfM);
            }
            if (grad_w) {
                dw.rows = ev ? E : (int)old;
                dw.cols = ev ? (int)old : E;
                dw.out = static_cast<T *>(grad_w) + (ev ? o0 : o0 * E);
                if (rc == HIPGPT_OK) rc = dz_map(ev ? &a.b[kDw] : &a.a[kDw], i - 1, kDeep);
            }
        }
        if (rc == HIPGPT_OK) rc = launch_loss_gemm<kBackward, T>(a, pairs, p.dev, st);
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
    const size_t ts = type == HIPGPT_TYPE_F32 ? 4 : 2, rows = (size_t)N * 4;
    const int clear = refuse_overlaps(2, {{d_loss, rows}, {d_lse, rows}, {d_x, (size_t)N * E * ts}, {d_w, (size_t)V * E * ts}, {d_targets, rows}});
    if (clear != HIPGPT_OK) return clear;
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
    const size_t ts = type == HIPGPT_TYPE_F32 ? 4 : 2, rows = (size_t)N * 4, xb = (size_t)N * E * ts, wb = (size_t)V * E * ts;
    const int clear = refuse_overlaps(2, {{d_grad_x, xb}, {d_grad_w, wb}, {d_x, xb}, {d_w, wb}, {d_targets, rows}, {d_lse, rows}, {d_grad_loss, rows}});
    if (clear != HIPGPT_OK) return clear;
    return type == HIPGPT_TYPE_F32
               ? backward<float>(d_x, d_w, d_targets, d_lse, d_grad_loss, d_grad_x, d_grad_w, accumulate_w, N, E, V, layout, st)
               : backward<__nv_bfloat16>(d_x, d_w, d_targets, d_lse, d_grad_loss, d_grad_x, d_grad_w, accumulate_w, N, E, V, layout, st);
}

}  // extern "C"
