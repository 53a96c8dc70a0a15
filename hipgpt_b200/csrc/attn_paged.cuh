// What the kernels of attention over a paged cache share: the cut of a ragged batch's work over the blocks of a grid, the parts that blocks leave where a cut goes
// through a row tile, and rows that are worked out again key by key.
//
// A row is one query (token and head); the rows of a sequence that share a head of the cache are numbered token * group + head in the group, and ROWS of them make a
// tile.  A tile's work is its keys in units of UNIT.  All units of all tiles, in order, are dealt to the blocks in equal runs, so a block has at most two tiles
// of which others have parts: the one that began before its run (its part is left in place 2 * block) and the one that goes on behind it (2 * block + 1).
// The block that has a tile's first unit notes it for the kernel that joins the parts.
#pragma once

#include "paged.cuh"

namespace hipgpt {

struct AttnArgs {
    PagedView c;
    const void *q;
    void *out;
    long long q_stride, out_stride;
    int group, causal;
    float cscale;                        // scale * log2 e
    int expire;                          // test hook (attn_paged.cu's kernels)
    float *parts;                        // [2 * blocks][ROWS][DP + 2]: sums, then reference maximum (log2 domain) and sum of exponentials of each row
    int4 *cuts;                          // [blocks]: the tile that begins here and goes on: sequence, head, tile, last block (w < 0: none)
    int *whole;                          // [blocks]: 0 where a wait ran out
    uint8_t *cut_k, *cut_v;              // [sequence][head][cut_units] places of the ring: fp32 cut into pieces before the attention
    int cut_units, cut_unit;             // keys a place (0: keys as they lie in the cache)
};

// The power of two that brings the largest value of a row of q to [2^14, 2^15) (2^126 at most); 1 for zeros, infinities and NaN
__device__ __forceinline__ float row_unit(float most) { return most <= 3.0e38f ? pow2_scale(most) : most <= 3.402823466e38f ? 0x1p-113f : 1.0f; }

// One tile's run of units in a block
struct Tile {
    int b, head, tile, units;            // units of the whole tile
    int from, to;                        // this block's
    Sequence s;
};

// Keys that a row sees: positions below this (the row's own included); 0 for rows behind the last
__device__ __forceinline__ int limit_of(const AttnArgs &a, const Sequence &s, int row)
{
    const int t = row / a.group;
    if (t >= s.n) return 0;
    return a.causal ? max(s.len - s.n + t + 1, 0) : s.len;
}
template <int ROWS>
__device__ __forceinline__ int tiles_of(const AttnArgs &a, const Sequence &s) { return (int)(((long long)s.n * a.group + ROWS - 1) / ROWS); }
// Keys that the tile's rows see
template <int ROWS>
__device__ __forceinline__ int tile_keys(const AttnArgs &a, const Sequence &s, int tile)
{
    const long long last = min((long long)(tile + 1) * ROWS, (long long)s.n * a.group) - 1;
    return limit_of(a, s, (int)last);
}
// A tile without keys has one unit all the same: its rows get zeros
template <int ROWS, int UNIT>
__device__ __forceinline__ int tile_units(const AttnArgs &a, const Sequence &s, int tile) { return max(1, (tile_keys<ROWS>(a, s, tile) + UNIT - 1) / UNIT); }

template <int THREADS>
__device__ __forceinline__ long long block_sum(long long v, long long *shared)
{
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = v;
    __syncthreads();
    long long sum = 0;
#pragma unroll
    for (int w = 0; w < THREADS / 32; ++w) sum += shared[w];
    return sum;
}

// The block's run through the batch: begin(), then next() until it says no.  All threads of the block call it together.
template <int ROWS, int UNIT, int THREADS>
struct Run {
    const AttnArgs &a;
    long long u, end;                    // units still to come: [u, end)
    long long start;                     // the run's first
    long long per;                       // units a block
    int b, tile, head;
    long long base;                      // the first unit of (b, tile, head)
    Sequence s;
    int units;

    // units of one head of the sequences b0 ...: of one in each thread, or, where there are no more sequences than warps, of one in the first lane of each warp (its lanes
    // share the tiles); `i`: which sequence
    __device__ __forceinline__ long long count(int b0, int &i) const
    {
        const bool few = a.c.B <= THREADS / 32;
        const int lane = threadIdx.x & 31;
        i = few ? (int)(threadIdx.x >> 5) : b0 + (int)threadIdx.x;
        long long n = 0;
        if (i < a.c.B) {
            const Sequence q = sequence_of(a.c, i);
            const int tiles = tiles_of<ROWS>(a, q);
            for (int t = few ? lane : 0; t < tiles; t += few ? 32 : 1) n += tile_units<ROWS, UNIT>(a, q, t);
        }
        if (few) {
#pragma unroll
            for (int o = 16; o; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
            if (lane) n = 0;
        }
        return n * a.c.heads;
    }

    __device__ __forceinline__ explicit Run(const AttnArgs &args) : a(args) {}

    __device__ __forceinline__ bool begin(long long *shared)
    {
        const int tid = threadIdx.x, lane = tid & 31;
        // all units
        int i = 0;
        long long n = count(0, i), mine = n;
        for (int b0 = THREADS; b0 < a.c.B; b0 += THREADS) { int x; mine += count(b0, x); }
        const long long total = block_sum<THREADS>(mine, shared);
        // (64-bit divisions take a hundred instructions)
        per = total < 1 << 30 ? (int)(((unsigned)total + gridDim.x - 1) / gridDim.x) : (total + gridDim.x - 1) / gridDim.x;
        per = max(per, 1LL);
        u = start = (long long)blockIdx.x * per;
        end = min(total, u + per);
        if (u >= end) return false;
        // the sequence that holds the first
        long long before = 0;
        for (int b0 = 0;; b0 += THREADS) {
            if (b0) n = count(b0, i);
            // running sums over the block
            long long upto = n;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const long long x = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= o) upto += x;
            }
            __syncthreads();
            if (lane == 31) shared[tid >> 5] = upto;
            if (tid == 0) shared[THREADS / 32 + 1] = -1;
            __syncthreads();
            long long chunk = 0;
            for (int w = 0; w < THREADS / 32; ++w) {
                if (w < tid >> 5) upto += shared[w];
                chunk += shared[w];
            }
            if (u >= before + upto - n && u < before + upto) {
                shared[THREADS / 32] = before + upto - n;
                shared[THREADS / 32 + 1] = i;
            }
            __syncthreads();
            b = (int)shared[THREADS / 32 + 1];
            if (b >= 0) { base = shared[THREADS / 32]; break; }
            before += chunk;
            if (b0 + THREADS >= a.c.B) return false;                  // (not reached: u < total)
        }
        s = sequence_of(a.c, b);
        // tile after tile, all heads of one before the next; 32 tiles at a time
        const int tiles = tiles_of<ROWS>(a, s);
        for (tile = 0;; tile += 32) {
            const int mine_units = tile + lane < tiles ? tile_units<ROWS, UNIT>(a, s, tile + lane) : 0;
            long long upto = (long long)mine_units * a.c.heads;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const long long x = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= o) upto += x;
            }
            const unsigned behind = __ballot_sync(0xffffffffu, u < base + upto);
            if (behind) {
                const int at = __ffs((int)behind) - 1;
                units = __shfl_sync(0xffffffffu, mine_units, at);
                base += __shfl_sync(0xffffffffu, upto, at) - (long long)units * a.c.heads;
                tile += at;
                break;
            }
            base += __shfl_sync(0xffffffffu, upto, 31);
        }
        head = u - base < 1 << 30 ? (int)((unsigned)(u - base) / (unsigned)units) : (int)((u - base) / units);
        base += (long long)head * units;
        return true;
    }

    // The tile at hand
    __device__ __forceinline__ Tile at() const
    {
        return {b, head, tile, units, (int)(u - base), (int)(min(end, base + units) - base), s};
    }
    // The next one; false when the run is at its end
    __device__ __forceinline__ bool next()
    {
        u = base + units;
        if (u >= end) return false;
        base = u;
        if (++head < a.c.heads) return true;
        head = 0;
        if (++tile >= tiles_of<ROWS>(a, s)) {
            do { s = sequence_of(a.c, ++b); } while (s.n == 0 && b + 1 < a.c.B);
            tile = 0;
        }
        units = tile_units<ROWS, UNIT>(a, s, tile);
        return true;
    }
    // Where the part of the tile at hand goes: -1: it is whole here
    __device__ __forceinline__ int part() const
    {
        if (base >= start && base + units <= end) return -1;
        return 2 * (int)blockIdx.x + (base >= start ? 1 : 0);
    }
    // The run once more: thread 0 keeps in shared memory where it began (behind begin())
    struct Start { long long start, end, per, base; int b, tile, head, units; };
    __device__ __forceinline__ void keep(Start *to) const { if (threadIdx.x == 0) *to = {start, end, per, base, b, tile, head, units}; }
    __device__ __forceinline__ Run(const AttnArgs &args, const Start &from)
        : a(args), u(from.start), end(from.end), start(from.start), per(from.per), b(from.b), tile(from.tile), head(from.head), base(from.base), s(sequence_of(args.c, from.b)), units(from.units) {}
    // Noted by the block that has the first unit of a tile that goes on
    __device__ __forceinline__ int4 cut() const { return make_int4(b, head, tile, (int)((base + units - 1) / per)); }
};

// ---- rows worked out again ---------------------------------------------------------------------------------------------
// A product over a tile of keys takes every row's probabilities times every key's values, zero times what a row must not see.  Where that is an infinity or NaN the
// sum is NaN.  Sums over the keys are divided by the probabilities' sum at their end, so they also pass fp32's range where the values come near its largest number.  Such a row is found by its result, and is
// worked out again over the keys that it sees: when the block's whole run is done and nobody in it waits for anything any more (a long row
// takes longer than a wait may), or where parts are joined.

// Sixteen values in a row of the cache, of codes without their scale
template <typename T, int FMT>
__device__ __forceinline__ void cached16(const uint8_t *base, long long row, int D, int d, float (&x)[16])
{
    if constexpr (FMT == HIPGPT_CACHE_PLAIN) {
        constexpr int W = kPer16<T>;
#pragma unroll
        for (int i = 0; i < 16 / W; ++i) {
            float y[W];
            load_values<T, W>(reinterpret_cast<const T *>(base) + row * D + d + i * W, y);
#pragma unroll
            for (int e = 0; e < W; ++e) x[i * W + e] = y[e];
        }
    } else {
        const uint4 c = *reinterpret_cast<const uint4 *>(base + row * D + d);
        const uint32_t w[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint32_t lo, hi;
            codes_to_half<FMT>(w[i], lo, hi);
            const float2 p = floats_of(lo), q = floats_of(hi);
            x[4 * i] = p.x; x[4 * i + 1] = p.y; x[4 * i + 2] = q.x; x[4 * i + 3] = q.y;
        }
    }
}

__device__ __forceinline__ bool finite(float x) { return fabsf(x) <= 3.402823466e38f; }

// The last position of [from, to) with a value that is not finite, -1: none.  A lane a position, 32 after 32 of them for each of the block's warps.
template <typename T, int FMT>
__device__ __forceinline__ int last_wild(const AttnArgs &a, int b, int head, int from, int to, int warp, int warps)
{
    int top = -1;
    for (int p0 = from + 32 * warp; p0 < to; p0 += 32 * warps) {
        const int p = p0 + (threadIdx.x & 31);
        const long long row = p < to ? row_of(a.c, b, head, p) : -1;
        bool wild = false;
        if (row >= 0) {
            const float unit = FMT == HIPGPT_CACHE_PLAIN ? 1.0f : a.c.vs[row];
#pragma unroll 4
            for (int d = 0; d < a.c.D; d += 16) {
                float x[16];
                cached16<T, FMT>(a.c.v, row, a.c.D, d, x);
#pragma unroll
                for (int e = 0; e < 16; ++e) wild = wild || !finite(x[e] * unit);
            }
        }
        const unsigned who = __ballot_sync(0xffffffffu, wild);
        if (who) top = p0 + 31 - __clz((int)who);
    }
    return top;
}

// Four values from column `d` on in a row of the cache, of codes without their scale
template <typename T, int FMT>
__device__ __forceinline__ float4 cached4(const uint8_t *base, long long row, int D, int d)
{
    if constexpr (FMT != HIPGPT_CACHE_PLAIN) {
        uint32_t lo, hi;
        codes_to_half<FMT>(*reinterpret_cast<const uint32_t *>(base + row * D + d), lo, hi);
        const float2 p = floats_of(lo), q = floats_of(hi);
        return make_float4(p.x, p.y, q.x, q.y);
    } else {
        float x[4];
        load_values<T, 4>(reinterpret_cast<const T *>(base) + row * D + d, x);
        return make_float4(x[0], x[1], x[2], x[3]);
    }
}

// One warp: values c0 .. c1 of one or two rows (-1: none) of (sequence b, head of the cache), 32 keys at a time: a lane a key for the scores, a lane four values for the sums over the keys, which are added up
// 32 by 32 and kept as half of their average so far: nothing passes fp32's range that does not end outside it.  What is fetched serves both rows, and four keys' values are on their way at once.
// (More of either takes registers that the kernels which call it then do not have: fp32 prompts 78 -> 90 us.)
template <typename T, int FMT>
__device__ __noinline__ void rows_again(const AttnArgs &a, int b, int head, int2 which, int c0, int c1)
{
    constexpr bool CODED = FMT != HIPGPT_CACHE_PLAIN;
    constexpr int N = 2, kAhead = 4;
    const int lane = threadIdx.x & 31, D = a.c.D, d0 = 4 * lane, row[N] = {which.x, which.y};
    const Sequence s = sequence_of(a.c, b);
    int limit[N], most = 0;
    float q[N][4], o[N][4], factor[N], m[N], l[N];
    auto place = [&](int n, long long stride) { return (s.first + row[n] / a.group) * stride + (long long)(head * a.group + row[n] % a.group) * D + d0; };
#pragma unroll
    for (int n = 0; n < N; ++n) {
        limit[n] = row[n] >= 0 ? limit_of(a, s, row[n]) : 0;
        most = max(most, limit[n]);
        float largest = 0.0f;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            q[n][e] = row[n] >= 0 && d0 < D ? to_float((static_cast<const T *>(a.q) + place(n, a.q_stride))[e]) : 0.0f;
            largest = fmaxf(largest, fabsf(q[n][e]));
            o[n][e] = 0.0f;
        }
        factor[n] = a.cscale;
        if constexpr (CODED) {                       // (as in the kernels: small queries and large scales, or the other way round)
#pragma unroll
            for (int off = 16; off; off >>= 1) largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, off));
            const float unit = row_unit(largest);
            factor[n] *= pow2_inverse(unit);
#pragma unroll
            for (int e = 0; e < 4; ++e) q[n][e] *= unit;
        }
        m[n] = -INFINITY;
        l[n] = 0.0f;
    }
    for (int p0 = 0; p0 < most; p0 += 32) {
        const int p = p0 + lane;
        const long long mine = p < most ? row_of(a.c, b, head, p) : -1;
        const unsigned there = __ballot_sync(0xffffffffu, mine >= 0);
        if (!there) continue;
        // (a lane without a key reads another's: loads without conditions go out together)
        const long long other = __shfl_sync(0xffffffffu, mine, __ffs((int)there) - 1), r = mine >= 0 ? mine : other;
        float z[N] = {0.0f, 0.0f};
#pragma unroll 4
        for (int c = 0; c < D; c += 16) {
            float k[16];
            cached16<T, FMT>(a.c.k, r, D, c, k);
#pragma unroll
            for (int n = 0; n < N; ++n) {
                float sum = 0.0f;
#pragma unroll
                for (int e = 0; e < 16; ++e) sum = fmaf(__shfl_sync(0xffffffffu, q[n][e & 3], c / 4 + (e >> 2)), k[e], sum);
                z[n] += sum;
            }
        }
        float unit = 1.0f, weight = 0.5f;
        if constexpr (CODED) {
            unit = a.c.ks[r];
            weight *= a.c.vs[r];
        }
        unsigned seen[N];
        float f[N], keep[N];
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const bool sees = mine >= 0 && p < limit[n];
            seen[n] = __ballot_sync(0xffffffffu, sees);
            const float score = sees ? z[n] * (unit * factor[n]) : -INFINITY;
            float top = score;
#pragma unroll
            for (int off = 16; off; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
            const float now = fmaxf(m[n], top), base = now == -INFINITY ? 0.0f : now;
            const float e = exp2f(score - base), before = l[n] * exp2f(m[n] - base);
            m[n] = now;
            float sum = e;
#pragma unroll
            for (int off = 16; off; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
            l[n] = before + sum;
            const float inv = l[n] == 0.0f ? 0.0f : 1.0f / l[n];
            keep[n] = before * inv;
            f[n] = e * inv * weight;                 // (of the keys that the row sees)
        }
        float x[N][4] = {};
#pragma unroll 1
        for (int j0 = 0; j0 < 32; j0 += kAhead) {
            float4 v[kAhead];
#pragma unroll
            for (int j = 0; j < kAhead; ++j) v[j] = cached4<T, FMT>(a.c.v, __shfl_sync(0xffffffffu, r, j0 + j), D, min(d0, D - 4));
#pragma unroll
            for (int j = 0; j < kAhead; ++j)
#pragma unroll
                for (int n = 0; n < N; ++n) {
                    const float fj = __shfl_sync(0xffffffffu, f[n], j0 + j);
                    if (seen[n] >> (j0 + j) & 1) {
                        x[n][0] = fmaf(fj, v[j].x, x[n][0]);
                        x[n][1] = fmaf(fj, v[j].y, x[n][1]);
                        x[n][2] = fmaf(fj, v[j].z, x[n][2]);
                        x[n][3] = fmaf(fj, v[j].w, x[n][3]);
                    }
                }
        }
        bool number = false;
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                o[n][e] = fmaf(o[n][e], keep[n], x[n][e]);
                number = number || (row[n] >= 0 && d0 < D && o[n][e] == o[n][e]);
            }
        // NaN stays NaN: where all are, the rest of a long sequence need not be gone through
        if (!__any_sync(0xffffffffu, number)) break;
    }
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            // (an average of finite values that rounding took beyond the largest)
            const float y = l[n] != l[n] ? l[n] : finite(o[n][e]) ? fminf(fmaxf(2.0f * o[n][e], -3.402823466e38f), 3.402823466e38f) : o[n][e];
            if (row[n] >= 0 && d0 + e >= c0 && d0 + e < min(c1, D)) (static_cast<T *>(a.out) + place(n, a.out_stride))[e] = from_float<T>(y);
        }
}

// The keys that a tile's rows have been multiplied with: those they see, and where these were cut before, to the end of the last place
__device__ __forceinline__ int keys_met(const AttnArgs &a, const Sequence &s, int keys) { return a.cut_unit ? (int)min((long long)s.len, ((long long)keys + a.cut_unit - 1) / a.cut_unit * a.cut_unit) : keys; }

// The tile's rows from `first` on, every `step`th, one a warp, that hold something that is not finite in their values c0 .. c1 and were touched by keys that they do not see, or see finite values alone.  The block's
// `warps` warps call it together (meet() is their barrier), with their rows stored.
template <typename T, int FMT, int ROWS, typename Meet>
__device__ __forceinline__ void mend_tile(const AttnArgs &a, int b, int head, int tile, const Sequence &s, int first, int step, int warp, int warps, int *tops, Meet meet, int c0 = 0, int c1 = 128)
{
    const int lane = threadIdx.x & 31, row0 = tile * ROWS;
    const int rows = (int)min((long long)s.n * a.group - row0, (long long)ROWS), keys = keys_met(a, s, tile_keys<ROWS>(a, s, tile)), least = limit_of(a, s, row0);
    auto last = [&](int from, int to) {
        int top = last_wild<T, FMT>(a, b, head, from, to, warp, warps);
        meet();                                      // (everybody's rows are stored, and what was there before has been read)
        if (lane == 0) tops[warp] = top;
        meet();
        for (int w = 0; w < warps; ++w) top = max(top, tops[w]);
        return top;
    };
    const int top = last(least, keys);               // (rows that see it see all of them)
    if (top < 0 && last(0, least) >= 0) return;
    int found = -1;                                  // rows are worked out two at a time
    for (int r = first; r < rows; r += step) {
        const int row = row0 + r;
        if (top >= 0 && limit_of(a, s, row) > top) break;
        const T *out = static_cast<const T *>(a.out) + (long long)(s.first + row / a.group) * a.out_stride + (long long)(head * a.group + row % a.group) * a.c.D;
        bool wild = false;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int d = lane + 32 * i;
            if (d >= c0 && d < min(c1, a.c.D)) wild = wild || !finite(to_float(out[d]));
        }
        if (!__any_sync(0xffffffffu, wild)) continue;
        if (found >= 0) rows_again<T, FMT>(a, b, head, make_int2(found, row), c0, c1);
        found = found >= 0 ? -1 : row;
    }
    if (found >= 0) rows_again<T, FMT>(a, b, head, make_int2(found, -1), c0, c1);
}

// The tiles of a block's run whose number (modulo 32) is in `which`
template <typename T, int FMT, int ROWS, int UNIT, int THREADS, typename Meet>
__device__ __noinline__ void mend_run(const AttnArgs &a, const typename Run<ROWS, UNIT, THREADS>::Start *from, uint32_t which, int warp, int warps, int *tops, Meet meet)
{
    Run<ROWS, UNIT, THREADS> run(a, *from);
    int k = 0;
    do {
        if ((which >> (k & 31) & 1) && run.part() < 0) mend_tile<T, FMT, ROWS>(a, run.b, run.head, run.tile, run.s, warp, warps, warp, warps, tops, meet);
        ++k;
    } while (run.next());
}

// ---- joining the parts ----------------------------------------------------------------------------------------------------
// One block a block of the kernel before it: the tile that began there, if it went on.  A warp takes a row; parts in ascending order.
template <typename T, int FMT, int ROWS, int DP>
__global__ void __launch_bounds__(256)
paged_join_kernel(const __grid_constant__ AttnArgs a)
{
    dependency_wait();
    dependents_may_start();
    const int4 cut = a.cuts[blockIdx.x];
    if (cut.w < 0) return;
    for (int blk = blockIdx.x; blk <= cut.w; ++blk) if (!a.whole[blk]) return;
    __shared__ int tops[8];
    const Sequence s = sequence_of(a.c, cut.x);
    const int lane = threadIdx.x & 31, D = a.c.D;
    constexpr int E = DP / 32;
    const long long rows = (long long)s.n * a.group;
    bool wild = false;
    for (int r = blockIdx.y * 8 + (threadIdx.x >> 5); r < ROWS; r += 8 * gridDim.y) {
        const long long row = (long long)cut.z * ROWS + r;
        if (row >= rows) break;
        float m = -INFINITY, l = 0.0f, o[E];
#pragma unroll
        for (int i = 0; i < E; ++i) o[i] = 0.0f;
        for (int blk = blockIdx.x; blk <= cut.w; ++blk) {
            const float *p = a.parts + ((size_t)(2 * blk + (blk == (int)blockIdx.x)) * ROWS) * (DP + 2);
            const float m2 = p[ROWS * DP + 2 * r], l2 = p[ROWS * DP + 2 * r + 1];
            const float mn = fmaxf(m, m2), base = mn == -INFINITY ? 0.0f : mn;
            const float f1 = ex2_approx(m - base), f2 = ex2_approx(m2 - base);
            m = mn;
            l = fmaf(l, f1, l2 * f2);
#pragma unroll
            for (int i = 0; i < E; ++i) o[i] = fmaf(o[i], f1, p[(size_t)r * DP + lane + 32 * i] * f2);
        }
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        const long long t = s.first + row / a.group;
        T *out = static_cast<T *>(a.out) + t * a.out_stride + (long long)(cut.y * a.group + (int)(row % a.group)) * D;
#pragma unroll
        for (int i = 0; i < E; ++i) {
            const float y = l == 0.0f ? 0.0f : o[i] * inv;
            wild = wild || (!finite(y) && l == l);
            if (lane + 32 * i < D) out[lane + 32 * i] = from_float<T>(y);
        }
    }
    if (__syncthreads_or(wild)) {
        const int warp = threadIdx.x >> 5;
        mend_tile<T, FMT, ROWS>(a, cut.x, cut.y, cut.z, s, blockIdx.y * 8 + warp, 8 * gridDim.y, warp, 8, tops, [] { __syncthreads(); });
    }
}

int launch_paged_tc(int format, const AttnArgs &a, cudaStream_t st);

}  // namespace hipgpt
