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
    float scale, cscale;                 // and scale * log2 e
    int least;                           // units a block takes at least
    float *parts;                        // [2 * blocks][ROWS][DP + 2]: sums, then reference maximum (log2 domain) and sum of exponentials of each row
    int4 *cuts;                          // [blocks]: the tile that begins here and goes on: sequence, head, tile, last block (w < 0: none)
    int *whole;                          // [blocks]: 0 where a wait ran out
    uint8_t *cut_k, *cut_v;              // [sequence][head][cut_units] places of the ring: fp32 cut into pieces before the attention
    int cut_units, cut_unit;             // keys a place (0: keys as they lie in the cache)
};

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
        per = max(per, (long long)a.least);
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
    // Noted by the block that has the first unit of a tile that goes on
    __device__ __forceinline__ int4 cut() const { return make_int4(b, head, tile, (int)((base + units - 1) / per)); }
};

// ---- rows worked out key by key ----------------------------------------------------------------------------------------
// A product over a tile of keys takes every row's probabilities times every key's values, zero times what a row must not see.  Where that is an infinity or NaN the
// sum is NaN.  Such a row is found by its result, and is worked out again without the keys that it does not see.

// One value of a row of the cache
template <typename T, int FMT>
__device__ __forceinline__ float cached(const uint8_t *base, const float *scale, long long row, int D, int d)
{
    if constexpr (FMT == HIPGPT_CACHE_PLAIN) {
        return to_float(reinterpret_cast<const T *>(base)[row * D + d]);
    } else {
        uint32_t lo, hi;
        codes_to_half<FMT>(base[row * D + d], lo, hi);
        return floats_of(lo).x * scale[row];
    }
}

template <typename T, int FMT>
__device__ __forceinline__ bool any_wild(const AttnArgs &a, int b, int head, int from, int to)
{
    const int lane = threadIdx.x & 31;
    bool wild = false;
    for (int p = from; p < to && !wild; ++p) {
        const long long row = row_of(a.c, b, head, p);
        bool w = false;
        if (row >= 0)
            for (int d = lane; d < a.c.D; d += 32) w = w || !(fabsf(cached<T, FMT>(a.c.v, a.c.vs, row, a.c.D, d)) <= 3.402823466e38f);
        wild = __any_sync(0xffffffffu, w);
    }
    return wild;
}

// One warp: values c0 .. c1 of row `row` of (sequence b, head of the cache)
template <typename T, int FMT>
__device__ __noinline__ void row_again(const AttnArgs &a, int b, int head, const Sequence &s, int row, int c0, int c1)
{
    const int lane = threadIdx.x & 31, D = a.c.D, limit = limit_of(a, s, row);
    const long long t = s.first + row / a.group;
    const int h = head * a.group + row % a.group;
    const T *q = static_cast<const T *>(a.q) + t * a.q_stride + (long long)h * D;
    float qv[4], o[4], m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        qv[i] = lane + 32 * i < D ? to_float(q[lane + 32 * i]) : 0.0f;
        o[i] = 0.0f;
    }
    for (int p = 0; p < limit; ++p) {
        const long long r = row_of(a.c, b, head, p);
        if (r < 0) continue;
        float z = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i) if (lane + 32 * i < D) z = fmaf(qv[i], cached<T, FMT>(a.c.k, a.c.ks, r, D, lane + 32 * i), z);
#pragma unroll
        for (int off = 16; off; off >>= 1) z += __shfl_xor_sync(0xffffffffu, z, off);
        z *= a.cscale;
        const float mn = fmaxf(m, z), base = mn == -INFINITY ? 0.0f : mn;
        const float alpha = exp2f(m - base), e = exp2f(z - base);
        m = mn;
        l = fmaf(l, alpha, e);
#pragma unroll
        for (int i = 0; i < 4; ++i) if (lane + 32 * i < D) o[i] = fmaf(e, cached<T, FMT>(a.c.v, a.c.vs, r, D, lane + 32 * i), o[i] * alpha);
        // NaN stays NaN: where all are, the rest of a long sequence need not be gone through
        bool number = false;
#pragma unroll
        for (int i = 0; i < 4; ++i) number = number || (lane + 32 * i < D && o[i] == o[i]);
        if (l != l || !__any_sync(0xffffffffu, number)) break;
    }
    T *out = static_cast<T *>(a.out) + t * a.out_stride + (long long)h * D;
#pragma unroll
    for (int i = 0; i < 4; ++i) if (lane + 32 * i >= c0 && lane + 32 * i < min(c1, D)) out[lane + 32 * i] = from_float<T>(l == 0.0f ? 0.0f : o[i] / l);
}

// Whether a row whose result is not finite was touched by keys that it does not see (its tile's keys go up to `keys`)
template <typename T, int FMT>
__device__ __forceinline__ void mend_row(const AttnArgs &a, int b, int head, const Sequence &s, int row, int keys, int c0 = 0, int c1 = 128)
{
    const int limit = limit_of(a, s, row);
    if (limit < keys && any_wild<T, FMT>(a, b, head, limit, keys)) row_again<T, FMT>(a, b, head, s, row, c0, c1);
}

// The keys that a tile's rows have been multiplied with: those they see, and where these were cut before, to the end of the last place
__device__ __forceinline__ int keys_met(const AttnArgs &a, const Sequence &s, int keys) { return a.cut_unit ? (int)min((long long)s.len, ((long long)keys + a.cut_unit - 1) / a.cut_unit * a.cut_unit) : keys; }

// ---- joining the parts ----------------------------------------------------------------------------------------------------
// One block a block of the kernel before it: the tile that began there, if it went on.  A warp takes a row; parts in ascending order.
template <typename T, int FMT, int ROWS, int DP>
__global__ void __launch_bounds__(256)
paged_join_kernel(const AttnArgs a)
{
    dependency_wait();
    dependents_may_start();
    const int4 cut = a.cuts[blockIdx.x];
    if (cut.w < 0) return;
    for (int blk = blockIdx.x; blk <= cut.w; ++blk) if (!a.whole[blk]) return;
    const Sequence s = sequence_of(a.c, cut.x);
    const int lane = threadIdx.x & 31, D = a.c.D;
    constexpr int E = DP / 32;
    const long long rows = (long long)s.n * a.group;
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
        bool wild = false;
#pragma unroll
        for (int i = 0; i < E; ++i) {
            const float y = l == 0.0f ? 0.0f : o[i] * inv;
            wild = wild || !(fabsf(y) <= 3.402823466e38f);
            if (lane + 32 * i < D) out[lane + 32 * i] = from_float<T>(y);
        }
        if (__any_sync(0xffffffffu, wild)) {
            __syncwarp();
            mend_row<T, FMT>(a, cut.x, cut.y, s, (int)row, keys_met(a, s, tile_keys<ROWS>(a, s, cut.z)));
        }
    }
}

int launch_paged_tc(int format, const AttnArgs &a, cudaStream_t st);

}  // namespace hipgpt
