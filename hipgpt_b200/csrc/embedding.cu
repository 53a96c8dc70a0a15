// Embedding lookup with a scale, for fp32 and bf16 tables, and its gradient (HipGPT's launch_embedding_lookup and
// embedding_backward_kernel, src/hip_kernels.cpp:537-599 and :1064-1088; the reference adds its gradients with atomics, in any order).
//
//   out[t]      = scale tok[id_t] + pos[t mod S]                       an id outside [0, V) gives a row of zeros
//   grad_tok[v] = scale * sum of g[t] over the t with id_t = v         (+ what it held, when accumulating)
//   grad_pos[s] = sum of g[b S + s] over the b whose id is inside      (likewise)
//
// Both are bound by HBM: rows read once, rows written once.
//
// The gradient sums every row of the table in a fixed order, without atomics on values: the tokens are sorted by id first.
//   sort_ids_kernel   one cluster of up to sixteen blocks sorts (id, t) by id, stable (so equal ids keep ascending t): two passes of
//                     counting sort for vocabularies below 2^20, three from there on; then writes where the entries of each row begin.
//                     Within a pass a block counts its part's digits, the cluster's counts become offsets through
//                     distributed shared memory, and every warp ranks 32 keys at a time among themselves by votes.
//   zero_table_kernel stores zeros, beside the sort.
//   embed_sum_kernel  a group of threads fetches the rows of a piece of the sorted entries into shared memory, adds them up in order and stores each row of the table that
//                     begins and ends in the piece.  Words are not spread evenly (one id may take a tenth of the tokens, padding half of them): pieces are
//                     equal, not rows.  Of a row that falls to several pieces each leaves a sum in fp32, and the group that comes last adds them in
//                     ascending order, whichever group it is.  The positions' table is summed
//                     in the same way over the batch.
#include "elem_types.cuh"
#include "stream_workspace.hpp"

#include <algorithm>

namespace hipgpt {
namespace {

// ---- lookup -----------------------------------------------------------------------------------------------------------

// One warp per row, 16 bytes a lane (W = 1: value by value).
template <typename T, int W, bool POS>
__global__ void __launch_bounds__(256)
embedding_scaled_kernel(const int *__restrict__ ids, const T *__restrict__ tok, const T *__restrict__ pos, T *__restrict__ out, float scale, long long n, int S, int V, int E)
{
    dependency_wait();
    dependents_may_start();
    const int lane = threadIdx.x & 31;
    const long long t = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (t >= n) return;
    const int id = ids[t];
    const bool ok = id >= 0 && id < V;
    const T *src = tok + (size_t)(ok ? id : 0) * E, *prow = POS ? pos + (size_t)(t % S) * E : nullptr;
    T *dst = out + (size_t)t * E;
#pragma unroll 4
    for (int e = lane * W; e < E; e += 32 * W) {
        float x[W], p[W];
#pragma unroll
        for (int j = 0; j < W; ++j) x[j] = p[j] = 0.0f;
        if (ok) {
            load_values<T, W>(src + e, x);
            if constexpr (POS) load_values<T, W>(prow + e, p);
#pragma unroll
            for (int j = 0; j < W; ++j) x[j] = POS ? __fadd_rn(__fmul_rn(scale, x[j]), p[j]) : __fmul_rn(scale, x[j]);
        }
        store_values<T, W>(dst + e, x);
    }
}

template <typename T>
int launch_embedding_scaled(const int *ids, const void *tok, const void *pos, void *out, float scale, long long n, int S, int V, int E, cudaStream_t st)
{
    constexpr int W = kPer16<T>;
    const bool vec = E % W == 0 && all_aligned16({tok, pos, out});
    const auto kern = pos ? (vec ? embedding_scaled_kernel<T, W, true> : embedding_scaled_kernel<T, 1, true>)
                          : (vec ? embedding_scaled_kernel<T, W, false> : embedding_scaled_kernel<T, 1, false>);
    const cudaError_t e = launch_overlapped(kern, dim3((unsigned)((n + 7) / 8)), dim3(256), 0, st, ids, static_cast<const T *>(tok), static_cast<const T *>(pos), static_cast<T *>(out),
                                            scale, n, S, V, E);
    return e == cudaSuccess ? check_launch("embedding_scaled_kernel") : fail(HIPGPT_ERR_CUDA, "embedding_scaled_kernel: %s", cudaGetErrorString(e));
}

// ---- the tokens in the order of their ids -----------------------------------------------------------------------------

constexpr int kMostSortBlocks = 16, kSortThreads = 1024, kSortWarps = kSortThreads / 32;
constexpr int kKeysPerLane = 4, kTileKeys = kSortThreads * kKeysPerLane;
constexpr int kMostBits = 10, kMostBins = 1 << kMostBits;

struct SortShared {
    int hist[kMostBins];                    // digits of this block's part; read by the other blocks
    int base[kMostBins];                    // where this block's next key of each digit goes
    unsigned short warp_count[kSortWarps][kMostBins];
    int warp_sum[kSortWarps];
};

__device__ __forceinline__ int read_peer_int(const int *p, int rank)
{
    int v;
    asm volatile("ld.shared::cluster.b32 %0, [%1];" : "=r"(v) : "r"(peer_addr(smem_u32(p), rank)));
    return v;
}

// ids [n] -> (id, t) sorted in `sorted` (ids outside [0, V) as V, last), row_start[v] = first entry of row v (v <= V; row_start[V] = entries inside), and
// counters[0 .. ncounters) = 0.  `other`: a second buffer of n entries.  npass passes of `bits` bits; the last one ends in `sorted`.
__global__ void __launch_bounds__(kSortThreads)
sort_ids_kernel(const int *__restrict__ ids, int n, int V, int blocks, int bits, int npass, int2 *sorted, int2 *other, int *row_start, int *counters, int ncounters)
{
    extern __shared__ __align__(16) uint8_t sort_smem[];
    SortShared &s = *reinterpret_cast<SortShared *>(sort_smem);
    const int rank = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int bins = 1 << bits;
    dependency_wait();
    dependents_may_start();
    for (int i = rank * kSortThreads + tid; i < ncounters; i += blocks * kSortThreads) counters[i] = 0;
    const int per = ((n + blocks - 1) / blocks + 31) / 32 * 32;
    const int from = min((long long)rank * per, (long long)n), to = min((long long)from + per, (long long)n);
    // Where a block's part is one tile (up to 65536 tokens) the entries stay in registers between counting and placing, and the warps' counts are the block's
    const bool single = per <= kTileKeys;
    const int lane_keys = single ? (per + kSortThreads - 1) / kSortThreads : kKeysPerLane, warp_keys = 32 * lane_keys, warps = single ? (per + warp_keys - 1) / warp_keys : kSortWarps;
    const int2 *src = nullptr;
    int2 e[kKeysPerLane];
    int place[kKeysPerLane];
    for (int pass = 0; pass < npass; ++pass) {
        const int shift = pass * bits;
        int2 *dst = (npass - pass) & 1 ? sorted : other;
        auto entry = [&](int i) {
            if (pass) return __ldcg(src + i);
            const int id = ids[i];
            return make_int2(id >= 0 && id < V ? id : V, i);
        };
        // the entries of a tile, and each one's place among those of its digit in its warp; the warps' counts
        auto rank_tile = [&](int t0) {
            const int used = bins / 2;                // (two counts a word)
#pragma unroll
            for (int k = 0; k < kKeysPerLane; ++k) {
                const int i = t0 + warp * warp_keys + k * 32 + lane;
                e[k] = k < lane_keys && i < to ? entry(i) : make_int2(-1, 0);
            }
            if (warp < warps) {
                uint32_t *mine = reinterpret_cast<uint32_t *>(s.warp_count[warp]);
                for (int d = lane; d < used; d += 32) mine[d] = 0;
                __syncwarp();
#pragma unroll
                for (int k = 0; k < kKeysPerLane; ++k) {
                    if (k >= lane_keys) break;
                    const int d = e[k].x < 0 ? -1 : e[k].x >> shift & (bins - 1);
                    // the lanes with the same digit, bit by bit (a match of the whole digits takes several times as long: it goes by the different ones)
                    unsigned same = __ballot_sync(0xffffffffu, d >= 0);
                    for (int b = 0; b < bits; ++b) {
                        const unsigned with = __ballot_sync(0xffffffffu, d >> b & 1);
                        same &= d >> b & 1 ? with : ~with;
                    }
                    const int before_me = __popc(same & ((1u << lane) - 1));
                    const int seen = d >= 0 ? s.warp_count[warp][d] : 0;
                    __syncwarp();
                    place[k] = seen + before_me;
                    if (d >= 0 && before_me == 0) s.warp_count[warp][d] = (unsigned short)(seen + __popc(same));
                    __syncwarp();
                }
            }
            __syncthreads();
        };
        // counts of the warps -> offsets among them; the sum
        auto over_warps = [&] {
            int all = 0;
            if (tid < bins) {
#pragma unroll 8
                for (int w = 0; w < warps; ++w) {
                    const int c = s.warp_count[w][tid];
                    s.warp_count[w][tid] = (unsigned short)all;
                    all += c;
                }
            }
            return all;
        };
        if (single) {
            rank_tile(from);
            const int all = over_warps();
            if (tid < bins) s.hist[tid] = all;
        } else {
            for (int d = tid; d < bins; d += kSortThreads) s.hist[d] = 0;
            __syncthreads();
            for (int i = from + tid; i < to; i += kSortThreads) atomicAdd(&s.hist[entry(i).x >> shift & (bins - 1)], 1);
        }
        cluster_sync();
        // digit d = tid: keys of smaller digits anywhere, and of this digit in the blocks before
        int total = 0, before = 0;
        if (tid < bins) {
            int h[kMostSortBlocks];              // (all of them on their way before the first is used)
#pragma unroll
            for (int r = 0; r < kMostSortBlocks; ++r) h[r] = read_peer_int(&s.hist[tid], r < blocks ? r : rank);
#pragma unroll
            for (int r = 0; r < kMostSortBlocks; ++r) {
                total += r < blocks ? h[r] : 0;
                before += r < rank ? h[r] : 0;
            }
        }
        int incl = total;
#pragma unroll
        for (int o = 1; o < 32; o *= 2) {
            const int up = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += up;
        }
        if (lane == 31) s.warp_sum[warp] = incl;
        __syncthreads();
        int prev = 0;
        for (int w = 0; w < warp && w < bins / 32; ++w) prev += s.warp_sum[w];
        if (tid < bins) s.base[tid] = prev + incl - total + before;
        __syncthreads();
        for (int t0 = from; t0 < to; t0 += kTileKeys) {
            int all = 0;
            if (!single) {
                rank_tile(t0);
                all = over_warps();
                __syncthreads();
            }
#pragma unroll
            for (int k = 0; k < kKeysPerLane; ++k)
                if (e[k].x >= 0) {
                    const int d = e[k].x >> shift & (bins - 1);
                    __stcg(dst + s.base[d] + s.warp_count[warp][d] + place[k], e[k]);
                }
            if (!single) {
                __syncthreads();
                if (tid < bins) s.base[tid] += all;
                __syncthreads();
            }
        }
        cluster_sync();                      // the pass's entries are all there, and nobody reads this block's counts any more
        src = dst;
    }
    // rows between one entry's id and the next begin at the next; a warp fills long gaps together
    for (int i0 = from + warp * 32; i0 < to; i0 += kSortThreads) {
        const int i = i0 + lane;
        const int key = i < n ? __ldcg(&src[i].x) : V, prev = i == 0 ? -1 : i <= n ? __ldcg(&src[i - 1].x) : V;
        const bool live = i < to;
        if (live && key - prev <= 8)          // short gaps by the lane itself
            for (int v = prev + 1; v <= key; ++v) row_start[v] = i;
        unsigned gaps = __ballot_sync(0xffffffffu, live && key - prev > 8);
        while (gaps) {
            const int l = __ffs(gaps) - 1;
            gaps &= gaps - 1;
            const int a = __shfl_sync(0xffffffffu, prev, l) + 1, b = __shfl_sync(0xffffffffu, key, l), at = i0 + l;
            for (int v = a + lane; v <= b; v += 32) row_start[v] = at;
        }
    }
    if (rank == 0) {                          // rows behind the last entry
        const int last = __ldcg(&src[n - 1].x);
        for (int v = last + 1 + tid; v <= V; v += kSortThreads) row_start[v] = n;
    }
}

// ---- sums of rows -----------------------------------------------------------------------------------------------------

// Zeros for the whole table, beside the sort (which leaves most of the GPU alone and has seen the work before it complete, in every block, when it lets this kernel in; this one reads nothing); the rows that have
// entries are stored over them.  16 x 2048 tokens, 50021 x 1024 fp32: 79 us, and 88 with zeros
// for the empty rows only, behind the sort and beside the sums (82 - 102 with zeros by further clusters of the sort's launch, of which seven fit at a time)
template <typename G>
__global__ void __launch_bounds__(256)
zero_table_kernel(G *table, long long count)
{
    dependents_may_start();
    const long long i0 = (long long)blockIdx.x * 256 + threadIdx.x, step = (long long)gridDim.x * 256;
    const long long head = min(count, (long long)((16 - (reinterpret_cast<uintptr_t>(table) & 15)) % 16 / sizeof(G))), words = (count - head) / (16 / sizeof(G)), tail = head + words * (16 / sizeof(G));
    if (i0 < head) table[i0] = from_float<G>(0.0f);
    if (tail + i0 < count) table[tail + i0] = from_float<G>(0.0f);
    uint4 *to = reinterpret_cast<uint4 *>(table + head);
#pragma unroll 4
    for (long long i = i0; i < words; i += step) to[i] = make_uint4(0u, 0u, 0u, 0u);
    dependency_wait();
}

// A block has kSumThreads threads, each 16 bytes of a row of gradients; they form groups of 2^row_log threads that cover a slice of a row (at most kSliceBytes).  A
// group's task: a piece of the sorted entries, or of the batch at one position.  The rows of kRound entries at a time come into shared memory by
// one bulk copy each, so that a group has all of them on their way at once without a register.  (kRound 8, 16, 32: 32768 tokens and a table of 50021 x 1024 92, 88, 87 us; 20 x 1024 89, 64, 67; 8192 tokens,
// 5000 x 256 fp32 25.6, 25.2, 26.5.)
constexpr int kSumThreads = 128, kSliceBytes = 16 * kSumThreads, kRound = 16, kSuper = 64;
constexpr size_t kSumRows = (size_t)kSumThreads * 16 * kRound;          // bytes of a round's rows; behind them the entries

__device__ int g_embed_status = 0;            // 1: a round's copies did not come

struct SumPlan {
    int n, V, E, B, S;
    int slice, slices, row_log;               // columns of a slice, slices of a row, threads of a group
    int units;                                // groups of at most a warp that cover a row
    int piece, pieces;                        // entries of a piece, and how many
    int pos_piece, pos_pieces;                // batches of a piece of a position's row, and how many; 0: no positions' table
    long long pos_first, tasks;
    int part_row;                             // values of a row of partial sums
    int bulk, vec_out;                        // rows of gradients that a bulk copy can fetch; rows of the tables that take 16 bytes at a time
};

// Sums of rows that fall to several pieces are joined twice: those of up to kSuper pieces that follow one another, then what these give.  Places:
// [2 piece + whether the row begins in it][part_row], and the same for each kSuper pieces
struct Parts {
    float *piece, *super;
    int *piece_arrived, *super_arrived;
};

// Whether this group (a warp or a part of one) is the last of `count` that came here with what it stored; the others' sums are then visible
__device__ __forceinline__ bool last_of(int *arrived, int count, unsigned mask, int leader)
{
    __threadfence();
    __syncwarp(mask);
    int seen = 0;
    if ((int)(threadIdx.x & 31) == leader) seen = atomicAdd(arrived, 1);
    seen = __shfl_sync(mask, seen, leader);
    __threadfence();
    return seen == count - 1;
}

template <typename G, int W>
__device__ __forceinline__ void put_row(G *p, const float (&sum)[W], float scale, bool accumulate, int left, bool vec)
{
    if (vec && left >= W) {
        float v[W];
#pragma unroll
        for (int j = 0; j < W; ++j) v[j] = __fmul_rn(sum[j], scale);
        if (accumulate) {
            float old[W];
            load_values<G, W>(p, old);
#pragma unroll
            for (int j = 0; j < W; ++j) v[j] = __fadd_rn(old[j], v[j]);
        }
        store_values<G, W>(p, v);
    } else {
#pragma unroll
        for (int j = 0; j < W; ++j)
            if (j < left) {
                const float v = __fmul_rn(sum[j], scale);
                p[j] = from_float<G>(accumulate ? __fadd_rn(to_float(p[j]), v) : v);
            }
    }
}

// Five blocks an SM (four, five, six: 32768 tokens and a table of 50021 x 1024 79, 76, 82 us; 20 x 1024 63, 56, 58; rows of 64 bf16 values 110, 112, 119: the joins' loads on their way
// are registers)
template <typename T, typename G>
__global__ void __launch_bounds__(kSumThreads, 5)
embed_sum_kernel(const T *__restrict__ g, const int *__restrict__ ids, const int2 *__restrict__ sorted, const int *__restrict__ row_start, Parts tok_parts, Parts pos_parts,
                 G *grad_tok, G *grad_pos, float scale, int accumulate, SumPlan p)
{
    constexpr int W = kPer16<T>;
    extern __shared__ __align__(128) uint8_t rows_s[];       // [group][entry of the round][16 bytes a thread]
    __shared__ uint64_t landed;
    const int tid = threadIdx.x, lane = tid & 31;
    if (tid == 0) mbar_init(&landed, kSumThreads);
    __syncthreads();
    dependency_wait();
    dependents_may_start();
    int2 (*entry_s)[kRound] = reinterpret_cast<int2 (*)[kRound]>(rows_s + kSumRows);         // [group][entry of the round]: row of the table, token (-1: not to be added)
    const int size = 1 << p.row_log, groups = kSumThreads >> p.row_log, group = tid >> p.row_log, sub = tid & (size - 1);
    const long long task = (long long)blockIdx.x * groups + group;
    const bool live = task < p.tasks, pos = task >= p.pos_first;
    const long long r = pos ? task - p.pos_first : task;
    const int sl = (int)(r % p.slices), at = sl * p.slice, cols = min(p.slice, p.E - at), e = at + sub * W, left = at + cols - e;      // this thread's columns: e ... e + min(W, left)
    const int s = (int)(r / p.slices % max(1, p.S)), c = (int)(pos ? r / p.slices / p.S : r / p.slices);
    const int i0 = c * (pos ? p.pos_piece : p.piece), i1 = !live ? i0 : min(pos ? p.B : p.n, i0 + (pos ? p.pos_piece : p.piece));
    const int longest = max(p.pos_pieces ? p.pos_piece : 0, p.piece);
    // groups of at most a warp count for themselves
    const unsigned mask = size >= 32 ? 0xffffffffu : ((1u << size) - 1) << (lane & ~(size - 1));
    const int leader = size >= 32 ? 0 : lane & ~(size - 1), unit = sl * max(1, size / 32) + sub / 32;

    const int key_before = !live || pos || i0 == 0 ? -1 : __ldg(&sorted[i0 - 1].x), key_behind = !live || pos || i1 == p.n ? -1 : __ldg(&sorted[i1].x);

    float acc[W];
    auto clear = [&] {
#pragma unroll
        for (int j = 0; j < W; ++j) acc[j] = 0.0f;
    };
    // (rows of sums are padded: whole 16-byte words, whatever E)
    auto store = [&](float *row) {
        if (left <= 0) return;
#pragma unroll
        for (int j = 0; j < W; j += 4) __stcg(reinterpret_cast<float4 *>(row + e + j), make_float4(acc[j], acc[j + 1], acc[j + 2], acc[j + 3]));
    };
    // acc = rows first, first + stride, ... of sums
    auto add_sums = [&](const float *first, size_t stride, int count) {
        clear();
        if (left <= 0) return;
#pragma unroll (W == 4 ? 8 : 4)
        for (int i = 0; i < count; ++i)
#pragma unroll
            for (int j = 0; j < W; j += 4) {
                const float4 x = __ldcg(reinterpret_cast<const float4 *>(first + i * stride + e + j));
                acc[j] = __fadd_rn(acc[j], x.x);
                acc[j + 1] = __fadd_rn(acc[j + 1], x.y);
                acc[j + 2] = __fadd_rn(acc[j + 2], x.z);
                acc[j + 3] = __fadd_rn(acc[j + 3], x.w);
            }
    };
    // the sums of pieces `from` ... `to` of places that follow one another; the row begins in piece `begins` (or before)
    auto join = [&](const float *places, size_t stride, int from, int to, int begins) {
        if (from != begins) { add_sums(places + (size_t)(2 * from) * stride, 2 * stride, to - from + 1); return; }
        add_sums(places + (size_t)(2 * from + 1) * stride, 0, 1);
        float head[W];
#pragma unroll
        for (int j = 0; j < W; ++j) head[j] = acc[j];
        add_sums(places + (size_t)(2 * (from + 1)) * stride, 2 * stride, to - from);
#pragma unroll
        for (int j = 0; j < W; ++j) acc[j] = __fadd_rn(head[j], acc[j]);
    };
    // acc is the sum of what piece c has of a row that lies in pieces `first` ... `last`: true where this group then has the whole row's in acc.  stride: of the parts' rows
    auto complete = [&](const Parts &parts, size_t stride, int first, int last) {
        if (first == last) return true;
        store(parts.piece + (size_t)(2 * c + (c == first)) * stride);
        const int super = c / kSuper, from = max(first, super * kSuper), to = min(last, super * kSuper + kSuper - 1);
        if (!last_of(parts.piece_arrived + (size_t)(2 * from + (from == first)) * p.units + unit, to - from + 1, mask, leader)) return false;
        join(parts.piece, stride, from, to, first);
        const int super0 = first / kSuper, super1 = last / kSuper;
        if (super0 == super1) return true;
        store(parts.super + (size_t)(2 * super + (super == super0)) * stride);
        if (!last_of(parts.super_arrived + (size_t)(2 * super0 + 1) * p.units + unit, super1 - super0 + 1, mask, leader)) return false;
        join(parts.super, stride, super0, super1, super0);
        return true;
    };
    auto flush = [&](int v) {
        if (pos) {
            // places of a position's pieces: [place][S][row]
            Parts q = pos_parts;
            q.piece += (size_t)s * p.part_row;
            q.super += (size_t)s * p.part_row;
            q.piece_arrived += (size_t)s * 2 * p.pos_pieces * p.units;
            q.super_arrived += (size_t)s * 2 * ((p.pos_pieces + kSuper - 1) / kSuper) * p.units;
            if (complete(q, (size_t)p.S * p.part_row, 0, p.pos_pieces - 1)) put_row<G, W>(grad_pos + (size_t)s * p.E + e, acc, 1.0f, accumulate != 0, left, p.vec_out != 0);
        } else {
            int first = c, last = c;
            if (v == key_before || v == key_behind) {        // it falls to several pieces
                first = __ldg(row_start + v) / p.piece;
                last = (__ldg(row_start + v + 1) - 1) / p.piece;
            }
            if (complete(tok_parts, p.part_row, first, last)) put_row<G, W>(grad_tok + (size_t)v * p.E + e, acc, scale, accumulate != 0, left, p.vec_out != 0);
        }
    };

    clear();
    int v = -1;                              // the row that acc belongs to
    bool gone = false;                       // a round's copies have not come in time: nothing more is added or stored
    for (int round = 0; round * kRound < longest; ++round) {
        const int j0 = i0 + round * kRound, here = max(0, min(kRound, i1 - j0));
        if (round) __syncthreads();          // the round before has been read
        // the entries, and their rows on their way
        uint32_t bytes = 0;
        for (int k = sub; k < here; k += size) {
            int2 en;
            if (pos) {
                const int t = (j0 + k) * p.S + s, id = __ldg(ids + t);
                en = make_int2(s, id >= 0 && id < p.V ? t : -1);
            } else {
                en = __ldg(sorted + j0 + k);
                if (en.x >= p.V) en.y = -1;
            }
            entry_s[group][k] = en;
            if (p.bulk && !gone && en.y >= 0) bytes += (uint32_t)(cols * sizeof(T));
        }
        if (p.bulk && !gone) {
            mbar_arrive_expect_tx(&landed, bytes);
            for (int k = sub; k < here; k += size) {
                const int t = entry_s[group][k].y;
                if (t >= 0) bulk_load(rows_s + ((size_t)(group * kRound + k) << p.row_log) * 16, g + (size_t)t * p.E + at, (uint32_t)(cols * sizeof(T)), &landed);
            }
            __syncthreads();                 // the entries
            gone = !__all_sync(0xffffffffu, mbar_wait(&landed, (uint32_t)(round & 1)));        // (a warp as a whole: its lanes meet again in last_of)
            if (gone) {
                atomicCAS(&g_embed_status, 0, 1);
                linger();
            }
        } else {
            __syncthreads();
            for (int k = 0; k < here; ++k) {
                const int t = entry_s[group][k].y;
                T *to = reinterpret_cast<T *>(rows_s + ((size_t)(group * kRound + k) << p.row_log) * 16) + sub * W;
#pragma unroll
                for (int j = 0; j < W; ++j) if (t >= 0 && j < left) to[j] = g[(size_t)t * p.E + e + j];
            }
        }
        // (an entry's values are read while the one before it is added)
        int2 ahead = entry_s[group][0];
        float x_ahead[W];
        auto read = [&](int k) { load_values<T, W>(reinterpret_cast<const T *>(rows_s + ((size_t)(group * kRound + k) << p.row_log) * 16) + sub * W, x_ahead); };
        read(0);
#pragma unroll 1
        for (int k = 0; k < here && !gone; ++k) {
            const int2 en = ahead;
            float x[W];
#pragma unroll
            for (int j = 0; j < W; ++j) x[j] = x_ahead[j];
            const int behind = min(k + 1, kRound - 1);
            ahead = entry_s[group][behind];
            read(behind);
            if (en.y < 0 && !pos) continue;
            if (en.x != v) {
                if (v >= 0) flush(v);
                v = en.x;
                clear();
            }
            if (en.y < 0) continue;
#pragma unroll
            for (int j = 0; j < W; ++j) acc[j] = __fadd_rn(acc[j], x[j]);
        }
    }
    if (v >= 0 && !gone) flush(v);
}

StreamWorkspace g_embed_ws;

int ceil_div(long long a, long long b) { return (int)std::min<long long>((a + b - 1) / b, 2147483647); }
size_t padded(size_t bytes) { return (bytes + 255) & ~(size_t)255; }

template <typename T, typename G>
int launch_embedding_backward(const void *grad_out, const int *ids, void *grad_tok, void *grad_pos, float scale, int accumulate, int B, int S, int V, int E, cudaStream_t st)
{
    const int n = B * S;
    SumPlan p = {};
    p.n = n; p.V = V; p.E = E; p.B = B; p.S = S;
    p.slice = std::min(E, kSliceBytes / (int)sizeof(T));
    p.slices = ceil_div(E, p.slice);
    while ((1 << p.row_log) * kPer16<T> < p.slice) ++p.row_log;
    p.units = p.slices * std::max(1, (1 << p.row_log) / 32);
    // a piece: one round of copies, or as many as leave 65536 threads at work (2048 to 8192 pieces, so that joining twice is enough).  131072 rows of 256 bf16 values: 111 us in 2048 pieces,
    // 114 in 4096, 120 in 8192; 262144 rows of 64 values: 163, 128, 110
    p.piece = kRound * std::max(1, ceil_div(n, (long long)std::max(2048, std::min(8192, 65536 >> p.row_log)) * kRound));
    p.pieces = ceil_div(n, p.piece);
    p.pos_piece = kRound * std::max(1, ceil_div(B, 2048 * kRound));
    p.pos_pieces = grad_pos ? ceil_div(B, p.pos_piece) : 0;
    p.pos_first = grad_tok ? (long long)p.pieces * p.slices : 0;
    p.tasks = p.pos_first + (long long)p.pos_pieces * S * p.slices;
    p.bulk = E * sizeof(T) % 16 == 0 && all_aligned16({grad_out});
    p.vec_out = E % kPer16<T> == 0 && all_aligned16({grad_tok, grad_pos});
    const int groups = kSumThreads >> p.row_log;
    const long long blocks = (p.tasks + groups - 1) / groups;
    p.part_row = (E + 7) / 8 * 8;
    const int supers = ceil_div(p.pieces, kSuper), pos_supers = ceil_div(p.pos_pieces, kSuper);
    const bool pos_parts = p.pos_pieces > 1;
    const long long ncounters = 2LL * p.units * (p.pieces + supers + (pos_parts ? (long long)S * (p.pos_pieces + pos_supers) : 0));
    if (blocks > 2147483647LL || ncounters > 2147483647LL) return fail(HIPGPT_ERR_UNSUPPORTED, "a table of %d rows of %d values is beyond one call", V, E);

    const size_t entry_bytes = padded((size_t)n * sizeof(int2)), start_bytes = padded(((size_t)V + 1) * sizeof(int)), counter_bytes = padded((size_t)ncounters * sizeof(int));
    const size_t row = (size_t)p.part_row * sizeof(float), part_bytes = padded(2 * (p.pieces + supers) * row), pos_bytes = pos_parts ? padded(2 * (p.pos_pieces + pos_supers) * S * row) : 0;
    StreamWorkspace::Lease ws;
    int rc = g_embed_ws.enter(st, 2 * entry_bytes + start_bytes + counter_bytes + part_bytes + pos_bytes, &ws);
    if (rc != HIPGPT_OK) return rc;
    uint8_t *at = ws.get();
    auto take = [&](size_t bytes) { uint8_t *r = at; at += bytes; return r; };
    int2 *sorted = reinterpret_cast<int2 *>(take(entry_bytes)), *other = reinterpret_cast<int2 *>(take(entry_bytes));
    int *row_start = reinterpret_cast<int *>(take(start_bytes)), *counters = reinterpret_cast<int *>(take(counter_bytes));
    Parts tok, pos;
    tok.piece = reinterpret_cast<float *>(take(part_bytes));
    tok.super = tok.piece + (size_t)2 * p.pieces * p.part_row;
    tok.piece_arrived = counters;
    tok.super_arrived = counters + (size_t)2 * p.pieces * p.units;
    pos.piece = reinterpret_cast<float *>(take(pos_bytes));
    pos.super = pos.piece + (size_t)2 * p.pos_pieces * S * p.part_row;
    pos.piece_arrived = tok.super_arrived + (size_t)2 * supers * p.units;
    pos.super_arrived = pos.piece_arrived + (size_t)2 * p.pos_pieces * S * p.units;

    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    static std::atomic<unsigned long long> done{0};
    if (e == cudaSuccess) e = once_per_device(done, dev, [] {
        cudaError_t r = cudaFuncSetAttribute(sort_ids_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(SortShared));
        if (r == cudaSuccess) r = cudaFuncSetAttribute(sort_ids_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        return r;
    });
    int key_bits = 1;
    while (key_bits < 31 && (V >> key_bits)) ++key_bits;                   // keys 0 ... V
    const int npass = ceil_div(key_bits, kMostBits), bits = ceil_div(key_bits, npass);
    if (!grad_tok) {                                                       // no order is asked for; nothing of the long rows runs
        if (e == cudaSuccess) e = cudaMemsetAsync(counters, 0, (size_t)ncounters * sizeof(int), st);
    } else if (e == cudaSuccess) {
        const int sort_blocks = n <= 1024 ? 1 : kMostSortBlocks;           // a cluster meets twice a pass, half a microsecond each: not for as few as one round of one block's threads
        e = launch_overlapped_clusters(sort_ids_kernel, sort_blocks, dim3((unsigned)sort_blocks), dim3(kSortThreads), sizeof(SortShared), st, ids, n, V, sort_blocks, bits, npass, sorted, other,
                                       row_start, counters, (int)ncounters);
    }
    if (e != cudaSuccess) return fail(HIPGPT_ERR_CUDA, "sort_ids_kernel: %s", cudaGetErrorString(e));
    rc = check_launch("sort_ids_kernel");
    if (rc != HIPGPT_OK) return rc;
    if (grad_tok && !accumulate && V > 0) {
        e = launch_overlapped(zero_table_kernel<G>, dim3((unsigned)std::min(ceil_div((long long)V * E, 8192), 148 * 4)), dim3(256), 0, st, static_cast<G *>(grad_tok), (long long)V * E);
        if (e != cudaSuccess) return fail(HIPGPT_ERR_CUDA, "zero_table_kernel: %s", cudaGetErrorString(e));
    }
    static std::atomic<unsigned long long> sum_done{0};
    e = once_per_device(sum_done, dev, [] { return cudaFuncSetAttribute(embed_sum_kernel<T, G>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(kSumRows + kSumThreads * kRound * sizeof(int2))); });
    if (e == cudaSuccess) e = launch_overlapped(embed_sum_kernel<T, G>, dim3((unsigned)blocks), dim3(kSumThreads), kSumRows + groups * kRound * sizeof(int2), st, static_cast<const T *>(grad_out), ids, (const int2 *)sorted,
                                                (const int *)row_start, tok, pos, static_cast<G *>(grad_tok), static_cast<G *>(grad_pos), scale, accumulate, p);
    return e == cudaSuccess ? check_launch("embed_sum_kernel") : fail(HIPGPT_ERR_CUDA, "embed_sum_kernel: %s", cudaGetErrorString(e));
}

int check_embedding_sizes(int B, int S, int V, int E, int type)
{
    if (type != HIPGPT_TYPE_F32 && type != HIPGPT_TYPE_BF16) return fail(HIPGPT_ERR_BAD_ARG, "unknown type %d", type);
    if (B < 0 || S < 0 || V < 0 || E < 0) return fail(HIPGPT_ERR_BAD_ARG, "negative size: B=%d S=%d V=%d E=%d", B, S, V, E);
    if (V >= 1 << 30 || E >= 1 << 30) return fail(HIPGPT_ERR_UNSUPPORTED, "tables of %d rows of %d values are beyond one call", V, E);
    if ((long long)B * S > 1LL << 30) return fail(HIPGPT_ERR_UNSUPPORTED, "%lld tokens are beyond one call", (long long)B * S);
    return HIPGPT_OK;
}

}  // namespace

void embedding_release_scratch() { g_embed_ws.release(); }

int embedding_status_fetch(int *status)
{
    int v = 0;
    const cudaError_t e = cudaMemcpyFromSymbol(&v, g_embed_status, sizeof(v));
    if (e != cudaSuccess) return fail(HIPGPT_ERR_CUDA, "cudaMemcpyFromSymbol: %s", cudaGetErrorString(e));
    if (v) { const int zero = 0; cudaMemcpyToSymbol(g_embed_status, &zero, sizeof(zero)); }
    *status = v;
    return HIPGPT_OK;
}

}  // namespace hipgpt

using namespace hipgpt;

extern "C" {

int hipgpt_embedding_scaled(const int *d_ids, const void *d_tok, const void *d_pos, void *d_out, float scale, int B, int S, int V, int E, int type, void *stream)
{
    const int rc = check_embedding_sizes(B, S, V, E, type);
    if (rc != HIPGPT_OK) return rc;
    if (B == 0 || S == 0 || E == 0) return HIPGPT_OK;
    if (!d_ids || !d_out || (V > 0 && !d_tok)) return fail(HIPGPT_ERR_NULL, "ids, tok and out must not be NULL");
    const size_t ts = type == HIPGPT_TYPE_F32 ? 4 : 2, row = (size_t)E * ts, n = (size_t)B * S;
    const int clear = refuse_overlaps(1, {{d_out, n * row}, {d_ids, n * sizeof(int)}, {d_tok, V * row}, {d_pos, S * row}});
    if (clear != HIPGPT_OK) return clear;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    return type == HIPGPT_TYPE_F32 ? launch_embedding_scaled<float>(d_ids, d_tok, d_pos, d_out, scale, (long long)B * S, S, V, E, st)
                                   : launch_embedding_scaled<__nv_bfloat16>(d_ids, d_tok, d_pos, d_out, scale, (long long)B * S, S, V, E, st);
}

int hipgpt_embedding_backward(const void *d_grad_out, const int *d_ids, void *d_grad_tok, void *d_grad_pos, float scale, int accumulate,
                              int B, int S, int V, int E, int type, int grad_type, void *stream)
{
    const int rc = check_embedding_sizes(B, S, V, E, type);
    if (rc != HIPGPT_OK) return rc;
    if (grad_type != HIPGPT_TYPE_F32 && grad_type != HIPGPT_TYPE_BF16) return fail(HIPGPT_ERR_BAD_ARG, "unknown type %d", grad_type);
    if (type == HIPGPT_TYPE_F32 && grad_type == HIPGPT_TYPE_BF16) return fail(HIPGPT_ERR_UNSUPPORTED, "fp32 gradients are not summed into bf16 tables");
    if (E == 0 || (!d_grad_tok && !d_grad_pos)) return HIPGPT_OK;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    const size_t gs = grad_type == HIPGPT_TYPE_F32 ? 4 : 2;
    if (B == 0 || S == 0) {                              // no token: gradients of zero
        if (accumulate) return HIPGPT_OK;
        cudaError_t e = d_grad_tok && V ? cudaMemsetAsync(d_grad_tok, 0, (size_t)V * E * gs, st) : cudaSuccess;
        if (e == cudaSuccess && d_grad_pos && S) e = cudaMemsetAsync(d_grad_pos, 0, (size_t)S * E * gs, st);
        return e == cudaSuccess ? HIPGPT_OK : fail(HIPGPT_ERR_CUDA, "cudaMemsetAsync: %s", cudaGetErrorString(e));
    }
    if (!d_grad_out || !d_ids) return fail(HIPGPT_ERR_NULL, "grad_out and ids must not be NULL");
    const size_t n = (size_t)B * S, row = (size_t)E * gs;
    const int clear = refuse_overlaps(2, {{d_grad_tok, V * row}, {d_grad_pos, S * row}, {d_grad_out, n * E * (type == HIPGPT_TYPE_F32 ? 4 : 2)}, {d_ids, n * sizeof(int)}});
    if (clear != HIPGPT_OK) return clear;
    if (type == HIPGPT_TYPE_F32) return launch_embedding_backward<float, float>(d_grad_out, d_ids, d_grad_tok, d_grad_pos, scale, accumulate, B, S, V, E, st);
    return grad_type == HIPGPT_TYPE_F32 ? launch_embedding_backward<__nv_bfloat16, float>(d_grad_out, d_ids, d_grad_tok, d_grad_pos, scale, accumulate, B, S, V, E, st)
                                        : launch_embedding_backward<__nv_bfloat16, __nv_bfloat16>(d_grad_out, d_ids, d_grad_tok, d_grad_pos, scale, accumulate, B, S, V, E, st);
}

}  // extern "C"
